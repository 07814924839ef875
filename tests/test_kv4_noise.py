"""CPU: the bound on the outputs' noise sees a single operand that was rounded to fp16 where it should not have been (the mistake is planted in a
statement of its own, on the inputs' distribution that the GPU tests have)."""
import math

import numpy as np
import pytest

import kv4_noise as noise
import kv4_util as kv

HOW = ["right", "weights", "values", "keys"]


def fp16(x):
    return np.asarray(x).astype(np.float16).astype(np.float64)


def sequence(rng, kh, n, loud=False):
    codes, scale, low = kv.snap(noise.loud_rows(rng, kh, n, 64) if loud else rng.standard_normal((kh, n, 64)))[1:]
    return kv.values(codes, scale, low), np.abs(np.repeat(scale, 64, -1) * (codes - 8))


def attend(q, k, v, scale, how, lift=10):
    """With one of the operands rounded to fp16 (weights before their products, as 2^lift of the largest)."""
    if how == "keys":
        k = fp16(k)
    if how == "values":
        v = fp16(v)
    n, heads, d = q.shape
    out, L, g = np.zeros_like(q), k.shape[1], heads // k.shape[0]
    for i in range(n):
        see = L - n + i + 1
        for h in range(heads):
            s = (k[h // g, :see] @ q[i, h]) * scale
            p = np.exp(s - s.max())
            l = p.sum()
            out[i, h] = (fp16(p * 2.0 ** lift) / 2.0 ** lift if how == "weights" else p) @ v[h // g, :see] / l
    return out


@pytest.mark.parametrize("counts,lens,loud", [([1] * 32, [2, 3, 4, 5, 7, 9, 12, 17] * 4, False), ([60] * 3, [60, 61, 70], False), ([60] * 3, [60, 61, 70], True)],
                         ids=["tokens", "portions", "portions, loud channels"])
def test_the_bound_sees_an_operand_of_fp16(counts, lens, loud):
    seen = {}
    for how in HOW:
        rng = np.random.default_rng(0)
        got, ref, before = [], [], []
        for n, L in zip(counts, lens):
            k, _ = sequence(rng, 8, L, loud)
            v, spread = sequence(rng, 8, L)
            q = noise.rounded(rng.standard_normal((n, 8, 64)) * (1.0 if loud else 0.02), "fp16")
            r, b = noise.statement(q, k, v, 1 / 8, spread)
            ref.append(r), before.append(np.broadcast_to(b, r.shape)), got.append(noise.rounded(attend(q, k, v, 1 / 8, how), "fp16"))
        got, ref, before = (np.concatenate([x.reshape(-1) for x in t]) for t in (got, ref, before))
        seen[how] = noise.too_far(got, ref, before, "fp16")
    print(seen)
    assert seen["right"] < 1
    for how in HOW[3:] if loud else HOW[1:3]:
        assert seen[how] > 1, seen
