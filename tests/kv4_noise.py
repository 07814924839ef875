"""How far outputs may be from the 64-bit statement in the mean: rounding an output once has a noise of its own, and what comes before it is bounded.

With x = ref + e the output is round(x), and round(x) - ref = (round(x) - x) + e, so its root mean square is at most that of round(x) - x and
that of e together.  round(x) - x is distributed as round(ref) - ref is (e is far below a step); the mean square of N such numbers, uniform
between two halves of a step, has a relative deviation of 0.9 / sqrt(N), its root half that, and two of them differ by 3.2 / sqrt(N) in five
deviations.

e, where weights and values are held in 22 bits or more (a pair of fp16, or fp32): products and their sums in 32 bits are off by less than
2^-18 of sum p max(|v|, |scale (code - 8)|), and a score's error ds multiplies a weight by exp(2 ds) at most.  A score is a sum of 16 exact
products at a time, 2 d / 16 times for a pair of fp16: each of the 17 numbers that a step adds up may lose 2^-24 of the largest."""
import math

import numpy as np
import torch

import kv4_util as kv

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def rounded(x, dtype):
    return torch.from_numpy(np.asarray(x, np.float64)).to(TYPES[dtype]).double().numpy()


def rms(x):
    return math.sqrt(float(np.mean(np.square(x))))


def too_far(got, ref, before, dtype):
    """got, ref: float64, before: bound on |e|, elementwise -> the noise over its limit."""
    assert ref.size > 10000
    return rms(got - ref) / (rms(rounded(ref, dtype) - ref) * (1 + 3.2 / math.sqrt(ref.size)) + rms(before))


def score_error(q, k, scale):
    """q [n, heads, d], k [kv heads, L, d] -> [n, heads, 1]."""
    if k.shape[1] == 0:
        return np.zeros((*q.shape[:2], 1))
    n, heads, d = q.shape
    out, g = np.zeros((n, heads, 1)), heads // k.shape[0]
    for h in range(heads):
        terms = q[:, h, None, :] * k[h // g][None]                # [n, L, d]
        sums = np.abs(terms.reshape(*terms.shape[:2], -1, 16).sum(-1).cumsum(-1)).max((1, 2))
        out[:, h, 0] = scale * (d // 8 + 2) * 17 * 2.0 ** -24 * np.maximum(sums, np.abs(terms).max((1, 2)))
    return out


def statement(q, k, v, scale, spread):
    """-> ref and the bound on e."""
    ref, w, size = kv.attend(q, k, v, scale, spread)
    return ref, (2.0 ** -18 + np.expm1(2 * score_error(q, k, scale))) * size


def loud_rows(rng, *shape):
    """Rows with one channel of each group far from 0, as keys have it where a projection's bias is large: 100 +- 20 beside 1."""
    x = rng.standard_normal(shape)
    x[..., ::64] = 100 + 20 * x[..., ::64]
    return x
