"""GPU: attention over a 4-bit cache holds its operands in as many bits as its outputs show, by the noise of the outputs (kv4_noise)."""
import math

import numpy as np
import pytest
import torch

import kv4_noise as noise
import kv4_util as kv
from test_gpu_kv4 import host

pytestmark = pytest.mark.gpu


def caches(qh, kh, d, dtype, lens, loud):
    """Rows appended from normal numbers; keys with a loud channel a group if wanted."""
    c = kv.KV4(qh, kh, d, [0] * len(lens), lens, dtype, seed=qh + d)
    n = sum(lens)
    k = noise.loud_rows(c.rng, n, kh * d) if loud else c.rng.standard_normal((n, kh * d))
    k, v = torch.from_numpy(k.astype(np.float32)).to(c.dev).to(c.dtype), c.normal(n, kh * d)
    out = c.ints([0] * len(lens))
    c.do("append", c.append_args(lens, out, None, k, v))
    torch.cuda.synchronize()
    assert out.tolist() == lens and c.status.item() == 0
    c.lens = out
    return c


def outputs(c, counts, lens, q_scale, mass):
    q = c.normal(sum(counts), c.qh, c.d, scale=q_scale)
    out = torch.zeros_like(q)
    m = torch.zeros(c.n_pages, c.kh, 64, device=c.dev) if mass else None
    c.do("attention", c.attention_args(counts, c.lens, q, out, mass=m))
    torch.cuda.synchronize()
    assert c.status.item() == 0
    ref, before, size, row = [], [], [], 0
    for b, (n, L) in enumerate(zip(counts, lens)):
        k, v = c.held(b, L)
        x = host(q[row:row + n])
        r, e = noise.statement(x, k, v, 1 / math.sqrt(c.d), c.spread(b, L))
        ref.append(r), before.append(e)
        size.append(kv.attend(x, k, v, 1 / math.sqrt(c.d), c.spread(b, L))[2])
        row += n
    return host(out), np.concatenate(ref), np.concatenate(before), np.concatenate(size)


TOKENS, PORTIONS = ([1] * 32, [2, 3, 4, 5, 7, 9, 12, 17] * 4), ([60] * 6, [60, 61, 70, 60, 60, 64])


@pytest.mark.parametrize("qh,kh,d", [(8, 8, 64), (16, 4, 128), (48, 4, 64)])
@pytest.mark.parametrize("mass", [False, True])
def test_fp16_tokens(qh, kh, d, mass):
    """One row a sequence, and (48 heads on 4) more than a warp's tile of them."""
    got, ref, before, _ = outputs(caches(qh, kh, d, "fp16", TOKENS[1], False), *TOKENS, 0.02, mass)
    assert noise.too_far(got, ref, before, "fp16") < 1


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("loud", [False, True])
def test_fp16_portions(d, mass, loud):
    got, ref, before, _ = outputs(caches(16, 16, d, "fp16", PORTIONS[1], loud), *PORTIONS, 1.0 if loud else 0.02, mass)
    assert noise.too_far(got, ref, before, "fp16") < 1


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("portions", [False, True])
def test_bf16_keys_where_a_channel_is_loud(d, portions):
    """Weights (and many rows' values) of bf16 outputs may be rounded to fp16; keys not where a row's weights are one token's, or summed."""
    counts, lens = PORTIONS if portions else TOKENS
    got, ref, before, size = outputs(caches(16, 16, d, "bf16", lens, True), counts, lens, 1.0, portions)
    assert noise.too_far(got, ref, before + (2 if portions else 1) * 2.0 ** -11 * size, "bf16") < 1


@pytest.mark.parametrize("rows,others", [(1, 1), (1, 60)])
def test_fp16_rows_do_not_depend_on_their_neighbours_rows(rows, others):
    """A token is as near the formula beside other tokens as beside portions."""
    counts, lens = [rows] * 20 + [others] * 6, [2, 3, 4, 5, 7, 9, 12, 17, 6, 8] * 2 + [60] * 6
    c = caches(32, 32, 64, "fp16", lens, False)
    got, ref, before, _ = outputs(c, counts, lens, 0.02, False)
    assert noise.too_far(got[:20 * rows], ref[:20 * rows], before[:20 * rows], "fp16") < 1
