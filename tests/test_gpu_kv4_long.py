"""GPU: attention over a 4-bit cache at lengths and scores that the other tests do not come to: caches behind one warp's, one round's and one
block's limits of joining, and rows whose largest score comes pages after their first (tolerances: test_gpu_kv4; a weight is off by its score's error as well, kv4_noise)."""
import math

import numpy as np
import pytest
import torch

import kv4_util as kv
from test_gpu_kv4 import attention_bound, host

pytestmark = pytest.mark.gpu


class Long:
    """One sequence per length on random tiles made on the GPU (codes any, scales and minima of normal numbers), and the statement with torch in
    64 bits, row by row of queries."""

    def __init__(self, qh, kh, d, lens, dtype, seed):
        self.c = c = kv.KV4(qh, kh, d, lens, None, dtype, seed=seed)
        g = torch.Generator(device=c.dev).manual_seed(seed)
        c.pool.random_(0, 256, generator=g)
        for a, e in (kv.parts(d)[1], kv.parts(d)[3]):
            n = (e - a) // 4
            scale = torch.rand(c.n_pages, kh, n, generator=g, device=c.dev) * 0.2 + 0.2
            low = torch.randn(c.n_pages, kh, n, generator=g, device=c.dev) * 0.3 - 7.5 * scale
            c.pool[:, :, a:e] = torch.stack((scale, low), -1).half().contiguous().view(torch.uint8).reshape(c.n_pages, kh, e - a)
        for d_key in (True, False):
            setattr(self, "place_k" if d_key else "place_v", torch.from_numpy(kv.nibble_place(d, d_key)).to(c.dev))

    def held(self, b, n):
        """[kv heads, n, d] keys, values, and |scale (code - 8)| of the values, in 64 bits."""
        c, d = self.c, self.c.d
        t = c.pool[torch.from_numpy(c.np_table[b, :-(-n // 64)].astype(np.int64)).to(c.dev)]
        out = []
        for place, (a, e), (p0, p1) in ((self.place_k, *kv.parts(d)[:2]), (self.place_v, *kv.parts(d)[2:])):
            w = t[:, :, a:e].reshape(len(t), c.kh, 64, d // 2)
            codes = torch.stack((w & 15, w >> 4), -1).reshape(len(t), c.kh, 64, d)[..., place].double()
            par = t[:, :, p0:p1].contiguous().view(torch.float16).reshape(len(t), c.kh, 64, d // 64, 2).double()
            scale, low = (par[..., i].repeat_interleave(64, -1) for i in (0, 1))
            out.append((low + scale * codes).transpose(0, 1).reshape(c.kh, -1, d)[:, :n])
            spread = (scale * (codes - 8)).abs().transpose(0, 1).reshape(c.kh, -1, d)[:, :n]
        return *out, spread

    def statement(self, q, b, n, L, scale):
        """q [n, heads, d] -> out, sum of p max(|v|, spread), weights summed over rows and heads of a group [kv heads, L]."""
        k, v, spread = self.held(b, L)
        g = q.shape[1] // self.c.kh
        out, size, mass = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(self.c.kh, L, dtype=torch.float64, device=q.device)
        big = torch.maximum(v.abs(), spread)
        for i in range(n):
            see = L - n + i + 1
            for h in range(self.c.kh):
                p = torch.softmax(q[i, h * g:(h + 1) * g] @ k[h, :see].T * scale, -1)
                out[i, h * g:(h + 1) * g], size[i, h * g:(h + 1) * g] = p @ v[h, :see], p @ big[h, :see]
                mass[h, :see] += p.sum(0)
        return out, size, mass, k


def score_error(q, k, scale):
    """kv4_noise.score_error, the largest of all, in torch."""
    d, g, top = q.shape[-1], q.shape[1] // k.shape[0], 0.0
    for h in range(q.shape[1]):
        s = torch.zeros(q.shape[0], k.shape[1], dtype=torch.float64, device=q.device)
        top = max(top, (q[:, h].abs().amax(0) * k[h // g].abs().amax(0)).max().item())
        for c in range(0, d, 16):
            s += q[:, h, c:c + 16] @ k[h // g, :, c:c + 16].T
            top = max(top, s.abs().max().item())
    return scale * (d // 8 + 2) * 17 * 2.0 ** -24 * top


def check(x, counts, lens, dtype, mass, q, shared=False):
    c = x.c
    out = torch.full_like(q, 9.0)
    m_in = torch.rand(c.n_pages, c.kh, 64, device=c.dev) if mass else None
    m_out = torch.full_like(m_in, -1.0) if mass else None
    a = c.attention_args(counts, c.ints(lens), q, out, mass=m_in, mass_out=m_out)
    c.do("attention", a)
    torch.cuda.synchronize()
    assert c.status.item() == 0
    row, scale = 0, 1 / math.sqrt(c.d)
    for b, (n, L) in enumerate(zip(counts, lens)):
        ref, size, w, kt = x.statement(q[row:row + n].double(), b, n, L, scale)
        ref, size, w, k = (t.cpu().numpy() for t in (ref, size, w, kt))
        bound = attention_bound(dtype, ref, size, host(q[row:row + n]), k, scale, shared)
        off = np.abs(host(out[row:row + n]) - ref)
        assert (off <= bound).all(), (b, float((off / bound).max()))
        if mass:
            want = c.rows_of(m_in, b, L).astype(np.float64) + w
            weights_off = math.expm1(2 * score_error(q[row:row + n].double(), kt, scale))
            assert (np.abs(c.rows_of(m_out, b, L) - want) <= 2.0 ** -15 * max(1.0, np.abs(want).max()) + weights_off * w).all()
        row += n
    first = out.clone()
    c.do("attention", a)
    assert torch.equal(out, first)


@pytest.mark.parametrize("qh,kh,d,dtype,counts,lens", [
    (7, 1, 128, "bf16", [1], [131000]),                # one kv head: its pages on all warps, more pieces than a round of factors
    (28, 4, 128, "bf16", [1, 1, 1], [40001, 64, 3]),   # pieces beyond 256, beside short ones
    (16, 1, 64, "fp16", [1], [70003]), (2, 2, 64, "bf16", [1], [33000]), (16, 2, 128, "bf16", [2, 1], [50000, 20000])])
@pytest.mark.parametrize("mass", [False, True])
def test_tokens_behind_long_caches(qh, kh, d, dtype, counts, lens, mass):
    x = Long(qh, kh, d, lens, dtype, seed=qh)
    check(x, counts, lens, dtype, mass, x.c.normal(sum(counts), qh, d))


@pytest.mark.parametrize("qh,kh,d,dtype", [(8, 1, 128, "bf16"), (8, 1, 128, "fp16"), (14, 2, 64, "bf16")])
@pytest.mark.parametrize("mass", [False, True])
def test_portions_behind_long_caches(qh, kh, d, dtype, mass):
    counts, lens = [200, 40], [21000, 9000]
    x = Long(qh, kh, d, lens, dtype, seed=d)
    check(x, counts, lens, dtype, mass, x.c.normal(sum(counts), qh, d), shared=True)


def loudest_last(x, b, L, qh):
    """A query whose scores rise along the cache, above all from page to page: many times its first page's maximum times 2^8."""
    c = x.c
    k = x.held(b, L)[0]
    g = qh // c.kh
    q = torch.empty(qh, c.d, dtype=torch.float64, device=c.dev)
    for h in range(qh):
        pages = [k[h // g, min(L - 1, 64 * j + 7 * (h % 9))] for j in range(-(-L // 64))]
        # the direction of the last pages' keys, less that of the earlier ones
        q[h] = sum((j + 1) * p / p.norm() for j, p in enumerate(pages)) / len(pages)
        q[h] *= 14.0 / q[h].norm() * math.sqrt(c.d) / 4
    return q


def rescales(x, b, n, L, q, scale):
    """(row, head, page) at which a row's weights have to be scaled: its maximum has passed what they are relative to by more than 2^8."""
    k = x.held(b, L)[0]
    g, count = q.shape[1] // x.c.kh, 0
    for h in range(q.shape[1]):
        s = (q[:, h].double() @ k[h // g].T * scale * math.log2(math.e)).cpu().numpy()
        for i in range(n):
            see, m = L - n + i + 1, -np.inf
            for j in range(0, see, 64):
                top = s[i, j:min(see, j + 64)].max()
                if top > m + 8:
                    count += j > 0
                    m = top
    return count


@pytest.mark.parametrize("qh,kh,d,dtype,counts,lens", [(16, 2, 128, "bf16", [150, 40], [700, 333]), (8, 8, 64, "fp16", [100] * 8, [500 + 9 * i for i in range(8)]),
                                                       (28, 4, 128, "bf16", [128], [3000])])
@pytest.mark.parametrize("mass", [False, True])
def test_many_rows_whose_maximum_grows(qh, kh, d, dtype, counts, lens, mass):
    """Outputs in tensor memory are scaled where a maximum grows by more than 2^8 after a row's first page; the inputs do that often."""
    x = Long(qh, kh, d, lens, dtype, seed=3)
    q = x.c.normal(sum(counts), qh, d, scale=0.3).double()
    row, grown = 0, 0
    for b, (n, L) in enumerate(zip(counts, lens)):
        q[row:row + n] += loudest_last(x, b, L, qh)
        row += n
    q = q.to(x.c.dtype)
    row = 0
    for b, (n, L) in enumerate(zip(counts, lens)):
        grown += rescales(x, b, n, L, q[row:row + n], 1 / math.sqrt(d))
        row += n
    assert grown > 100, grown
    check(x, counts, lens, dtype, mass, q, shared=True)
