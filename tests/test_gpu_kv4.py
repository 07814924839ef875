"""GPU: the operators of the 4-bit cache through the C ABI against the plain 64-bit statement in kv4_util.

Tolerances.  An output rounded to bf16 or fp16 is off by half a step, eps/2 of its value.  Before that, attention's weights may be rounded to
fp16, 2^-11 of each.  With v = c + scale (code - 8), c = min + 8 scale, a rounded weight p (1 + e) may stand before all of v, which is off by
e p |v|, or before scale (code - 8) alone while c keeps the unrounded one, which is off by e p |scale (code - 8)|: at most 2^-11 times the sum
of p max(|v|, |scale (code - 8)|).  Everything else is 32 bits: scores of up to some tens come out within 2^-18, which multiplies a weight by
at most 1 + 2^-17.  Where many rows share tiles the dequantised k and v are rounded to fp16 as well: another 2^-11 of sum p |v|, and a score
is off by 2^-11 sum |q k| scale at most.  attention_bound() is that sum."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import kv4_util as kv

pytestmark = pytest.mark.gpu

HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
TINY = {"bf16": 0.0, "fp16": 2.0 ** -25}               # half a step below fp16's normal range


def host(t):
    return t.double().cpu().numpy()


def attention_bound(dtype, ref, size, q, k, scale, shared_tiles=False):
    """q [n, heads, d], k [kv heads, L, d] -> [n, heads, d]."""
    rel = 2.0 ** -11 + 2.0 ** -16
    if shared_tiles:
        kmax = np.abs(k).max(axis=1) if k.shape[1] else np.zeros((k.shape[0], k.shape[2]))
        g = q.shape[1] // k.shape[0]
        ds = scale * 2.0 ** -11 * (np.abs(q) * kmax.repeat(g, 0)[None]).sum(-1, keepdims=True)
        rel = rel + 2.0 ** -11 + np.expm1(2 * ds)
    return HALF_STEP[dtype] * np.abs(ref) + rel * size * (1 + HALF_STEP[dtype]) + TINY[dtype]


# ---- append ----------------------------------------------------------------------------------------------------------------
def append_reference(c, x, kw, rows, q_heads):
    """Normed and turned heads of the projected rows [n, heads, d]; v heads as they are."""
    y = x.copy()
    qk = q_heads + c.kh
    if kw.get("norm"):
        y[:, :q_heads] = kv.normed(x[:, :q_heads], kw["norm_eps"], host(kw["q_norm"]) if "q_norm" in kw else 1.0)
        y[:, q_heads:qk] = kv.normed(x[:, q_heads:qk], kw["norm_eps"], host(kw["k_norm"]) if "k_norm" in kw else 1.0)
    if kw.get("rot_dims"):
        pos, freq = kw["positions"].cpu().numpy().reshape(kw["axes"], -1), kw["inv_freq"].cpu().numpy()
        for i in range(rows):
            y[i, :qk] = kv.turned(y[i, :qk], pos[:, i], freq, kw["rot_dims"], kw["rot_kind"], kw.get("sections") if kw["axes"] == 3 else None)
    return y


def check_snapped(got, want, dtype):
    """got [n, heads, d] rounded values against unrounded 64-bit ones: equal to rounding, or one code off where the code lay on a border."""
    ok = np.zeros(got.shape, bool)
    for ds, dl in ((0, 0), (1e-6, 0), (-1e-6, 0), (0, 1e-6), (0, -1e-6)):          # scale and minimum may lie on a border of their own rounding
        raw, codes, scale, low = kv.snap(want, ds, dl)
        near = np.abs(raw - np.floor(raw) - 0.5) < 1e-3          # 32-bit arithmetic may fall on the other side
        for step in (0, -1, 1):
            val = kv.values(np.clip(codes + step, 0, 15), scale, low)
            fits = np.abs(got - val) <= HALF_STEP[dtype] * np.abs(val) + TINY[dtype] + 1e-6 * np.repeat(scale, 64, -1)
            ok |= fits & (near if step else True)
    _, codes, scale, low = kv.snap(want)
    assert ok.mean() == 1.0, (np.argwhere(~ok)[:5], got[~ok][:5], want[~ok][:5])
    exact = np.abs(got - kv.values(codes, scale, low)) <= HALF_STEP[dtype] * np.abs(got) * 1.01 + TINY[dtype] + 1e-6 * np.repeat(scale, 64, -1)
    assert exact.mean() > 0.995                                   # borders are rare


APPEND = [
    # q heads, kv heads, d, dtype, held, counts, norm, rot_dims, kind, axes
    (14, 2, 64, "bf16", [0], [1], False, 64, 0, 1),
    (28, 4, 128, "bf16", [63, 0, 64], [2, 0, 130], False, 128, 0, 3),
    (32, 8, 128, "fp16", [5, 200, 1, 0], [1, 7, 64, 1], True, 96, 1, 1),
    (5, 5, 64, "fp16", [10, 127], [65, 1], True, 32, 1, 3),
    (7, 1, 128, "bf16", [100], [3], True, 16, 0, 1),
    (3, 3, 128, "bf16", [0, 0, 0], [0, 0, 1], False, 0, 0, 1),
]


@pytest.mark.parametrize("qh,kh,d,dtype,held,counts,norm,rot,kind,axes", APPEND)
@pytest.mark.parametrize("weights", [True, False])
def test_append(qh, kh, d, dtype, held, counts, norm, rot, kind, axes, weights):
    full = [h + n for h, n in zip(held, counts)]
    c = kv.KV4(qh, kh, d, held, full, dtype, seed=qh + d).fill()
    before = c.pool.clone()
    n, pad = sum(counts), 2
    R = n + pad
    x = c.normal(R, (qh + 2 * kh) * d + 8, scale=1.5)                       # rows of another stride
    x[0, qh * d] = 40.0                                                       # a loud channel
    qo = torch.full((R, qh, d), 7.0, dtype=c.dtype, device=c.dev)
    ko, vo = (torch.full((R, kh, d), 7.0, dtype=c.dtype, device=c.dev) for _ in range(2))
    kw = dict(norm=int(norm), norm_eps=1e-6, rot_dims=rot, rot_kind=kind, axes=axes)
    if norm and weights:
        kw.update(q_norm=c.normal(d) * 0.1 + 1, k_norm=c.normal(d) * 0.1 + 1)
    half = rot // 2
    if rot:
        freq = torch.tensor([1e4 ** (-i / half) for i in range(half)], dtype=torch.float64, device=c.dev)
        kw.update(inv_freq=freq, positions=c.ints(c.rng.integers(0, 200000, axes * R)))
        if axes == 3:
            kw["sections"] = (half // 4, half // 4, half - 2 * (half // 4))
    tok = c.ints(c.rng.integers(0, 10 ** 6, R))
    if weights:
        kw["token_index"] = tok
    lens_out = torch.full((len(held),), -3, dtype=torch.int32, device=c.dev)
    q, k, v = x[:, :qh * d], x[:, qh * d:(qh + kh) * d], x[:, (qh + kh) * d:(qh + 2 * kh) * d]
    c.do("append", c.append_args(counts, lens_out, q, k, v, R, q_out=qo, k_held=ko, v_held=vo, index=c.index, mass=c.mass, **kw))
    torch.cuda.synchronize()
    assert lens_out.tolist() == full and c.status.item() == 0
    y = append_reference(c, host(x[:, :(qh + 2 * kh) * d]).reshape(R, -1, d), kw, n, qh)
    got = host(qo)
    assert (got[n:] == 7.0).all() and (host(ko)[n:] == 7.0).all() and (host(vo)[n:] == 7.0).all()       # rows behind the last sequence
    assert (np.abs(got[:n] - y[:n, :qh]) <= HALF_STEP[dtype] * np.abs(y[:n, :qh]) + 1e-5).all()
    check_snapped(host(ko)[:n], y[:n, qh:qh + kh], dtype)
    check_snapped(host(vo)[:n], y[:n, qh + kh:], dtype)
    # the tiles hold what was reported, every other byte is as it was
    expect = before.cpu().numpy()
    now = c.pool.cpu().numpy()
    row = 0
    for b, (h0, m) in enumerate(zip(held, counts)):
        kk, vv = c.held(b, full[b])
        for i in range(m):
            for t, o in ((kk, ko), (vv, vo)):
                val, rep = t[:, h0 + i], host(o)[row]
                assert (np.abs(val - rep) <= HALF_STEP[dtype] * np.abs(val) * (1 + 1e-6) + TINY[dtype]).all()
            page, r = c.np_table[b, (h0 + i) // 64], (h0 + i) % 64
            for (a, e) in kv.parts(d):
                w = (e - a) // 64
                expect[page, :, a + r * w:a + (r + 1) * w] = now[page, :, a + r * w:a + (r + 1) * w]
            row += 1
        idx, ms = c.rows_of(c.index, b, full[b]), c.rows_of(c.mass, b, full[b])
        assert (ms[:, h0:] == 0).all() and np.isnan(ms[:, :h0]).all() and (idx[:, :h0] == -1).all()
        want = tok.cpu().numpy()[row - m:row] if weights else np.arange(h0, full[b])
        assert (idx[:, h0:] == want[None]).all()
    assert (now == expect).all()


def test_append_is_the_same_whatever_the_launch():
    """All rows at once, row by row, and without q: the same bytes."""
    qh, kh, d, n = 12, 2, 128, 600
    c = kv.KV4(qh, kh, d, [0], [n], "bf16", seed=3)
    x = c.normal(n, (qh + 2 * kh) * d)
    freq = torch.tensor([1e6 ** (-i / 64) for i in range(64)], dtype=torch.float64, device=c.dev)
    pos = c.ints(np.arange(n) * 97)
    w = c.normal(d) * 0.2 + 1
    pools, qs = [], []
    for way in range(3):
        c.pool.fill_(255)
        qo = torch.zeros(n, qh, d, dtype=c.dtype, device=c.dev)
        if way != 1:
            out = c.ints([0])
            a = c.append_args([n], out, x[:, :qh * d] if way == 0 else None, x[:, qh * d:(qh + kh) * d], x[:, (qh + kh) * d:], norm=1, norm_eps=1e-5, q_norm=w, k_norm=w,
                              rot_dims=128, axes=1, inv_freq=freq, positions=pos, **({"q_out": qo} if way == 0 else {}))
            c.do("append", a)
        else:
            start = c.lens
            for i in range(n):
                out = c.ints([0])
                xi, p = x[i:i + 1], pos[i:i + 1]
                c.do("append", c.append_args([1], out, xi[:, :qh * d], xi[:, qh * d:(qh + kh) * d], xi[:, (qh + kh) * d:], norm=1, norm_eps=1e-5, q_norm=w, k_norm=w,
                                             rot_dims=128, axes=1, inv_freq=freq, positions=p, q_out=qo[i:i + 1]))
                c.lens = out
            c.lens = start
            assert out.item() == n
        pools.append(c.pool.clone())
        qs.append(qo)
    assert torch.equal(pools[0], pools[1]) and torch.equal(pools[0], pools[2]) and torch.equal(qs[0], qs[1])


def test_append_values_that_no_code_can_hold():
    c = kv.KV4(1, 1, 64, [0], [4], "bf16")
    x = torch.zeros(4, 64 * 3, dtype=torch.bfloat16, device=c.dev)
    x[0, 64:] = 5.5                                        # constant: the minimum alone
    x[1, 64:] = float("nan")
    x[2, 70], x[2, 71], x[2, 140] = float("inf"), float("-inf"), 3e38
    x[3, 64:66] = 1e-9
    ko, vo = (torch.empty(4, 1, 64, dtype=torch.bfloat16, device=c.dev) for _ in range(2))
    out = c.ints([0])
    c.do("append", c.append_args([4], out, None, x[:, 64:128], x[:, 128:], k_held=ko, v_held=vo))
    k, v = host(ko)[:, 0], host(vo)[:, 0]
    assert (k[0] == 5.5).all() and (v[0] == 5.5).all() and (k[1] == 0).all() and np.isfinite(k).all() and np.isfinite(v).all()
    for val, lim in ((k[2, 6], 65504), (k[2, 7], -65504), (v[2, 12], 65504)):
        assert abs(val - lim) <= 65504 * 2 / 15
    assert np.abs(k[3]).max() <= 2.0 ** -24
    check_snapped(k[:, None], host(x)[:, None, 64:128], "bf16")


def test_append_full_cache_and_bad_pages():
    c = kv.KV4(2, 1, 64, [60, 64], [64, 64], "bf16").fill()
    before = c.pool.clone()
    x = c.normal(12, 64 * 4)
    qo = torch.zeros(12, 2, 64, dtype=c.dtype, device=c.dev)
    out = c.ints([0, 0])
    c.do("append", c.append_args([8, 4], out, x[:, :128], x[:, 128:192], x[:, 192:], q_out=qo, index=c.index, mass=c.mass))
    assert out.tolist() == [64, 64] and c.status.item() == kv.FULL
    changed = (c.pool != before).any(-1).nonzero().tolist()
    assert changed == [[int(c.np_table[0, 0]), 0]]                         # four rows stored, the rest dropped
    assert torch.equal(qo.view(12, 128), x[:, :128])                       # q of dropped rows all the same
    for wrong in (-1, c.n_pages, 2 ** 31 - 1):
        c.status.zero_()
        c.pool.copy_(before)
        c.table[1, 0] = wrong
        c.lens = c.ints([60, 3])
        c.do("append", c.append_args([1, 1], out, x[:2, :128], x[:2, 128:192], x[:2, 192:], q_out=qo[:2]))
        assert c.status.item() == kv.BAD_PAGE and out.tolist() == [61, 4]
        assert (c.pool != before).any(-1).nonzero().tolist() == [[int(c.np_table[0, 0]), 0]]
    c.status.zero_()
    c.lens = c.ints([-5, 1000])
    c.do("append", c.append_args([0, 0], out, x[:2, :128], x[:2, 128:192], x[:2, 192:], max_rows=2, q_out=qo[:2]))
    assert out.tolist() == [0, 64] and c.status.item() == kv.BAD_COUNT


# ---- attention -------------------------------------------------------------------------------------------------------------
def run_attention(c, counts, lens, dtype, mass=False, pad=2, max_len=0, shared_tiles=False, q_scale=1.0, **over):
    n = sum(counts)
    R = n + pad
    c.lens_t = c.ints(lens)
    q = c.normal(R, c.qh, c.d, scale=q_scale)
    out = torch.full((R, c.qh, c.d), 9.0, dtype=c.dtype, device=c.dev)
    m_in = torch.rand(c.n_pages, c.kh, 64, device=c.dev) if mass else None
    m_out = torch.full_like(m_in, -1.0) if mass else None
    a = c.attention_args(counts, c.lens_t, q, out, R, max_len, mass=m_in, mass_out=m_out, **over)
    c.do("attention", a)
    torch.cuda.synchronize()
    assert c.status.item() == 0
    got, row = host(out), 0
    assert (got[n:] == 9.0).all()
    scale = 1.0 / math.sqrt(c.d)
    touched = np.zeros((c.n_pages, 64), bool)
    for b, (m, L) in enumerate(zip(counts, lens)):
        k, v = c.held(b, L)
        x = host(q[row:row + m])
        ref, w, size = kv.attend(x, k, v, scale, c.spread(b, L))
        if m and L:
            off = np.abs(got[row:row + m] - ref)
            bound = attention_bound(dtype, ref, size, x, k, scale, shared_tiles)
            assert (off <= bound).all(), (b, L, m, float((off / np.maximum(bound, 1e-30)).max()), np.argwhere(off > bound)[:4])
        if m:
            assert (got[row:row + m][[i for i in range(m) if L - m + i < 0]] == 0).all()
        if mass and L:
            g = c.qh // c.kh
            want = c.rows_of(m_in, b, L).astype(np.float64) + w.reshape(c.kh, g * m, L).sum(1)
            have = c.rows_of(m_out, b, L)
            assert np.abs(have - want).max() <= 2.0 ** -15 * max(1.0, np.abs(want).max()), (b, np.abs(have - want).max())
            for r in range(L):
                touched[c.np_table[b, r // 64], r % 64] = True
        row += m
    if mass:
        assert (m_out.cpu().numpy().swapaxes(1, 2)[~touched] == -1.0).all()
    return q, out, m_in, m_out, a


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 1000]


@pytest.mark.parametrize("qh,kh,d,dtype", [(14, 2, 64, "bf16"), (28, 4, 128, "bf16"), (8, 8, 128, "fp16"), (16, 1, 64, "fp16"), (12, 1, 128, "bf16"), (40, 2, 128, "fp16")])
@pytest.mark.parametrize("mass", [False, True])
def test_attention_single_tokens(qh, kh, d, dtype, mass):
    c = kv.KV4(qh, kh, d, LENGTHS, None, dtype, seed=qh * d).fill()
    run_attention(c, [1] * len(LENGTHS), LENGTHS, dtype, mass, max_len=max(LENGTHS))
    run_attention(c, [1] * len(LENGTHS), LENGTHS, dtype, mass, q_scale=6.0)              # peaked weights; split sized by the table


@pytest.mark.parametrize("qh,kh,d,dtype", [(14, 2, 64, "bf16"), (28, 4, 128, "bf16"), (6, 6, 128, "fp16"), (20, 1, 64, "fp16")])
def test_attention_few_rows_and_rows_that_see_nothing(qh, kh, d, dtype):
    counts, lens = [2, 0, 3, 1, 5, 4, 2, 0], [70, 40, 3, 0, 2, 200, 64, 0]                 # 5 rows on 2 cached ones, 1 on none, none at all
    c = kv.KV4(qh, kh, d, lens, None, dtype, seed=d).fill()
    many = max(counts) * qh // kh > 32                       # one of the sequences is dealt as many rows
    run_attention(c, counts, lens, dtype, True, shared_tiles=many)
    run_attention(c, counts, lens, dtype, False, shared_tiles=many)


@pytest.mark.parametrize("qh,kh,d,dtype", [(14, 2, 64, "bf16"), (28, 4, 128, "bf16"), (4, 4, 128, "fp16"), (8, 1, 64, "fp16")])
@pytest.mark.parametrize("mass", [False, True])
def test_attention_portions(qh, kh, d, dtype, mass):
    counts, lens = [150, 1, 64, 0, 33, 128], [150, 333, 65, 20, 500, 100]
    c = kv.KV4(qh, kh, d, lens, None, dtype, seed=3).fill()
    run_attention(c, counts, lens, dtype, mass, shared_tiles=True)


def test_attention_scales_of_every_size():
    """Values and scales from the smallest fp16 to the largest: no weight overflows, none is lost."""
    c = kv.KV4(4, 1, 64, [200, 130], None, "bf16", seed=9).fill()
    pool = c.pool.cpu().numpy()
    for b, f in ((0, 1.0), (1, 2.0 ** -18)):
        for j, page in enumerate(c.np_table[b, :4 if b == 0 else 3]):
            a, e = kv.parts(64)[3]
            par = np.ascontiguousarray(pool[page, :, a:e]).view(np.float16).reshape(1, 64, 2)
            par[..., 0] = (f * (1.0 if b else 10.0 ** (j - 1)) * np.linspace(0.5, 400.0, 64)[None]).astype(np.float16)
            with np.errstate(over="ignore"):               # only behind the rows held
                par[..., 1] = -par[..., 0] * np.float16(7.0)
            pool[page, :, a:e] = par.view(np.uint8).reshape(1, -1)
    c.pool.copy_(torch.from_numpy(pool))
    run_attention(c, [1, 1], [200, 130], "bf16", True)
    run_attention(c, [40, 50], [200, 130], "bf16", False, shared_tiles=True)


def test_attention_large_and_small_queries():
    c = kv.KV4(6, 2, 128, [100], None, "bf16", seed=4).fill()
    for s in (1e-30, 1e-4, 300.0, 1e6):
        n = 1
        q = c.normal(n, 6, 128, scale=s)
        out = torch.zeros_like(q)
        lens = c.ints([100])
        c.do("attention", c.attention_args([1], lens, q, out, 1))
        ref, _, size = kv.attend(host(q), *c.held(0, 100), 1.0 / math.sqrt(128), c.spread(0, 100))
        if s < 1000:                                       # scores of thousands: only the order of the two largest counts
            slack = 2.0 ** -18 * max(1.0, s * 30)
            assert (np.abs(host(out) - ref) <= HALF_STEP["bf16"] * np.abs(ref) + (2.0 ** -11 + 2 * slack) * size).all()
        assert torch.isfinite(out.float()).all()


def test_attention_offsets_beyond_32_bits():
    d, kh = 128, 8
    pages = (1 << 32) // (kh * kv.tile_bytes(d)) + 40
    c = kv.KV4(16, kh, d, [130, 64], None, "bf16", seed=1, n_pages=pages).fill()
    assert int(c.np_table.max()) * kh * kv.tile_bytes(d) > 1 << 32
    run_attention(c, [1, 3], [130, 64], "bf16", False)
    x = c.normal(2, 32 * d)
    ko = torch.zeros(2, kh, d, dtype=c.dtype, device=c.dev)
    out = c.ints([0, 0])
    c.lens = c.ints([129, 63])
    c.do("append", c.append_args([1, 1], out, None, x[:, 16 * d:24 * d], x[:, 24 * d:], k_held=ko))
    for b, n in ((0, 130), (1, 64)):
        assert np.abs(c.held(b, n)[0][:, -1] - host(ko)[b]).max() < 0.05


def test_attention_bad_pages_and_counts():
    c = kv.KV4(4, 2, 64, [200, 64], None, "bf16", seed=2).fill()
    q = c.normal(2, 4, 64)
    out = torch.zeros_like(q)
    lens = c.ints([200, 64])
    m_in = torch.zeros(c.n_pages, 2, 64, device=c.dev)
    for wrong in (-1, c.n_pages, -2 ** 31):
        c.status.zero_()
        c.table[0, 1] = wrong
        m_out = torch.full_like(m_in, -1.0)
        c.do("attention", c.attention_args([1, 1], lens, q, out, mass=m_in, mass_out=m_out))
        assert c.status.item() == kv.BAD_PAGE
        kk, vv = c.held(1, 64)
        ref = kv.attend(host(q[1:]), kk, vv, 0.125)[0]
        assert np.abs(host(out[1:]) - ref).max() < 0.02               # the other sequence is whole
        c.table[0, 1] = int(c.np_table[0, 1])
        k, v = c.held(0, 200)
        stay = [r for r in range(200) if r // 64 != 1]
        ref, w, _ = kv.attend(host(q[:1]), k[:, stay], v[:, stay], 0.125)
        assert np.abs(host(out[:1]) - ref).max() < 0.02               # the page's rows count as absent
        got = c.rows_of(m_out, 0, 200)
        assert (got[:, 64:128] == -1.0).all() and np.abs(got[:, stay] - w[:, 0].reshape(2, 2, -1).sum(1)).max() < 1e-4
    c.status.zero_()
    c.do("attention", c.attention_args([1, 1], c.ints([-3, 5000]), q, out))
    assert c.status.item() == kv.BAD_COUNT | kv.BAD_PAGE and (host(out[0]) == 0).all()      # cut to the table, whose last columns name no page


def test_attention_is_the_same_every_time():
    for counts in ([1, 1, 1], [40, 3, 100]):
        lens = [700, 64, 300]
        c = kv.KV4(28, 4, 128, lens, None, "bf16", seed=5).fill()
        q, out, m_in, m_out, a = run_attention(c, counts, lens, "bf16", True, shared_tiles=True)
        first = (out.clone(), m_out.clone())
        for _ in range(3):
            out.fill_(9.0)
            c.do("attention", a)
            assert torch.equal(out, first[0]) and torch.equal(m_out, first[1])
        in_place = m_in.clone()
        c.do("attention", c.attention_args(counts, c.lens_t, q, out, q.shape[0], mass=in_place))
        for b, L in enumerate(lens):
            assert np.array_equal(c.rows_of(in_place, b, L), c.rows_of(first[1], b, L))


# ---- eviction --------------------------------------------------------------------------------------------------------------
def set_rows(c, t, b, rows):
    """rows [kv heads, n] into t [pages, kv heads, 64]."""
    n = rows.shape[1]
    for k in range(-(-n // 64)):
        t[int(c.np_table[b, k]), :, :min(64, n - 64 * k)] = torch.from_numpy(np.ascontiguousarray(rows[:, 64 * k:64 * k + 64])).to(t)


def run_evict(c, lens, index, mass, budget, limit, keep_first, keep_last, in_place):
    for b, n in enumerate(lens):
        if n:
            set_rows(c, c.index, b, index[b])
            set_rows(c, c.mass, b, mass[b])
    before = [c.held(b, n) for b, n in enumerate(lens)]
    idx_before, mass_before, pool_before = c.index.clone(), c.mass.clone(), c.pool.clone()
    io = c.index if in_place else torch.full_like(c.index, -5)
    mo = c.mass if in_place else torch.full_like(c.mass, -5.0)
    out = c.ints([0] * len(lens))
    c.do("evict", c.evict_args(c.ints(lens), out, budget, limit, keep_first, keep_last, None if in_place else io, None if in_place else mo))
    torch.cuda.synchronize()
    assert c.status.item() == 0
    assert out.tolist() == [budget if n > limit else n for n in lens]
    for b, n in enumerate(lens):
        left = budget if n > limit else n
        now, gi, gm = c.held(b, left), c.rows_of(io, b, left), c.rows_of(mo, b, left)
        for h in range(c.kh):
            rows = kv.evicted(index[b][h], mass[b][h], budget, keep_first, keep_last) if n > limit else list(range(n))
            assert gi[h].tolist() == [index[b][h][r] for r in rows], (b, h)
            assert np.array_equal(gm[h], mass[b][h][rows].astype(np.float32), equal_nan=True)
            for x, y in zip(now, before[b]):
                assert np.array_equal(x[h], y[h, rows])
        if n > limit:                                            # rows behind the budget are as they were
            for t, old in ((c.held(b, n)[0], before[b][0]), (c.held(b, n)[1], before[b][1])):
                assert np.array_equal(t[:, budget:], old[:, budget:])
            fill_i, fill_m = (c.rows_of(idx_before, b, n), c.rows_of(mass_before, b, n)) if in_place else (np.full((c.kh, n), -5), np.full((c.kh, n), -5.0))
            assert np.array_equal(c.rows_of(io, b, n)[:, budget:], fill_i[:, budget:]) and np.array_equal(c.rows_of(mo, b, n)[:, budget:], fill_m[:, budget:], equal_nan=True)
    used = {int(p) for b, n in enumerate(lens) for p in c.np_table[b, :-(-n // 64)]}
    other = [p for p in range(c.n_pages) if p not in used]
    assert torch.equal(c.pool[other], pool_before[other])


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kh,d,lens,budget,limit,first,last", [
    (2, 64, [100, 65, 64, 0, 1], 64, 64, 4, 16), (1, 128, [300, 1000], 1, 1, 0, 0), (3, 128, [700, 699, 130], 129, 600, 2, 50),
    (2, 64, [2500], 2000, 2000, 100, 300), (2, 128, [90], 89, 89, 0, 1), (1, 64, [500], 40, 60, 30, 30)])
def test_evict(kh, d, lens, budget, limit, first, last, in_place):
    c = kv.KV4(kh, kh, d, lens, [max(n, 1) for n in lens], "bf16", seed=budget).fill()
    index, mass = [], []
    for n in lens:
        index.append(np.stack([c.rng.permutation(3 * n + 1)[:n] for _ in range(kh)]).astype(np.int32))
        mass.append((c.rng.random((kh, n)) ** 6 * 30).astype(np.float32))
    run_evict(c, lens, index, mass, budget, limit, first, last, in_place)


@pytest.mark.parametrize("in_place", [True, False])
def test_evict_ties_and_odd_masses(in_place):
    n, kh = 900, 4
    c = kv.KV4(kh, kh, 64, [n], None, "bf16", seed=8).fill()
    index = np.tile(np.arange(n, dtype=np.int32), (kh, 1))
    mass = np.zeros((kh, n), np.float32)
    mass[1] = c.rng.integers(0, 3, n)                                # few distinct values: ties at the border
    mass[2] = c.rng.random(n)
    mass[2][::7], mass[2][::11], mass[2][3::50] = np.nan, np.inf, -np.inf
    mass[3] = np.where(np.arange(n) % 2, -0.0, 0.0)                  # equal numbers of two signs
    mass[3][500:] = np.float32(1e-42)                                # below the normal range
    for budget, first, last in ((300, 0, 0), (500, 10, 450), (128, 200, 0)):
        run_evict(c, [n], [index], [mass], budget, budget, first, last, in_place)
        c.fill()


def test_evict_longer_than_shared_memory_holds():
    n = 70000
    c = kv.KV4(1, 1, 64, [n], None, "bf16", seed=6)
    c.pool.random_(0, 256)
    a, e = kv.parts(64)[1]
    c.pool[:, :, a:e] = 0
    a, e = kv.parts(64)[3]
    c.pool[:, :, a:e] = 0                                             # finite parameters
    index = np.arange(n, dtype=np.int32)[None]
    mass = c.rng.integers(0, 5000, (1, n)).astype(np.float32)
    for page, rows in enumerate(np.array_split(np.arange(1094 * 64), 1094)):
        rows = rows[rows < n]
        c.index[int(c.np_table[0, page]), 0, :len(rows)] = torch.from_numpy(index[0, rows]).to(c.dev)
        c.mass[int(c.np_table[0, page]), 0, :len(rows)] = torch.from_numpy(mass[0, rows]).to(c.dev)
    before = c.pool[c.table[0].long()].clone()
    out = c.ints([0])
    c.do("evict", c.evict_args(c.ints([n]), out, 9000, 9000, 5, 1000))
    rows = kv.evicted(index[0], mass[0], 9000, 5, 1000)
    assert c.rows_of(c.index, 0, 9000)[0].tolist() == rows and np.array_equal(c.rows_of(c.mass, 0, 9000)[0], mass[0, rows])
    after = c.pool[c.table[0].long()]
    w = 64 // 2
    old, new = (t[:, 0, :64 * w].reshape(-1, w).cpu().numpy() for t in (before, after))
    assert np.array_equal(new[:9000], old[rows])


def test_evict_bad_pages():
    n = 256
    c = kv.KV4(1, 1, 64, [n], None, "bf16", seed=8).fill()
    set_rows(c, c.index, 0, np.arange(n, dtype=np.int32)[None])
    set_rows(c, c.mass, 0, np.ones((1, n), np.float32))
    c.table[0, 0] = c.n_pages + 5
    others, out = c.pool.clone(), c.ints([0])
    c.do("evict", c.evict_args(c.ints([n]), out, 200, 200, 0, 0))
    assert c.status.item() == kv.BAD_PAGE and out.item() == 200
    assert torch.equal(c.pool[int(c.np_table[0, 0])], others[int(c.np_table[0, 0])])


# ---- read, and all of them together ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("kh,d,dtype", [(2, 64, "bf16"), (5, 128, "fp16"), (1, 128, "bf16")])
def test_read(kh, d, dtype):
    lens = [200, 0, 64, 1, 130]
    c = kv.KV4(kh, kh, d, lens, None, dtype, seed=d).fill()
    for first, rows in ((0, 200), (0, 64), (63, 3), (64, 100), (130, 500), (0, 1), (5, 0), (10 ** 6, 4)):
        k, v = (torch.full((len(lens), rows, kh, d), 3.0, dtype=c.dtype, device=c.dev) for _ in range(2))
        r = kv.Read(C.sizeof(kv.Read), first, rows, 0, c.lens.data_ptr(), k.data_ptr() or c.lens.data_ptr(), v.data_ptr() or None)
        if rows == 0:
            r.k_out = c.pool.data_ptr()
        c.do("read", r)
        for b, n in enumerate(lens):
            m = max(0, min(n, first + rows) - first)
            for got, want in zip((k, v), c.held(b, n)):
                w = want[:, first:first + m].swapaxes(0, 1)
                assert (np.abs(host(got)[b, :m] - w) <= HALF_STEP[dtype] * np.abs(w) * (1 + 1e-6) + TINY[dtype] + 1e-7).all()
                assert (host(got)[b, m:] == 3.0).all()
    v = torch.full((len(lens), 64, kh, d), 3.0, dtype=c.dtype, device=c.dev)
    c.do("read", kv.Read(C.sizeof(kv.Read), 0, 64, 0, c.lens.data_ptr(), None, v.data_ptr()))
    assert np.abs(host(v)[0] - c.held(0, 64)[1].swapaxes(0, 1)).max() < 0.05
    c.table[0, 0] = -1
    c.do("read", kv.Read(C.sizeof(kv.Read), 0, 64, 0, c.lens.data_ptr(), None, v.data_ptr()))
    assert c.status.item() == kv.BAD_PAGE


class Loop:
    """Decoding with a budget: append, attend with weights, evict; buffers stay where they are, so that a step can be captured."""

    def __init__(self, qh=8, kh=2, d=64, batch=3, budget=100, limit=140, dtype="bf16", seed=0, device="cuda:0"):
        self.c = c = kv.KV4(qh, kh, d, [0] * batch, [limit + 64] * batch, dtype, seed=seed, device=device)
        self.budget, self.limit, self.batch = budget, limit, batch
        self.a, self.b = c.ints([0] * batch), c.ints([0] * batch)
        self.x = torch.zeros(batch, (qh + 2 * kh) * d, dtype=c.dtype, device=c.dev)
        self.q, self.out = (torch.zeros(batch, qh, d, dtype=c.dtype, device=c.dev) for _ in range(2))
        self.pos = c.ints([0] * batch)
        self.freq = torch.tensor([1e4 ** (-i / (d // 2)) for i in range(d // 2)], dtype=torch.float64, device=c.dev)
        c.lens = self.a
        x = self.x
        self.append = c.append_args([1] * batch, self.b, x[:, :qh * d], x[:, qh * d:(qh + kh) * d], x[:, (qh + kh) * d:], q_out=self.q, rot_dims=d, axes=1,
                                    inv_freq=self.freq, positions=self.pos, token_index=self.pos, index=c.index, mass=c.mass)
        cu = c.cu
        self.attend = c.attention_args([1] * batch, self.b, self.q, self.out, mass=c.mass)
        self.cu = (cu, c.cu)
        self.evict = c.evict_args(self.b, self.a, budget, limit, 4, 16)

    def step(self):
        self.c.do("append", self.append)
        self.c.do("attention", self.attend)
        self.c.do("evict", self.evict)

    def feed(self, t, gen):
        self.x.copy_(torch.randn(self.x.shape, generator=gen, device=self.x.device))
        self.pos.fill_(t)


def state(lp):
    c, n = lp.c, lp.a.tolist()
    return [lp.out.clone()] + [torch.from_numpy(np.concatenate([c.rows_of(t, b, m).reshape(-1) for b, m in enumerate(n)])) for t in (c.index, c.mass)], n


def test_decoding_under_a_budget_eager_and_captured():
    """230 steps, five evictions: a captured step replayed gives bit for bit what the calls give, and both follow the plain statement."""
    eager, graph = Loop(seed=1), Loop(seed=1)
    c = eager.c
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        graph.step()
        s.synchronize()
        graph.a.zero_(); graph.b.zero_(); graph.c.mass.fill_(float("nan")); graph.c.index.fill_(-1); graph.c.pool.fill_(255)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            graph.step()
    torch.cuda.synchronize()
    gens = [torch.Generator(device="cuda").manual_seed(2) for _ in range(2)]
    model = [[dict(k=np.zeros((0, c.d)), v=np.zeros((0, c.d)), i=np.zeros(0, int), m=np.zeros(0)) for _ in range(c.kh)] for _ in range(eager.batch)]
    for t in range(230):
        eager.feed(t, gens[0])
        graph.feed(t, gens[1])
        n0 = eager.a.tolist()
        eager.step()
        g.replay()
        if t % 23 == 22 or t in (0, 1, 64):
            (o1, n1), (o2, n2) = state(eager), state(graph)
            assert n1 == n2 and all(torch.equal(x, y) for x, y in zip(o1, o2)), t
        # the statement, from the cache's own keys and values (what a row holds is test_append's matter)
        q = host(eager.q)
        for b in range(eager.batch):
            n = n0[b] + 1
            got = eager.a.tolist()[b]
            assert got == (eager.budget if n > eager.limit else n)
            if got == n and t % 10 == 0:
                k, v = c.held(b, n)
                ref, _, size = kv.attend(q[b:b + 1], k, v, 1 / 8, c.spread(b, n))
                assert (np.abs(host(eager.out)[b:b + 1] - ref) <= attention_bound("bf16", ref, size, q[b:b + 1], k, 1 / 8)).all()
    n = eager.a.tolist()
    assert eager.c.status.item() == 0 and n == [100 + (230 - 141) % 41] * 3
    for b in range(3):
        idx, ms = c.rows_of(c.index, b, n[b]), c.rows_of(c.mass, b, n[b])
        for h in range(c.kh):
            assert set(range(4)) <= set(idx[h]) and set(range(214, 230)) <= set(idx[h]) and len(set(idx[h])) == n[b]
        assert (ms >= 0).all() and (ms > 0).any()


def test_masses_of_a_run_add_up():
    """Without evictions every new row and q head hands out a weight of one."""
    lp = Loop(limit=200, budget=200, seed=5)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for t in range(150):
        lp.feed(t, gen)
        lp.step()
    for b in range(lp.batch):
        m = lp.c.rows_of(lp.c.mass, b, 150).astype(np.float64)
        assert np.abs(m.sum(1) - 150 * 4).max() < 1e-2


def test_two_streams_with_a_workspace_each():
    loops = [Loop(seed=s) for s in (3, 4)]
    alone = [Loop(seed=s) for s in (3, 4)]
    streams = [torch.cuda.Stream() for _ in loops]
    gens = [torch.Generator(device="cuda").manual_seed(7) for _ in range(4)]
    torch.cuda.synchronize()
    for t in range(60):
        for lp, s, g in zip(loops, streams, gens[:2]):
            with torch.cuda.stream(s):
                lp.feed(t, g)
                lp.step()
    torch.cuda.synchronize()
    for t in range(60):
        for lp, g in zip(alone, gens[2:]):
            lp.feed(t, g)
            lp.step()
    for a, b in zip(loops, alone):
        (x, n), (y, m) = state(a), state(b)
        assert n == m and all(torch.equal(u, w) for u, w in zip(x, y))


def test_portions_and_decoded_tokens_of_one_prompt_agree():
    """A prompt appended and attended whole, in portions of unequal length, and token by token: the same cache bytes, outputs to rounding."""
    qh, kh, d, n = 8, 2, 128, 150
    outs, pools = [], []
    for cuts in ([n], [64, 1, 37, 48], [1] * n):
        c = kv.KV4(qh, kh, d, [0], [n], "bf16", seed=2)
        x = torch.randn(n, (qh + 2 * kh) * d, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(torch.bfloat16)
        q, out = (torch.zeros(n, qh, d, dtype=c.dtype, device=c.dev) for _ in range(2))
        at = 0
        for m in cuts:
            lens_out = c.ints([0])
            xi = x[at:at + m]
            c.do("append", c.append_args([m], lens_out, xi[:, :qh * d], xi[:, qh * d:(qh + kh) * d], xi[:, (qh + kh) * d:], q_out=q[at:at + m]))
            c.do("attention", c.attention_args([m], lens_out, q[at:at + m], out[at:at + m]))
            c.lens = lens_out
            at += m
        outs.append(host(out))
        pools.append(c.pool.clone())
        k, v = c.held(0, n)
        ref, _, size = kv.attend(host(q), k, v, 1 / math.sqrt(d), c.spread(0, n))
        assert (np.abs(outs[-1] - ref) <= attention_bound("bf16", ref, size, host(q), k, 1 / math.sqrt(d), True)).all()
    assert torch.equal(pools[0], pools[1]) and torch.equal(pools[0], pools[2])


def test_empty_calls():
    c = kv.KV4(2, 1, 64, [10], None, "bf16").fill()
    x = c.normal(1, 64 * 4)
    out = c.ints([-1])
    a = c.append_args([0], out, x[:, :128], x[:, 128:192], x[:, 192:], max_rows=0)
    a.q = a.k = a.v = None
    c.do("append", a)
    assert out.item() == 10
    m = torch.rand(c.n_pages, 1, 64, device=c.dev)
    mo = torch.full_like(m, -1.0)
    q = c.normal(1, 2, 64)
    at = c.attention_args([0], c.lens, q, q, 0, mass=m, mass_out=mo, max_new=0)
    c.do("attention", at)
    assert np.array_equal(c.rows_of(mo, 0, 10), c.rows_of(m, 0, 10)) and (mo >= 0).sum().item() == 10
