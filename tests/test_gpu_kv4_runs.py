"""GPU: the operators of the 4-bit cache where sizes, batches and orders of calls change what is launched (helpers and tolerances: test_gpu_kv4)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import kv4_util as kv
from test_gpu_kv4 import HALF_STEP, attention_bound, host, run_attention, set_rows

pytestmark = pytest.mark.gpu

COUNTS, LENS = [70, 1, 64, 0, 33, 128, 26, 300], [70, 333, 65, 20, 500, 100, 26, 290]


@pytest.mark.parametrize("qh,kh,d,dtype", [(28, 4, 128, "bf16"), (28, 4, 128, "fp16"), (14, 7, 64, "bf16"), (12, 4, 64, "fp16"), (8, 8, 128, "fp16"), (40, 2, 128, "bf16")])
@pytest.mark.parametrize("mass", [False, True])
def test_attention_batches_of_portions(qh, kh, d, dtype, mass):
    """Enough sequences and rows that the longer portions go to the kernel for many rows and the shorter ones do not."""
    c = kv.KV4(qh, kh, d, LENS, None, dtype, seed=qh + d).fill()
    run_attention(c, COUNTS, LENS, dtype, mass, shared_tiles=True)


@pytest.mark.parametrize("qh,kh,d,dtype,counts,lens", [
    (64, 1, 128, "bf16", [1], [3001]), (192, 1, 64, "fp16", [2], [129]), (48, 1, 128, "fp16", [1] * 5, [1, 700, 64, 63, 130]), (28, 4, 128, "bf16", [60], [700]),
    (14, 2, 64, "bf16", [250], [900]), (1024, 1, 64, "bf16", [1, 4], [90, 10])])
@pytest.mark.parametrize("mass", [False, True])
def test_attention_wide_groups_and_short_portions(qh, kh, d, dtype, counts, lens, mass):
    c = kv.KV4(qh, kh, d, lens, None, dtype, seed=qh).fill()
    run_attention(c, counts, lens, dtype, mass, shared_tiles=True)


@pytest.mark.parametrize("counts,lens", [([128] * 8, [400 + 7 * i for i in range(8)]), ([128] * 8, [150, 150, 900, 150, 150, 150, 150, 150]), ([300, 2, 40], [2000, 2, 1200])])
@pytest.mark.parametrize("mass", [False, True])
def test_attention_even_and_uneven_blocks_of_rows(counts, lens, mass):
    """Blocks of rows of much the same length, which stay whole, and one far longer than the rest, which does not."""
    c = kv.KV4(16, 2, 128, lens, None, "bf16", seed=3).fill()
    run_attention(c, counts, lens, "bf16", mass, shared_tiles=True)


def test_attention_more_pages_than_a_warp_asks_for_at_once():
    """64 sequences of up to 7100 rows on the same pages: every warp has more than 32 of a row's."""
    B, kh, d, L = 64, 8, 64, 7100
    c = kv.KV4(16, kh, d, [L], None, "bf16", seed=4).fill()
    c.batch, c.np_table = B, np.tile(c.np_table, (B, 1))
    c.table = torch.from_numpy(c.np_table).to(c.dev)
    lens = [L - 13 * b for b in range(B)]
    q = c.normal(B, 16, d)
    out = torch.zeros_like(q)
    c.do("attention", c.attention_args([1] * B, c.ints(lens), q, out))
    assert c.status.item() == 0
    for b in (0, 17, 40, 63):
        k, v = c.held(b, lens[b])
        ref, _, size = kv.attend(host(q[b:b + 1]), k, v, 1 / 8, c.spread(b, lens[b]))
        assert (np.abs(host(out[b:b + 1]) - ref) <= attention_bound("bf16", ref, size, host(q[b:b + 1]), k, 1 / 8)).all()


@pytest.mark.parametrize("qh,kh,d", [(2, 1, 64), (6, 2, 128)])
def test_batches_of_hundreds(qh, kh, d):
    """300 sequences of unequal length, one new row each but every seventh, which has none or three."""
    B = 300
    lens = [(37 * b) % 201 for b in range(B)]
    counts = [1 if b % 7 else 3 * (b % 2) for b in range(B)]
    full = [a + n for a, n in zip(lens, counts)]
    c = kv.KV4(qh, kh, d, lens, [n + 70 for n in full], "bf16", seed=d).fill()
    n = sum(counts)
    x = c.normal(n, (qh + 2 * kh) * d)
    out, ko = c.ints([0] * B), torch.zeros(n, kh, d, dtype=c.dtype, device=c.dev)
    q = x[:, :qh * d].contiguous()
    c.do("append", c.append_args(counts, out, None, x[:, qh * d:(qh + kh) * d], x[:, (qh + kh) * d:], k_held=ko, index=c.index, mass=c.mass))
    assert out.tolist() == full
    row = 0
    for b in range(B):
        k = c.held(b, full[b])[0]
        for i in range(counts[b]):
            assert (np.abs(k[:, lens[b] + i] - host(ko[row])) <= HALF_STEP["bf16"] * np.abs(k[:, lens[b] + i]) * (1 + 1e-6)).all()
            row += 1
    run_attention(c, counts, full, "bf16", True)
    run_attention(c, counts, full, "bf16", False, max_len=max(full))
    for b in range(B):
        if full[b]:
            set_rows(c, c.index, b, np.tile(np.arange(full[b], dtype=np.int32), (kh, 1)))
            set_rows(c, c.mass, b, c.rng.random((kh, full[b])).astype(np.float32))
    mass = [c.rows_of(c.mass, b, full[b]) for b in range(B)]
    left = c.ints([0] * B)
    c.do("evict", c.evict_args(c.ints(full), left, 90, 120, 2, 9))
    assert left.tolist() == [90 if m > 120 else m for m in full]
    for b in range(B):
        m = left[b].item()
        for h in range(kh):
            rows = kv.evicted(np.arange(full[b]), mass[b][h], 90, 2, 9) if full[b] > 120 else list(range(full[b]))
            assert c.rows_of(c.index, b, m)[h].tolist() == rows
    k = torch.full((B, 90, kh, d), 3.0, dtype=c.dtype, device=c.dev)
    c.do("read", kv.Read(C.sizeof(kv.Read), 0, 90, 0, left.data_ptr(), k.data_ptr(), None))
    for b in range(0, B, 11):
        m = min(90, left[b].item())
        w = c.held(b, m)[0].swapaxes(0, 1)
        assert (np.abs(host(k[b, :m]) - w) <= HALF_STEP["bf16"] * np.abs(w) * (1 + 1e-6)).all() and (k[b, m:] == 3.0).all()
    assert c.status.item() == 0


class Chain:
    """append -> attention with weights -> evict with portions of any size; everything a step needs lies ready, so calls follow each other closely."""

    def __init__(self, counts, steps, qh=16, kh=2, d=64, budget=256, limit=320, dtype="bf16"):
        self.B, self.n, self.budget = len(counts), sum(counts), budget
        self.c = c = kv.KV4(qh, kh, d, [0] * self.B, [limit + max(counts)] * self.B, dtype, seed=7)
        self.a, self.b = c.ints([0] * self.B), c.ints([0] * self.B)
        c.lens = self.a
        self.xs = [c.normal(self.n, (qh + 2 * kh) * d) for _ in range(steps)]
        self.outs = [torch.zeros(self.n, qh, d, dtype=c.dtype, device=c.dev) for _ in range(steps)]
        self.calls = []
        for t in range(steps):
            x, q = self.xs[t], torch.zeros_like(self.outs[t])
            tok = c.ints(np.full(self.n, t))
            ap = c.append_args(counts, self.b, x[:, :qh * d], x[:, qh * d:(qh + kh) * d], x[:, (qh + kh) * d:], q_out=q, token_index=tok, index=c.index, mass=c.mass)
            self.calls.append((("append", ap), ("attention", c.attention_args(counts, self.b, q, self.outs[t], mass=c.mass)), ("evict", c.evict_args(self.b, self.a, budget, limit, 1, 2))))

    def run(self, between=lambda: None):
        c = self.c
        self.a.zero_(); self.b.fill_(3); c.mass.fill_(-1.0); c.index.fill_(-1); c.pool.fill_(255)
        torch.cuda.synchronize()
        for calls in self.calls:
            for name, args in calls:
                c.do(name, args)
                between()
        torch.cuda.synchronize()
        assert c.status.item() == 0
        n = self.a.tolist()
        return [o.clone() for o in self.outs] + [c.pool.clone()] + [torch.from_numpy(c.rows_of(t, b, m)) for t in (c.index, c.mass) for b, m in enumerate(n)], n


@pytest.mark.parametrize("counts,steps,kw", [
    ([1, 1, 1], 330, {}), ([3, 0, 2], 120, dict(dtype="fp16")), ([40, 3, 100], 12, dict(kh=16)), ([90] * 4, 10, dict(qh=32, kh=16, d=128)), ([90] * 6, 10, dict(qh=32, kh=16, dtype="fp16"))])
def test_calls_that_follow_each_other_see_what_was_before(counts, steps, kw):
    """Lengths, pages and sums come from the call before, which may still be running when the next is launched: the same as with a pause
    after every call, and the same again from a graph."""
    ch = Chain(counts, steps, **kw)
    apart, n0 = ch.run(torch.cuda.synchronize)
    assert max(n0) >= ch.budget
    for _ in range(3):
        close, n1 = ch.run()
        assert n0 == n1 and all(torch.equal(x, y) for x, y in zip(apart, close))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for calls in ch.calls:
                for name, args in calls:
                    ch.c.do(name, args)
    ch.calls, calls = [], ch.calls
    ch.run()                                                 # back to the beginning
    for o in ch.outs:
        o.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        g.replay()
    torch.cuda.synchronize()
    assert ch.c.status.item() == 0 and ch.a.tolist() == n0
    assert all(torch.equal(x, y) for x, y in zip(apart, ch.outs + [ch.c.pool]))
    ch.calls = calls


def test_no_new_rows_right_after_an_append():
    """A call that only hands its sums on must take the lengths that the append before it leaves."""
    c = kv.KV4(4, 2, 64, [0], [2000], "bf16", seed=1)
    x = c.normal(2000, 64 * 8)
    m_in = torch.rand(c.n_pages, 2, 64, device=c.dev)
    out = c.ints([0])
    ap = c.append_args([2000], out, None, x[:, 256:384], x[:, 384:])
    q = c.normal(1, 4, 64)
    m_out = torch.full_like(m_in, -1.0)
    for max_len in (0, 2000):
        at = c.attention_args([0], out, q, torch.zeros_like(q), 1, max_len=max_len, mass=m_in, mass_out=m_out, max_new=0)
        for _ in range(20):
            out.zero_(); m_out.fill_(-1.0)
            c.do("append", ap)
            c.do("attention", at)
            assert np.array_equal(c.rows_of(m_out, 0, 2000), c.rows_of(m_in, 0, 2000)) and int((m_out >= 0).sum()) == 4000


def test_captured_calls_that_share_a_workspace_in_turn():
    """A graph of a portion and one of single tokens on one stream and one workspace: either may come first."""
    lens = [500, 64, 700]
    c = kv.KV4(28, 4, 128, lens, None, "bf16", seed=5).fill()
    t_lens = c.ints(lens)
    made = []
    for counts in ([1, 1, 1], [120, 64, 200]):
        q = c.normal(sum(counts), 28, 128)
        m = torch.rand(c.n_pages, 4, 64, device=c.dev)
        made.append([c.attention_args(counts, t_lens, q, torch.zeros_like(q), mass=m, mass_out=torch.zeros_like(m)), None])
        made[-1][1] = c.keep[-5:]
    ws = torch.empty(max(a.workspace_bytes for a, _ in made), dtype=torch.uint8, device=c.dev)
    s = torch.cuda.Stream()
    want, graphs = [], []
    outs = [[k for k in keep if k is not None and k.dim() == 3][1:] for _, keep in made]          # (q,) out, (mass,) mass_out
    for (a, keep), o in zip(made, outs):
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        c.do("attention", a)
        torch.cuda.synchronize()
        want.append([t.clone() for t in o])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
            c.do("attention", a)
        graphs.append(g)
    for order in ((0, 1, 0, 0, 1, 1), (1, 0, 1, 1, 0, 0)):
        for t in (x for o in outs for x in (o[0], o[-1])):
            t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            for i in order:
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for o, w in zip(outs, want) for x, y in zip(o, w))


def test_many_rows_a_hundred_times_over():
    """Launches of the kernel for many rows one behind the other: the same every time, and no wait gives up."""
    c = kv.KV4(28, 4, 128, [900, 350, 128], None, "bf16", seed=2).fill()
    for counts in ([300, 350, 128], [640, 1, 127]):
        for mass in (None, torch.rand(c.n_pages, 4, 64, device=c.dev)):
            q = c.normal(sum(counts), 28, 128)
            outs = [torch.zeros_like(q) for _ in range(100)]
            m_out = torch.zeros_like(mass) if mass is not None else None
            args = c.attention_args(counts, c.lens, q, outs[0], mass=mass, mass_out=m_out)
            for o in outs:
                args.out = o.data_ptr()
                c.do("attention", args)
            torch.cuda.synchronize()
            assert c.status.item() == 0 and all(torch.equal(o, outs[0]) for o in outs)


def test_bad_pages_under_many_rows():
    c = kv.KV4(16, 16, 64, [300] * 6, None, "bf16", seed=3).fill()
    counts = [200] * 6
    q = c.normal(1200, 16, 64)
    m_in = torch.zeros(c.n_pages, 16, 64, device=c.dev)
    for wrong in (-1, c.n_pages, 2 ** 31 - 1):
        out, m_out = torch.zeros_like(q), torch.full_like(m_in, -1.0)
        c.status.zero_()
        c.table[0, 1] = wrong
        c.do("attention", c.attention_args(counts, c.lens, q, out, mass=m_in, mass_out=m_out))
        assert c.status.item() == kv.BAD_PAGE
        c.table[0, 1] = int(c.np_table[0, 1])
        k, v = c.held(0, 300)
        stay = [r for r in range(300) if r // 64 != 1]
        for i in (60, 199):                                      # rows that see all but a few of the pages
            see = [r for r in stay if r <= 100 + i]
            ref = kv.attend(host(q[i:i + 1]), k[:, see], v[:, see], 0.125)[0]
            assert np.abs(host(out[i:i + 1]) - ref).max() < 0.02
        ref = kv.attend(host(q[200:400]), *c.held(1, 300), 0.125)[0]
        assert np.abs(host(out[200:400]) - ref).max() < 0.02          # the other sequences are whole
        got = c.rows_of(m_out, 0, 300)
        assert (got[:, 64:128] == -1.0).all() and np.abs(got[:, stay].sum(1) - 200).max() < 1e-2


@pytest.mark.parametrize("counts,kh", [([1, 1, 1], 4), ([30, 1, 200], 4), ([130, 90, 200], 28)])
def test_queries_that_are_not_numbers_stay_with_their_rows(counts, kh):
    lens = [400, 90, 300]
    c = kv.KV4(28, kh, 128, lens, None, "bf16", seed=6).fill()
    n = sum(counts)
    q = c.normal(n, 28, 128)
    out = [torch.zeros_like(q) for _ in range(2)]
    c.do("attention", c.attention_args(counts, c.lens, q, out[0]))
    bad = torch.zeros(n, 28, dtype=torch.bool, device=c.dev)
    bad[0, 3] = bad[n - 1, 27] = bad[n // 2, 10] = True
    q[0, 3], q[n - 1, 27, 5], q[n // 2, 10, 7] = float("nan"), float("nan"), float("inf")
    c.do("attention", c.attention_args(counts, c.lens, q, out[1]))
    torch.cuda.synchronize()
    assert c.status.item() == 0 and torch.equal(out[0][~bad], out[1][~bad])
    assert torch.isnan(out[1][0, 3]).all() and torch.isnan(out[1][n - 1, 27]).all()


def test_counts_and_lengths_that_lie():
    """Row counts that fall, pass the buffers or max_new: cut to them, reported, nothing else is touched."""
    c = kv.KV4(8, 8, 64, [200] * 4, None, "bf16", seed=9).fill()
    for per, max_new in ((2, 2), (90, 90)):
        R = 4 * per
        q = c.normal(R, 8, 64)
        for cu, rows in (([0, per, 2 * per, 3 * per, 4 * per + 5], R), ([0, per, 0, per, 2 * per], 2 * per), ([-4, per, 2 * per, 3 * per, 4 * per], R), ([0, 2 * per, 2 * per, 2 * per, 2 * per], per)):
            out = torch.full_like(q, 9.0)
            a = c.attention_args([per] * 4, c.lens, q, out, max_new=max_new)
            cu_t = c.ints(cu)
            a.cu_rows = cu_t.data_ptr()
            c.status.zero_()
            c.do("attention", a)
            torch.cuda.synchronize()
            assert c.status.item() == kv.BAD_COUNT
            assert torch.isfinite(out.float()).all() and (out[rows:] == 9.0).all() and (out[:per] != 9.0).any()


def test_the_same_token_number_twice():
    """Token numbers need not be different: rows that share one are kept or ordered as rows."""
    n, kh = 400, 2
    c = kv.KV4(kh, kh, 64, [n], None, "bf16", seed=1).fill()
    index = np.stack([np.arange(n) // 5, np.full(n, 7)]).astype(np.int32)
    mass = c.rng.integers(0, 6, (kh, n)).astype(np.float32)
    set_rows(c, c.index, 0, index)
    set_rows(c, c.mass, 0, mass)
    out = c.ints([0])
    c.do("evict", c.evict_args(c.lens, out, 150, 150, 3, 4))
    for h in range(kh):
        rows = kv.evicted(index[h], mass[h], 150, 3, 4)
        assert c.rows_of(c.index, 0, 150)[h].tolist() == index[h][rows].tolist() and np.array_equal(c.rows_of(c.mass, 0, 150)[h], mass[h][rows])


def extreme(c, b, seed):
    """Every row of sequence b from values as large as fp16 goes: some groups span all of it, some lie at its upper end, some at its lower."""
    rng, d = np.random.default_rng(seed), c.d
    pages = c.np_table[b, :-(-c.lens.tolist()[b] // 64)]
    pool = c.pool.cpu().numpy()
    for page in pages:
        tile = np.full((c.kh, kv.tile_bytes(d)), 255, np.uint8)
        for key, (a, e), (p0, p1) in ((True, *kv.parts(d)[:2]), (False, *kv.parts(d)[2:])):
            x = rng.standard_normal((c.kh, 64, d // 64, 64))
            x = x / np.abs(x).max(-1, keepdims=True)
            kind = rng.integers(0, 4, (c.kh, 64, d // 64, 1))
            x = np.choose(kind, [x * 65504 * 1.2, 65504 - np.abs(x) * 500, np.abs(x) * 500 - 65504, x * 30000])
            _, codes, scale, low = kv.snap(x.reshape(c.kh, 64, d))
            nib = np.zeros((c.kh, 64, d), np.uint8)
            nib[..., kv.nibble_place(d, key)] = codes
            tile[:, a:e] = (nib[..., 0::2] | (nib[..., 1::2] << 4)).reshape(c.kh, -1)
            tile[:, p0:p1] = np.ascontiguousarray(np.stack((scale, low), -1).astype(np.float16)).view(np.uint8).reshape(c.kh, -1)
        pool[page] = tile
    c.pool.copy_(torch.from_numpy(pool))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("counts,kh", [([1, 2], 2), ([130, 200], 16)])
@pytest.mark.parametrize("mass", [False, True])
def test_values_at_the_ends_of_fp16(dtype, counts, kh, mass):
    """Parameters whose value lies beyond 65504 by their rounding, or whose scale times a code does: finite everywhere, and near the formula,
    with values that stop at 65504 where the header allows it."""
    lens = [190, 200]
    c = kv.KV4(2 * kh, kh, 64, lens, None, dtype, seed=8).fill()
    for b in range(2):
        extreme(c, b, b)
    q = c.normal(sum(counts), 2 * kh, 64, scale=2e-6)                         # scores of some units
    out = torch.zeros_like(q)
    m = torch.zeros(c.n_pages, kh, 64, device=c.dev) if mass else None
    c.do("attention", c.attention_args(counts, c.lens, q, out, mass=m))
    assert c.status.item() == 0 and torch.isfinite(out.float()).all()
    row = 0
    for b, n in enumerate(counts):
        k, v = c.held(b, lens[b])
        x = host(q[row:row + n])
        ok, end = False, 65504.0
        for kk, vv in ((k, v), (k, np.minimum(v, end)), (np.minimum(k, end), np.minimum(v, end)))[:3 if n > 2 else 1]:
            ref, _, size = kv.attend(x, kk, vv, 1 / 8, c.spread(b, lens[b]))
            ok |= np.abs(host(out[row:row + n]) - ref) <= attention_bound(dtype, ref, size, x, kk, 1 / 8, n > 2)
        assert ok.all()
        if mass:
            w = kv.attend(x, k, v, 1 / 8)[1]
            want = w.reshape(kh, 2 * n, lens[b]).sum(1)
            assert np.abs(c.rows_of(m, b, lens[b]) - want).max() <= 2.0 ** -15 * max(1.0, want.max())
        row += n
    held = [torch.zeros(2, 256, kh, 64, dtype=c.dtype, device=c.dev) for _ in range(2)]
    c.do("read", kv.Read(C.sizeof(kv.Read), 0, 256, 0, c.lens.data_ptr(), held[0].data_ptr(), held[1].data_ptr()))
    for b in range(2):
        for got, want in zip(held, c.held(b, lens[b])):
            want = np.minimum(want.swapaxes(0, 1), 65504.0 if dtype == "fp16" else np.inf)
            assert torch.isfinite(got.float()).all()
            assert (np.abs(host(got[b, :lens[b]]) - want) <= HALF_STEP[dtype] * np.abs(want) * (1 + 1e-6) + 1e-6).all()


def test_portions_on_two_streams_at_once():
    """Kernels with tensor memory of their own side by side, and single tokens between them: what they give alone."""
    made = [Chain([90] * 4, 8, qh=32, kh=16, d=128), Chain([200, 3, 41], 8, qh=28, kh=4, d=128, dtype="fp16"), Chain([1] * 5, 40)]
    alone = [ch.run() for ch in made]
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(3):
        for ch in made:
            ch.a.zero_(); ch.b.fill_(3); ch.c.mass.fill_(-1.0); ch.c.index.fill_(-1); ch.c.pool.fill_(255)
            for o in ch.outs:
                o.zero_()
        torch.cuda.synchronize()
        for t in range(40):
            for ch, s in zip(made, streams):
                if t < len(ch.calls):
                    with torch.cuda.stream(s):
                        for name, args in ch.calls[t]:
                            ch.c.do(name, args)
        torch.cuda.synchronize()
        for ch, (want, n) in zip(made, alone):
            assert ch.c.status.item() == 0 and ch.a.tolist() == n
            assert all(torch.equal(x, y) for x, y in zip(want, ch.outs + [ch.c.pool]))
