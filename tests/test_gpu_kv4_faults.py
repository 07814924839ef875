"""GPU: the operators of the 4-bit cache where a call's own numbers are wrong, or a wait inside a kernel runs out."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import kv4_util as kv

pytestmark = pytest.mark.gpu


def effective(cu, max_rows):
    """What an append makes of row counts: cut to the buffers, never falling."""
    out = [min(max(cu[0], 0), max_rows)]
    for x in cu[1:]:
        out.append(max(out[-1], min(max(x, 0), max_rows)))
    return out


@pytest.mark.parametrize("cu", [[0, 4, 2, 6], [0, 6, 0, 6], [-3, 2, 4, 6], [0, 2, 4, 9], [5, 3, 1, 6], [0, -1, -7, -2], [4, 2, 2 ** 31 - 1, -2 ** 31], [0, 2, 2, 2 ** 31 - 1]])
@pytest.mark.parametrize("q_heads", [2, 40])
def test_append_row_counts_that_lie(cu, q_heads):
    """Reported, and the same bytes, lengths and outputs as the counts cut to what they can be; no held row is touched."""
    kh, d, R = 1, 64, 6
    held = [62, 5, 10]
    c = kv.KV4(q_heads, kh, d, held, [128] * 3, "bf16", seed=11).fill()
    start = c.pool.clone()
    x = c.normal(R, (q_heads + 2) * d)
    q, k, v = x[:, :q_heads * d], x[:, q_heads * d:(q_heads + 1) * d], x[:, (q_heads + 1) * d:]
    good, got = effective(cu, R), []
    for counts in (good, cu):
        for _ in range(20 if counts is cu else 1):
            c.pool.copy_(start); c.index.fill_(-1); c.mass.fill_(-1.0); c.status.zero_()
            out, qo = c.ints([-1] * 3), torch.full((R, q_heads, d), 9.0, dtype=c.dtype, device=c.dev)
            ko = torch.full((R, kh, d), 9.0, dtype=c.dtype, device=c.dev)
            a = c.append_args([0, 0, 0], out, q, k, v, R, q_out=qo, k_held=ko, index=c.index, mass=c.mass)
            cu_t = c.ints(np.asarray(counts, np.int64))
            a.cu_rows = cu_t.data_ptr()
            c.do("append", a)
            torch.cuda.synchronize()
            assert c.status.item() == (0 if counts is good else kv.BAD_COUNT)
            got.append([t.clone() for t in (c.pool, c.index, c.mass, out, qo, ko)])
    assert got[0][3].tolist() == [h + b - a for h, a, b in zip(held, good, good[1:])]
    for g in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], g))
    for b, n in enumerate(held):                                  # what was held is what it was
        now, before = c.pool[c.table[b].long()], start[c.table[b].long()]
        for a, e in kv.parts(d):
            w = (e - a) // 64
            assert torch.equal(now[0, :, a:a + n * w], before[0, :, a:a + n * w])


def test_append_falling_counts_of_many_sequences():
    """More sequences than a block has threads; one count falls far behind the first ones."""
    B, d = 300, 64
    c = kv.KV4(1, 1, d, [3] * B, [64] * B, "bf16", seed=2).fill()
    R = 2 * B
    x = c.normal(R, 3 * d)
    cu = list(range(0, 2 * B + 1, 2))
    cu[200] = 7
    good, got = effective(cu, R), []
    start = c.pool.clone()
    for counts in (good, cu):
        c.pool.copy_(start); c.status.zero_()
        out, qo = c.ints([0] * B), torch.zeros(R, 1, d, dtype=c.dtype, device=c.dev)
        a = c.append_args([0] * B, out, x[:, :d], x[:, d:2 * d], x[:, 2 * d:], R, q_out=qo)
        cu_t = c.ints(counts)
        a.cu_rows = cu_t.data_ptr()
        c.do("append", a)
        torch.cuda.synchronize()
        got.append((c.status.item(), [t.clone() for t in (c.pool, out, qo)]))
    assert [g[0] for g in got] == [0, kv.BAD_COUNT] and all(torch.equal(a, b) for a, b in zip(got[0][1], got[1][1]))


@pytest.mark.parametrize("counts,mass", [([60] * 6, False), ([60] * 6, True), ([1] * 6, False)])
@pytest.mark.parametrize("held", [1.0, 0.0])
def test_scores_beyond_all_numbers_show(counts, mass, held):
    """An infinite query channel meets one key (of any place in a page) that is positive or 0 there, all others negative: weights of inf - inf, or
    of 0 inf.  NaN like every row whose scores are no numbers, and no other row changes."""
    kh, d, L = 16, 64, 60
    for place in (0, 3, 6, 7, 38, 55):
        c = kv.KV4(kh, kh, d, [0] * 6, [L] * 6, "bf16", seed=place)
        x = c.normal(6 * L, kh * d)
        k = x.clone().view(6, L, kh, d)
        k[..., 0] = -1.0 - k[..., 0].abs()
        k[:, place] = 0.0
        k[:, place, :, 0] = held
        out = c.ints([0] * 6)
        c.do("append", c.append_args([L] * 6, out, None, k.view(6 * L, kh * d), x))
        q = c.normal(sum(counts), kh, d)
        got = [torch.zeros_like(q) for _ in range(2)]
        m = torch.zeros(c.n_pages, kh, 64, device=c.dev) if mass else None
        c.do("attention", c.attention_args(counts, out, q, got[0], mass=m))
        row = counts[0] - 1                                       # sees every key
        q[row, 5] = 0.0
        q[row, 5, 0] = float("inf")
        c.do("attention", c.attention_args(counts, out, q, got[1], mass=m))
        torch.cuda.synchronize()
        assert c.status.item() == 0 and torch.isnan(got[1][row, 5]).all()
        got[1][row, 5] = got[0][row, 5]
        assert torch.equal(got[0], got[1])


# ---- waits that run out ----------------------------------------------------------------------------------------------------
def hasty_calls():
    """In a process of its own, since the library looks for the variable once.  Waits give up after a few polls: copies and products on their
    way, tensor memory and shared memory are seen to, a status says so, sums of weights are whole or as they were, and the next call is right."""
    seen = {}
    for qh, kh, d, dtype, counts, lens in ((28, 4, 128, "bf16", [1, 1, 1], [700, 64, 300]), (28, 4, 128, "bf16", [1] * 40, [50 * b + 1 for b in range(40)]),
                                           (28, 4, 128, "bf16", [4, 3, 2], [150, 1000, 2]), (28, 4, 128, "bf16", [300, 350, 128], [900, 350, 128]),
                                           (16, 16, 64, "fp16", [200] * 6, [300] * 6), (16, 16, 64, "fp16", [1] * 30, [40 * b + 7 for b in range(30)])):
        c = kv.KV4(qh, kh, d, lens, None, dtype, seed=5).fill()
        q = c.normal(sum(counts), qh, d)
        m_in = torch.rand(c.n_pages, kh, 64, device=c.dev)
        for mass in (False, True):
            out, m = torch.zeros_like(q), m_in.clone()
            args = c.attention_args(counts, c.lens, q, out, mass=m if mass else None)

            def run(which):
                os.environ["EFM_B200_KV4_HASTY"] = str(which)
                out.zero_()
                m.copy_(m_in)
                c.status.zero_()
                c.do("attention", args)
                torch.cuda.synchronize()
                return c.status.item(), out.clone(), m.clone()
            st, want, want_m = run(0)
            assert st == 0
            for which in (1, 2, 4, 7):
                for _ in range(10):
                    st, got, got_m = run(which)
                    assert st in (0, kv.WAIT)
                    assert ((got_m == m_in) | (got_m == want_m)).all()
                    if st == 0:
                        assert torch.equal(got, want) and torch.equal(got_m, want_m)
                    elif which == 2:
                        assert torch.equal(got_m, m_in)
                    seen[which, max(counts) > 4, mass] = seen.get((which, max(counts) > 4, mass), 0) + (st != 0)
                    st, got, got_m = run(0)
                    assert st == 0 and torch.equal(got, want) and torch.equal(got_m, want_m)
    print("seen", seen)
    assert all(seen[k] > 0 for k in ((1, False, False), (1, False, True), (2, True, False), (2, True, True), (4, True, True)))


def test_waits_that_run_out():
    r = subprocess.run([sys.executable, os.path.abspath(__file__)], capture_output=True, text=True, timeout=600, env=dict(os.environ, EFM_B200_KV4_HASTY="0"))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


if __name__ == "__main__":
    hasty_calls()
