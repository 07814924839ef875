"""GPU: the operators of the 4-bit cache where a call's own numbers are wrong, or a wait inside a kernel runs out."""
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
