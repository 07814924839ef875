"""GPU: attention over a 4-bit cache where its workspace is laid out by the call's rows or the pool's pages instead of so much a sequence
(helpers and tolerances: test_gpu_kv4)."""
import ctypes as C

import numpy as np
import pytest
import torch

import kv4_util as kv
from test_gpu_kv4 import host, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qh,kh,d,dtype", [(28, 4, 128, "bf16"), (16, 16, 64, "fp16"), (40, 2, 128, "bf16")])
@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("pad", [0, 3, 5000])
def test_one_portion_among_tokens(qh, kh, d, dtype, mass, pad):
    counts = [1, 1, 0, 203, 1, 3] + [1] * 20 + [130, 0, 1]
    lens = [n + (31 * b) % 170 for b, n in enumerate(counts)]
    c = kv.KV4(qh, kh, d, lens, None, dtype, seed=qh).fill()
    run_attention(c, counts, lens, dtype, mass, pad=pad, shared_tiles=True)


@pytest.mark.parametrize("qh,kh,d,dtype", [(28, 4, 128, "bf16"), (14, 2, 64, "fp16"), (32, 2, 128, "bf16")])
@pytest.mark.parametrize("new", [1, 2])
def test_weights_of_tokens_whose_limit_is_far(qh, kh, d, dtype, new):
    """Scores by the pool's pages: sequences that may be long by the table, but are not."""
    lens = [700, 1, 64, 130, 257, 5, 300, 63, 65, 0]
    counts = [min(n, new) for n in lens]
    c = kv.KV4(qh, kh, d, lens, None, dtype, seed=qh, spare=1).fill()
    c.max_pages = 400                                             # columns behind a sequence's rows are not read
    c.np_table = np.concatenate((c.np_table, np.full((c.batch, 400 - c.np_table.shape[1]), -7, np.int32)), 1)
    c.table = torch.from_numpy(c.np_table).to(c.dev)
    run_attention(c, counts, lens, dtype, True)
    run_attention(c, counts, lens, dtype, True, max_len=max(lens))


def test_weights_by_pages_with_a_bad_page():
    lens = [200, 64, 700, 130]
    c = kv.KV4(8, 2, 64, lens, None, "bf16", seed=2).fill()
    assert c.batch * c.max_pages > c.n_pages                      # scores are kept by pages
    q = c.normal(4, 8, 64)
    m_in = torch.rand(c.n_pages, 2, 64, device=c.dev)
    whole, got = torch.full_like(m_in, -1.0), torch.full_like(m_in, -1.0)
    c.do("attention", c.attention_args([1] * 4, c.ints(lens), q, torch.zeros_like(q), mass=m_in, mass_out=whole))
    for wrong in (-1, c.n_pages, 2 ** 31 - 1):
        c.status.zero_()
        got.fill_(-1.0)
        c.table[2, 3] = wrong
        c.do("attention", c.attention_args([1] * 4, c.ints(lens), q, torch.zeros_like(q), mass=m_in, mass_out=got))
        assert c.status.item() == kv.BAD_PAGE
        c.table[2, 3] = int(c.np_table[2, 3])
        for b in (0, 1, 3):
            assert np.array_equal(c.rows_of(got, b, lens[b]), c.rows_of(whole, b, lens[b]))
        k, v = c.held(2, 700)
        stay = [r for r in range(700) if r // 64 != 3]
        w = kv.attend(host(q[2:3]), k[:, stay], v[:, stay], 0.125)[1].reshape(2, 4, -1).sum(1)
        have = c.rows_of(got, 2, 700)
        assert (have[:, 192:256] == -1.0).all() and np.abs(have[:, stay] - w - c.rows_of(m_in, 2, 700)[:, stay]).max() <= 2.0 ** -15 * 4


@pytest.mark.parametrize("counts,lens,max_new", [([1] * 6, [300, 1, 64, 900, 2, 77], 1), ([200, 1, 1, 1], [260, 90, 1, 300], 200), ([200, 1, 1, 1], [260, 90, 1, 300], 400),
                                                 ([3, 300, 2], [1000, 300, 2], 300)])
@pytest.mark.parametrize("mass", [False, True])
def test_nothing_is_written_behind_the_workspace(counts, lens, max_new, mass):
    c = kv.KV4(28, 4, 128, lens, None, "bf16", seed=4).fill()
    q = c.normal(sum(counts), 28, 128)
    m = torch.zeros(c.n_pages, 4, 64, device=c.dev) if mass else None
    a = c.attention_args(counts, c.lens, q, torch.zeros_like(q), mass=m, max_new=max_new)
    need = C.c_int64()
    assert kv.lib().efm_b200_kv4_attention_workspace(C.byref(c.cache()), C.byref(a), C.byref(need)) == 0
    ws = torch.full((need.value + (1 << 20),), 0x5a, dtype=torch.uint8, device=c.dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
    c.do("attention", a)
    torch.cuda.synchronize()
    assert c.status.item() == 0 and (ws[need.value:] == 0x5a).all()
