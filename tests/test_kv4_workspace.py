"""CPU: what attention over a 4-bit cache asks for beside the cache stays in proportion to what a call's buffers and the pool can hold."""
import ctypes as C

import pytest

import cabi
import kv4_util as kv

MB = 1 << 20
FAKE = 1 << 20


def need(batch, max_rows, max_new, max_len, n_pages, mass, heads=(28, 4, 128), dtype=cabi.EFM_BF16):
    c = kv.Cache(C.sizeof(kv.Cache), dtype, *heads, n_pages, batch, -(-max_len // 64), FAKE, FAKE, None)
    a = kv.Attention(C.sizeof(kv.Attention), max_rows, max_new, max_len, FAKE, FAKE, FAKE, FAKE, 0.1, 0, FAKE if mass else None, FAKE if mass else None, None, 0)
    n = C.c_int64()
    assert kv.lib().efm_b200_kv4_attention_workspace(C.byref(c), C.byref(a), C.byref(n)) == 0, kv.error()
    return n.value


# what 148 blocks (or twice as many of 4 warps) leave of the rows that they begin and end in, whatever the call
PIECES = 2 * 148 * 256 * (128 + 2) * 4 + 2 * 2 * 148 * 4 * 16 * (128 + 2) * 4


@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("dtype", [cabi.EFM_BF16, cabi.EFM_F16])
def test_one_long_portion_among_many_tokens(built, mass, dtype):
    q = 2111 * 28 * 128 * 2
    n = need(64, 2111, 2048, 4096, 4000, mass, dtype=dtype)
    assert n <= PIECES + 2 * q + 64 * 4 * 128 * (128 * 2 + 8)          # operands of the rows there are, and a tile that is not full a sequence and head
    more = need(128, 2175, 2048, 4096, 4000, mass, dtype=dtype)
    assert more - n < 16 * MB
    assert need(64, 4 * 2048, 2048, 4096, 4000, mass, dtype=dtype) <= PIECES + 2 * 4 * 2048 * 28 * 128 * 2 + 10 * MB


def test_scores_of_many_tokens_that_could_be_long(built):
    pool = 4000 * 4 * kv.tile_bytes(128)
    n = need(64, 64, 1, 131072, 4000, True)
    assert n < pool // 2
    assert need(500, 500, 1, 131072, 4000, True) < pool // 2
    assert need(64, 64, 1, 131072, 4000, False) < 20 * MB


def test_a_token_beside_a_large_pool(built):
    """Nor does it grow with a pool of which a call can use little."""
    assert need(1, 1, 1, 1500, 1 << 20, True) < 2 * MB
    assert need(2, 1 << 20, 1, 1500, 1 << 20, True, heads=(80, 2, 64)) < 64 * MB


def test_sizes_do_not_fall_when_a_call_may_bring_more(built):
    last = 0
    for max_len in (1, 64, 65, 257, 1000, 20000):
        n = need(3, 3, 1, max_len, 10000, True)
        assert n >= last
        last = n
