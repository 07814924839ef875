"""CPU: the header of the 4-bit cache against its binding, the statement of the format against itself, refusals before anything reaches a GPU."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

import cabi
import kv4_util as kv

HEADER = os.path.join(cabi.ROOT, "include", "efm_b200_kv4.h")


def test_header_binding_and_library_agree(built, tmp_path):
    declared = sorted(set(re.findall(r"\b(efm_b200_\w*kv4_\w+)\s*\(", open(HEADER).read())))
    assert declared == sorted(kv.SIGNATURES)
    L = kv.lib()
    for n in declared:
        assert hasattr(L, n)
    names = {"cache": kv.Cache, "append": kv.Append, "attention": kv.Attention, "evict": kv.Evict, "read": kv.Read}
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "efm_b200_kv4.h"\nint main(void) {\n'
    for n, s in names.items():
        src += f'printf("%zu", sizeof(efm_kv4_{n}));\n' + "".join(f'printf(" %zu", offsetof(efm_kv4_{n}, {f[0]}));\n' for f in s._fields_) + 'printf("\\n");\n'
    (tmp_path / "t.c").write_text(src + "return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.dirname(HEADER), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    lines = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.splitlines()
    for line, s in zip(lines, names.values()):
        assert [int(x) for x in line.split()] == [C.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]


@pytest.mark.parametrize("d", [64, 128])
def test_every_channel_has_a_nibble_of_its_own(d):
    for key in (True, False):
        assert sorted(kv.nibble_place(d, key)) == list(range(d))
    assert kv.parts(d)[3][1] == kv.tile_bytes(d)
    n = C.c_int64()
    assert kv.lib().efm_b200_kv4_tile_bytes(d, C.byref(n)) == 0 and n.value == kv.tile_bytes(d)


def test_the_format_is_off_by_half_a_step_at_most():
    rng = np.random.default_rng(0)
    x = np.concatenate((rng.standard_normal((50, 128)), rng.uniform(-1e-3, 1e-3, (50, 128)), np.exp(3 * rng.standard_normal((50, 128)))))
    _, codes, scale, low = kv.snap(x)
    off = np.abs(kv.values(codes, scale, low) - np.clip(x, -65504, 65504)).reshape(len(x), -1, 64)
    # half a step, the minimum's rounding, and 15 times the scale's (fp16: 2^-11 relative, 2^-25 below its normal range)
    bound = scale / 2 + np.abs(low) * 2.0 ** -11 + 15 * scale * 2.0 ** -11 + 16 * 2.0 ** -25
    assert (off <= bound[..., None] * (1 + 1e-9)).all()
    raw, codes, scale, low = kv.snap(np.full((1, 64), 3.25))
    assert (scale == 0).all() and (kv.values(codes, scale, low) == 3.25).all()
    _, codes, scale, low = kv.snap(np.array([[np.nan, np.inf, -np.inf] + [0.0] * 61]))
    got = kv.values(codes, scale, low)
    assert np.isfinite(got).all() and abs(got[0, 1] - 65504) <= 65504 / 15 and abs(got[0, 2] + 65504) <= 65504 / 15


def test_eviction_statement():
    assert kv.evicted([0, 1, 2, 3, 4], [0, 5, 1, 9, 0], 3, 0, 1) == [3, 1, 4]       # newest and the two heaviest; late rows into the holes in order
    assert kv.evicted([0, 1, 2, 3], [1, 1, 1, 1], 2, 0, 0) == [0, 1]                # ties: lower rows
    assert kv.evicted([7, 5, 6, 0], [float("nan"), 0, 0, 0], 2, 1, 0) == [3, 1]     # first token kept, NaN last
    assert kv.evicted([0, 1, 2, 3], [0, 0, 0, 9], 2, 4, 4) == [0, 1]                # more protected rows than the budget: lower ones


FAKE = 1 << 20                                              # a number that looks like an aligned address; never looked at by a refused call


def cache(**over):
    c = kv.Cache(C.sizeof(kv.Cache), cabi.EFM_BF16, 8, 2, 128, 10, 2, 4, FAKE, FAKE, None)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def append(**over):
    a = kv.Append(C.sizeof(kv.Append), 3, FAKE, FAKE, 2 * FAKE, FAKE, FAKE, FAKE, 1024, 256, 256, 1, 1e-6, FAKE, FAKE, 128, 0, 3, (C.c_int32 * 3)(16, 24, 24),
                  FAKE, FAKE, None, FAKE, None, None, FAKE, FAKE)
    for k, v in over.items():
        setattr(a, k, (C.c_int32 * 3)(*v) if k == "sections" else v)
    return a


def attention(**over):
    a = kv.Attention(C.sizeof(kv.Attention), 3, 2, 200, FAKE, FAKE, FAKE, FAKE, 0.1, 0, FAKE, FAKE, FAKE, 1 << 40)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def evict(**over):
    a = kv.Evict(C.sizeof(kv.Evict), 64, 128, 4, 16, 0, FAKE, 2 * FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def read(**over):
    a = kv.Read(C.sizeof(kv.Read), 0, 64, 0, FAKE, FAKE, FAKE)
    for k, v in over.items():
        setattr(a, k, v)
    return a


INVALID, UNSUPPORTED = 1, 5
CACHE_FAULTS = [(dict(struct_size=8), INVALID), (dict(dtype=cabi.EFM_F32), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(q_heads=7), INVALID),
                (dict(kv_heads=0), INVALID), (dict(q_heads=0), INVALID), (dict(q_heads=2048), INVALID), (dict(n_pages=0), INVALID), (dict(n_pages=(1 << 24) + 1), INVALID), (dict(batch=0), INVALID),
                (dict(batch=65536), INVALID), (dict(max_pages=0), INVALID), (dict(max_pages=1 << 24), INVALID), (dict(pool=None), INVALID),
                (dict(pool=FAKE + 8), INVALID), (dict(page_table=None), INVALID), (dict(status=FAKE + 1), INVALID)]
FAULTS = [
    ("append", append, [dict(struct_size=0), dict(max_rows=-1), dict(cu_rows=None), dict(lens_in=None), dict(lens_out=None), dict(lens_out=FAKE), dict(k=None), dict(v=None),
                        dict(q=None), dict(q_out=None), dict(q_stride=1016), dict(q_stride=1028), dict(k_stride=255), dict(v_stride=128), dict(q=FAKE + 2), dict(k=FAKE + 8),
                        dict(k_held=FAKE + 4), dict(norm=2), dict(norm_eps=-1.0), dict(norm_eps=float("nan")), dict(rot_dims=8), dict(rot_dims=144), dict(rot_dims=-16),
                        dict(rot_kind=2), dict(axes=2), dict(sections=(16, 24, 23)), dict(sections=(-1, 33, 32)), dict(inv_freq=None), dict(inv_freq=FAKE + 4),
                        dict(positions=None), dict(mass=FAKE + 2), dict(index=FAKE + 1)]),
    ("attention", attention, [dict(struct_size=1), dict(max_rows=-1), dict(max_new=-1), dict(max_len=-1), dict(max_len=257), dict(cu_rows=None), dict(lens=None), dict(q=None),
                              dict(out=None), dict(q=FAKE + 8), dict(out=FAKE + 2), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                              dict(mass_in=None), dict(mass_out=None), dict(workspace=None), dict(workspace_bytes=8), dict(workspace=FAKE + 8), dict(mass_in=FAKE + 1)]),
    ("evict", evict, [dict(struct_size=1), dict(budget=0), dict(budget=-3), dict(limit=63), dict(keep_first=-1), dict(keep_last=-1), dict(lens_in=None), dict(lens_out=None),
                      dict(lens_out=FAKE), dict(index_in=None), dict(index_out=None), dict(mass_in=None), dict(mass_out=None), dict(workspace=None),
                      dict(workspace_bytes=8), dict(workspace=FAKE + 4), dict(mass_out=FAKE + 2)]),
    ("read", read, [dict(struct_size=1), dict(first=-1), dict(rows=-1), dict(first=1 << 30, rows=1), dict(lens=None), dict(k_out=None, v_out=None), dict(k_out=FAKE + 8)]),
]


@pytest.mark.parametrize("name,make,faults", FAULTS, ids=[f[0] for f in FAULTS])
def test_refusals(built, name, make, faults):
    fn = getattr(kv.lib(), "efm_b200_op_kv4_" + name)
    for over in faults:
        assert fn(C.byref(cache()), C.byref(make(**over)), None) == INVALID, over
        assert kv.error().startswith("op_kv4_" + name), over
    assert fn(C.byref(cache()), None, None) == INVALID and fn(None, C.byref(make()), None) == INVALID
    for over, st in CACHE_FAULTS:
        assert fn(C.byref(cache(**over)), C.byref(make()), None) == st, over


def test_workspace_sizes(built):
    n = C.c_int64()
    L = kv.lib()
    assert L.efm_b200_kv4_evict_workspace(C.byref(cache()), C.byref(evict()), C.byref(n)) == 0 and n.value >= 2 * 2 * 64 * 8
    assert L.efm_b200_kv4_attention_workspace(C.byref(cache()), C.byref(attention(workspace=None)), C.byref(n)) == 0 and n.value > 0
    assert L.efm_b200_kv4_attention_workspace(C.byref(cache()), C.byref(attention(scale=0.0)), C.byref(n)) == INVALID
    assert L.efm_b200_kv4_evict_workspace(C.byref(cache()), C.byref(evict(budget=0)), C.byref(n)) == INVALID
    assert L.efm_b200_kv4_evict_workspace(C.byref(cache()), C.byref(evict()), None) == INVALID
    assert L.efm_b200_kv4_tile_bytes(96, C.byref(n)) == INVALID and L.efm_b200_kv4_tile_bytes(64, None) == INVALID
    # large batches: sizes pass 32 bits
    big = cache(q_heads=1024, kv_heads=1024, batch=60000, max_pages=1 << 20)
    assert L.efm_b200_kv4_evict_workspace(C.byref(big), C.byref(evict(budget=1 << 16, limit=1 << 20)), C.byref(n)) == 0 and n.value > 1024 * 60000 * 65536 * 8


@pytest.mark.skipif(__import__("torch").cuda.is_available(), reason="checks the no-device failure mode")
def test_without_a_gpu_the_calls_fail(built):
    for name, make, _ in FAULTS:
        assert getattr(kv.lib(), "efm_b200_op_kv4_" + name)(C.byref(cache()), C.byref(make()), None) == 2       # EFM_ERR_CUDA
