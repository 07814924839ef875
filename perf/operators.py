"""The operators of the 4-bit key/value cache, as calls that can be timed and checked.

A pool of pages holds 64 rows of a kv head per tile: keys and values in 4 bits with a scale and a minimum (16 bits each) for 64 channels
of a row.  Five kinds of case, each one pass as an engine makes it over the C interface (include/efm_b200_kv4.h):

  append  projected q, k, v rows of a batch: norm of every head, rotation, q out, k and v quantised behind what their sequences hold
  attend  new rows against the cache, with the attention weights summed per cached row where they are kept for an eviction
  step    append and attend of one decoded token per sequence
  evict   caches that ran full brought back to a budget of rows by accumulated weight, and what is left of them read back
  read    cached rows as 16-bit values

Everything a program has before the call is on the GPU: pool, page table, lengths, projections, frequencies.  Pages lie in random order, and
what no sequence holds is filled with bits that read as NaN.
"""
import ctypes as C
import math
import os

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE = GROUP = 64
LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "edge-fm-x_b200", "lib", "libefm_b200.so")
TYPES = {"bf16": (torch.bfloat16, 2), "fp16": (torch.float16, 1)}
NIBBLE = (0, 4, 1, 5, 2, 6, 3, 7)          # which nibble of a 32-bit word holds channel 0 .. 7 of its eight


# ---- the interface ---------------------------------------------------------------------------------------------------------
class Cache(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("struct_size", "dtype", "q_heads", "kv_heads", "head_dim", "n_pages", "batch", "max_pages")] + \
        [(n, C.c_void_p) for n in ("pool", "page_table", "status")]


class Append(C.Structure):
    _fields_ = [("struct_size", C.c_int32), ("max_rows", C.c_int32)] + [(n, C.c_void_p) for n in ("cu_rows", "lens_in", "lens_out", "q", "k", "v")] + \
        [(n, C.c_int64) for n in ("q_stride", "k_stride", "v_stride")] + [("norm", C.c_int32), ("norm_eps", C.c_float)] + \
        [(n, C.c_void_p) for n in ("q_norm", "k_norm")] + [(n, C.c_int32) for n in ("rot_dims", "rot_kind", "axes")] + [("sections", C.c_int32 * 3)] + \
        [(n, C.c_void_p) for n in ("inv_freq", "positions", "token_index", "q_out", "k_held", "v_held", "index", "mass")]


class Attention(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("struct_size", "max_rows", "max_new", "max_len")] + [(n, C.c_void_p) for n in ("cu_rows", "lens", "q", "out")] + \
        [("scale", C.c_float), ("reserved", C.c_int32)] + [(n, C.c_void_p) for n in ("mass_in", "mass_out", "workspace")] + [("workspace_bytes", C.c_int64)]


class Evict(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("struct_size", "budget", "limit", "keep_first", "keep_last", "reserved")] + \
        [(n, C.c_void_p) for n in ("lens_in", "lens_out", "index_in", "index_out", "mass_in", "mass_out", "workspace")] + [("workspace_bytes", C.c_int64)]


class Read(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("struct_size", "first", "rows", "reserved")] + [(n, C.c_void_p) for n in ("lens", "k_out", "v_out")]


_lib = None


def lib():
    global _lib
    if _lib is None:
        L = C.CDLL(LIB)
        for n in ("append", "attention", "evict", "read"):
            f = getattr(L, "efm_b200_op_kv4_" + n)
            f.restype, f.argtypes = C.c_int32, [C.c_void_p, C.c_void_p, C.c_void_p]
        for n in ("attention", "evict"):
            f = getattr(L, "efm_b200_kv4_%s_workspace" % n)
            f.restype, f.argtypes = C.c_int32, [C.c_void_p, C.c_void_p, C.POINTER(C.c_int64)]
        L.efm_b200_last_error.restype, L.efm_b200_last_error.argtypes = C.c_char_p, [C.c_void_p]
        _lib = L
    return _lib


def ok(st):
    if st:
        raise RuntimeError(lib().efm_b200_last_error(None).decode())


def call(name, s, args):
    L = lib()
    if hasattr(args, "workspace") and not args.workspace:      # kept by the program, like its captured graphs
        need = C.c_int64()
        ok(getattr(L, "efm_b200_kv4_%s_workspace" % name)(C.byref(s.cache), C.byref(args), C.byref(need)))
        ws = torch.empty(max(need.value, 16), dtype=torch.uint8, device=DEV)
        s.keep.append(ws)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need.value
    ok(getattr(L, "efm_b200_op_kv4_" + name)(C.byref(s.cache), C.byref(args), torch.cuda.current_stream().cuda_stream))


# ---- cases -----------------------------------------------------------------------------------------------------------------
def case(name, kind, heads, dtype="bf16", batch=1, rows=(1, 1), held=(0, 0), norm=False, rot="halves", axes=1, weights=False, budget=0, keep=(4, 32)):
    c = {"name": name, "kind": kind, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2], "dtype": dtype, "batch": batch,
         "rows_min": rows[0], "rows_max": rows[1], "held_min": held[0], "held_max": held[1]}
    if kind in ("append", "step"):
        c.update(norm=norm, rot=rot, axes=axes)
    if kind in ("attend", "step"):
        c.update(weights=weights)
    if kind == "evict":
        c.update(budget=budget, keep_first=keep[0], keep_last=keep[1])
    return c


# heads of the four text towers of the benchmark (q heads, kv heads, head size) and a generic layout
H05, H15, H3, H7, HG = (14, 2, 64), (12, 2, 128), (16, 2, 128), (28, 4, 128), (32, 8, 128)


def listed():
    return [
        case("step_0p5b", "step", H05, held=(192, 192)),                                      # one decoded token of the smallest tower
        case("step_7b_weights", "step", H7, held=(1451, 1451), axes=3, weights=True),         # one token behind the image prompt, weights kept
        case("append_prompt_7b", "append", H7, rows=(1324, 1324), axes=3),                    # the image prompt into an empty cache
        case("append_batch", "append", HG, "fp16", 64, rows=(1, 96), held=(0, 2000), norm=True, rot="neighbours"),   # portions of many live requests
        case("attend_long", "attend", H7, held=(131000, 131000), weights=True),               # one token behind a very long context
        case("attend_batch", "attend", H7, batch=64, held=(300, 4000), weights=True),         # a decode step of 64 requests of unequal length
        case("attend_batch_fp16", "attend", (16, 16, 64), "fp16", 48, held=(1, 3000)),         # the same with a kv head per head
        case("attend_portions", "attend", H3, batch=16, rows=(1, 256), held=(0, 1800), weights=True),   # portions of prompts beside decoded tokens
        case("attend_prompt", "attend", H7, rows=(2048, 2048), held=(12289, 12289)),          # a large portion of a long prompt
        case("evict_small", "evict", H15, held=(600, 600), budget=512),                       # one request at its limit
        case("evict_batch", "evict", H7, batch=64, held=(900, 4100), budget=1024),            # many requests shrunk in one call
        case("read_prefix", "read", H7, batch=8, held=(1000, 1452)),                          # cached prefixes handed to the 16-bit kernels
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "step", "evict", "read"))
    d = rng.choice((64, 128, 128))
    g = rng.choice((1, 2, 4, 5, 7, 8, 12, 16))
    kv = _log(rng, 1, 16 if g <= 4 else 4)
    heads, dtype = (g * kv, kv, d), rng.choice(("bf16", "bf16", "fp16"))
    if kind == "append":
        b = _log(rng, 1, 64)
        top = max(1, min(1400, 3000 * 28 // (heads[0] * b)))
        hi = _log(rng, 1, top)
        return _bare(case("", kind, heads, dtype, b, (rng.choice((0, 1, hi)), hi), (0, _log(rng, 1, 3000)), rng.random() < 0.5,
                          rng.choice(("halves", "neighbours")), rng.choice((1, 3))))
    if kind in ("attend", "step"):
        b = _log(rng, 1, 64)
        hi = 1 if kind == "step" or rng.random() < 0.5 else _log(rng, 2, max(2, 2000 // b))
        room = 500_000 * 128 // d if hi == 1 else 200_000_000 // (hi * heads[0])     # cached rows of all kv heads together, or rows x keys
        most = max(16, min(120_000, room // (b * kv) if hi == 1 else min(16_000, room // b)))
        top = _log(rng, 8, most)
        return _bare(case("", kind, heads, dtype, b, (hi if kind == "step" else rng.choice((1, hi)), hi), (rng.choice((0, top // 3, top)), top), rng.random() < 0.5,
                          rng.choice(("halves", "neighbours")), 1, rng.random() < 0.5))
    b = _log(rng, 1, 64)
    top = _log(rng, 64, max(64, min(30_000, 700_000 // (b * kv))))
    if kind == "evict":
        return _bare(case("", kind, heads, dtype, b, held=(top // rng.choice((1, 2, 4)), top), budget=max(1, int(top * rng.uniform(0.1, 1.0))),
                          keep=(rng.choice((0, 1, 4, 16)), rng.choice((0, 1, 16, 32)))))
    return _bare(case("", kind, heads, dtype, b, held=(top // 3, top)))


def _bare(c):
    del c["name"]
    return c


def _spread(lo, hi, n):
    """n whole numbers over [lo, hi], the largest first, without a pattern."""
    return [lo + min(hi - lo, int((hi - lo + 1) * ((0.99999 - i * 0.6180339887) % 1.0))) for i in range(n)]


def _lengths(c):
    """New rows and rows already held of every sequence."""
    return _spread(c["rows_min"], c["rows_max"], c["batch"]), _spread(c["held_min"], c["held_max"], c["batch"])


# ---- layout of a tile ------------------------------------------------------------------------------------------------------
def tile_bytes(d):
    return 2 * PAGE * (d // 2 + d // 16)


def _parts(d):
    """First 32-bit word of a tile's key codes, key parameters, value codes, value parameters."""
    codes, params = PAGE * d // 8, PAGE * d // 64
    return 0, codes, codes + params, 2 * codes + params


def _quantise(x):
    """x fp32 [..., d] -> codes int32 [..., d], scale and minimum fp16 [..., d / 64]."""
    x = torch.nan_to_num(x, nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504.0, 65504.0).unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(-1), x.amax(-1)
    scale, low = ((hi - lo) * (1.0 / 15.0)).half(), lo.half()
    s = scale.float()[..., None]
    code = torch.where(s > 0, torch.round((x - low.float()[..., None]) / s), torch.zeros_like(x)).clamp(0, 15)
    return code.flatten(-2).int(), scale, low


def _words(codes, key):
    """codes int32 [..., d] -> the 32-bit words of a row, in the order of the tile."""
    w = codes.unflatten(-1, (-1, 8))
    shift = torch.tensor([4 * n for n in NIBBLE], dtype=torch.int64, device=codes.device)
    w = (w.long() << shift).sum(-1)
    w = torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()
    return w.unflatten(-1, (-1, 4, 2)).transpose(-3, -2).flatten(-3) if key else w     # keys: groups of a quarter lie side by side


def _codes(words, key):
    if key:
        words = words.unflatten(-1, (4, -1, 2)).transpose(-3, -2).flatten(-3)
    shift = torch.tensor([4 * n for n in NIBBLE], dtype=torch.int32, device=words.device)
    return ((words[..., None] >> shift) & 15).flatten(-2)


def _pair(scale, low):
    return torch.stack((scale, low), -1).view(torch.int32).flatten(-2)


def _values(words, params, key):
    """words int32 [..., d / 8], params int32 [..., d / 64] -> fp32 [..., d]."""
    p = params[..., None].contiguous().view(torch.float16).float()
    return (p[..., 1:] + p[..., :1] * _codes(words, key).float().unflatten(-1, (-1, GROUP))).flatten(-2)


def _tiles(pool, d):
    """pool uint8 [..., tile] -> keys, values fp32 [..., 64, d]."""
    w = pool.view(torch.int32)
    a, b, c, e = _parts(d)
    rows = lambda lo, hi: w[..., lo:hi].unflatten(-1, (PAGE, -1))  # noqa: E731
    return _values(rows(a, b), rows(b, c), True), _values(rows(c, e), rows(e, w.shape[-1]), False)


# ---- inputs ----------------------------------------------------------------------------------------------------------------
class State:
    pass


def _ptr(t):
    return None if t is None else t.data_ptr()


def prepare(case, seed):
    c, s = case, State()
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    kind, B, qh, kh, d = c["kind"], c["batch"], c["q_heads"], c["kv_heads"], c["head_dim"]
    s.case, s.dtype = c, TYPES[c["dtype"]][0]
    s.keep = []
    new, held = _lengths(c)
    if kind in ("evict", "read"):
        new = [0] * B
    s.max_new, total = max(new), sum(new)
    full = [h + n for h, n in zip(held, new)]                   # rows once the new ones are in
    s.max_len = max(max(full), 1)
    s.max_pages = (s.max_len + PAGE - 1) // PAGE + 1
    pages = [(n + PAGE - 1) // PAGE for n in full]
    s.n_pages = sum(pages) + 3
    order = torch.randperm(s.n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = np.zeros((B, s.max_pages), np.int32)
    filled = np.zeros((s.n_pages, PAGE), bool)
    at = 0
    here = held if kind in ("append", "step") else full         # rows the cache holds before the call
    for b in range(B):
        table[b, :pages[b]] = order[at:at + pages[b]]
        for p in range((here[b] + PAGE - 1) // PAGE):
            filled[order[at + p], :max(0, here[b] - p * PAGE)] = True
        at += pages[b]
    s.table = torch.from_numpy(table).to(DEV)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s.lens_in, s.lens_out, s.lens_full = ints(held), ints([0] * B), ints(full)
    s.cu = ints(np.concatenate(([0], np.cumsum(new))).tolist())
    # keys with a few loud channels per head, values without
    loud = torch.exp(0.5 * rnd(kh, 1, d))
    mask = torch.from_numpy(filled).to(DEV)
    s.pool = torch.full((s.n_pages, kh, tile_bytes(d)), 255, dtype=torch.uint8, device=DEV)
    w32 = s.pool.view(torch.int32)
    a, b_, c_, e = _parts(d)
    step = max(1, 40_000_000 // (kh * PAGE * d))
    for p in range(0, s.n_pages, step):
        n = min(step, s.n_pages - p)
        for key, at_codes, at_params, end in ((True, a, b_, c_), (False, c_, e, w32.shape[-1])):
            x = rnd(n, kh, PAGE, d) * (loud if key else 1.0)
            codes, scale, low = _quantise(x)
            for t, lo, hi in ((_words(codes, key), at_codes, at_params), (_pair(scale, low), at_params, end)):
                keep = mask[p:p + n, None, :, None].expand(-1, kh, -1, t.shape[-1])
                w32[p:p + n, :, lo:hi] = torch.where(keep, t, torch.full_like(t, -1)).flatten(-2)
    s.index = torch.zeros(s.n_pages, kh, PAGE, dtype=torch.int32, device=DEV)
    s.index_out = torch.zeros_like(s.index)
    s.mass = torch.rand(s.n_pages, kh, PAGE, generator=g, device=DEV) ** 4
    s.mass_out = torch.zeros_like(s.mass)
    for b in range(B):                                           # token numbers of what is held: the cache was filled in order
        n = pages[b]
        s.index[s.table[b, :n].long()] = torch.arange(n * PAGE, dtype=torch.int32, device=DEV).view(n, 1, PAGE)
    s.max_rows = total + (3 if B > 1 else 0)                     # a padded batch: rows behind the last sequence
    R = max(s.max_rows, 1)
    s.cache = Cache(C.sizeof(Cache), TYPES[c["dtype"]][1], qh, kh, d, s.n_pages, B, s.max_pages, _ptr(s.pool), _ptr(s.table), None)
    loudest = float(loud.square().mean().sqrt())
    s.scale = 1.0 / math.sqrt(d)
    if kind in ("append", "step"):
        s.qkv = rnd(R, (qh + 2 * kh) * d)
        s.qkv[:, :qh * d] *= 2.0 / loudest
        s.qkv = s.qkv.to(s.dtype)
        s.q_norm, s.k_norm = ((1.0 + 0.1 * rnd(d)).to(s.dtype) for _ in range(2))
        # head sizes of 128 turn three quarters of their channels with neighbours, all of them by halves
        s.rot_dims = 3 * d // 4 if c["rot"] == "neighbours" and d == 128 else d
        half = s.rot_dims // 2
        s.inv_freq = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        s.sections = [half, 0, 0] if c["axes"] == 1 else [half // 4, half // 4 + half // 8, half - 2 * (half // 4) - half // 8]
        place = np.concatenate([np.arange(n) + h for n, h in zip(new, held)] + [np.zeros(R - total)]).astype(np.int32)
        s.token_index = torch.from_numpy(place).to(DEV)
        pos = [place] if c["axes"] == 1 else [place // 3, place // 46, place % 46]       # images: time, row and column
        s.positions = torch.from_numpy(np.stack(pos).astype(np.int32)).to(DEV)
        s.q_out = torch.zeros(R, qh, d, dtype=s.dtype, device=DEV)
        s.k_held, s.v_held = (torch.zeros(R, kh, d, dtype=s.dtype, device=DEV) for _ in range(2))
        row, size = (qh + 2 * kh) * d, s.qkv.element_size()
        s.append = Append(C.sizeof(Append), s.max_rows, _ptr(s.cu), _ptr(s.lens_in), _ptr(s.lens_out), _ptr(s.qkv), _ptr(s.qkv) + qh * d * size,
                          _ptr(s.qkv) + (qh + kh) * d * size, row, row, row, 1 if c["norm"] else 0, 1e-6, _ptr(s.q_norm), _ptr(s.k_norm), s.rot_dims,
                          1 if c["rot"] == "neighbours" else 0, c["axes"], (C.c_int32 * 3)(*s.sections), _ptr(s.inv_freq), _ptr(s.positions),
                          _ptr(s.token_index), _ptr(s.q_out), _ptr(s.k_held), _ptr(s.v_held), _ptr(s.index), _ptr(s.mass))
    if kind in ("attend", "step"):
        if kind == "attend":
            s.q = (rnd(R, qh, d) * (2.0 / loudest)).to(s.dtype)
        s.out = torch.zeros(R, qh, d, dtype=s.dtype, device=DEV)
        s.weights = c["weights"]
        lens = s.lens_out if kind == "step" else s.lens_full
        s.attention = Attention(C.sizeof(Attention), s.max_rows, max(s.max_new, 1), s.max_len, _ptr(s.cu), _ptr(lens), _ptr(s.q_out if kind == "step" else s.q),
                                _ptr(s.out), s.scale, 0, _ptr(s.mass) if s.weights else None, _ptr(s.mass_out) if s.weights else None, None, 0)
    if kind in ("evict", "read"):
        rows = c["budget"] if kind == "evict" else s.max_len
        s.k_out, s.v_out = (torch.zeros(B, rows, kh, d, dtype=s.dtype, device=DEV) for _ in range(2))
        if kind == "evict":
            s.evict = Evict(C.sizeof(Evict), rows, rows, c["keep_first"], c["keep_last"], 0, _ptr(s.lens_in), _ptr(s.lens_out), _ptr(s.index), _ptr(s.index_out),
                            _ptr(s.mass), _ptr(s.mass_out), None, 0)
        s.read = Read(C.sizeof(Read), 0, rows, 0, _ptr(s.lens_out if kind == "evict" else s.lens_in), _ptr(s.k_out), _ptr(s.v_out))
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------------
def _owner(s):
    """Of the rows that belong to a sequence: row, sequence, place among the sequence's new rows."""
    row = torch.arange(s.max_rows, device=DEV)
    row = row[row < s.cu[-1]]
    b = torch.searchsorted(s.cu[1:].contiguous(), row.int(), right=True)
    return row, b, row - s.cu[b]


def _turn(s, x, row):
    """x fp32 [rows, heads, d], turned by the rows' positions."""
    half = s.rot_dims // 2
    axis = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(s.sections, device=DEV))
    angle = s.positions[:, row][axis % s.positions.shape[0]].double().T * s.inv_freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if s.append.rot_kind == 0:
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)
    a, b, rest = x[..., 0:2 * half:2], x[..., 1:2 * half:2], x[..., 2 * half:]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), rest), -1)


def _normed(s, x, w):
    if not s.case["norm"]:
        return x
    mean = x.double().square().mean(-1, keepdim=True).float()
    return x * (1.0 / torch.sqrt(mean + 1e-6)) * w.float()


def _append(s):
    c, qh, kh, d = s.case, s.case["q_heads"], s.case["kv_heads"], s.case["head_dim"]
    row, b, i = _owner(s)
    x = s.qkv[row].float().unflatten(-1, (-1, d))
    q = _turn(s, _normed(s, x[:, :qh], s.q_norm), row)
    k = _turn(s, _normed(s, x[:, qh:qh + kh], s.k_norm), row)
    v = x[:, qh + kh:]
    s.q_out[row] = q.to(s.dtype)
    place = s.lens_in[b] + i
    page, r = s.table[b, place // PAGE].long(), (place % PAGE).long()
    w32 = s.pool.view(torch.int32)
    head = torch.arange(kh, device=DEV)[None, :, None]
    a, b_, c_, e = _parts(d)
    for x, key, at_codes, at_params, held in ((k, True, a, b_, s.k_held), (v, False, c_, e, s.v_held)):
        codes, scale, low = _quantise(x)
        words, params = _words(codes, key), _pair(scale, low)
        for t, at in ((words, at_codes), (params, at_params)):
            n = t.shape[-1]
            w32[page[:, None, None], head, at + r[:, None, None] * n + torch.arange(n, device=DEV)] = t
        held[row] = _values(words, params, key).to(s.dtype)
    s.index[page, :, r] = s.token_index[row][:, None].expand(-1, kh)
    s.mass[page, :, r] = 0.0
    s.lens_out.copy_(s.lens_in + (s.cu[1:] - s.cu[:-1]))


def _gathered(s, t):
    """t [pages, ...] -> [batch, pages of the longest, ...]."""
    n = (s.max_len + PAGE - 1) // PAGE
    return t[s.table[:, :n].long()]


def _attend(s, q, lens):
    c, kh, d = s.case, s.case["kv_heads"], s.case["head_dim"]
    B, g, n = c["batch"], c["q_heads"] // kh, max(s.max_new, 1)
    k, v = _tiles(_gathered(s, s.pool), d)                       # [B, pages, kv heads, 64, d]
    k, v = (t.transpose(1, 2).flatten(2, 3) for t in (k, v))     # [B, kv heads, rows, d]
    L = k.shape[2]
    seen = torch.arange(L, device=DEV)[None] < lens[:, None]
    k, v = (torch.where(seen[:, None, :, None], t, torch.zeros((), device=DEV)) for t in (k, v))
    row, b, i = _owner(s)
    x = torch.zeros(B, n, c["q_heads"], d, device=DEV)
    x[b, i] = q[row].float()
    x = x.view(B, n, kh, g, d).permute(0, 2, 3, 1, 4).reshape(B, kh, g * n, d)
    score = (torch.matmul(x, k.transpose(-1, -2)) * s.scale).view(B, kh, g, n, L)
    count = s.cu[1:] - s.cu[:-1]
    i_ = torch.arange(n, device=DEV)
    last = (lens - count)[:, None] + i_[None]                    # last cached row that a new row sees
    see = (torch.arange(L, device=DEV)[None, None] <= last[..., None]) & (i_[None] < count[:, None])[..., None] & seen[:, None]
    see = see[:, None, None]
    score = torch.where(see, score, torch.full((), -math.inf, device=DEV))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top.isinf(), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p.view(B, kh, g * n, L), v).view(B, kh, g, n, d).permute(0, 3, 1, 2, 4).reshape(B, n, c["q_heads"], d)
    s.out[row] = o[b, i].to(s.dtype)
    if s.weights:
        w = p.sum((2, 3))                                        # [B, kv heads, rows]
        at = seen.nonzero(as_tuple=True)
        page, r = s.table[at[0], at[1] // PAGE].long(), at[1] % PAGE
        s.mass_out[page, :, r] = s.mass[page, :, r] + w[at[0], :, at[1]]


def _evict(s):
    c, kh, d = s.case, s.case["kv_heads"], s.case["head_dim"]
    budget = c["budget"]
    per_row = lambda t: _gathered(s, t).transpose(1, 2).flatten(2)  # noqa: E731
    index, mass = per_row(s.index), per_row(s.mass)              # [B, kv heads, rows]
    L = index.shape[-1]
    row = torch.arange(L, device=DEV)
    lens = s.lens_in.long()[:, None, None]
    seen = row < lens
    newest = torch.where(seen, index, torch.full_like(index, -1)).amax(-1, keepdim=True)
    always = (index < c["keep_first"]) | (index > newest - c["keep_last"])
    key = torch.where(mass.isnan(), torch.full((), -3e38, device=DEV), mass)
    key = torch.where(always, torch.full((), math.inf, device=DEV), key)
    key = torch.where(seen, key, torch.full((), -math.inf, device=DEV))
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.zeros_like(seen.expand_as(key)).scatter(-1, best, True)
    over = lens > budget
    kept = torch.where(over, kept & seen, seen.expand_as(kept))
    hole, extra = (~kept & (row < budget) & over).nonzero(as_tuple=True), (kept & (row >= budget) & over).nonzero(as_tuple=True)
    place = lambda h: (s.table[h[0], h[2] // PAGE].long(), h[1], h[2] % PAGE)  # noqa: E731
    (pd, hd, rd), (ps, hs, rs) = place(hole), place(extra)       # as many of one as of the other, head by head
    w32 = s.pool.view(torch.int32)
    for lo, n in zip(_parts(d), (d // 8, d // 64, d // 8, d // 64)):
        col = lo + torch.arange(n, device=DEV)[None]
        w32[pd[:, None], hd[:, None], col + rd[:, None] * n] = w32[ps[:, None], hs[:, None], col + rs[:, None] * n]
    s.lens_out.copy_(torch.where(s.lens_in > budget, torch.full_like(s.lens_in, budget), s.lens_in))
    left = (row < s.lens_out[:, None, None]).expand_as(kept).nonzero(as_tuple=True)
    pl = place(left)
    for src, dst in ((s.index, s.index_out), (s.mass, s.mass_out)):
        dst[pl] = src[pl]
        dst[pd, hd, rd] = src[ps, hs, rs]


def _read(s, lens):
    rows = s.k_out.shape[1]
    seen = (torch.arange(rows, device=DEV)[None] < lens[:, None]).nonzero(as_tuple=True)
    for t, out in zip(_tiles(_gathered(s, s.pool), s.case["head_dim"]), (s.k_out, s.v_out)):
        t = t.transpose(2, 3).flatten(1, 2)                      # [B, rows, kv heads, d]
        out[seen] = t[seen].to(s.dtype)


# ---- one pass --------------------------------------------------------------------------------------------------------------
def run(s):
    kind = s.case["kind"]
    if own:
        if kind in ("append", "step"):
            call("append", s, s.append)
        if kind in ("attend", "step"):
            call("attention", s, s.attention)
        if kind == "evict":
            call("evict", s, s.evict)
        if kind in ("evict", "read"):
            call("read", s, s.read)
    else:
        if kind in ("append", "step"):
            _append(s)
        if kind in ("attend", "step"):
            _attend(s, s.q_out if kind == "step" else s.q, s.lens_out if kind == "step" else s.lens_full)
        if kind == "evict":
            _evict(s)
        if kind in ("evict", "read"):
            _read(s, s.lens_out if kind == "evict" else s.lens_in)
    out = {}
    if kind in ("append", "step"):
        out.update(q=s.q_out, k=s.k_held, v=s.v_held, lens=s.lens_out, index=s.index)
    if kind in ("attend", "step"):
        out["out"] = s.out
        if s.weights:
            out["mass"] = s.mass_out
    if kind == "evict":
        out.update(lens=s.lens_out, index=s.index_out, mass=s.mass_out)
    if kind in ("evict", "read"):
        out.update(k=s.k_out, v=s.v_out)
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    c = case
    kind, qh, kh, d = c["kind"], c["q_heads"], c["kv_heads"], c["head_dim"]
    row = 2 * (d // 2 + d // 16)                                 # bytes of a cached row of one kv head, keys and values
    new, held = _lengths(c)
    by, fl = 0, 0
    if kind in ("append", "step"):
        n = sum(new)
        by += n * ((qh + 2 * kh) * d * 2 + qh * d * 2 + kh * (row + 8) + 2 * kh * d * 2)
        fl += n * (qh + 2 * kh) * d * 8
    if kind in ("attend", "step"):
        by += sum(n + h for n, h in zip(new, held) if n) * kh * row + sum(new) * qh * d * 2 * (1 if kind == "step" else 2)
        if c["weights"]:
            by += sum(n + h for n, h in zip(new, held)) * kh * 8
        fl += sum(4 * d * qh * (n * h + n * (n + 1) // 2) for n, h in zip(new, held))
    if kind == "evict":
        m = c["budget"]
        for h in held:
            if h > m:
                by += kh * (8 * h + 8 * m + 2 * row * (m * (h - m) // h))
        held = [min(h, m) for h in held]
    if kind in ("evict", "read"):
        by += sum(held) * kh * (row + 2 * d * 2)
        fl += sum(held) * kh * d * 4
    return {"bytes": by, "flops": fl}


# ---- 64 bits ---------------------------------------------------------------------------------------------------------------
def _tile64(tile, d, part):
    """One tile as bytes on the host side of the definition: float64 [64, d] of its keys (part 0) or values (part 1)."""
    half = PAGE * (d // 2 + d // 16)
    t = tile[..., part * half:(part + 1) * half]
    code, par = t[..., :PAGE * d // 2].unflatten(-1, (PAGE, d // 2)), t[..., PAGE * d // 2:].contiguous().view(torch.float16).double().unflatten(-1, (PAGE, d // 64, 2))
    both = torch.stack((code & 15, code >> 4), -1).double()      # [..., 64, byte, nibble]
    ch = torch.arange(d)
    word = ch // 8 if part else (ch % 64 // 16) * (2 * (d // 64)) + (ch // 64) * 2 + ch % 16 // 8
    nib = ch % 8 // 2 + 4 * (ch % 2)
    x = both.flatten(-2)[..., (word * 8 + nib).to(tile.device)]
    g = (ch // 64).to(tile.device)
    return par[..., g, 1] + par[..., g, 0] * x


def _held64(s, b, n):
    """Keys and values of sequence b's first n cached rows, float64 [kv heads, n, d]."""
    t = s.pool[s.table[b, :(n + PAGE - 1) // PAGE].long()]
    return [_tile64(t, s.case["head_dim"], p).transpose(0, 1).flatten(1, 2)[:, :n] for p in (0, 1)]


def _snap64(x):
    """float64 [..., d] as 4 bits hold it."""
    y = torch.nan_to_num(x, nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504.0, 65504.0).unflatten(-1, (-1, GROUP))
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    sc, mn = ((hi - lo) / 15).half().double(), lo.half().double()
    code = ((y - mn) / torch.where(sc > 0, sc, torch.ones_like(sc))).round().clamp(0, 15) * (sc > 0)
    return (mn + sc * code).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    c, kind, qh, kh, d = case, case["kind"], case["q_heads"], case["kv_heads"], case["head_dim"]
    new, held = _lengths(c)
    cu = s.cu.tolist()
    out = {}
    if kind in ("append", "step"):
        R = s.q_out.shape[0]
        x = s.qkv.double().view(R, -1, d)

        def head(t, w):
            if c["norm"]:
                t = t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double()
            t, half = t.clone(), s.rot_dims // 2
            for j in range(half):
                axis = 0 if j < s.sections[0] else 1 if j < s.sections[0] + s.sections[1] else 2
                ang = s.positions[axis if c["axes"] == 3 else 0].double() * s.inv_freq[j]
                u, v = (j, j + half) if c["rot"] == "halves" else (2 * j, 2 * j + 1)
                co, si = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
                a, b = t[..., u].clone(), t[..., v].clone()
                t[..., u], t[..., v] = a * co - b * si, b * co + a * si
            return t
        live = (torch.arange(R, device=DEV) < cu[-1])[:, None, None]
        q = head(x[:, :qh], s.q_norm) * live
        k, v = _snap64(head(x[:, qh:qh + kh], s.k_norm)) * live, _snap64(x[:, qh + kh:]) * live
        out.update(q=q, k=k, v=v, lens=s.lens_full, index=None)
    if kind in ("attend", "step"):
        o = torch.zeros(s.out.shape, dtype=torch.float64, device=DEV)
        mass = torch.zeros(s.mass.shape, dtype=torch.float64, device=DEV)
        if sum(4 * d * qh * n * (n + h) for n, h in zip(new, held)) > 1e13:
            return None
        for b in range(c["batch"]):
            n, have = new[b], held[b] + (new[b] if kind == "attend" else 0)
            K, V = _held64(s, b, have)
            if kind == "step":
                at = slice(cu[b], cu[b + 1])
                K, V = torch.cat((K, k[at].transpose(0, 1)), 1), torch.cat((V, v[at].transpose(0, 1)), 1)
            L = K.shape[1]
            if not L:
                continue
            w = torch.zeros(kh, L, dtype=torch.float64, device=DEV)
            limit = (torch.arange(n, device=DEV) + L - n)[:, None]
            far = torch.arange(L, device=DEV)[None] > limit
            for h in range(qh if n else 0):
                x = (q.to(s.dtype) if kind == "step" else s.q)[cu[b]:cu[b + 1], h].double()      # q is rounded once, by definition
                p = torch.softmax((x @ K[h // (qh // kh)].T * s.scale).masked_fill(far, -math.inf), -1)
                o[cu[b]:cu[b + 1], h] = p @ V[h // (qh // kh)]
                w[h // (qh // kh)] += p.sum(0)
            if s.weights:
                r = torch.arange(L, device=DEV)
                page = s.table[b, r // PAGE].long()
                before = s.mass[page, :, r % PAGE].double()
                if kind == "step":
                    before[held[b]:] = 0
                mass[page, :, r % PAGE] = before + w.T
        out["out"] = o
        if s.weights:
            # a step's sums follow the rounded q, whose last bit two exact computations may place differently
            out["mass"] = mass if kind == "attend" else None
    if kind == "evict":
        m, first, last = c["budget"], c["keep_first"], c["keep_last"]
        mass = torch.zeros(s.mass.shape, dtype=torch.float64, device=DEV)
        kv = [torch.zeros(s.k_out.shape, dtype=torch.float64, device=DEV) for _ in range(2)]
        for b in range(c["batch"]):
            n = held[b]
            r = torch.arange(n, device=DEV)
            page = s.table[b, r // PAGE].long()
            ms, ix = s.mass[page, :, r % PAGE].T.double().cpu().numpy(), s.index[page, :, r % PAGE].T.cpu().numpy()
            K, V = _held64(s, b, n)
            for h in range(kh):
                rows = np.arange(n)
                if n > m:
                    safe = (ix[h] < first) | (ix[h] > ix[h].max() - last)
                    keep = np.zeros(n, bool)
                    keep[np.lexsort((rows, np.where(safe, -np.inf, -ms[h])))[:m]] = True
                    rows = np.arange(m)
                    rows[~keep[:m]] = m + np.flatnonzero(keep[m:])
                to = torch.arange(len(rows), device=DEV)
                src = torch.from_numpy(rows).to(DEV)
                mass[s.table[b, to // PAGE].long(), h, to % PAGE] = s.mass[page[src], h, src % PAGE].double()
                for t, dst in zip((K, V), kv):
                    dst[b, :min(len(rows), m), h] = t[h, src[:m]]
        out.update(lens=None, index=None, mass=mass, k=kv[0], v=kv[1])
    if kind == "read":
        kv = [torch.zeros(s.k_out.shape, dtype=torch.float64, device=DEV) for _ in range(2)]
        for b in range(c["batch"]):
            for t, dst in zip(_held64(s, b, held[b]), kv):
                dst[b, :held[b]] = t.transpose(0, 1)
        out.update(k=kv[0], v=kv[1])
    return out
