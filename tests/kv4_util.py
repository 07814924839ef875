"""Binding of include/efm_b200_kv4.h and a plain 64-bit statement of what its operators do (numpy, row by row, from the header's text)."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np

import cabi

P, I32, I64 = C.c_void_p, C.c_int32, C.c_int64
ROWS = GROUP = 64
BAD_PAGE, FULL, BAD_COUNT, WAIT = 1, 2, 4, 8


class Cache(C.Structure):
    _fields_ = [(n, I32) for n in ("struct_size", "dtype", "q_heads", "kv_heads", "head_dim", "n_pages", "batch", "max_pages")] + \
        [(n, P) for n in ("pool", "page_table", "status")]


class Append(C.Structure):
    _fields_ = [("struct_size", I32), ("max_rows", I32)] + [(n, P) for n in ("cu_rows", "lens_in", "lens_out", "q", "k", "v")] + \
        [(n, I64) for n in ("q_stride", "k_stride", "v_stride")] + [("norm", I32), ("norm_eps", C.c_float)] + [(n, P) for n in ("q_norm", "k_norm")] + \
        [(n, I32) for n in ("rot_dims", "rot_kind", "axes")] + [("sections", I32 * 3)] + \
        [(n, P) for n in ("inv_freq", "positions", "token_index", "q_out", "k_held", "v_held", "index", "mass")]


class Attention(C.Structure):
    _fields_ = [(n, I32) for n in ("struct_size", "max_rows", "max_new", "max_len")] + [(n, P) for n in ("cu_rows", "lens", "q", "out")] + \
        [("scale", C.c_float), ("reserved", I32)] + [(n, P) for n in ("mass_in", "mass_out", "workspace")] + [("workspace_bytes", I64)]


class Evict(C.Structure):
    _fields_ = [(n, I32) for n in ("struct_size", "budget", "limit", "keep_first", "keep_last", "reserved")] + \
        [(n, P) for n in ("lens_in", "lens_out", "index_in", "index_out", "mass_in", "mass_out", "workspace")] + [("workspace_bytes", I64)]


class Read(C.Structure):
    _fields_ = [(n, I32) for n in ("struct_size", "first", "rows", "reserved")] + [(n, P) for n in ("lens", "k_out", "v_out")]


SIGNATURES = {
    "efm_b200_kv4_tile_bytes": [I32, C.POINTER(I64)],
    "efm_b200_kv4_attention_workspace": [P, P, C.POINTER(I64)],
    "efm_b200_kv4_evict_workspace": [P, P, C.POINTER(I64)],
    "efm_b200_op_kv4_append": [P, P, P],
    "efm_b200_op_kv4_attention": [P, P, P],
    "efm_b200_op_kv4_evict": [P, P, P],
    "efm_b200_op_kv4_read": [P, P, P],
}


def lib():
    L = cabi.lib()
    if not hasattr(L, "_kv4"):
        for n, args in SIGNATURES.items():
            f = getattr(L, n)
            f.restype, f.argtypes = I32, args
        L._kv4 = True
    return L


def error():
    return cabi.lib().efm_b200_last_error(None).decode()


def tile_bytes(d):
    return 2 * ROWS * (d // 2 + d // 16)


# ---- the format, in 64 bits ------------------------------------------------------------------------------------------------
def nibble_place(d, key):
    """Of every channel of a row: its nibble, counted from the row's first byte (low nibble first)."""
    ch = np.arange(d)
    word = (ch % 64 // 16) * (2 * (d // 64)) + (ch // 64) * 2 + ch % 16 // 8 if key else ch // 8
    order = [0, 2, 4, 6, 1, 3, 5, 7]                   # channels of a word's nibbles, lowest first
    return word * 8 + np.array([order.index(i) for i in range(8)])[ch % 8]


def parts(d):
    codes, params = ROWS * d // 2, ROWS * d // 64 * 4
    return (0, codes), (codes, codes + params), (codes + params, 2 * codes + params), (2 * codes + params, 2 * (codes + params))


def unpack(tile, d):
    """uint8 [..., tile] -> codes, scales, minima of keys, then of values: ([..., 64, d], [..., 64, d/64], [..., 64, d/64])."""
    out = []
    for key, (a, b), (c, e) in ((True, *parts(d)[:2]), (False, *parts(d)[2:])):
        t = tile[..., a:b].reshape(*tile.shape[:-1], ROWS, d // 2)
        nib = np.stack((t & 15, t >> 4), -1).reshape(*t.shape[:-1], d)
        par = np.ascontiguousarray(tile[..., c:e]).view(np.float16).reshape(*tile.shape[:-1], ROWS, d // 64, 2).astype(np.float64)
        out.append((nib[..., nibble_place(d, key)].astype(np.int64), par[..., 0], par[..., 1]))
    return out


def values(codes, scale, low):
    return np.repeat(low, GROUP, -1) + np.repeat(scale, GROUP, -1) * codes


def snap(x, ds=0.0, dl=0.0):
    """float64 [..., d] -> unrounded codes, codes, scale, minimum; the last two as they round when they are off by ds and dl before."""
    x = np.clip(np.nan_to_num(x, nan=0.0, posinf=65504.0, neginf=-65504.0), -65504.0, 65504.0).reshape(*x.shape[:-1], -1, GROUP)
    low, scale = (x.min(-1) * (1 + dl)).astype(np.float16).astype(np.float64), ((x.max(-1) - x.min(-1)) / 15 * (1 + ds)).astype(np.float16).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        raw = np.where(scale[..., None] > 0, (x - low[..., None]) / scale[..., None], 0.0)
    shape = (*x.shape[:-2], -1)
    return raw.reshape(shape), np.clip(np.rint(raw), 0, 15).reshape(shape).astype(np.int64), scale, low


def turned(x, pos, inv_freq, rot_dims, kind, sections=None):
    """x [heads, d]; pos: positions of the axes."""
    y, half = x.copy(), rot_dims // 2
    for i in range(half):
        axis = 0 if sections is None or i < sections[0] else 1 if i < sections[0] + sections[1] else 2
        c, s = math.cos(float(pos[axis]) * float(inv_freq[i])), math.sin(float(pos[axis]) * float(inv_freq[i]))
        a, b = (i, i + half) if kind == 0 else (2 * i, 2 * i + 1)
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
    return y


def normed(x, eps, w):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def attend(q, k, v, scale, spread=None):
    """q [n, heads, d], k / v [kv heads, L, d] (float64), row i sees L - n + i + 1 rows.  -> out, weights [heads, n, L], sum of p max(|v|, spread)."""
    big = np.abs(v) if spread is None else np.maximum(np.abs(v), spread)
    n, qh, d = q.shape
    L, g = k.shape[1], qh // k.shape[0]
    out, size, w = np.zeros((n, qh, d)), np.zeros((n, qh, d)), np.zeros((qh, n, L))
    for i in range(n):
        see = min(L, L - n + i + 1)
        for h in range(qh if see > 0 else 0):
            s = (k[h // g, :see] @ q[i, h]) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            w[h, i, :see] = p
            out[i, h], size[i, h] = p @ v[h // g, :see], p @ big[h // g, :see]
    return out, w, size


def evicted(index, mass, budget, keep_first, keep_last):
    """Rows of one head that stay, as the list of old rows by new row."""
    n = len(index)
    newest = max(int(i) for i in index)
    rank = []
    for r in range(n):
        always = index[r] < keep_first or index[r] > newest - keep_last
        m = float(mass[r])
        rank.append((0, 0.0, r) if always else (2, 0.0, r) if math.isnan(m) else (1, -m, r))
    keep = sorted(r for _, _, r in sorted(rank)[:budget])
    stay, extra = [r for r in keep if r < budget], [r for r in keep if r >= budget]
    out = dict((r, r) for r in stay)
    for hole, r in zip([r for r in range(budget) if r not in out], extra):
        out[hole] = r
    return [out[r] for r in range(budget)]


# ---- a cache on the GPU ----------------------------------------------------------------------------------------------------
class KV4:
    """Pool, table and lengths of a batch, with the calls.  Unused rows and pages hold bits that read as NaN."""

    def __init__(self, q_heads, kv_heads, head_dim, lens, capacity=None, dtype="bf16", seed=0, n_pages=None, spare=3, device="cuda:0"):
        import torch
        self.torch, self.dev, self.dtype = torch, device, {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
        self.qh, self.kh, self.d, self.batch = q_heads, kv_heads, head_dim, len(lens)
        need = [max(1, -(-max(n, 1) // ROWS)) for n in (capacity or lens)]
        self.max_pages = max(need)
        total = sum(need)
        self.n_pages = n_pages or total + spare
        rng = np.random.default_rng(seed)
        order = rng.permutation(total + spare) + (self.n_pages - total - spare)
        table = np.full((self.batch, self.max_pages), -7, np.int32)          # columns that must not be read
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.np_table = table
        if n_pages is None:
            self.pool = torch.full((self.n_pages, kv_heads, tile_bytes(head_dim)), 255, dtype=torch.uint8, device=device)
        else:
            self.pool = torch.empty((self.n_pages, kv_heads, tile_bytes(head_dim)), dtype=torch.uint8, device=device)
        self.table = torch.from_numpy(table).to(device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.lens = self.ints(lens)
        self.index = torch.full((self.n_pages, kv_heads, ROWS), -1, dtype=torch.int32, device=device) if n_pages is None else None
        self.mass = torch.full((self.n_pages, kv_heads, ROWS), float("nan"), device=device) if n_pages is None else None
        self.rng = rng
        self.code = {"bf16": cabi.EFM_BF16, "fp16": cabi.EFM_F16}[dtype]
        self.keep = []

    def ints(self, v):
        return self.torch.tensor([int(x) for x in np.asarray(v).reshape(-1)], dtype=self.torch.int32, device=self.dev)

    def normal(self, *shape, scale=1.0):
        return self.torch.from_numpy((self.rng.standard_normal(shape) * scale).astype(np.float32)).to(self.dev).to(self.dtype)

    def cache(self, **over):
        c = Cache(C.sizeof(Cache), self.code, self.qh, self.kh, self.d, self.n_pages, self.batch, self.max_pages, self.pool.data_ptr(), self.table.data_ptr(),
                  self.status.data_ptr())
        for k, v in over.items():
            setattr(c, k, v)
        return c

    def stream(self):
        return self.torch.cuda.current_stream().cuda_stream

    def do(self, name, args, want=0, **over):
        st = getattr(lib(), "efm_b200_op_kv4_" + name)(C.byref(self.cache(**over)), C.byref(args), self.stream())
        assert st == want, (st, error())

    def fill(self, loud=0.5):
        """Rows below lens hold snapped normal numbers, written straight into the tiles."""
        d, lens = self.d, self.lens.tolist()
        pool = self.pool.cpu().numpy() if self.n_pages < 4096 else None
        gain = np.exp(loud * self.rng.standard_normal((self.kh, 1, d)))
        for b, n in enumerate(lens):
            for k in range(-(-n // ROWS)):
                page, m = self.np_table[b, k], min(ROWS, n - k * ROWS)
                tile = np.full((self.kh, tile_bytes(d)), 255, np.uint8)
                for key, (a, e), (p0, p1) in ((True, *parts(d)[:2]), (False, *parts(d)[2:])):
                    _, codes, scale, low = snap(self.rng.standard_normal((self.kh, m, d)) * (gain if key else 1.0))
                    nib = np.zeros((self.kh, m, d), np.uint8)
                    nib[..., nibble_place(d, key)] = codes
                    tile[:, a:e].reshape(self.kh, ROWS, d // 2)[:, :m] = nib[..., 0::2] | (nib[..., 1::2] << 4)
                    par = np.stack((scale, low), -1).astype(np.float16)
                    tile[:, p0:p1].reshape(self.kh, ROWS, d // 64 * 4)[:, :m] = np.ascontiguousarray(par).view(np.uint8).reshape(self.kh, m, -1)
                if pool is not None:
                    pool[page] = tile
                else:
                    self.pool[page] = self.torch.from_numpy(tile).to(self.dev)
        if pool is not None:
            self.pool.copy_(self.torch.from_numpy(pool))
        return self

    def held(self, b, n):
        """Keys and values of sequence b, float64 [kv heads, n, d]."""
        if n == 0:
            return [np.zeros((self.kh, 0, self.d))] * 2
        pages = self.np_table[b, :-(-n // ROWS)]
        tiles = self.pool[self.torch.from_numpy(pages.astype(np.int64)).to(self.dev)].cpu().numpy()
        return [values(*u).swapaxes(0, 1).reshape(self.kh, -1, self.d)[:, :n] for u in unpack(tiles, self.d)]

    def spread(self, b, n):
        """|scale (code - 8)| of sequence b's values: what a weight multiplies once the centre of the codes is taken out."""
        if n == 0:
            return np.zeros((self.kh, 0, self.d))
        tiles = self.pool[self.torch.from_numpy(self.np_table[b, :-(-n // ROWS)].astype(np.int64)).to(self.dev)].cpu().numpy()
        codes, scale, _ = unpack(tiles, self.d)[1]
        return np.abs(np.repeat(scale, GROUP, -1) * (codes - 8)).swapaxes(0, 1).reshape(self.kh, -1, self.d)[:, :n]

    def rows_of(self, t, b, n):
        """t [pages, kv heads, 64] -> [kv heads, n] of sequence b."""
        pages = self.np_table[b, :max(1, -(-n // ROWS))].astype(np.int64)
        return t[self.torch.from_numpy(pages).to(self.dev)].cpu().numpy().swapaxes(0, 1).reshape(self.kh, -1)[:, :n]

    def append_args(self, counts, lens_out, q, k, v, max_rows=None, **kw):
        self.cu = self.ints(np.concatenate(([0], np.cumsum(counts))))
        self.keep += [self.cu, q, k, v, lens_out]
        a = Append(C.sizeof(Append), max_rows if max_rows is not None else int(sum(counts)), self.cu.data_ptr(), self.lens.data_ptr(), lens_out.data_ptr(),
                   q.data_ptr() if q is not None else None, k.data_ptr(), v.data_ptr(), q.stride(0) if q is not None else 0, k.stride(0), v.stride(0))
        for n, x in kw.items():
            if hasattr(x, "data_ptr"):
                self.keep.append(x)
                x = x.data_ptr()
            setattr(a, n, (I32 * 3)(*x) if n == "sections" else x)
        return a

    def attention_args(self, counts, lens, q, out, max_rows=None, max_len=0, scale=None, mass=None, mass_out=None, workspace=None, max_new=None):
        self.cu = self.ints(np.concatenate(([0], np.cumsum(counts))))
        a = Attention(C.sizeof(Attention), max_rows if max_rows is not None else q.shape[0], max_new if max_new is not None else max(max(counts), 1), max_len,
                      self.cu.data_ptr(), lens.data_ptr(), q.data_ptr(), out.data_ptr(), scale or 1.0 / math.sqrt(self.d), 0,
                      mass.data_ptr() if mass is not None else None, (mass_out if mass_out is not None else mass).data_ptr() if mass is not None else None, None, 0)
        self.keep += [self.cu, lens, q, out, mass, mass_out]
        return self.with_workspace("attention", a, workspace)

    def with_workspace(self, name, a, ws=None):
        need = I64()
        st = getattr(lib(), f"efm_b200_kv4_{name}_workspace")(C.byref(self.cache()), C.byref(a), C.byref(need))
        assert st == 0, error()
        if ws is None:
            ws = self.torch.empty(max(need.value, 16), dtype=self.torch.uint8, device=self.dev)
            ws.random_(0, 256)                               # its contents do not matter
        assert ws.numel() >= need.value
        self.keep.append(ws)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        return a

    def evict_args(self, lens_in, lens_out, budget, limit, keep_first, keep_last, index_out=None, mass_out=None):
        a = Evict(C.sizeof(Evict), budget, limit, keep_first, keep_last, 0, lens_in.data_ptr(), lens_out.data_ptr(), self.index.data_ptr(),
                  (index_out if index_out is not None else self.index).data_ptr(), self.mass.data_ptr(), (mass_out if mass_out is not None else self.mass).data_ptr(), None, 0)
        self.keep += [lens_in, lens_out, index_out, mass_out]
        return self.with_workspace("evict", a)
