// Bringing a 4-bit cache back to a budget of rows (kv4_cache.cuh), each kv head by itself.
//
// Rows are ordered by (protected, mass, lower row first); the budget-th key is found digit by digit (11 + 11 + 10 bits of a 32-bit key,
// a histogram each), rows equal to it are taken from the lowest up.  Kept rows below the budget stay, those behind it move into the
// free rows, so that at most min(budget, rows - budget) rows move and no row that is written is read by another: one pass in place.
// Two launches: a block per sequence and head orders and writes the list of moves (bound by its walks over 8 bytes a row, latency on
// small caches), then blocks of 16 lanes a row move codes, parameters, token number and mass (bound by bytes).
#pragma once
#include "kv4_cache.cuh"

namespace efm {
namespace kv4 {

struct EvictParams {
    int budget, limit, keep_first, keep_last;
    const int32_t *lens_in, *index_in;
    int32_t *lens_out, *index_out;
    const float* mass_in;
    float* mass_out;
    int2* moves;              // [batch, kv_heads, most_moves] (from, to)
    int32_t* n_moves;         // [batch, kv_heads]
    int most_moves;
    int keys_cap;             // keys that fit in shared memory; a longer sequence computes them again on every walk
};

constexpr int kEvictThreads = 1024, kBins = 2048, kMoveThreads = 256;

// Ascending order of masses as unsigned numbers: NaN 0, protected rows the largest.
__device__ __forceinline__ uint32_t evict_key(float mass, bool always) {
    if (always) return 0xffffffffu;
    if (mass != mass) return 0u;
    const uint32_t u = __float_as_uint(mass + 0.0f);      // -0 is 0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Sum of v over the threads below this one; *total: over all.
__device__ __forceinline__ int block_prefix(int v, int* sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int y = sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        sums[lane] = y;
    }
    __syncthreads();
    const int before = (warp > 0 ? sums[warp - 1] : 0) + x - v;
    *total = sums[31];
    __syncthreads();
    return before;
}

// grid (kv heads, batch)
__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(const Cache c, const EvictParams p) {
    extern __shared__ uint32_t keys[];
    __shared__ int hist[kBins], sums[32], found[2], newest_s;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    const int n = held(c, p.lens_in, b, c.max_pages * kRows);
    const bool over = n > p.limit;
    const int left = over ? p.budget : n;
    if (h == 0 && tid == 0) p.lens_out[b] = left;
    auto slot = [&](int row, size_t& at) {
        const int page = page_of(c, b, row / kRows);
        at = page < 0 ? 0 : row_slot(c, page, h, row % kRows);
        return page >= 0;
    };
    if (!over) {
        if (tid == 0) p.n_moves[b * c.kv_heads + h] = 0;
        if (p.index_out != p.index_in || p.mass_out != p.mass_in)
            for (int row = tid; row < n; row += kEvictThreads) {
                size_t at;
                if (!slot(row, at)) continue;
                const int ix = p.index_in[at];
                const float ms = p.mass_in[at];
                p.index_out[at] = ix;
                p.mass_out[at] = ms;
            }
        return;
    }
    if (tid == 0) newest_s = INT32_MIN;
    __syncthreads();
    int newest = INT32_MIN;
    for (int row = tid; row < n; row += kEvictThreads) {
        size_t at;
        if (slot(row, at)) newest = max(newest, p.index_in[at]);
    }
    atomicMax(&newest_s, newest);
    __syncthreads();
    newest = newest_s;
    auto make_key = [&](int row) -> uint32_t {
        size_t at;
        if (!slot(row, at)) return 0u;                           // rows of a bad page count as the least
        const int ix = p.index_in[at];
        return evict_key(p.mass_in[at], ix < p.keep_first || (long long)ix > (long long)newest - p.keep_last);
    };
    const bool cached = n <= p.keys_cap;
    if (cached) for (int row = tid; row < n; row += kEvictThreads) keys[row] = make_key(row);
    __syncthreads();
    auto key_of = [&](int row) { return cached ? keys[row] : make_key(row); };

    // the budget-th largest key; `want` of the rows equal to it are kept
    uint32_t prefix = 0;
    int want = p.budget;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11, bins = 1 << bits;
        for (int i = tid; i < kBins; i += kEvictThreads) hist[i] = 0;
        __syncthreads();
        for (int row = tid; row < n; row += kEvictThreads) {
            const uint32_t k = key_of(row);
            if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
        }
        __syncthreads();
        const int d1 = kBins - 1 - 2 * tid, d0 = d1 - 1;         // this thread's two digits, the largest digits first
        const int c1 = hist[d1], c0 = hist[d0];
        int total;
        const int before = block_prefix(c1 + c0, sums, &total);
        if (before < want && want <= before + c1) { found[0] = d1; found[1] = before; }
        else if (before + c1 < want && want <= before + c1 + c0) { found[0] = d0; found[1] = before + c1; }
        __syncthreads();
        prefix = (prefix << bits) | (uint32_t)found[0];
        want -= found[1];
        __syncthreads();
    }
    const uint32_t border = prefix;

    int ties = 0, holes = 0, extra = 0;                          // of the rows before this round's
    int2* moves = p.moves + (size_t)(b * c.kv_heads + h) * p.most_moves;
    for (int base = 0; base < n; base += kEvictThreads) {
        const int row = base + tid;
        const bool in = row < n;
        const uint32_t k = in ? key_of(row) : 0u;
        const bool tie = in && k == border;
        int total;
        const int rank = ties + block_prefix(tie, sums, &total);
        ties += total;
        const bool kept = in && (k > border || (tie && rank < want));
        const bool hole = in && !kept && row < p.budget, ext = kept && row >= p.budget;
        const int both = block_prefix((hole ? 1 : 0) + (ext ? 1 << 16 : 0), sums, &total);
        if (hole) moves[holes + (both & 0xffff)].y = row;
        if (ext) moves[extra + (both >> 16)].x = row;
        holes += total & 0xffff;
        extra += total >> 16;
        if (kept && row < p.budget && (p.index_out != p.index_in || p.mass_out != p.mass_in)) {
            size_t at;
            if (slot(row, at)) {
                const int ix = p.index_in[at];
                const float ms = p.mass_in[at];
                p.index_out[at] = ix;
                p.mass_out[at] = ms;
            }
        }
    }
    if (tid == 0) p.n_moves[b * c.kv_heads + h] = holes;
}

// grid (parts of the list, kv heads, batch); 16 lanes a row
template <int D>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const Cache c, const EvictParams p) {
    using L = Tile<D>;
    constexpr int Q = D / 32;                                    // 16-byte pieces of a row's codes
    const int h = blockIdx.y, b = blockIdx.z;
    pdl_launch_dependents();
    pdl_wait();
    const int n = p.n_moves[b * c.kv_heads + h];
    const int2* moves = p.moves + (size_t)(b * c.kv_heads + h) * p.most_moves;
    const int part = threadIdx.x & 15;
    for (int i = blockIdx.x * (kMoveThreads / 16) + threadIdx.x / 16; i < n; i += gridDim.x * (kMoveThreads / 16)) {
        const int2 m = moves[i];
        const int from = page_of(c, b, m.x / kRows), to = page_of(c, b, m.y / kRows);
        if (from < 0 || to < 0) continue;
        const uint8_t* src = tile_of<D>(c, from, h);
        uint8_t* dst = tile_of<D>(c, to, h);
        const int r = m.x % kRows, w = m.y % kRows;
        if (part < 2 * Q) {
            const int at = part < Q ? L::K_CODES : L::V_CODES, q = part % Q;
            reinterpret_cast<uint4*>(dst + at)[w * Q + q] = reinterpret_cast<const uint4*>(src + at)[r * Q + q];
        } else if (part < 2 * Q + 2 * L::G) {
            const int at = part < 2 * Q + L::G ? L::K_PARAMS : L::V_PARAMS, g = (part - 2 * Q) % L::G;
            reinterpret_cast<uint32_t*>(dst + at)[w * L::G + g] = reinterpret_cast<const uint32_t*>(src + at)[r * L::G + g];
        } else if (part == 14) {
            p.index_out[row_slot(c, to, h, w)] = p.index_in[row_slot(c, from, h, r)];
        } else if (part == 15) {
            p.mass_out[row_slot(c, to, h, w)] = p.mass_in[row_slot(c, from, h, r)];
        }
    }
}

}  // namespace kv4
}  // namespace efm
