// Bringing a 4-bit cache back to a budget of rows (kv4_cache.cuh), each kv head by itself.
//
// Rows are ordered by (protected, mass, lower row first); the budget-th key is found digit by digit (four of 8 bits, a histogram each in
// eight copies: masses share their exponents, and the rows of a warp queue at a few bins), rows equal to it are taken from the lowest up.
// Kept rows below the budget stay, those behind it move into the free rows, so that at most min(budget, rows - budget) rows move and no row that is written is read by another: one pass in place.
// A block per sequence and head orders and lists the moves (bound by its walks over 8 bytes a row, latency on small caches); 16 lanes a row
// move codes, parameters, token number and mass: the same block where few rows can move at all, else a second launch of as many blocks
// as fill the GPU (bound by bytes).
// 64 caches of 900 .. 4100 rows, 4 kv heads of 128, down to 1024: 19 us to order, 22 us to move 38 MB there and as many back; one of 600 rows
// 6 us.
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
    int2* moves;              // [batch, kv_heads, most_moves] (from, to), each 64 x page + row, or -1 in a page that is none
    int32_t* n_moves;         // [batch, kv_heads]
    int most_moves, head_dim, inline_moves;      // inline_moves: no second launch
    int keys_cap;             // keys that fit in shared memory; a longer sequence computes them again on every walk
};

constexpr int kEvictThreads = 512, kEvictWarps = kEvictThreads / 32, kBins = 256, kCopies = 8, kMoveThreads = 256;
constexpr int kInlineMoves = 256;         // rows: two rounds of a block's 128 rows, below the cost of a launch
// Rows a thread holds in registers, a round's 512: 5120 a round, or 1024 where a sequence cannot have more, which leaves out most of what
// is unrolled over them.
constexpr int kKeepMany = 10, kKeepFew = 2;

// Ascending order of masses as unsigned numbers: NaN 0, protected rows the largest.
__device__ __forceinline__ uint32_t evict_key(float mass, bool always) {
    if (always) return 0xffffffffu;
    if (mass != mass) return 0u;
    const uint32_t u = __float_as_uint(mass + 0.0f);      // -0 is 0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Rows by 16 lanes each, RUN of them on their way at a time: codes, parameters, token number and mass.
template <int D, int RUN>
__device__ __forceinline__ void move_rows(const Cache& c, const EvictParams& p, int h, const int2* moves, int first, int step, int n, int part) {
    using L = Tile<D>;
    constexpr int Q = D / 32;                                    // 16-byte pieces of a row's codes
    const bool codes = part < 2 * Q, pars = !codes && part < 2 * Q + 2 * L::G;
    const int piece = codes ? part % Q : (part - 2 * Q) % L::G;
    const int at = codes ? (part < Q ? L::K_CODES : L::V_CODES) : part < 2 * Q + L::G ? L::K_PARAMS : L::V_PARAMS;
    for (int i = first; i < n; i += RUN * step) {
        int2 m[RUN];
        uint4 v[RUN];
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
            m[k] = i + k * step < n ? moves[i + k * step] : make_int2(-1, -1);
            if (m[k].x < 0 || m[k].y < 0) m[k] = make_int2(-1, -1);
        }
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
            if (m[k].x < 0) continue;
            const int from = m[k].x / kRows, r = m[k].x % kRows;
            const uint8_t* src = tile_of<D>(c, from, h) + at;
            if (codes) v[k] = reinterpret_cast<const uint4*>(src)[r * Q + piece];
            else if (pars) v[k].x = reinterpret_cast<const uint32_t*>(src)[r * L::G + piece];
            else if (part == 14) v[k].x = (uint32_t)p.index_in[row_slot(c, from, h, r)];
            else if (part == 15) v[k].x = __float_as_uint(p.mass_in[row_slot(c, from, h, r)]);
        }
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
            if (m[k].x < 0) continue;
            const int to = m[k].y / kRows, r = m[k].y % kRows;
            uint8_t* dst = tile_of<D>(c, to, h) + at;
            if (codes) reinterpret_cast<uint4*>(dst)[r * Q + piece] = v[k];
            else if (pars) reinterpret_cast<uint32_t*>(dst)[r * L::G + piece] = v[k].x;
            else if (part == 14) p.index_out[row_slot(c, to, h, r)] = (int32_t)v[k].x;
            else if (part == 15) p.mass_out[row_slot(c, to, h, r)] = __uint_as_float(v[k].x);
        }
    }
}

// grid (kv heads, batch).  Barriers cost more than arithmetic here: rows are counted by ballots, and every warp adds up the warps' counts
// for itself.
template <int kKeep>
__global__ void __launch_bounds__(kEvictThreads, 2) evict_select_kernel(const Cache c, const EvictParams p) {
    extern __shared__ uint32_t keys[];
    __shared__ int hist[kBins * kCopies], counts[2][kKeep * kEvictWarps + 1], digit_sums[2][kEvictWarps], found[2], newest_s;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) newest_s = INT32_MIN;
    for (int i = tid; i < kBins * kCopies; i += kEvictThreads) hist[i] = 0;
    pdl_wait();
    pdl_launch_dependents();
    const int n = held(c, p.lens_in, b, c.max_pages * kRows);
    const bool over = n > p.limit, apart = p.index_out != p.index_in || p.mass_out != p.mass_in;
    if (h == 0 && tid == 0) p.lens_out[b] = over ? p.budget : n;
    auto place = [&](int row) {                                  // 64 x page + row, -1 where the page is none
        const int page = page_of(c, b, row / kRows);
        return page < 0 ? -1 : page * kRows + row % kRows;
    };
    auto slot = [&](int at) { return row_slot(c, at / kRows, h, at % kRows); };
    if (!over) {
        if (tid == 0) p.n_moves[b * c.kv_heads + h] = 0;
        if (apart)
            for (int row = tid; row < n; row += kEvictThreads) {
                const int at = place(row);
                if (at < 0) continue;
                const int ix = p.index_in[slot(at)];
                const float ms = p.mass_in[slot(at)];
                p.index_out[slot(at)] = ix;
                p.mass_out[slot(at)] = ms;
            }
        return;
    }
    // One walk over the rows: keys into shared memory where they fit (a longer sequence computes them again), those of the first round
    // in registers.  Where the outputs are other arrays every row below the budget is copied: the free ones are written by their moves.
    const bool cached = n <= p.keys_cap;
    int at[kKeep], newest = INT32_MIN;
    uint32_t key[kKeep];
    for (int base = 0; base < n; base += kKeep * kEvictThreads) {
        int a[kKeep], ix[kKeep];
        float ms[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) { const int row = base + i * kEvictThreads + tid; a[i] = row < n ? place(row) : -1; }
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            ix[i] = a[i] >= 0 ? p.index_in[slot(a[i])] : INT32_MIN;
            ms[i] = a[i] >= 0 ? p.mass_in[slot(a[i])] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const int row = base + i * kEvictThreads + tid;
            const uint32_t k = a[i] >= 0 ? evict_key(ms[i], ix[i] < p.keep_first) : 0u;      // rows of a bad page count as the least
            newest = max(newest, ix[i]);
            if (apart && a[i] >= 0 && row < p.budget) { p.index_out[slot(a[i])] = ix[i]; p.mass_out[slot(a[i])] = ms[i]; }
            if (cached && row < n) keys[row] = k;
            if (base == 0) { at[i] = a[i]; key[i] = k; }
        }
    }
    newest = __reduce_max_sync(0xffffffffu, newest);
    __syncthreads();
    if (lane == 0) atomicMax(&newest_s, newest);
    __syncthreads();
    const long long recent = (long long)newest_s - p.keep_last;  // token numbers above are kept
    if (p.keep_last > 0) {                                       // few rows: their numbers are read again
#pragma unroll
        for (int i = 0; i < kKeep; ++i)
            if (at[i] >= 0 && p.index_in[slot(at[i])] > recent) key[i] = 0xffffffffu;
        if (cached)
            for (int row = tid + kKeep * kEvictThreads; row < n; row += kEvictThreads) {
                const int x = place(row);
                if (x >= 0 && p.index_in[slot(x)] > recent) keys[row] = 0xffffffffu;
            }
    }
    auto key_of = [&](int row) -> uint32_t {                     // of the rows behind those in registers
        if (cached) return keys[row];
        const int x = place(row);
        if (x < 0) return 0u;
        const int ix = p.index_in[slot(x)];
        return evict_key(p.mass_in[slot(x)], ix < p.keep_first || ix > recent);
    };

    // the budget-th largest key; `want` of the rows equal to it are kept
    uint32_t prefix = 0;
    int want = p.budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
        auto count = [&](uint32_t k) {
            if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift & 255u) * kCopies + (tid & (kCopies - 1))], 1);
        };
#pragma unroll
        for (int i = 0; i < kKeep; ++i) if (tid + i * kEvictThreads < n) count(key[i]);
        for (int row = tid + kKeep * kEvictThreads; row < n; row += kEvictThreads) count(key_of(row));
        __syncthreads();
        const int digit = kBins - 1 - tid / 2;                   // two threads a digit, the largest digits first
        int4* from = reinterpret_cast<int4*>(hist) + digit * 2 + (tid & 1);
        const int4 v = *from;
        *from = make_int4(0, 0, 0, 0);
        int mine = v.x + v.y + v.z + v.w;
        mine += __shfl_xor_sync(0xffffffffu, mine, 1);
        int before = (tid & 1) == 0 ? mine : 0;                  // of the digits above this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += y; }
        int* sums = digit_sums[shift >> 3 & 1];
        if (lane == 31) sums[warp] = before;
        __syncthreads();
        const int ahead = lane < warp ? sums[lane] : 0;
        before += __reduce_add_sync(0xffffffffu, ahead) - mine;
        if ((tid & 1) == 0 && before < want && want <= before + mine) { found[0] = digit; found[1] = before; }
        __syncthreads();
        prefix = prefix << 8 | (uint32_t)found[0];
        want -= found[1];
    }
    const uint32_t border = prefix;

    // Ties, then free rows below the budget and kept ones behind it, numbered in the order of the rows: round by round, within a
    // round by (row of the thread, warp), within a warp by lane.
    int2* moves = p.moves + (size_t)(b * c.kv_heads + h) * p.most_moves;
    int ties = 0, holes = 0, extra = 0;                          // of the rounds before
    auto number = [&](int* cnt) {                                // counts in the rows' order become sums of those ahead, the last entry the total
        __syncthreads();
        if (warp == 0) {
            constexpr int PER = kKeep * kEvictWarps / 32;
            int v[PER], sum = 0;
#pragma unroll
            for (int k = 0; k < PER; ++k) { v[k] = cnt[lane * PER + k]; sum += v[k]; }
            int before = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += y; }
            if (lane == 31) cnt[kKeep * kEvictWarps] = before;
            before -= sum;
#pragma unroll
            for (int k = 0; k < PER; ++k) { cnt[lane * PER + k] = before; before += v[k]; }
        }
        __syncthreads();
    };
    const uint32_t below = (1u << lane) - 1u;
    for (int base = 0; base < n; base += kKeep * kEvictThreads) {
        if (base > 0) {
#pragma unroll
            for (int i = 0; i < kKeep; ++i) {
                const int row = base + i * kEvictThreads + tid;
                at[i] = row < n ? place(row) : -1;
                key[i] = row < n ? key_of(row) : 0u;
            }
            __syncthreads();                                     // the last round's counts have been read
        }
        uint32_t kept = 0;                                       // bit per row of the thread
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const bool in = base + i * kEvictThreads + tid < n;
            const uint32_t m = __ballot_sync(0xffffffffu, in && key[i] == border);
            if (lane == 0) counts[0][i * kEvictWarps + warp] = __popc(m);
            if (in && key[i] > border) kept |= 1u << i;
        }
        number(counts[0]);
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const int row = base + i * kEvictThreads + tid;
            const bool in = row < n, tie = in && key[i] == border;
            const uint32_t m = __ballot_sync(0xffffffffu, tie);
            if (tie && ties + counts[0][i * kEvictWarps + warp] + __popc(m & below) < want) kept |= 1u << i;
            const bool k = kept >> i & 1u;
            const uint32_t mh = __ballot_sync(0xffffffffu, in && !k && row < p.budget), me = __ballot_sync(0xffffffffu, in && k && row >= p.budget);
            if (lane == 0) counts[1][i * kEvictWarps + warp] = __popc(mh) | __popc(me) << 16;
        }
        ties += counts[0][kKeep * kEvictWarps];
        number(counts[1]);
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const int row = base + i * kEvictThreads + tid;
            const bool in = row < n, k = kept >> i & 1u, hole = in && !k && row < p.budget, ext = in && k && row >= p.budget;
            const uint32_t mh = __ballot_sync(0xffffffffu, hole), me = __ballot_sync(0xffffffffu, ext);
            const int off = counts[1][i * kEvictWarps + warp];
            if (hole) moves[holes + (off & 0xffff) + __popc(mh & below)].y = at[i];
            if (ext) moves[extra + (off >> 16) + __popc(me & below)].x = at[i];
        }
        holes += counts[1][kKeep * kEvictWarps] & 0xffff;
        extra += counts[1][kKeep * kEvictWarps] >> 16;
    }
    if (!p.inline_moves) {
        if (tid == 0) p.n_moves[b * c.kv_heads + h] = holes;     // as many as extra
        return;
    }
    __syncthreads();
    if (p.head_dim == 64) move_rows<64, 4>(c, p, h, moves, tid / 16, kEvictThreads / 16, holes, tid & 15);
    else move_rows<128, 4>(c, p, h, moves, tid / 16, kEvictThreads / 16, holes, tid & 15);
}

// grid (parts of the list, kv heads, batch)
template <int D>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const Cache c, const EvictParams p) {
    const int h = blockIdx.y, b = blockIdx.z;
    pdl_wait();
    pdl_launch_dependents();
    const int2* moves = p.moves + (size_t)(b * c.kv_heads + h) * p.most_moves;
    move_rows<D, 4>(c, p, h, moves, blockIdx.x * (kMoveThreads / 16) + threadIdx.x / 16, gridDim.x * (kMoveThreads / 16), p.n_moves[b * c.kv_heads + h], threadIdx.x & 15);
}

}  // namespace kv4
}  // namespace efm
