// Attention over a 4-bit cache (kv4_cache.cuh): new rows of a ragged batch against the pages of their sequences.
//
// The codes go to the tensor cores as they are: a key is min + scale * code = c + scale * (code - 8) with c = min + 8 scale, so that
//     q . k = sum over groups g of  scale_g (q_g . (code - 8)_g + 8 (sum of q_g)) + min_g (sum of q_g),
// and code - 8 is exact in fp16.  q is scaled by a power of two per row and is exact there too, but for channels 2^17 (bf16 2^20) below the
// row's largest, which lose bits below fp16's normal range: scores carry fp32 rounding only.  Values: o = sum over tokens of
// (p scale_g) (code - 8) + sum of p c_g, with p scale_g rounded to fp16 below a power of two that keeps the largest scale seen at 2^14 .. 2^15,
// so that neither large nor small scales leave its range.  That is 2^-11 of a weight, well below the half step of a bf16 output (2^-8); for
// fp16 outputs, whose half step it is, p scale_g is a pair high + low (2^-22).
#pragma once
#include "gemm_tc.cuh"
#include "kv4_cache.cuh"

namespace efm {
namespace kv4 {

struct AttnParams {
    int max_rows, max_new, max_len;
    const int32_t *cu_rows, *lens;
    const void* q;
    void* out;
    float scale_log2;         // scale * log2(e): scores in units of log2
    const float* mass_in;
    float* mass_out;
    int few_rows;             // sequences with at most this many packed rows (new rows x heads of a group) are attend_few's
    int warps, unit_shift;    // attend_few's warps; pages of a unit of work: 1 << unit_shift
    uint32_t group_inv;       // ceil(2^32 / heads of a group), 0 for one: what packed rows are divided by
    float2* stats;            // [rows, q_heads] (maximum, sum) of a row's weights, where one warp had all its keys; null: not wanted
    int rows, row_tiles;      // rows and tiles of 128 packed rows that a sequence has in stats and images; rows 0: they follow each other as
                              // in the call's buffers, and a sequence's first tile is row0 x group / 128 + b (one has at most n x group / 128 + 1)
    float2* part_stats;       // [8 nt][2 warps] the same of the keys a warp had, and
    float* part;              // [2 warps][8 nt][D] its weighted values: slot 0 is the piece its range begins with, slot 1 the one it ends with
    int32_t* starts;          // [batch + 1] units ahead of every sequence, and all of them
    int32_t* lost;            // [n_lost] of attend_few's blocks, then of attend_many's: 1 where a wait gave up.  Weights are not summed then
    int few_blocks, n_lost;
    uint8_t* images;          // [tiles, kv_heads][128 x D fp16] packed rows as operands, and
    float* units;             // [tiles, kv_heads][128] what their scores are multiplied with; where many rows are a sequence's
    int many_tiles, many_blocks;      // blocks of 256 packed rows a sequence may have; blocks of attend_many
    int32_t* many_starts;     // [batch x many_tiles + 2] its units ahead, all of them, and those of each if blocks of rows stay whole
    float2* many_stats;       // [2 many_blocks][256] and
    float* many_part;         // [2 many_blocks][D / 4][256][4] what part_stats and part are, of its pieces
    float* scores;            // [pages, kv_heads][64][8 nt] scores in units of log2; null: not wanted
    int score_pages;          // pages a sequence has there; 0: they are the pool's
};

// New rows and cache rows of sequence b, cut to what the call was given.
struct Entry { int row0, n, len; };
__device__ __forceinline__ Entry entry_of(const Cache& c, const AttnParams& p, int b) {
    Entry e;
    const int lo = p.cu_rows[b], hi = p.cu_rows[b + 1];
    e.row0 = min(max(lo, 0), p.max_rows);
    e.n = min(max(hi, e.row0), p.max_rows) - e.row0;
    if (lo < 0 || hi < lo || hi > p.max_rows || e.n > p.max_new) raise(c, kBadCount);
    e.n = min(e.n, p.max_new);
    e.len = held(c, p.lens, b, min(p.max_len, c.max_pages * kRows));
    return e;
}
__device__ __forceinline__ size_t stat_row(const Cache& c, const AttnParams& p, const Entry& e, int b, int i, int head) {
    return ((p.rows > 0 ? (size_t)b * p.rows : (size_t)e.row0) + i) * c.q_heads + head;
}

constexpr int kWarps = 4;

// Wait of a whole warp for a phase, bounded; false when it gave up.  The limit (some seconds) is a constant: read from the parameters it
// cost attend_many 5 % and attend_few 3, since warps that poll take issue slots from the others.  kHasty: for tests of what follows.
constexpr int kPolls = 1 << 25, kHasty = 2;
template <int POLLS>
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    for (int i = 0; i < POLLS; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (__all_sync(0xffffffffu, ok)) return true;
        if ((i & 0xff) == 0xff && __any_sync(0xffffffffu, *abort_flag != 0)) return false;      // another role already gave up
    }
    return false;
}
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// How attend_few's work is dealt: the pages of every (sequence, kv head, tile of R packed rows) in units of p.unit, in that order; warp w
// has the units [w step, (w + 1) step).  Lengths are known on the device only, so every block adds them up for itself.
struct Deal { int before, all; };          // units ahead of sequence b, and altogether
struct Share { int units, tiles, each; };      // of a sequence; row tiles; units of a tile and head
template <int R>
__device__ __forceinline__ Share share_of(const Cache& c, const AttnParams& p, const Entry& e, int group) {
    const int rows = e.n * group;
    Share s;
    s.each = max(1, ((e.len + kRows - 1) / kRows + (1 << p.unit_shift) - 1) >> p.unit_shift);      // a row that sees nothing is somebody's to clear
    s.tiles = rows <= p.few_rows ? (rows + R - 1) / R : 0;
    s.units = s.tiles * s.each * c.kv_heads;
    return s;
}
__device__ __forceinline__ int step_of(const AttnParams& p, int all) { return max(1, (all + p.warps - 1) / p.warps); }

// ---- fragments -------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// d = a b + (c0, c1, c0, c1)
__device__ __forceinline__ void mma16816_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Nibbles at bits 0 and 16 (4 and 20) of w as a pair of fp16 code - 8: 1024 + n (1024 + 16 n) by setting the exponent, then exact arithmetic.
__device__ __forceinline__ uint32_t low_pair(uint32_t w) {
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(0x000f000fu), "r"(0x64006400u));     // (w & mask) | 1024 in one instruction
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(v) : "r"(0x64086408u));                       // 1032
    return v;
}
__device__ __forceinline__ uint32_t high_pair(uint32_t w) {
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(0x00f000f0u), "r"(0x64006400u));
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(v) : "r"(0x2c002c00u), "r"(0xd480d480u));   // / 16, - 72
    return v;
}
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
    uint32_t v;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(b), "f"(a));
    return v;
}

// Eight query rows in the B operand's layout: lane (n, j) has row n's channels g * 64 + 16 j .. + 15.
template <int D>
struct QueryTile {
    static constexpr int G = D / kGroup;
    uint32_t f[G][4][2];
    float sum[G][2], eight[G][2], unit[2];      // of the lane's two columns 2 j, 2 j + 1: sums of the scaled q, 8 times those, what a score is multiplied with

    struct Raw { uint4 w[G][2]; };
    template <typename T>
    static __device__ __forceinline__ Raw fetch(const T* row, bool have) {                  // row: of column lane / 4
        Raw r;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h) r.w[g][h] = have ? *reinterpret_cast<const uint4*>(row + g * 64 + (threadIdx.x & 3) * 16 + h * 8) : make_uint4(0u, 0u, 0u, 0u);
        return r;
    }
    template <typename T>
    __device__ __forceinline__ void take(const Raw& raw, float scale_log2) {
        const int j = threadIdx.x & 3;
        float x[G][16], top = 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t v[4] = {raw.w[g][h].x, raw.w[g][h].y, raw.w[g][h].z, raw.w[g][h].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 t = Num<T>::two(v[i]);
                    x[g][h * 8 + 2 * i] = t.x;
                    x[g][h * 8 + 2 * i + 1] = t.y;
                    top = fmaxf(top, fmaxf(fabsf(t.x), fabsf(t.y)));
                }
            }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // exponent of the largest magnitude; infinities keep the factor 1, rows below 2^-100 count as that large
        const int bits = (int)(__float_as_uint(top) >> 23), e = bits == 255 ? 3 : max(bits - 127, -100);
        const float up = __uint_as_float((uint32_t)(130 - e) << 23), down = __uint_as_float((uint32_t)(max(e, -100) + 124) << 23);
        float s[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            s[g] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t v = half_pair(x[g][4 * i + 2 * k] * up, x[g][4 * i + 2 * k + 1] * up);
                    f[g][i][k] = v;
                    const float2 t = Num<__half>::two(v);
                    s[g] += t.x + t.y;
                }
            s[g] += __shfl_xor_sync(0xffffffffu, s[g], 1);
            s[g] += __shfl_xor_sync(0xffffffffu, s[g], 2);
#pragma unroll
            for (int k = 0; k < 2; ++k) { sum[g][k] = __shfl_sync(0xffffffffu, s[g], (2 * j + k) * 4); eight[g][k] = 8.0f * sum[g][k]; }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) unit[k] = __shfl_sync(0xffffffffu, fmaxf(down * scale_log2, 1.2e-38f), (2 * j + k) * 4);     // times -inf: -inf
    }
};

// Token of a 16-token tile that the operand layouts' row (or column) l stands for; chosen so that four neighbouring lanes read rows
// next to each other.
__device__ __forceinline__ int token_of(int l) { return (l & 8) + ((l & 7) >> 1) + 4 * (l & 1); }

// Parameters of a row and group: scale and centre of the codes.
__device__ __forceinline__ float2 centred(uint32_t par) {
    const float2 t = Num<__half>::two(par);
    return make_float2(t.x, fmaf(8.0f, t.x, t.y));
}
// Rows of a page in shared memory that are not held: parameters of nothing, whatever bits were there (the whole warp calls).
template <int D>
__device__ __forceinline__ void clear_rows(uint8_t* page, int valid, bool values) {
    using L = Tile<D>;
    __syncwarp();
    for (int i = valid * L::G + (threadIdx.x & 31); i < kRows * L::G; i += 32) {
        reinterpret_cast<uint32_t*>(page + L::K_PARAMS)[i] = 0u;
        if (values) reinterpret_cast<uint32_t*>(page + L::V_PARAMS)[i] = 0u;
    }
    __syncwarp();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");                  // ahead of the next copy into this place
}

// Scores, unscaled, of the 16 tokens of tile u of a page against NT query tiles: s[t][0..1] of token token_of(lane / 4) and the lane's
// two columns, s[t][2..3] of the token 8 behind.
template <int D, int NT>
__device__ __forceinline__ void score_tile(const uint8_t* page, int u, const QueryTile<D> (&q)[NT], float (&s)[NT][4]) {
    using L = Tile<D>;
    constexpr int G = L::G;
    const int lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
    const int ta = u * 16 + token_of(r), tb = ta + 8;
    uint32_t ka[G][2], kb[G][2], pa[G], pb[G];
    if constexpr (G == 2) {
        const uint4 a = *reinterpret_cast<const uint4*>(page + L::K_CODES + ta * (D / 2) + j * 16), b = *reinterpret_cast<const uint4*>(page + L::K_CODES + tb * (D / 2) + j * 16);
        ka[0][0] = a.x; ka[0][1] = a.y; ka[1][0] = a.z; ka[1][1] = a.w;
        kb[0][0] = b.x; kb[0][1] = b.y; kb[1][0] = b.z; kb[1][1] = b.w;
        const uint2 x = *reinterpret_cast<const uint2*>(page + L::K_PARAMS + ta * 8), y = *reinterpret_cast<const uint2*>(page + L::K_PARAMS + tb * 8);
        pa[0] = x.x; pa[1] = x.y; pb[0] = y.x; pb[1] = y.y;
    } else {
        const uint2 a = *reinterpret_cast<const uint2*>(page + L::K_CODES + ta * (D / 2) + j * 8), b = *reinterpret_cast<const uint2*>(page + L::K_CODES + tb * (D / 2) + j * 8);
        ka[0][0] = a.x; ka[0][1] = a.y;
        kb[0][0] = b.x; kb[0][1] = b.y;
        pa[0] = *reinterpret_cast<const uint32_t*>(page + L::K_PARAMS + ta * 4);
        pb[0] = *reinterpret_cast<const uint32_t*>(page + L::K_PARAMS + tb * 4);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        float acc[NT][4];                                        // begin with 8 (sum of q): products with the codes themselves
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint32_t a0[4] = {low_pair(ka[g][w]), low_pair(kb[g][w]), high_pair(ka[g][w]), high_pair(kb[g][w])};
            const uint32_t a1[4] = {low_pair(ka[g][w] >> 8), low_pair(kb[g][w] >> 8), high_pair(ka[g][w] >> 8), high_pair(kb[g][w] >> 8)};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (w == 0) mma16816_from(acc[t], a0, q[t].f[g][0][0], q[t].f[g][0][1], q[t].eight[g][0], q[t].eight[g][1]);
                else mma16816(acc[t], a0, q[t].f[g][2][0], q[t].f[g][2][1]);
                mma16816(acc[t], a1, q[t].f[g][2 * w + 1][0], q[t].f[g][2 * w + 1][1]);
            }
        }
        const float2 a = Num<__half>::two(pa[g]), b = Num<__half>::two(pb[g]);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                s[t][k] = fmaf(a.x, acc[t][k], g == 0 ? a.y * q[t].sum[g][k] : fmaf(a.y, q[t].sum[g][k], s[t][k]));
                s[t][2 + k] = fmaf(b.x, acc[t][2 + k], g == 0 ? b.y * q[t].sum[g][k] : fmaf(b.y, q[t].sum[g][k], s[t][2 + k]));
            }
    }
}

template <int D, int NT>
struct FewCfg {
    static constexpr int STAGES = D == 128 ? 2 : 4;
    static constexpr int BLOCKS = NT == 1 ? 3 : 2;                               // per SM
    static constexpr size_t RING = (size_t)kWarps * STAGES * Tile<D>::BYTES;
    static constexpr size_t SMEM = RING + kWarps * STAGES * 8 + 16;
};

// Few query rows.  A warp works for itself on the pages of its units, each page (one kv head's tile) one bulk copy into a ring of its own;
// where a row's keys are dealt over several warps it leaves its sums, and attend_merge joins them.  Blocks whose warps shared a row and
// joined it in shared memory spent a third of their time on barriers and waiting for queries behind their own copies.
// The MMA's 16 rows are tokens (channels in P V) and its 8 columns query rows -- the heads of a group, times the new rows -- so that a
// single token of up to 8 heads per kv head fills it: m16n8k16 the other way round would leave half of it empty.
// Bound: instruction issue, 1280 a page of 64 x 128 (a third of them on the integer pipe, which takes the codes apart, half floating point),
// of which three blocks an SM, as many as registers allow, reach 57 % of the slots; then bytes.  One token, 28 heads on 4 kv heads of 128, on
// 131000 rows: 28 us, 2.8 TB/s; on 64 caches of 300 .. 4000: 30 us, 2.7 TB/s.
template <typename T, int D, int NT, int POLLS = kPolls>
__global__ void __launch_bounds__(kWarps * 32, FewCfg<D, NT>::BLOCKS) attend_few_kernel(const Cache c, const AttnParams p) {
    using L = Tile<D>;
    using C = FewCfg<D, NT>;
    constexpr int G = L::G, R = 8 * NT;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int sums[kWarps], before_s[kWarps], first_s[kWarps];
    __shared__ Entry entry_s[kWarps];
    __shared__ volatile int stage_page_s[kWarps][C::STAGES];                     // the page in a stage, -1: none of the pool's
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::RING);
    volatile int* abort_s = reinterpret_cast<volatile int*>(bars + kWarps * C::STAGES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3, group = c.q_heads / c.kv_heads;
    unsigned char* ring = smem + (size_t)warp * C::STAGES * L::BYTES;
    const uint32_t bar0 = tc::smem_u32(bars + warp * C::STAGES);
    if (lane == 0) {
        for (int i = 0; i < C::STAGES; ++i) tc::mbar_init(bar0 + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 0) *abort_s = 0;
    pdl_wait();
    pdl_launch_dependents();
    // the warps' ranges of the units, and the sequences they begin in
    const int me = blockIdx.x * kWarps + warp;
    if (threadIdx.x == 0) p.lost[blockIdx.x] = 0;
    int all = 0, b = 0, start = 0;                                               // b: sequence, start: unit that it begins with
    Entry e0;
    if (c.batch == 1) {
        e0 = entry_of(c, p, 0);
        all = share_of<R>(c, p, e0, group).units;
        if (blockIdx.x == 0 && threadIdx.x == 0) { p.starts[0] = 0; p.starts[1] = all; }      // for attend_merge
        __syncthreads();                                                         // barriers and the abort word are set up
    } else {
        const int per = (c.batch + kWarps * 32 - 1) / (kWarps * 32), b_lo = min(c.batch, (int)threadIdx.x * per), b_hi = min(c.batch, b_lo + per);
        int own = 0;
        for (int i = b_lo; i < b_hi; ++i) own += share_of<R>(c, p, e0 = entry_of(c, p, i), group).units;
        int upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) { if (w < warp) upto += sums[w]; all += sums[w]; }
        const int step = step_of(p, all);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const int u = (int)min((int64_t)all, ((int64_t)blockIdx.x * kWarps + w) * step);
            if (upto - own <= u && u < upto) {
                int at = upto - own, i = b_lo;
                if (per > 1)
                    for (int n; at + (n = share_of<R>(c, p, e0 = entry_of(c, p, i), group).units) <= u; ++i) at += n;
                first_s[w] = i;
                before_s[w] = at;
                entry_s[w] = e0;
            }
        }
        if (blockIdx.x == 0) {
            if (threadIdx.x == 0) p.starts[c.batch] = all;
            int at = upto - own;
            for (int i = b_lo; i < b_hi; ++i) { p.starts[i] = at; at += share_of<R>(c, p, entry_of(c, p, i), group).units; }
        }
        __syncthreads();
        b = first_s[warp];
        start = before_s[warp];
        e0 = entry_s[warp];
    }
    const int step = step_of(p, all), u1 = (int)min((int64_t)all, ((int64_t)me + 1) * step);
    int u = (int)min((int64_t)all, (int64_t)me * step), slot = 0;                // slot: of the copies and their barriers
    if (u >= u1) return;
    auto by_group = [&](int row) { return p.group_inv != 0u ? (int)__umulhi((uint32_t)row, p.group_inv) : row; };      // row / group, exact below 2^22

    // one piece after the other: pages of a (sequence, kv head, tile of rows)
    struct Piece { Entry e; int b, h, tile, p0, mine; bool from_start, to_end; };
    auto next_piece = [&]() {
        Share sh = share_of<R>(c, p, e0, group);
        while (u >= start + sh.units) { start += sh.units; sh = share_of<R>(c, p, e0 = entry_of(c, p, ++b), group); }
        Piece x;
        x.b = b;
        x.e = e0;
        const int in = u - start, i = in / sh.each, first = in - i * sh.each, last = min(sh.each, first + (u1 - u));
        x.h = sh.tiles == 1 ? i : i / sh.tiles;
        x.tile = i - x.h * sh.tiles;
        x.p0 = first << p.unit_shift;
        x.mine = max(0, min(last << p.unit_shift, (x.e.len + kRows - 1) / kRows) - x.p0);
        x.from_start = first == 0;
        x.to_end = last == sh.each;
        u += last - first;
        return x;
    };
    auto value_params = [&](const uint8_t* page, int t, uint32_t (&w)[G]) {      // read for the largest scale and again for the values: kept they take 16 registers
        const uint32_t at = tc::smem_u32(page) + (uint32_t)(L::V_PARAMS + t * G * 4);
        if constexpr (G == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[G - 1]) : "r"(at));
        else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at));
    };
    auto row_at = [&](const Piece& x, int row) { return ((size_t)(x.e.row0 + by_group(row)) * c.q_heads + x.h * group + row - by_group(row) * group) * D; };
    int lane_page = -1;
    auto request = [&](const Piece& x, int i) {
        if ((i & 31) == 0) {                                                     // a lane knows one page of 32
            const bool in = i + lane < x.mine;
            lane_page = in ? c.page_table[(size_t)x.b * c.max_pages + x.p0 + i + lane] : -1;
            if ((unsigned)lane_page >= (unsigned)c.n_pages) { if (in) raise(c, kBadPage); lane_page = -1; }
        }
        const int page = __shfl_sync(0xffffffffu, lane_page, i & 31), st = (slot + i) % C::STAGES;
        if (lane == 0) {
            stage_page_s[warp][st] = page;
            if (page >= 0) {
                tc::mbar_expect_tx(bar0 + 8 * st, L::BYTES);
                bulk_copy(tc::smem_u32(ring) + st * L::BYTES, tile_of<D>(c, page, x.h), L::BYTES, bar0 + 8 * st);
            } else {
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar0 + 8 * st) : "memory");
            }
        }
    };
    typename QueryTile<D>::Raw raw[NT];
    auto ask = [&](const Piece& x) {                                             // queries ahead of the pages, which they would queue behind
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int row = x.tile * R + t * 8 + r;
            const bool have = row < x.e.n * group;
            raw[t] = QueryTile<D>::fetch((const T*)p.q + (have ? row_at(x, row) : 0), have);
        }
        for (int i = 0; i < min(x.mine, C::STAGES); ++i) request(x, i);
        __syncwarp();
    };
    Piece x = next_piece();
    ask(x);
    for (bool more = true; more;) {
        QueryTile<D> q[NT];
        int see[NT][2], least = INT32_MAX;                                       // cached rows that the lane's columns see
        const int rows = x.e.n * group;                                          // packed: new row x head of the group
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            q[t].template take<T>(raw[t], p.scale_log2);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int cr = x.tile * R + t * 8 + 2 * j + k;
                see[t][k] = cr < rows ? max(0, min(x.e.len, x.e.len - x.e.n + by_group(cr) + 1)) : 0;
                if (cr < rows) least = min(least, see[t][k]);
            }
        }
        least = min(least, __shfl_xor_sync(0xffffffffu, least, 1));
        least = min(least, __shfl_xor_sync(0xffffffffu, least, 2));
        float o[G][4][NT][4], pc[G][NT][2], m[NT][2], l[NT][2];                  // m: maximum, in units of log2
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                m[t][k] = -INFINITY;
                l[t][k] = 0.f;
#pragma unroll
                for (int g = 0; g < G; ++g) pc[g][t][k] = 0.f;
            }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[g][y][t][k] = 0.f;
        int ev = -40;                                                            // exponent of the largest value scale seen

        for (int i = 0; i < x.mine; ++i) {
            const int st = (slot + i) % C::STAGES, first = (x.p0 + i) * kRows;
            if (!warp_wait<POLLS>(bar0 + 8 * st, (uint32_t)((slot + i) / C::STAGES) & 1u, abort_s)) {      // given up: the warp's copies in flight land first (bounded)
                *abort_s = 1;
                if (lane == 0) {
                    volatile int go_on = 0;
                    for (int k = slot + i; k < slot + min(x.mine, i + C::STAGES); ++k) (void)tc::mbar_wait(bar0 + 8 * (k % C::STAGES), (uint32_t)(k / C::STAGES) & 1u, &go_on);
                    raise(c, kWait);
                    p.lost[blockIdx.x] = 1;
                }
                return;
            }
            if (stage_page_s[warp][st] >= 0) {
                uint8_t* page = ring + (size_t)st * L::BYTES;
                if (x.e.len - first < kRows) clear_rows<D>(page, x.e.len - first, true);
                float s[4][NT][4];
#pragma unroll
                for (int u = 0; u < 4; ++u) score_tile<D, NT>(page, u, q, s[u]);
                if (first + kRows > least) {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (first + u * 16 + token_of(r) + 8 * (k >> 1) >= see[t][k & 1]) s[u][t][k] = -INFINITY;
                }
                if (p.scores != nullptr) {
                    const uint32_t at = (uint32_t)(p.score_pages > 0 ? x.b * p.score_pages + x.p0 + i : stage_page_s[warp][st]) * c.kv_heads + x.h;      // no more than the pool's tiles
                    float* to = p.scores + (size_t)at * (R * kRows) + token_of(r) * R + 2 * j;
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                            for (int t = 0; t < NT; ++t)
                                *reinterpret_cast<float2*>(to + (u * 16 + 8 * hf) * R + t * 8) = make_float2(s[u][t][2 * hf] * q[t].unit[0], s[u][t][2 * hf + 1] * q[t].unit[1]);
                }
                float top[NT][2];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        top[t][k] = fmaxf(s[0][t][k], s[0][t][2 + k]);
#pragma unroll
                        for (int u = 1; u < 4; ++u) top[t][k] = fmaxf(top[t][k], fmaxf(s[u][t][k], s[u][t][2 + k]));
                    }
                // parameters of the values; the largest scale is the low half of the largest pair
                uint32_t big2 = 0;
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        uint32_t vp[G];
                        value_params(page, u * 16 + token_of(r) + 8 * hf, vp);
#pragma unroll
                        for (int g = 0; g < G; ++g) asm("max.f16x2 %0, %0, %1;" : "+r"(big2) : "r"(vp[g]));
                    }
                int big = (int)(big2 & 0x7fffu);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    big = max(big, __shfl_xor_sync(0xffffffffu, big, off));
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int k = 0; k < 2; ++k) top[t][k] = fmaxf(top[t][k], __shfl_xor_sync(0xffffffffu, top[t][k], off));
                }
                const int en = max(ev, big > 0 ? max(big >> 10, 1) - 15 : -40);
                float base[NT][2];
                bool same = ev == en;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        base[t][k] = fmaxf(m[t][k], top[t][k] * q[t].unit[k]);
                        same = same && base[t][k] == m[t][k];
                    }
                if (!__all_sync(0xffffffffu, same)) {
                    const float fold = __uint_as_float((uint32_t)(127 + ev - en) << 23);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float alpha = m[t][k] == -INFINITY ? 0.f : ex2f(m[t][k] - base[t][k]), f = alpha * fold;
                            m[t][k] = base[t][k];
                            l[t][k] *= alpha;
#pragma unroll
                            for (int g = 0; g < G; ++g) {
                                pc[g][t][k] *= alpha;
#pragma unroll
                                for (int y = 0; y < 4; ++y) { o[g][y][t][k] *= f; o[g][y][t][2 + k] *= f; }
                            }
                        }
                    ev = en;
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (base[t][k] == -INFINITY) base[t][k] = 0.f;
                const float unit = __uint_as_float((uint32_t)(127 + 14 - ev) << 23);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    constexpr int PARTS = std::is_same<T, __half>::value ? 2 : 1;
                    uint32_t b0[PARTS][G][NT], b1[PARTS][G][NT], va[G], vb[G];
                    value_params(page, u * 16 + token_of(r), va);
                    value_params(page, u * 16 + token_of(r) + 8, vb);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            s[u][t][k] = ex2f(fmaf(s[u][t][k], q[t].unit[k & 1], -base[t][k & 1]));
                            l[t][k & 1] += s[u][t][k];
                        }
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float2 a = centred(va[g]), bb = centred(vb[g]);
                        const float sa = a.x * unit, sb = bb.x * unit;
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const float(&w)[4] = s[u][t];
                            pc[g][t][0] = fmaf(w[0], a.y, fmaf(w[2], bb.y, pc[g][t][0]));
                            pc[g][t][1] = fmaf(w[1], a.y, fmaf(w[3], bb.y, pc[g][t][1]));
                            float x[4] = {w[0] * sa, w[1] * sa, w[2] * sb, w[3] * sb};
#pragma unroll
                            for (int y = 0; y < PARTS; ++y) {
                                const uint32_t h0 = half_pair(x[0], x[1]), h1 = half_pair(x[2], x[3]);
                                b0[y][g][t] = transposed(h0);
                                b1[y][g][t] = transposed(h1);
                                const float2 f0 = Num<__half>::two(h0), f1 = Num<__half>::two(h1);
                                x[0] -= f0.x; x[1] -= f0.y; x[2] -= f1.x; x[3] -= f1.y;
                            }
                        }
                    }
                    // columns 2 j, 2 j + 1 (and 8 behind) of the operand are the tokens j, j + 4 (j + 8, j + 12)
                    const uint32_t* codes = reinterpret_cast<const uint32_t*>(page + L::V_CODES) + (u * 16 + j) * L::WORDS + r;
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const uint32_t w0 = codes[g * 8], w1 = codes[4 * L::WORDS + g * 8], w2 = codes[8 * L::WORDS + g * 8], w3 = codes[12 * L::WORDS + g * 8];
#pragma unroll
                        for (int hl = 0; hl < 2; ++hl) {
                            const uint32_t ta = __byte_perm(w0, w1, hl ? 0x7632 : 0x5410), tb = __byte_perm(w2, w3, hl ? 0x7632 : 0x5410);
                            const uint32_t a0[4] = {low_pair(ta), high_pair(ta), low_pair(tb), high_pair(tb)};
                            const uint32_t a1[4] = {low_pair(ta >> 8), high_pair(ta >> 8), low_pair(tb >> 8), high_pair(tb >> 8)};
#pragma unroll
                            for (int t = 0; t < NT; ++t)
#pragma unroll
                                for (int y = 0; y < PARTS; ++y) {
                                    mma16816(o[g][2 * hl][t], a0, b0[y][g][t], b1[y][g][t]);
                                    mma16816(o[g][2 * hl + 1][t], a1, b0[y][g][t], b1[y][g][t]);
                                }
                        }
                    }
                }
            }
            __syncwarp();                                                        // every lane has read the page
            if (i + C::STAGES < x.mine) request(x, i + C::STAGES);
        }
        slot += x.mine;
        const Piece done = x;
        more = u < u1;
        if (more) {                                                              // the next piece is on its way while this one is written
            x = next_piece();
            ask(x);
        }

#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    l[t][k] += __shfl_xor_sync(0xffffffffu, l[t][k], off);
#pragma unroll
                    for (int g = 0; g < G; ++g) pc[g][t][k] += __shfl_xor_sync(0xffffffffu, pc[g][t][k], off);
                }
        const float back = __uint_as_float((uint32_t)(127 + ev - 14) << 23);
        const bool alone = done.from_start && done.to_end;
        const int piece = 2 * me + (done.from_start ? 1 : 0);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int rr = t * 8 + 2 * j + k, row = done.tile * R + rr;
                if (row >= rows) continue;
                const float inv = alone ? (l[t][k] > 0.f ? 1.0f / l[t][k] : l[t][k] != l[t][k] ? l[t][k] : 0.f) : 1.0f;
                const size_t at = row_at(done, row);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    float v[8];                                                  // channels of word r of the group, see the nibbles' order
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int ch = (y & 1) * 4 + (y >> 1);
                        v[ch] = fmaf(o[g][y][t][k], back, pc[g][t][k]) * inv;
                        v[ch + 2] = fmaf(o[g][y][t][2 + k], back, pc[g][t][k]) * inv;
                    }
                    if (alone) {
                        *reinterpret_cast<uint4*>((T*)p.out + at + g * 64 + 8 * r) = make_uint4(within2<T>(v[0], v[1]), within2<T>(v[2], v[3]), within2<T>(v[4], v[5]), within2<T>(v[6], v[7]));
                    } else {
                        float4* dst = reinterpret_cast<float4*>(p.part + ((size_t)piece * R + rr) * D + g * 64 + 8 * r);
                        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                    }
                }
                if (r == 0) {
                    if (!alone) p.part_stats[(size_t)rr * 2 * p.warps + piece] = make_float2(m[t][k], l[t][k]);
                    else if (p.stats != nullptr) p.stats[stat_row(c, p, done.e, done.b, by_group(row), done.h * group + row - by_group(row) * group)] = make_float2(m[t][k], l[t][k]);
                }
            }
    }
}

// Where the keys of a tile of packed rows were dealt: to one warp, which finished the rows itself, or to warps [w0, w1].
struct Pieces { int w0, w1; };
__device__ __forceinline__ Pieces pieces_of(const AttnParams& p, const Share& s, const Deal& d, int h, int tile) {
    const int step = step_of(p, d.all), at = d.before + (h * s.tiles + tile) * s.each;
    return Pieces{at / step, (at + s.each - 1) / step};
}
__device__ __forceinline__ int piece_of(int w, const Pieces& x) { return 2 * w + (w == x.w0 ? 1 : 0); }

// Maximum and sum of packed row rr of a tile over its pieces, by a warp.
__device__ __forceinline__ float2 merged_stats(const AttnParams& p, const Pieces& x, int rr) {
    const int lane = threadIdx.x & 31;
    float top = -INFINITY, sum = 0.f;
    for (int base = x.w0; base <= x.w1; base += 256) {           // 256 pieces on their way at a time
        float2 s[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int w = base + k * 32 + lane;
            s[k] = w <= x.w1 ? p.part_stats[(size_t)rr * 2 * p.warps + piece_of(w, x)] : make_float2(-INFINITY, 0.f);
        }
        float mx = top;
#pragma unroll
        for (int k = 0; k < 8; ++k) mx = fmaxf(mx, s[k].x);
        if (mx == -INFINITY) continue;
        sum = top == -INFINITY ? 0.f : sum * ex2f(top - mx);
#pragma unroll
        for (int k = 0; k < 8; ++k) if (s[k].x != -INFINITY) sum = fmaf(s[k].y, ex2f(s[k].x - mx), sum);
        top = mx;
    }
    const float all = warp_max(top);
    return make_float2(all, warp_sum(top == -INFINITY ? 0.f : sum * ex2f(top - all)));
}

constexpr int kFactors = 512;         // pieces whose factors are at hand at a time
constexpr int kMassTokens = 512;      // cached rows of a block that sums weights from scores

// What needs the whole row.  grid (mass blocks + merging blocks, kv heads, batch): merging blocks join the pieces of rows that attend_few
// dealt over several warps, 32 channels of a row at a time; mass blocks sum the weights of 512 cached rows from the scores it left.
// Bound: the pieces' and scores' way through L2 and, with few rows, latency.  The caches above: 8 us without weights, 14 with.  Lengths are read
// behind the wait: what an earlier launch wrote is promised to a kernel by its own wait only, not by its predecessor's.  Read ahead of it they
// saved 0.5 us of one token on 1450 rows with weights (13.4), 0.8 of 41 on 131000, 2.6 of 36 on 64 caches without weights.
template <typename T, int D, int R>
__global__ void __launch_bounds__(kWarps * 32) attend_merge_kernel(const Cache c, const AttnParams p, int mass_blocks) {
    __shared__ float2 st_s[R];
    __shared__ float4 v_s[kWarps * 32];
    __shared__ float f_s[kFactors];
    const int h = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = c.q_heads / c.kv_heads;
    pdl_wait();
    pdl_launch_dependents();
    const Deal deal{p.starts[b], p.starts[c.batch]};             // on its way with the lengths; of no use where nothing was dealt
    const Entry e = entry_of(c, p, b);
    const Share sh = share_of<R>(c, p, e, group);
    const int rows = sh.tiles > 0 ? e.n * group : 0;
    if ((int)blockIdx.x < mass_blocks) {
        const int t0 = blockIdx.x * kMassTokens;
        if (t0 >= e.len) return;
        constexpr int PER = kMassTokens / (kWarps * 32);
        int page[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) { const int tk = t0 + threadIdx.x + k * kWarps * 32; page[k] = tk < e.len ? page_of(c, b, tk / kRows) : -1; }
        const Pieces x = rows > 0 ? pieces_of(p, sh, deal, h, 0) : Pieces{0, 0};
        bool lost = false;
        for (int i = x.w0 / kWarps + (int)threadIdx.x; rows > 0 && i <= x.w1 / kWarps; i += kWarps * 32) lost = lost || p.lost[i] != 0;
        for (int row = warp; row < rows; row += kWarps) {
            const float2 s = x.w0 == x.w1 ? p.stats[stat_row(c, p, e, b, row / group, h * group + row % group)] : merged_stats(p, x, row);
            if (lane == 0) st_s[row] = s.x == -INFINITY ? make_float2(0.f, 0.f) : make_float2(s.x, 1.0f / s.y);
        }
        if (__syncthreads_or(lost)) return;                      // not all scores are there
        float w[PER];
        const float* from[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int tk = t0 + threadIdx.x + k * kWarps * 32;
            w[k] = 0.f;
            from[k] = p.scores + ((p.score_pages > 0 ? (size_t)b * p.score_pages + tk / kRows : (size_t)max(page[k], 0)) * c.kv_heads + h) * (R * kRows) + tk % kRows * R;
        }
        for (int row = 0; row < rows; row += 4) {                // four rows' scores on their way at a time
            float s[4][PER];
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const float4 v = page[k] >= 0 ? *reinterpret_cast<const float4*>(from[k] + row) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                s[0][k] = v.x;
                s[1][k] = row + 1 < rows ? v.y : -INFINITY;
                s[2][k] = row + 2 < rows ? v.z : -INFINITY;
                s[3][k] = row + 3 < rows ? v.w : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 st = st_s[min(row + i, rows - 1)];
#pragma unroll
                for (int k = 0; k < PER; ++k) w[k] = fmaf(ex2f(s[i][k] - st.x), st.y, w[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            if (page[k] < 0) continue;
            const size_t at = row_slot(c, page[k], h, (t0 + threadIdx.x + k * kWarps * 32) % kRows);
            p.mass_out[at] = p.mass_in[at] + w[k];
        }
        return;
    }
    if (rows == 0) return;
    const int first = (int)blockIdx.x - mass_blocks, blocks = (int)gridDim.x - mass_blocks;
    constexpr int SLICES = D / 32, Q = 8, LANES = kWarps * 32 / Q;               // threads side by side, each with four channels of every LANES-th piece
    // few pieces, or more rows than there are blocks for: a row a warp, no barriers
    if (sh.each <= (blocks < rows * SLICES ? 64 : 12) * step_of(p, deal.all)) {
        for (int row = first * kWarps + warp; row < rows; row += blocks * kWarps) {
            const Pieces x = pieces_of(p, sh, deal, h, row / R);
            if (x.w0 == x.w1) continue;
            const int i = row / group, head = h * group + row % group, rr = row % R;
            const float2 st = merged_stats(p, x, rr);
            const float inv = st.y > 0.f ? 1.0f / st.y : st.y != st.y ? st.y : 0.f;
            constexpr int E = D / 32;
            float v[E];
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] = 0.f;
            for (int w0 = x.w0; w0 <= x.w1; w0 += 6) {
                float2 y[6][E / 2];
                float f[6];
#pragma unroll
                for (int s = 0; s < 6; ++s) {
                    const bool in = w0 + s <= x.w1;
                    const int piece = piece_of(w0 + s, x);
                    f[s] = in ? p.part_stats[(size_t)rr * 2 * p.warps + piece].x : -INFINITY;
#pragma unroll
                    for (int k = 0; k < E / 2; ++k) y[s][k] = in ? *reinterpret_cast<const float2*>(p.part + ((size_t)piece * R + rr) * D + lane * E + 2 * k) : make_float2(0.f, 0.f);
                }
#pragma unroll
                for (int s = 0; s < 6; ++s) {
                    const float a = f[s] == -INFINITY ? 0.f : ex2f(f[s] - st.x);
#pragma unroll
                    for (int k = 0; k < E / 2; ++k) { v[2 * k] = fmaf(y[s][k].x, a, v[2 * k]); v[2 * k + 1] = fmaf(y[s][k].y, a, v[2 * k + 1]); }
                }
            }
            T* dst = (T*)p.out + ((size_t)(e.row0 + i) * c.q_heads + head) * D + lane * E;
#pragma unroll
            for (int k = 0; k < E; k += 2) *reinterpret_cast<uint32_t*>(dst + k) = within2<T>(v[k] * inv, v[k + 1] * inv);
            if (lane == 0 && p.stats != nullptr && mass_blocks == 0) p.stats[stat_row(c, p, e, b, i, head)] = st;
        }
        return;
    }
    for (int job = first; job < rows * SLICES; job += blocks) {
        const int row = job / SLICES, d = job % SLICES * 32 + threadIdx.x % Q * 4;
        const Pieces x = pieces_of(p, sh, deal, h, row / R);
        if (x.w0 == x.w1) continue;
        const int i = row / group, head = h * group + row % group, rr = row % R;
        // every piece's factor once, in rounds of what fits
        const float2 st = merged_stats(p, x, rr);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int base = x.w0; base <= x.w1; base += kFactors) {
            const int n = min(kFactors, x.w1 + 1 - base);
            __syncthreads();
            for (int k = threadIdx.x; k < n; k += kWarps * 32) {
                const float m = p.part_stats[(size_t)rr * 2 * p.warps + piece_of(base + k, x)].x;
                f_s[k] = m == -INFINITY ? 0.f : ex2f(m - st.x);
            }
            __syncthreads();
            for (int k0 = threadIdx.x / Q; k0 < n; k0 += 8 * LANES) {            // eight loads on their way at a time
                float4 y[8];
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int k = k0 + i * LANES;
                    f[i] = k < n ? f_s[k] : 0.f;
                    y[i] = k < n ? *reinterpret_cast<const float4*>(p.part + ((size_t)piece_of(base + k, x) * R + rr) * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) { v.x = fmaf(y[i].x, f[i], v.x); v.y = fmaf(y[i].y, f[i], v.y); v.z = fmaf(y[i].z, f[i], v.z); v.w = fmaf(y[i].w, f[i], v.w); }
            }
        }
        v_s[threadIdx.x] = v;
        __syncthreads();
        if ((int)threadIdx.x < Q) {
            for (int k = 1; k < LANES; ++k) { const float4 y = v_s[k * Q + threadIdx.x]; v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w; }
            const float inv = st.y > 0.f ? 1.0f / st.y : st.y != st.y ? st.y : 0.f;
            *reinterpret_cast<uint2*>((T*)p.out + ((size_t)(e.row0 + i) * c.q_heads + head) * D + d) = make_uint2(within2<T>(v.x * inv, v.y * inv), within2<T>(v.z * inv, v.w * inv));
            if (threadIdx.x == 0 && d == 0 && p.stats != nullptr && mass_blocks == 0) p.stats[stat_row(c, p, e, b, i, head)] = st;
        }
        __syncthreads();
    }
}

}  // namespace kv4
}  // namespace efm
