// Attention over a 4-bit cache (kv4_cache.cuh): new rows of a ragged batch against the pages of their sequences.
//
// The codes go to the tensor cores as they are: a key is min + scale * code = c + scale * (code - 8) with c = min + 8 scale, so that
//     q . k = sum over groups g of  scale_g (q_g . (code - 8)_g) + c_g (sum of q_g),
// and code - 8 is exact in fp16.  q is scaled by a power of two per row and is exact there too (bf16 has fewer bits): scores carry fp32
// rounding only.  Values: o = sum over tokens of (p scale_g) (code - 8) + sum of p c_g, with p scale_g rounded to fp16 below a power of
// two that keeps the largest scale seen at 2^14 .. 2^15, so that neither large nor small scales leave its range.
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
    int chunk;                // pages a block takes
    int chunks;               // blocks of the longest sequence
    int rows;                 // new rows a sequence has in the buffers below
    float2* stats;            // [chunks, batch, rows, q_heads] (maximum, sum) of a row's weights in a chunk; null: not wanted
    float* part;              // [chunks, batch, rows, q_heads, D] its weighted values
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
__device__ __forceinline__ size_t part_row(const Cache& c, const AttnParams& p, int chunk, int b, int i, int head) {
    return (((size_t)chunk * c.batch + b) * p.rows + i) * c.q_heads + head;
}

constexpr int kWarps = 4, kMaxChunk = 32 * kWarps;      // a lane knows one page of its warp's

// ---- fragments -------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Nibbles at bits 0 and 16 (4 and 20) of w as a pair of fp16 code - 8: 1024 + n (1024 + 16 n) by setting the exponent, then exact arithmetic.
__device__ __forceinline__ uint32_t low_pair(uint32_t w) {
    uint32_t v = (w & 0x000f000fu) | 0x64006400u;
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(v) : "r"(0x64086408u));                       // 1032
    return v;
}
__device__ __forceinline__ uint32_t high_pair(uint32_t w) {
    uint32_t v = (w & 0x00f000f0u) | 0x64006400u;
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
    float sum[G][2], unit[2];      // of the lane's two columns 2 j, 2 j + 1: sums of the scaled q, and what a score is multiplied with

    template <typename T>
    __device__ __forceinline__ void load(const T* row, bool have, float scale_log2) {       // row: of column lane / 4
        const int lane = threadIdx.x & 31, j = lane & 3;
        float x[G][16], top = 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (have) w = *reinterpret_cast<const uint4*>(row + g * 64 + j * 16 + h * 8);
                const uint32_t v[4] = {w.x, w.y, w.z, w.w};
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
            for (int k = 0; k < 2; ++k) sum[g][k] = __shfl_sync(0xffffffffu, s[g], (2 * j + k) * 4);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) unit[k] = __shfl_sync(0xffffffffu, down * scale_log2, (2 * j + k) * 4);
    }
};

// Token of a 16-token tile that the operand layouts' row (or column) l stands for; chosen so that four neighbouring lanes read rows
// next to each other.
__device__ __forceinline__ int token_of(int l) { return (l & 8) + ((l & 7) >> 1) + 4 * (l & 1); }

// Parameters of a row and group: scale and centre of the codes; nothing where the row is not held.
__device__ __forceinline__ float2 centred(uint32_t par, bool have) {
    const float2 t = Num<__half>::two(have ? par : 0u);
    return make_float2(t.x, fmaf(8.0f, t.x, t.y));
}

// Scores, unscaled, of the 16 tokens of tile u of a page against NT query tiles: s[t][0..1] of token token_of(lane / 4) and the lane's
// two columns, s[t][2..3] of the token 8 behind.  valid: rows of the page that are held.
template <int D, int NT>
__device__ __forceinline__ void score_tile(const uint8_t* page, int u, int valid, const QueryTile<D> (&q)[NT], float (&s)[NT][4]) {
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
        float acc[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint32_t a0[4] = {low_pair(ka[g][w]), low_pair(kb[g][w]), high_pair(ka[g][w]), high_pair(kb[g][w])};
            const uint32_t a1[4] = {low_pair(ka[g][w] >> 8), low_pair(kb[g][w] >> 8), high_pair(ka[g][w] >> 8), high_pair(kb[g][w] >> 8)};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                mma16816(acc[t], a0, q[t].f[g][2 * w][0], q[t].f[g][2 * w][1]);
                mma16816(acc[t], a1, q[t].f[g][2 * w + 1][0], q[t].f[g][2 * w + 1][1]);
            }
        }
        const float2 a = centred(pa[g], ta < valid), b = centred(pb[g], tb < valid);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float x = fmaf(a.x, acc[t][k], a.y * q[t].sum[g][k]), y = fmaf(b.x, acc[t][2 + k], b.y * q[t].sum[g][k]);
                s[t][k] = g == 0 ? x : s[t][k] + x;
                s[t][2 + k] = g == 0 ? y : s[t][2 + k] + y;
            }
    }
}

// Pages of a warp through a ring of its own in shared memory, one bulk copy each.
template <int BYTES, int STAGES>
struct PageRing {
    uint32_t base, bars;
    int lane_page;               // of the warp's page number `lane`, -1: not a page of the pool
    __device__ __forceinline__ void init(unsigned char* smem, uint64_t* bar) {
        base = tc::smem_u32(smem);
        bars = tc::smem_u32(bar);
        if ((threadIdx.x & 31) == 0) {
            for (int i = 0; i < STAGES; ++i) tc::mbar_init(bars + 8 * i, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
    }
    template <int D>
    __device__ __forceinline__ int request(const Cache& c, int head, int i) {      // returns the page, by the whole warp
        const int page = __shfl_sync(0xffffffffu, lane_page, i & 31);
        if (page >= 0 && (threadIdx.x & 31) == 0) {
            tc::mbar_expect_tx(bars + 8 * (i % STAGES), BYTES);
            bulk_copy(base + (i % STAGES) * BYTES, tile_of<D>(c, page, head), BYTES, bars + 8 * (i % STAGES));
        }
        return page;
    }
};

template <int D, int NT>
struct FewCfg {
    static constexpr int STAGES = D == 128 ? 2 : 4;
    static constexpr int BLOCKS = NT == 1 ? 3 : 2;                               // per SM
    static constexpr size_t RING = (size_t)kWarps * STAGES * Tile<D>::BYTES;
    static constexpr int LD = D + 4;                                             // floats of a row in the merge of the warps
    static constexpr size_t MERGE = (size_t)kWarps * 8 * NT * LD * 4;
    static constexpr size_t SMEM = (RING > MERGE ? RING : MERGE) + kWarps * STAGES * 8 + kWarps * 8 * NT * 8 + 16;
};

// Few query rows.  grid (chunks x row tiles, kv heads, batch); a warp takes every fourth page of the chunk.  The MMA's 16 rows are
// tokens (channels in P V) and its 8 columns query rows -- the heads of a group, times the new rows -- so that a single token of up to 8
// heads per kv head fills it: m16n8k16 the other way round would leave half of it empty.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, FewCfg<D, NT>::BLOCKS) attend_few_kernel(const Cache c, const AttnParams p) {
    using L = Tile<D>;
    using C = FewCfg<D, NT>;
    constexpr int G = L::G, R = 8 * NT;
    extern __shared__ __align__(128) unsigned char smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (C::RING > C::MERGE ? C::RING : C::MERGE));
    float2* ml_s = reinterpret_cast<float2*>(bars + kWarps * C::STAGES);         // [warps][R]
    volatile int* abort_s = reinterpret_cast<volatile int*>(ml_s + kWarps * R);
    const int chunk = blockIdx.x % p.chunks, tile = blockIdx.x / p.chunks, h = blockIdx.y, b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3, group = c.q_heads / c.kv_heads;
    pdl_wait();
    pdl_launch_dependents();
    const int col = chunk * p.chunk + warp + kWarps * lane;                      // this lane's page of the warp's
    const int raw = col < c.max_pages && kWarps * lane + warp < p.chunk ? c.page_table[(size_t)b * c.max_pages + col] : -1;
    const Entry e = entry_of(c, p, b);
    const int rows = e.n * group;                                                // packed: new row x head of the group
    if (tile * R >= rows) return;
    const int pages = (e.len + kRows - 1) / kRows, p0 = chunk * p.chunk, mine = max(0, min(pages - p0, p.chunk) - warp + kWarps - 1) / kWarps;
    if (p0 >= pages && chunk > 0) return;
    PageRing<L::BYTES, C::STAGES> ring;
    ring.lane_page = (unsigned)raw < (unsigned)c.n_pages ? raw : -1;
    if (lane < mine && ring.lane_page < 0) raise(c, kBadPage);
    ring.init(smem + (size_t)warp * C::STAGES * L::BYTES, bars + warp * C::STAGES);
    if (threadIdx.x == 0) *abort_s = 0;
    for (int i = 0; i < min(mine, C::STAGES); ++i) ring.template request<D>(c, h, i);

    QueryTile<D> q[NT];
    int see[NT][2], least = INT32_MAX;                                           // cached rows that the lane's columns see
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row = tile * R + t * 8 + r;
        q[t].load((const T*)p.q + ((size_t)(e.row0 + row / group) * c.q_heads + h * group + row % group) * D, row < rows, p.scale_log2);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int cr = tile * R + t * 8 + 2 * j + k;
            see[t][k] = cr < rows ? max(0, min(e.len, e.len - e.n + cr / group + 1)) : 0;
            if (cr < rows) least = min(least, see[t][k]);
        }
    }
    least = min(least, __shfl_xor_sync(0xffffffffu, least, 1));
    least = min(least, __shfl_xor_sync(0xffffffffu, least, 2));
    float o[G][4][NT][4], pc[G][NT][2], m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) { m[t][k] = -INFINITY; l[t][k] = 0.f; for (int g = 0; g < G; ++g) pc[g][t][k] = 0.f; }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[g][x][t][k] = 0.f;
    int ev = -40;                                                                // exponent of the largest value scale seen
    __syncthreads();

    for (int i = 0; i < mine; ++i) {
        const int first = (p0 + warp + kWarps * i) * kRows, valid = min(kRows, e.len - first);
        const int page_no = __shfl_sync(0xffffffffu, ring.lane_page, i & 31);
        if (page_no >= 0) {
            if (!__all_sync(0xffffffffu, tc::mbar_wait(ring.bars + 8 * (i % C::STAGES), (uint32_t)(i / C::STAGES) & 1u, abort_s))) { *abort_s = 1; break; }
            const uint8_t* page = smem + ((size_t)warp * C::STAGES + i % C::STAGES) * L::BYTES;
            float s[4][NT][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) score_tile<D, NT>(page, u, valid, q, s[u]);
            const bool whole = first + kRows <= least;
            float top[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    top[t][k] = -INFINITY;
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            float& x = s[u][t][2 * hf + k];
                            x *= q[t].unit[k];
                            if (!whole && first + u * 16 + token_of(r) + 8 * hf >= see[t][k]) x = -INFINITY;
                            top[t][k] = fmaxf(top[t][k], x);
                        }
                }
            // parameters of the values, and the largest scale (positive halves order like whole numbers)
            uint32_t vp[4][2][G];
            int big = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int tk = u * 16 + token_of(r) + 8 * hf;
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        vp[u][hf][g] = tk < valid ? reinterpret_cast<const uint32_t*>(page + L::V_PARAMS)[tk * G + g] : 0u;
                        big = max(big, (int)(vp[u][hf][g] & 0x7fffu));
                    }
                }
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                big = max(big, __shfl_xor_sync(0xffffffffu, big, off));
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int k = 0; k < 2; ++k) top[t][k] = fmaxf(top[t][k], __shfl_xor_sync(0xffffffffu, top[t][k], off));
            }
            const int en = max(ev, big > 0 ? max(big >> 10, 1) - 15 : -40);
            const float fold = __uint_as_float((uint32_t)(127 + ev - en) << 23);
            float alpha[NT][2], base[NT][2];
            bool same = ev == en;
            ev = en;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float mn = fmaxf(m[t][k], top[t][k]);
                    base[t][k] = mn == -INFINITY ? 0.f : mn;
                    alpha[t][k] = m[t][k] == -INFINITY ? 0.f : ex2f(m[t][k] - base[t][k]);
                    same = same && (mn == m[t][k]);
                    m[t][k] = mn;
                }
            if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        l[t][k] *= alpha[t][k];
                        const float f = alpha[t][k] * fold;
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            pc[g][t][k] *= alpha[t][k];
#pragma unroll
                            for (int x = 0; x < 4; ++x) { o[g][x][t][k] *= f; o[g][x][t][2 + k] *= f; }
                        }
                    }
            }
            const float unit = __uint_as_float((uint32_t)(127 + 14 - en) << 23);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                uint32_t b0[G][NT], b1[G][NT];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        s[u][t][k] = ex2f(s[u][t][k] - base[t][k & 1]);
                        l[t][k & 1] += s[u][t][k];
                    }
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const float2 a = centred(vp[u][0][g], true), bb = centred(vp[u][1][g], true);
                    const float sa = a.x * unit, sb = bb.x * unit;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const float(&w)[4] = s[u][t];
                        pc[g][t][0] = fmaf(w[0], a.y, fmaf(w[2], bb.y, pc[g][t][0]));
                        pc[g][t][1] = fmaf(w[1], a.y, fmaf(w[3], bb.y, pc[g][t][1]));
                        b0[g][t] = transposed(half_pair(w[0] * sa, w[1] * sa));
                        b1[g][t] = transposed(half_pair(w[2] * sb, w[3] * sb));
                    }
                }
                // columns 2 j, 2 j + 1 (and 8 behind) of the operand are the tokens j, j + 4 (j + 8, j + 12)
                const uint32_t* codes = reinterpret_cast<const uint32_t*>(page + L::V_CODES) + (u * 16 + j) * L::WORDS + r;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint32_t w0 = codes[g * 8], w1 = codes[4 * L::WORDS + g * 8], w2 = codes[8 * L::WORDS + g * 8], w3 = codes[12 * L::WORDS + g * 8];
#pragma unroll
                    for (int hl = 0; hl < 2; ++hl) {
                        const uint32_t x = __byte_perm(w0, w1, hl ? 0x7632 : 0x5410), y = __byte_perm(w2, w3, hl ? 0x7632 : 0x5410);
                        const uint32_t a0[4] = {low_pair(x), high_pair(x), low_pair(y), high_pair(y)};
                        const uint32_t a1[4] = {low_pair(x >> 8), high_pair(x >> 8), low_pair(y >> 8), high_pair(y >> 8)};
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            mma16816(o[g][2 * hl][t], a0, b0[g][t], b1[g][t]);
                            mma16816(o[g][2 * hl + 1][t], a1, b0[g][t], b1[g][t]);
                        }
                    }
                }
            }
        }
        __syncwarp();                                                            // every lane has read the page
        if (i + C::STAGES < mine) ring.template request<D>(c, h, i + C::STAGES);
    }
    if (*abort_s != 0 && lane == 0)                                              // given up: let the copies in flight land (bounded)
        for (int i = 0; i < min(mine, C::STAGES); ++i) { volatile int go_on = 0; (void)tc::mbar_wait(ring.bars + 8 * i, 0, &go_on); (void)tc::mbar_wait(ring.bars + 8 * i, 1, &go_on); }

    // the warps' results: maxima first, then values relative to the block's
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
    if (r == 0)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) ml_s[warp * R + t * 8 + 2 * j + k] = make_float2(m[t][k], l[t][k]);
    __syncthreads();                                                             // the rings are free
    float* merge = reinterpret_cast<float*>(smem);
    const float back = __uint_as_float((uint32_t)(127 + ev - 14) << 23);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int rr = t * 8 + 2 * j + k;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml_s[w * R + rr].x);
            const float f = m[t][k] == -INFINITY ? 0.f : ex2f(m[t][k] - top);
            float* dst = merge + ((size_t)warp * R + rr) * C::LD + 8 * r;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float v[8];                                                      // channels of word r of the group, see the nibbles' order
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int at = (x & 1) * 4 + (x >> 1);
                    v[at] = fmaf(o[g][x][t][k], back, pc[g][t][k]) * f;
                    v[at + 2] = fmaf(o[g][x][t][2 + k], back, pc[g][t][k]) * f;
                }
                *reinterpret_cast<float4*>(dst + g * 64) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4*>(dst + g * 64 + 4) = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
    __syncthreads();
    if (*abort_s != 0) { if (threadIdx.x == 0) raise(c, kWait); return; }
    const bool alone = pages <= p.chunk;
    for (int i = threadIdx.x; i < R * (D / 4); i += kWarps * 32) {
        const int rr = i / (D / 4), d = i % (D / 4) * 4, row = tile * R + rr;
        if (row >= rows) continue;
        float top = -INFINITY, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml_s[w * R + rr].x);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 s = ml_s[w * R + rr];
            if (s.x != -INFINITY) sum = fmaf(s.y, ex2f(s.x - top), sum);
            const float4 x = *reinterpret_cast<const float4*>(merge + ((size_t)w * R + rr) * C::LD + d);
            v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        const int head = h * group + row % group;
        if (alone) {
            const float inv = sum > 0.f ? 1.0f / sum : 0.f;
            T* dst = (T*)p.out + ((size_t)(e.row0 + row / group) * c.q_heads + head) * D + d;
            *reinterpret_cast<uint2*>(dst) = make_uint2(Num<T>::pack(v.x * inv, v.y * inv), Num<T>::pack(v.z * inv, v.w * inv));
        } else {
            *reinterpret_cast<float4*>(p.part + part_row(c, p, chunk, b, row / group, head) * D + d) = v;
        }
        if (p.stats != nullptr && d == 0) p.stats[part_row(c, p, chunk, b, row / group, head)] = make_float2(top, sum);
    }
}

// Maximum and 1 / sum over the chunks of a row's weights.
__device__ __forceinline__ float2 row_stats(const Cache& c, const AttnParams& p, int n_chunks, int b, int i, int head) {
    float top = -INFINITY, sum = 0.f;
    for (int k = 0; k < n_chunks; ++k) top = fmaxf(top, p.stats[part_row(c, p, k, b, i, head)].x);
    if (top == -INFINITY) return make_float2(0.f, 0.f);
    for (int k = 0; k < n_chunks; ++k) {
        const float2 s = p.stats[part_row(c, p, k, b, i, head)];
        if (s.x != -INFINITY) sum = fmaf(s.y, ex2f(s.x - top), sum);
    }
    return make_float2(top, 1.0f / sum);
}

template <int D>
struct FinishCfg {
    static constexpr int K_BYTES = Tile<D>::V_CODES;                             // codes and parameters of the keys
    static constexpr size_t SMEM = (size_t)kWarps * K_BYTES + kWarps * 8 + 16;
};

// What needs the whole row: outputs of rows whose keys were dealt over several blocks, and the summed weights.  grid (page groups +
// merging blocks, kv heads, batch); in a page group a warp has a page of its own and walks the new rows in order.
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) attend_finish_kernel(const Cache c, const AttnParams p, int page_groups) {
    using L = Tile<D>;
    using C = FinishCfg<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (size_t)kWarps * C::K_BYTES);
    volatile int* abort_s = reinterpret_cast<volatile int*>(bars + kWarps);
    const int h = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3, group = c.q_heads / c.kv_heads;
    pdl_launch_dependents();
    if ((int)blockIdx.x >= page_groups) {                                        // merge: a warp per new row and head
        pdl_wait();
        const Entry e = entry_of(c, p, b);
        const int pages = (e.len + kRows - 1) / kRows, n_chunks = (pages + p.chunk - 1) / p.chunk;
        if (n_chunks <= 1) return;
        for (int row = ((int)blockIdx.x - page_groups) * kWarps + warp; row < e.n * group; row += ((int)gridDim.x - page_groups) * kWarps) {
            const int i = row / group, head = h * group + row % group;
            const float2 st = row_stats(c, p, n_chunks, b, i, head);
            constexpr int E = D / 32;
            float v[E];
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] = 0.f;
            for (int k = 0; k < n_chunks; ++k) {
                const size_t at = part_row(c, p, k, b, i, head);
                const float f = ex2f(p.stats[at].x - st.x);                      // 0 where the chunk has nothing to see
                const float* src = p.part + at * D + lane * E;
#pragma unroll
                for (int d = 0; d < E; ++d) v[d] = fmaf(src[d], f, v[d]);
            }
            T* dst = (T*)p.out + ((size_t)(e.row0 + i) * c.q_heads + head) * D + lane * E;
#pragma unroll
            for (int d = 0; d < E; d += 2) *reinterpret_cast<uint32_t*>(dst + d) = Num<T>::pack(v[d] * st.y, v[d + 1] * st.y);
        }
        return;
    }
    const Entry e = entry_of(c, p, b);
    const int pages = (e.len + kRows - 1) / kRows, pg = blockIdx.x * kWarps + warp, n_chunks = max(1, (pages + p.chunk - 1) / p.chunk);
    if (threadIdx.x == 0) *abort_s = 0;
    __syncthreads();
    if (pg >= pages) { pdl_wait(); return; }
    const int page = page_of(c, b, pg);
    if (page < 0) { pdl_wait(); return; }
    const uint32_t bar = tc::smem_u32(bars + warp);
    if (lane == 0) {
        tc::mbar_init(bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::mbar_expect_tx(bar, C::K_BYTES);
        bulk_copy(tc::smem_u32(smem) + warp * C::K_BYTES, tile_of<D>(c, page, h), C::K_BYTES, bar);
    }
    __syncwarp();
    pdl_wait();
    if (!__all_sync(0xffffffffu, tc::mbar_wait(bar, 0, abort_s))) { if (lane == 0) raise(c, kWait); return; }
    const uint8_t* tile = smem + (size_t)warp * C::K_BYTES;
    const int first = pg * kRows, valid = min(kRows, e.len - first), rows = e.n * group;
    float w[4][2];
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u][0] = w[u][1] = 0.f;
    const int row_first = max(0, first - (e.len - e.n)) * group;                 // earlier rows do not see the page
    for (int r0 = row_first & ~7; r0 < rows; r0 += 8) {
        QueryTile<D> q[1];
        const int row = r0 + r;
        q[0].load((const T*)p.q + ((size_t)(e.row0 + row / group) * c.q_heads + h * group + row % group) * D, row < rows, p.scale_log2);
        const float2 mine = row < rows ? row_stats(c, p, n_chunks, b, row / group, h * group + row % group) : make_float2(0.f, 0.f);
        float top[2], inv[2];
        int see[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            top[k] = __shfl_sync(0xffffffffu, mine.x, (2 * j + k) * 4);
            inv[k] = __shfl_sync(0xffffffffu, mine.y, (2 * j + k) * 4);
            const int cr = r0 + 2 * j + k;
            see[k] = cr < rows ? min(e.len, e.len - e.n + cr / group + 1) : 0;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float s[1][4];
            score_tile<D, 1>(tile, u, valid, q, s);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float x = ex2f(fmaf(s[0][k], q[0].unit[k & 1], -top[k & 1])) * inv[k & 1];
                if (first + u * 16 + token_of(r) + 8 * (k >> 1) < see[k & 1]) w[u][k >> 1] += x;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            float x = w[u][hf];
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            const int tk = u * 16 + token_of(r) + 8 * hf;
            if (j == 0 && tk < valid) {
                const size_t at = row_slot(c, page, h, tk);
                p.mass_out[at] = p.mass_in[at] + x;
            }
        }
}

}  // namespace kv4
}  // namespace efm
