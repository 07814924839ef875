// Many query rows against a 4-bit cache on the 5th-generation tensor cores.
//
// A block has 256 packed rows (new rows x heads of a group) of one sequence and kv head at a time, as two tiles of 128 that share the keys and
// values; 15 warps:
//   warps 0-3, 4-7   softmax of a tile, a thread per row: S from tensor memory, p = 2^(s - m), P back into tensor memory as fp16, where the
//                    product takes it as its A operand.  O stays in tensor memory; it is scaled only when a row's maximum has grown by
//                    more than 2^8 since it was last, which a row's first pages see and later ones hardly;
//   warp 14          asks for pages, a bulk copy each into a ring;
//   warps 8-11       codes to fp16 values (min + scale * code, rounded once), written in the
//                    operands' 128-byte-swizzled layout: K-major rows of K, and the same rows of V read MN-major;
//   warps 12, 13     one lane of each issues a tile's products: S = Q K^T (M 128, N 64, K = head size), O += P V (M 128, N = head size, K 64).  S has two
//                    buffers a tile and runs two pages ahead of P V; weights take the place of the scores they came from.  A wait costs
//                    that warp some 200 cycles even when it is over, so it polls for all that a page needs at once; one warp for both
//                    tiles left the tensor pipe idle half the time.
// q is scaled by a power of two per row to be exact in fp16.  k, v and p are rounded to fp16: v and p by 2^-11 of themselves, below the half step
// of a bf16 output (2^-8), and a score by 2^-11 of sum |q k| scale at most, as from a 16-bit cache of fp16 keys.  X 0, bf16 outputs without
// mass: on 2048 rows behind 12289 1.74e-3 from the formula, where rounding the outputs is 1.66e-3 (X 1 1.68e-3, but 540 us instead of 418).
// Pairs high + low hold more: k where row sums are wanted that summed weights are divided by (X 1: S = Q (Kh + Kl)), and all of them for fp16
// outputs, whose half step it would be (X 2: O += Ph Vh + Pl Vh + Ph Vl as well).
// A barrier is waited for by parity, which tells a phase from its neighbours only: every barrier here is either waited for in each of its
// phases by whoever its next phase needs, or (o_done) has a copy per page parity, whose next phase needs the waiting thread's weights of
// two pages later.
// Bound: the softmax warps (some 2000 cycles a page: 1600 of arithmetic, the rest waits), ahead of the tensor pipe (1280) and the exponential
// unit (770 after a quarter of the exponentials went to arithmetic).  2048 rows, 28 heads on 4 kv heads of 128, behind 12289: 370 - 411 us by
// the card's clock, 950 - 1060 TFLOP/s of 4 rows keys D; the whole call 400 - 450.
#pragma once
#include <type_traits>

#include "attention_tc.cuh"
#include "kv4_attention.cuh"

namespace efm {
namespace kv4 {

constexpr int kTileRows = 128, kManyThreads = 15 * 32;
constexpr float kLift = 7.0f;              // weights of many rows are relative to their maximum less this power of two

template <int D, int X>
struct ManyCfg {
    static constexpr int G = D / 64;
    static constexpr int KS = X >= 1 ? 2 : 3, VS = X == 2 ? 2 : 3, LEAD = KS - 1, RAW = LEAD + 2;          // K is converted LEAD pages ahead of V; pages in the ring of raw ones
    static constexpr int Q_BYTES = kTileRows * 128 * G, LOW = kRows * 128 * G;           // of one tile; of K or V of a page, and where its low half begins
    static constexpr int KB = X >= 1 ? 2 * LOW : LOW, VB = X == 2 ? 2 * LOW : LOW;       // bytes of a stage
    static constexpr int Q_AT = 0, K_AT = 2 * Q_BYTES, V_AT = K_AT + KS * KB, RAW_AT = V_AT + VS * VB, BARS = RAW_AT + RAW * Tile<D>::BYTES;
    static constexpr int S_COL = 0, O_COL = 256;                                         // S of (tile, page parity): 64 columns each, P in its place; O: 128 a tile
    static constexpr size_t SMEM = BARS + 352 + 1024;
};

// Pairs of fp16 codes of a word, in the order of the channels: as in low_pair / high_pair, without the 8.
__device__ __forceinline__ void half_codes(uint32_t w, __half2 (&n)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t x;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(i < 2 ? w : w >> 8), "r"((i & 1) ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));
        if (i & 1) asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(x) : "r"(0x2c002c00u), "r"(0xd400d400u));
        else asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x64006400u));
        n[i] = *reinterpret_cast<__half2*>(&x);
    }
}
__device__ __forceinline__ uint4 four(const __half2 (&x)[4]) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(x);
    return make_uint4(u[0], u[1], u[2], u[3]);
}
// Parameters whose products or sums could leave fp16's range (scale above 2048 or minimum beyond 32768): both tests in one addition.
__device__ __forceinline__ bool wide_range(__half2 par) {
    return (((*reinterpret_cast<const uint32_t*>(&par) & 0x7fff7fffu) + 0x07ff17ffu) & 0x80008000u) != 0u;
}
// (a whole warp asks once for all that it converts: a branch a word made attend_many a third slower)
// Their values by way of fp32, up to 65504 (the parameters' rounding may take them 80 beyond), and what is left of them.
__device__ __forceinline__ void wide_values(uint32_t w, __half2 par, uint4& high, uint4& low) {
    const float s = __low2float(par), m = __high2float(par);
    __half2 n[4], h[4];
    half_codes(w, n);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 c = __half22float2(n[i]);
        const float a = fmaf(c.x, s, m), b = fmaf(c.y, s, m);
        h[i] = __floats2half2_rn(fminf(a, 65504.0f), fminf(b, 65504.0f));
        const float2 f = __half22float2(h[i]);
        n[i] = __floats2half2_rn(a - f.x, b - f.y);
    }
    high = four(h);
    low = four(n);
}
// min + scale * code of a word's eight codes, rounded once
__device__ __forceinline__ uint4 half_values(uint32_t w, __half2 par) {
    const __half2 s = __low2half2(par), m = __high2half2(par);
    __half2 n[4];
    half_codes(w, n);
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = __hfma2(n[i], s, m);
    return four(n);
}
// the same as high + low: the product's and the sum's rounding errors, both exact, added up
__device__ __forceinline__ void half_pairs(uint32_t w, __half2 par, uint4& high, uint4& low) {
    const __half2 s = __low2half2(par), m = __high2half2(par);
    __half2 n[4], h[4];
    half_codes(w, n);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 x = __hmul2_rn(n[i], s), xl = __hfma2(n[i], s, __hneg2(x));
        h[i] = __hadd2_rn(m, x);
        const __half2 back = __hsub2_rn(h[i], m);
        n[i] = __hadd2_rn(__hadd2_rn(__hsub2_rn(m, __hsub2_rn(h[i], back)), __hsub2_rn(x, back)), xl);
    }
    high = four(h);
    low = four(n);
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}

__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&r)[64]) {
#pragma unroll
    for (int i = 0; i < 64; i += 32)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=f"(r[i]), "=f"(r[i + 1]), "=f"(r[i + 2]), "=f"(r[i + 3]), "=f"(r[i + 4]), "=f"(r[i + 5]), "=f"(r[i + 6]), "=f"(r[i + 7]), "=f"(r[i + 8]), "=f"(r[i + 9]), "=f"(r[i + 10]),
              "=f"(r[i + 11]), "=f"(r[i + 12]), "=f"(r[i + 13]), "=f"(r[i + 14]), "=f"(r[i + 15]), "=f"(r[i + 16]), "=f"(r[i + 17]), "=f"(r[i + 18]), "=f"(r[i + 19]), "=f"(r[i + 20]),
              "=f"(r[i + 21]), "=f"(r[i + 22]), "=f"(r[i + 23]), "=f"(r[i + 24]), "=f"(r[i + 25]), "=f"(r[i + 26]), "=f"(r[i + 27]), "=f"(r[i + 28]), "=f"(r[i + 29]), "=f"(r[i + 30]),
              "=f"(r[i + 31])
            : "r"(taddr + i) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Two 32-bit numbers a register pair, one instruction for both.
__device__ __forceinline__ uint64_t pair_of_floats(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float low_of(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float high_of(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^x of two numbers without the exponential unit: x = n + f, n the nearest integer (it is in the low bits of x + 1.5 2^23), 2^f on
// [-1/2, 1/2] by the polynomial of degree 4 of least largest relative error, 2^-18.5 (found by linear programming over 4001 Chebyshev
// points), n added to the exponent.  Below 2^-125 it stays there.
__device__ __forceinline__ void ex2_pair(uint64_t x, float& a, float& b) {
    const uint64_t big = pair_of_floats(12582912.0f, 12582912.0f);
    x = pair_of_floats(fmaxf(low_of(x), -125.0f), fmaxf(high_of(x), -125.0f));
    const uint64_t n = add2(x, big), f = fma2(add2(n, pair_of_floats(-12582912.0f, -12582912.0f)), pair_of_floats(-1.0f, -1.0f), x);
    uint64_t y = fma2(f, pair_of_floats(0.00957053154706955f, 0.00957053154706955f), pair_of_floats(0.05591866374015808f, 0.05591866374015808f));
    y = fma2(y, f, pair_of_floats(0.24024735391139984f, 0.24024735391139984f));
    y = fma2(y, f, pair_of_floats(0.6931216716766357f, 0.6931216716766357f));
    y = fma2(y, f, pair_of_floats(0.9999992847442627f, 0.9999992847442627f));
    a = __uint_as_float((uint32_t)y + ((uint32_t)n << 23));
    b = __uint_as_float((uint32_t)(y >> 32) + ((uint32_t)(n >> 32) << 23));
}
// Maxima that keep what is no number: ex2_pair does not.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max2(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Three waits at once: polled one behind the other a wait that is over takes some 200 cycles each.
struct Phase { uint32_t bar, parity; };
template <int POLLS>
__device__ __forceinline__ bool warp_wait(const Phase& a, const Phase& b, const Phase& c, volatile int* abort_flag) {
    for (int i = 0; i < POLLS; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n"
            ".reg .pred p, q, r;\n"
            "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "mbarrier.test_wait.parity.shared::cta.b64 q, [%3], %4;\n"
            "mbarrier.test_wait.parity.shared::cta.b64 r, [%5], %6;\n"
            "and.pred p, p, q;\n"
            "and.pred p, p, r;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(ok) : "r"(a.bar), "r"(a.parity), "r"(b.bar), "r"(b.parity), "r"(c.bar), "r"(c.parity) : "memory");
        if (__all_sync(0xffffffffu, ok)) return true;
        if ((i & 0xff) == 0xff && __any_sync(0xffffffffu, *abort_flag != 0)) return false;
    }
    return false;
}
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t lead;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(lead));
    return lead;
}
// 32 query rows into rows r0 .. r0 + 31 of a K-major operand of 128 rows, as fp16 scaled by a power of two, by a warp: neighbouring lanes
// have neighbouring channels (a thread per row took 6000 cycles over its strided loads).  mine: where the row of this lane begins, -1:
// no such row.  Returns what this lane's row's scores are to be multiplied with.
template <typename T, int D>
__device__ __forceinline__ float query_rows(const T* q, long long mine, unsigned char* to, int r0, float scale_log2) {
    constexpr int LANES = D / 8, PER = 32 / LANES;               // lanes of a row, rows at a time
    const int lane = threadIdx.x & 31, i = lane % LANES;
    uint4 w[LANES];
#pragma unroll
    for (int it = 0; it < LANES; ++it) {
        const long long at = __shfl_sync(0xffffffffu, mine, it * PER + lane / LANES);
        w[it] = at >= 0 ? *reinterpret_cast<const uint4*>(q + at + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
    }
    float unit = 0.f;
#pragma unroll
    for (int it = 0; it < LANES; ++it) {
        uint32_t v[4] = {w[it].x, w[it].y, w[it].z, w[it].w};
        float2 x[4];
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) { x[k] = Num<T>::two(v[k]); top = fmaxf(top, fmaxf(fabsf(x[k].x), fabsf(x[k].y))); }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int bits = (int)(__float_as_uint(top) >> 23), ex = bits == 255 ? 3 : max(bits - 127, -100);
        const float up = __uint_as_float((uint32_t)(130 - ex) << 23), down = fmaxf(__uint_as_float((uint32_t)(ex + 124) << 23) * scale_log2, 1.2e-38f);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = half_pair(x[k].x * up, x[k].y * up);
        const int r = r0 + it * PER + lane / LANES;
        *reinterpret_cast<uint4*>(to + (i >> 3) * (kTileRows * 128) + r * 128 + (((i & 7) ^ (r & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        const float u = __shfl_sync(0xffffffffu, down, (lane % PER) * LANES);
        if (lane / PER == it) unit = u;
    }
    return unit;
}
// The two words of a key row's quarter x of each group
template <int D, bool V>
__device__ __forceinline__ void quarter_words(const uint32_t* codes, int r, int x, uint32_t (&w)[D / 64][2]) {
    constexpr int W = D / 8;
    if constexpr (D == 128 && !V) {
        const uint4 v = *reinterpret_cast<const uint4*>(codes + r * W + x * 4);
        w[0][0] = v.x; w[0][1] = v.y; w[1][0] = v.z; w[1][1] = v.w;
    } else {
#pragma unroll
        for (int g = 0; g < D / 64; ++g) { const uint2 v = *reinterpret_cast<const uint2*>(codes + r * W + g * 8 + x * 2); w[g][0] = v.x; w[g][1] = v.y; }
    }
}

__device__ __forceinline__ size_t row_tile(const Cache& c, const AttnParams& p, const Entry& e, int b, int h, int tile) {
    const size_t first = p.rows > 0 ? (size_t)b * p.row_tiles : (size_t)e.row0 * (c.q_heads / c.kv_heads) / kTileRows + b;
    return (first + tile) * c.kv_heads + h;
}

// How attend_many's work is dealt: its units are the pages of every (sequence, block of 256 packed rows, kv head), in that order, block w of
// the grid has the units [w step, (w + 1) step).  Rows that begin or end inside such a range are joined by attend_join.
constexpr int kManyRows = 2 * kTileRows;
constexpr int64_t kMostUnits = 1 << 30;
constexpr int kManyStep = 4;               // at least that many pages a block: fewer cost more to join than they save
// Pages of a block of rows of a sequence, 0: nobody's, or attend_few's; rows that see nothing are somebody's to clear.
__device__ __forceinline__ int many_pages(const AttnParams& p, const Entry& e, int group, int tile) {
    const int rows = e.n * group;
    if (rows <= p.few_rows || tile * kManyRows >= rows) return 0;
    const int last = min(rows, (tile + 1) * kManyRows) - 1;
    return max(1, (min(e.len, e.len - e.n + last / group + 1) + kRows - 1) / kRows);
}
// Joining costs as much as some ten pages of a block.  Where every (block of rows, kv head) can have an SM and none has that many more than
// its even share they stay whole: they all get as many units as the longest then, which many_starts has behind the sums (otherwise 0).
// 8 sequences with 256 new rows on 1000, 16 query heads on 2 of 128 (128 blocks of 20 pages): 46 us whole, 57 dealt evenly; 4 of them
// (64 blocks, 8 pages an SM) 45 dealt evenly.
constexpr int kJoinPages = 10;
__device__ __forceinline__ int many_step(const AttnParams& p, int all, int whole) { return whole > 0 ? whole : max(kManyStep, (all + p.many_blocks - 1) / p.many_blocks); }
// many_starts[b * many_tiles + tile]: units ahead; all; units of each, if they stay whole.  By one block of kTileRows threads
__device__ __forceinline__ void lay_out_units(const Cache& c, const AttnParams& p) {
    __shared__ int64_t sums[kTileRows / 32], counts[kTileRows / 32];
    __shared__ int most_s;
    const int group = c.q_heads / c.kv_heads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t pairs = (int64_t)c.batch * p.many_tiles, per = (pairs + kTileRows - 1) / kTileRows, lo = min(pairs, (int64_t)threadIdx.x * per), hi = min(pairs, lo + per);
    if (threadIdx.x == 0) most_s = 0;
    __syncthreads();
    int64_t own = 0, count = 0;                                  // units, and blocks of rows that have any; most: of one
    int most = 0;
    auto walk = [&](auto&& visit) {
        int b = (int)(lo / p.many_tiles), tile = (int)(lo % p.many_tiles);
        Entry e{};
        if (lo < hi) e = entry_of(c, p, b);
        for (int64_t i = lo; i < hi; ++i) {
            visit(i, many_pages(p, e, group, tile));
            if (++tile == p.many_tiles) {
                tile = 0;
                if (++b < c.batch) e = entry_of(c, p, b);
            }
        }
    };
    walk([&](int64_t, int n) { own += (int64_t)n * c.kv_heads; count += n > 0 ? c.kv_heads : 0; most = max(most, n); });
    atomicMax(&most_s, most);
    int64_t upto = own, upto_n = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o), n = __shfl_up_sync(0xffffffffu, upto_n, o);
        if (lane >= o) { upto += v; upto_n += n; }
    }
    if (lane == 31) { sums[warp] = upto; counts[warp] = upto_n; }
    __syncthreads();
    int64_t all = 0, all_n = 0;
    for (int w = 0; w < kTileRows / 32; ++w) {
        if (w < warp) { upto += sums[w]; upto_n += counts[w]; }
        all += sums[w];
        all_n += counts[w];
    }
    const bool whole = all_n <= p.many_blocks && most_s <= (all + p.many_blocks - 1) / p.many_blocks + kJoinPages;
    // row counts that lie may add up to more than the caller's sizes allow: cut off there
    int64_t at = whole ? (upto_n - count) * most_s : upto - own;
    walk([&](int64_t i, int n) { p.many_starts[i] = (int)min(at, kMostUnits); at += (int64_t)(whole && n > 0 ? most_s : n) * c.kv_heads; });
    if (threadIdx.x == 0) {
        p.many_starts[pairs] = (int)min(whole ? all_n * most_s : all, kMostUnits);
        p.many_starts[pairs + 1] = whole ? most_s : 0;
    }
}
// Of a (sequence, block of rows) whose units begin at or before `from`, the one that has unit u, by a warp: 32 at a time.
__device__ __forceinline__ int pair_of(const int32_t* starts, int pairs, int from, int u) {
    const int lane = threadIdx.x & 31;
    int lo = from, hi = pairs;                                   // starts[lo] <= u < starts[hi]
    uint32_t later = __ballot_sync(0xffffffffu, starts[min(hi, lo + 1 + lane)] > u);         // mostly one of the next
    if (later != 0u) return lo + __ffs(later) - 1;
    for (lo += 32; hi - lo > 1;) {
        const int s = (hi - lo + 31) / 32;
        later = __ballot_sync(0xffffffffu, starts[min(hi, lo + (lane + 1) * s)] > u);
        const int k = __ffs(later) - 1;                          // lane 31 looks at hi
        hi = min(hi, lo + (k + 1) * s);
        lo += k * s;
    }
    return lo;
}
// Pages [p0, p0 + n) of a (sequence, block of rows, kv head), as a warp walks a block's range of units.
struct ManyPiece { Entry e; int b, h, r0, tiles, p0, n; bool from_start, to_end; };
struct ManyWalk {
    int u, u1, pair, base, pairs, whole;
    __device__ __forceinline__ ManyWalk(const Cache& c, const AttnParams& p, int block) : pair(0), base(0), pairs(c.batch * p.many_tiles) {
        whole = p.many_starts[pairs + 1];
        const int all = p.many_starts[pairs], step = many_step(p, all, whole);
        u = (int)min((int64_t)all, (int64_t)block * step);
        u1 = min(all, u + step);
    }
    __device__ __forceinline__ bool more() const { return u < u1; }
    __device__ __forceinline__ ManyPiece next(const Cache& c, const AttnParams& p) {
        ManyPiece x;
        pair = pair_of(p.many_starts, pairs, pair, u);
        base = p.many_starts[pair];
        x.b = pair / p.many_tiles;
        const int tile = pair - x.b * p.many_tiles, group = c.q_heads / c.kv_heads;
        x.e = entry_of(c, p, x.b);
        const int each = many_pages(p, x.e, group, tile), stride = whole > 0 ? whole : each, in = u - base;
        x.h = in / stride;
        x.p0 = in - x.h * stride;
        x.n = __shfl_sync(0xffffffffu, min(each - x.p0, u1 - u), 0);
        x.r0 = tile * kManyRows;
        x.tiles = x.e.n * group - x.r0 > kTileRows ? 2 : 1;
        x.from_start = x.p0 == 0;
        x.to_end = x.p0 + x.n == each;
        u += whole > 0 ? whole : x.n;
        return x;
    }
};

// Packed rows, 128 a tile, as the operands that attend_many and attend_weights copy in one piece (every block of theirs converting rows for
// itself took 4000 cycles a tile).  grid (tiles + 1, kv heads, batch): one block adds up attend_many's units of work instead.
template <typename T, int D>
__global__ void __launch_bounds__(kTileRows) attend_query_kernel(const Cache c, const AttnParams p) {
    pdl_wait();
    pdl_launch_dependents();
    if ((int)blockIdx.x == p.row_tiles) {
        if (blockIdx.y == 0 && blockIdx.z == 0 && p.many_tiles > 0) lay_out_units(c, p);
        return;
    }
    const int h = blockIdx.y, b = blockIdx.z, group = c.q_heads / c.kv_heads, row = blockIdx.x * kTileRows + threadIdx.x;
    const Entry e = entry_of(c, p, b);
    const int rows = e.n * group;
    if ((int)blockIdx.x * kTileRows >= rows) return;
    const size_t tile = row_tile(c, p, e, b, h, blockIdx.x);
    const long long at = row < rows ? ((long long)(e.row0 + row / group) * c.q_heads + h * group + row % group) * D : -1;
    p.units[tile * kTileRows + threadIdx.x] = query_rows<T, D>((const T*)p.q, at, p.images + tile * (kTileRows * D * 2), threadIdx.x & ~31, p.scale_log2);
}

// grid: one block an SM, each with its share of the units (above)
template <typename T, int D, int X, int POLLS = kPolls>
__global__ void __launch_bounds__(kManyThreads, 1) attend_many_kernel(const Cache c, const AttnParams p) {
    using C = ManyCfg<D, X>;
    using L = Tile<D>;
    constexpr int G = C::G;
    constexpr float kGrow = 8.0f;                                // p is up to 2^(8 + kLift): fp16 keeps weights down to 2^-21 of the largest whole
    extern __shared__ unsigned char many_smem[];
    const uint32_t raw_base = tc::smem_u32(many_smem), base = (raw_base + 1023u) & ~1023u;
    unsigned char* sm = many_smem + (base - raw_base);
    const uint32_t bars = base + C::BARS;
    const uint32_t q_full = bars, raw_full = bars + 16, raw_empty = bars + 48, k_full = bars + 80, k_empty = bars + 104, v_full = bars + 128, v_empty = bars + 152,
                   s_full = bars + 176, p_full = bars + 208, o_done = bars + 240, drain = bars + 272;     // q_full: [tile]; s_full, p_full, o_done: [tile][parity of its pages]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::BARS + 288);
    volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* valid_s = reinterpret_cast<volatile int*>(tmem_slot + 2);      // [8] rows held of the block's page number j % 8; 0: not one of the pool's
    volatile int* asked_s = valid_s + 8;                         // copies that warps 12, 13 and 14 asked for
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = c.q_heads / c.kv_heads;

    pdl_wait();
    if (tid == 0) p.lost[p.few_blocks + blockIdx.x] = 0;
    ManyWalk walk(c, p, blockIdx.x);
    if (!walk.more()) return;
    const int pages = walk.whole > 0 ? ManyWalk(walk).next(c, p).n : walk.u1 - walk.u;      // of all pieces
    if (tid == 0) {
        for (int i = 0; i < C::RAW; ++i) { tc::mbar_init(raw_full + 8 * i, 1); tc::mbar_init(raw_empty + 8 * i, 4); }
        for (int i = 0; i < 2; ++i) { tc::mbar_init(q_full + 8 * i, 1); tc::mbar_init(drain + 8 * i, 1); }
        for (int i = 0; i < C::KS; ++i) { tc::mbar_init(k_full + 8 * i, 4); tc::mbar_init(k_empty + 8 * i, 2); }
        for (int i = 0; i < C::VS; ++i) { tc::mbar_init(v_full + 8 * i, 4); tc::mbar_init(v_empty + 8 * i, 2); }
        for (int i = 0; i < 4; ++i) { tc::mbar_init(s_full + 8 * i, 1); tc::mbar_init(p_full + 8 * i, 4); tc::mbar_init(o_done + 8 * i, 1); }
        *abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();                                     // not before this block has its tensor memory

    if (warp < 8) {
        const int t = warp >> 2, tr = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t o_at = tmem + lanes + (uint32_t)(C::O_COL + t * 128);
        bool ok = true;
        for (int before = 0, mine = 0; ok && walk.more();) {     // pages of the pieces before: of all, and of this tile
            const ManyPiece x = walk.next(c, p);
            if (t >= x.tiles) { before += x.n; continue; }
            const int row = x.r0 + t * kTileRows + tr;
            const bool have = row < x.e.n * group;
            const int see = have ? max(0, min(x.e.len, x.e.len - x.e.n + row / group + 1)) - x.p0 * kRows : 0;     // counted from the piece's first key
            int least = have ? see : INT32_MAX;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
            const float unit = p.units[row_tile(c, p, x.e, x.b, x.h, x.r0 / kTileRows + t) * kTileRows + tr];
            float m = -INFINITY, l = 0.f;                        // m: what the row's weights are relative to
            int j = 0;
            for (; j < x.n; ++j) {
                const int buf = t * 2 + ((mine + j) & 1);
                const uint32_t s_at = tmem + lanes + (uint32_t)(C::S_COL + buf * 64);
                if (!warp_wait<POLLS>(s_full + 8 * buf, (uint32_t)((mine + j) >> 1) & 1u, abort_s)) { *abort_s = 1; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float s[64];
                tmem_ld64(s_at, s);
                const int held = valid_s[(before + j) & 7], seen = held != 0 ? see - j * kRows : 0;             // keys of the page that the row sees
                if (held == 0 || (j + 1) * kRows > least) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) if (i >= seen) s[i] = -INFINITY;
                }
                float mx[4] = {max2(s[0], s[1]), max2(s[2], s[3]), max2(s[4], s[5]), max2(s[6], s[7])};
#pragma unroll
                for (int i = 8; i < 64; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], s[i], s[i + 1]);
                const float mn = max2(max2(mx[0], mx[1]), max2(mx[2], mx[3])) * unit;
                const bool grow = !(mn <= m + kGrow);
                float alpha = 1.0f;
                if (grow) { alpha = at::ex2(m - mn); l *= alpha; m = mn + (mn - mn); }       // an infinite maximum has no weights: NaN
                const float off = m == -INFINITY ? kLift : kLift - m;
                uint32_t pk[32], pl[X == 2 ? 32 : 1];
                uint64_t sum = 0;
                const uint64_t unit2 = pair_of_floats(unit, unit), off2 = pair_of_floats(off, off);
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const uint64_t x2 = fma2(pair_of_floats(s[i], s[i + 1]), unit2, off2);
                    float a, bb;
                    if (X == 0 && (i & 6) == 6) {                // a quarter by arithmetic: the exponential unit is what the rest waits for
                        ex2_pair(x2, a, bb);
                    } else {
                        a = at::ex2(low_of(x2));
                        bb = at::ex2(high_of(x2));
                    }
                    sum = add2(sum, pair_of_floats(a, bb));
                    pk[i >> 1] = half_pair(a, bb);
                    if constexpr (X == 2) {
                        const float2 r = Num<__half>::two(pk[i >> 1]);
                        pl[i >> 1] = half_pair(a - r.x, bb - r.y);
                    }
                }
                l += low_of(sum) + high_of(sum);
                if (j > 0 && __any_sync(0xffffffffu, grow)) {    // O once P V of the page before is through
                    if (!warp_wait<POLLS>(o_done + 8 * (buf ^ 1), (uint32_t)((mine + j - 1) >> 1) & 1u, abort_s)) { *abort_s = 1; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                    for (int d = 0; d < D; d += 32) {
                        uint32_t y[32];
                        tc::tmem_ld32(o_at + d, y);
#pragma unroll
                        for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * alpha);
                        tmem_st32(o_at + d, y);
                    }
                }
                tmem_st32(s_at, pk);
                if constexpr (X == 2) tmem_st32(s_at + 32, pl);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                warp_arrive(p_full + 8 * buf);
            }
            before += x.n;
            mine += x.n;
            ok = j == x.n && warp_wait<POLLS>(o_done + 8 * (t * 2 + ((mine - 1) & 1)), (uint32_t)((mine - 1) >> 1) & 1u, abort_s);
            if (!ok) { *abort_s = 1; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int head = x.h * group + row % group;
            if (x.from_start && x.to_end) {
                const float inv = l > 0.f ? 1.0f / l : l != l ? l : 0.f;
                T* out = (T*)p.out + ((size_t)(x.e.row0 + row / group) * c.q_heads + head) * D;
#pragma unroll 1
                for (int d = 0; d < D; d += 32) {
                    uint32_t y[32];
                    tc::tmem_ld32(o_at + d, y);
                    if (have)
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint32_t z[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) z[k] = within2<T>(__uint_as_float(y[i + 2 * k]) * inv, __uint_as_float(y[i + 2 * k + 1]) * inv);
                            *reinterpret_cast<uint4*>(out + d + i) = make_uint4(z[0], z[1], z[2], z[3]);
                        }
                }
                if (have && p.stats != nullptr) p.stats[stat_row(c, p, x.e, x.b, row / group, head)] = make_float2(m == -INFINITY ? m : m - kLift, l);
            } else {                                             // [piece][channels / 4][256 rows][4]: neighbouring lanes side by side
                const size_t piece = (size_t)(2 * blockIdx.x + (x.from_start ? 1 : 0));
                float4* to = reinterpret_cast<float4*>(p.many_part) + piece * (D / 4) * kManyRows + t * kTileRows + tr;
#pragma unroll 1
                for (int d = 0; d < D; d += 32) {
                    uint32_t y[32];
                    tc::tmem_ld32(o_at + d, y);
                    if (have)
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            to[(d + i) / 4 * kManyRows] = make_float4(__uint_as_float(y[i]), __uint_as_float(y[i + 1]), __uint_as_float(y[i + 2]), __uint_as_float(y[i + 3]));
                }
                if (have) p.many_stats[piece * kManyRows + t * kTileRows + tr] = make_float2(m, l);
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");     // the next piece's products go where these were read
        }
    } else if (warp < 12) {
        const int dt = tid - 8 * 32;
        auto wait = [&](uint32_t bar, uint32_t parity) { return warp_wait<POLLS>(bar, parity, abort_s); };
        auto convert = [&](auto values, int j, uint32_t full) {  // K or V of page j, by all four warps
            constexpr bool V = decltype(values)::value;
            const uint8_t* page = sm + C::RAW_AT + (j % C::RAW) * L::BYTES;
            const int valid = valid_s[j & 7];
            unsigned char* to = sm + (V ? C::V_AT + (j % C::VS) * C::VB : C::K_AT + (j % C::KS) * C::KB);
            const uint32_t* codes = reinterpret_cast<const uint32_t*>(page + (V ? L::V_CODES : L::K_CODES));
            const __half2* pars = reinterpret_cast<const __half2*>(page + (V ? L::V_PARAMS : L::K_PARAMS));
            __half2 par[2][G];
            bool wide = false;
#pragma unroll
            for (int it = 0; it < 2; ++it)
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const int r = it * 32 + (dt >> 2);
                    par[it][g] = pars[r * G + g];
                    if (r >= valid) par[it][g] = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
                    wide = wide || wide_range(par[it][g]);
                }
            auto words = [&](auto by_fp32) {
#pragma unroll
                for (int it = 0; it < 2; ++it) {
                    const int r = it * 32 + (dt >> 2), x = dt & 3;               // row, quarter of its groups
                    uint32_t w[G][2];
                    quarter_words<D, V>(codes, r, x, w);
#pragma unroll
                    for (int g = 0; g < G; ++g)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            uint4* dst = reinterpret_cast<uint4*>(to + g * (kRows * 128) + r * 128 + (((2 * x + i) ^ (r & 7)) << 4));
                            constexpr bool pair = V ? X == 2 : X >= 1;
                            uint4 high, low;
                            if constexpr (decltype(by_fp32)::value) wide_values(w[g][i], par[it][g], high, low);
                            else if constexpr (pair) half_pairs(w[g][i], par[it][g], high, low);
                            else high = half_values(w[g][i], par[it][g]);
                            *dst = high;
                            if constexpr (pair) dst[C::LOW / 16] = low;
                        }
                }
            };
            if (!__any_sync(0xffffffffu, wide)) words(std::false_type());
            else words(std::true_type());
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            warp_arrive(full);
        };
        int i = 0;
        for (; i < pages + C::LEAD; ++i) {
            if (i < pages) {
                if (!wait(raw_full + 8 * (i % C::RAW), (uint32_t)(i / C::RAW) & 1u)) break;
                if (i >= C::KS && !wait(k_empty + 8 * (i % C::KS), (uint32_t)(i / C::KS - 1) & 1u)) break;
                convert(std::false_type(), i, k_full + 8 * (i % C::KS));
            }
            const int j = i - C::LEAD;
            if (j < 0) continue;
            if (j >= C::VS && !wait(v_empty + 8 * (j % C::VS), (uint32_t)(j / C::VS - 1) & 1u)) break;
            convert(std::true_type(), j, v_full + 8 * (j % C::VS));
            warp_arrive(raw_empty + 8 * (j % C::RAW));
        }
        if (i < pages + C::LEAD) *abort_s = 1;
    } else if (warp == 14) {
        bool ok = true;
        int j = 0;
        while (ok && walk.more()) {
            const ManyPiece x = walk.next(c, p);
            const int held = (x.e.len + kRows - 1) / kRows;      // pages; a row that sees nothing has one that is nobody's
            int lane_page = -1;
            for (int i = 0; i < x.n; ++i, ++j) {
                if ((i & 31) == 0) {                             // a lane knows one page of 32
                    const bool in = i + lane < x.n && x.p0 + i + lane < held;
                    lane_page = in ? c.page_table[(size_t)x.b * c.max_pages + x.p0 + i + lane] : -1;
                    if ((unsigned)lane_page >= (unsigned)c.n_pages) { if (in) raise(c, kBadPage); lane_page = -1; }
                }
                const int page = __shfl_sync(0xffffffffu, lane_page, i & 31);
                const uint32_t bar = raw_full + 8 * (j % C::RAW);
                if (j >= C::RAW && !warp_wait<POLLS>(raw_empty + 8 * (j % C::RAW), (uint32_t)(j / C::RAW - 1) & 1u, abort_s)) { *abort_s = 1; ok = false; break; }
                if (lane == 0) {
                    valid_s[j & 7] = page >= 0 ? min(kRows, x.e.len - (x.p0 + i) * kRows) : 0;
                    if (page >= 0) {
                        tc::mbar_expect_tx(bar, L::BYTES);
                        bulk_copy(base + C::RAW_AT + (j % C::RAW) * L::BYTES, tile_of<D>(c, page, x.h), L::BYTES, bar);
                    } else {
                        mbar_arrive(bar);
                    }
                }
                __syncwarp();
            }
        }
        if (lane == 0) asked_s[2] = j;
    } else {
        // The whole warp walks the loop, so that addresses and descriptors stay in uniform registers; one lane issues.
        constexpr uint32_t kDescS = at::instr_desc_f16(kTileRows, kRows), kDescO = at::instr_desc_f16(kTileRows, D) | (1u << 16);
        const int t = warp - 12;
        const uint32_t lead = elect_one();
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t qt = tc::umma_desc(base + C::Q_AT + t * C::Q_BYTES), kd = tc::umma_desc(base + C::K_AT), vd = at::umma_desc_mn(base + C::V_AT, (uint32_t)(kRows * 128), 1024u);
        const uint32_t s0 = tm + (uint32_t)(C::S_COL + t * 128), to = tm + (uint32_t)(C::O_COL + t * 128);
        int before = 0, mine = 0, begun = 0, asked = 0;          // pages of the pieces before, of all and of this tile; its pieces; copies of queries
        auto issue_s = [&](int j) {                              // of page j of the piece, into the buffer of the tile's page's parity
            if (lead) {
                const int k_slot = (before + j) % C::KS, buf = (mine + j) & 1;
                const uint64_t kt = kd + (uint64_t)(k_slot * (C::KB >> 4));
                const uint32_t s_to = s0 + (uint32_t)(buf * 64);
#pragma unroll
                for (int i = 0; i < (X >= 1 ? 2 : 1) * (D / 16); ++i) {
                    const int k = i % (D / 16), low = i / (D / 16);
                    at::umma_d(s_to, qt + (uint64_t)((k >> 2) * (kTileRows * 128 >> 4) + (k & 3) * 2), kt + (uint64_t)((low * C::LOW + (k >> 2) * (kRows * 128)) / 16 + (k & 3) * 2), kDescS, i != 0 ? 1u : 0u);
                }
                tc::umma_commit(s_full + 8 * (t * 2 + buf));
                tc::umma_commit(k_empty + 8 * k_slot);
            }
            __syncwarp();
        };
        auto wait = [&](uint32_t bar, uint32_t parity) { return warp_wait<POLLS>(bar, parity, abort_s); };
        auto k_of = [&](int j) { return Phase{k_full + 8 * ((before + j) % C::KS), (uint32_t)((before + j) / C::KS) & 1u}; };
        auto v_of = [&](int j) { return Phase{v_full + 8 * ((before + j) % C::VS), (uint32_t)((before + j) / C::VS) & 1u}; };
        auto wait_k = [&](int j) { return wait(k_of(j).bar, k_of(j).parity); };
        auto wait_v = [&](int j) { return wait(v_of(j).bar, v_of(j).parity); };
        auto ask = [&](const ManyPiece& x) {                     // the tile's queries, once no product reads those before
            if (t < x.tiles && lane == 0) {
                tc::mbar_expect_tx(q_full + 8 * t, C::Q_BYTES);
                bulk_copy(base + C::Q_AT + t * C::Q_BYTES, p.images + row_tile(c, p, x.e, x.b, x.h, x.r0 / kTileRows + t) * C::Q_BYTES, C::Q_BYTES, q_full + 8 * t);
            }
            asked += t < x.tiles ? 1 : 0;
            __syncwarp();
        };
        bool ok = true, more = true;
        ManyPiece x = walk.next(c, p);
        ask(x);
        while (ok && more) {
            ManyPiece y = x;
            more = walk.more();
            if (more) y = walk.next(c, p);
            if (t < x.tiles) {
                ok = wait(q_full + 8 * t, (uint32_t)(begun++) & 1u);
                for (int j = 0; j < min(x.n, 2) && ok; ++j) {
                    ok = wait_k(j);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    issue_s(j);
                }
                for (int j = 0; j < x.n && ok; ++j) {
                    const int buf = (mine + j) & 1;
                    const Phase weights{p_full + 8 * (t * 2 + buf), (uint32_t)((mine + j) >> 1) & 1u};
                    ok = warp_wait<POLLS>(v_of(j), j + 2 < x.n ? k_of(j + 2) : weights, weights, abort_s);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (j == x.n - 1 && more) ask(y);            // weights of the last page: all scores are through
                    if (lead) {
                        const int v_slot = (before + j) % C::VS;
                        const uint64_t vt = vd + (uint64_t)(v_slot * (C::VB >> 4));
                        const uint32_t from = s0 + (uint32_t)(buf * 64);
#pragma unroll
                        for (int i = 0; i < (X == 2 ? 3 : 1) * (kRows / 16); ++i) {
                            const int k = i % (kRows / 16), part = i / (kRows / 16);                       // Ph Vh, Pl Vh, Ph Vl
                            at::umma_ts(to, from + (uint32_t)((part == 1 ? 32 : 0) + 8 * k), vt + (uint64_t)((part == 2 ? C::LOW : 0) / 16 + k * (2048 >> 4)), kDescO, i != 0 || j > 0 ? 1u : 0u);
                        }
                        tc::umma_commit(o_done + 8 * (t * 2 + buf));
                        tc::umma_commit(v_empty + 8 * v_slot);
                    }
                    __syncwarp();
                    if (j + 2 < x.n) issue_s(j + 2);             // behind P V, which reads the weights in that place
                }
                mine += x.n;
            } else {                                             // no rows in this tile: keys and values are let go as they come
                if (more) ask(y);
                for (int j = 0; j < x.n && ok; ++j) {
                    ok = wait_k(j);
                    if (ok && lead) mbar_arrive(k_empty + 8 * ((before + j) % C::KS));
                    ok = ok && wait_v(j);
                    if (ok && lead) mbar_arrive(v_empty + 8 * ((before + j) % C::VS));
                    __syncwarp();
                }
            }
            before += x.n;
            x = y;
        }
        if (!ok) *abort_s = 1;
        if (lane == 0) asked_s[t] = asked;
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*abort_s != 0) {                                         // given up: products and copies on their way end before the block leaves (bounded)
        volatile int go_on = 0;
        if (warp == 12 || warp == 13) {
            const int t = warp - 12, asked = asked_s[t];
            if (elect_one()) tc::umma_commit(drain + 8 * t);     // the lane that issued the products
            __syncwarp();
            (void)tc::mbar_wait(drain + 8 * t, 0, &go_on);
            if (asked > 0) (void)tc::mbar_wait(q_full + 8 * t, (uint32_t)(asked - 1) & 1u, &go_on);
        } else if (warp == 14) {
            const int asked = asked_s[2];
            for (int j = max(0, asked - C::RAW); j < asked; ++j) (void)tc::mbar_wait(raw_full + 8 * (j % C::RAW), (uint32_t)(j / C::RAW) & 1u, &go_on);
        }
        if (tid == 0) { raise(c, kWait); p.lost[p.few_blocks + blockIdx.x] = 1; }
    }
    __syncthreads();
    if (warp == 12) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Rows whose pages attend_many dealt over several blocks: maximum, sum and values of their pieces put together.  Block (w - 1, s) looks at
// the boundary ahead of block w; if that is the first one inside a block of rows it joins 16 channels of those, a thread a row.  Bound: 39 MB of
// pieces through L2 where every block leaves two; 8 us behind its predecessor.
// grid (blocks of attend_many - 1, D / 16).
template <typename T, int D>
__global__ void __launch_bounds__(kManyRows) attend_join_kernel(const Cache c, const AttnParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int pairs = c.batch * p.many_tiles, all = p.many_starts[pairs], step = many_step(p, all, 0), w = blockIdx.x + 1, group = c.q_heads / c.kv_heads;
    if (p.many_starts[pairs + 1] > 0) return;                    // they stayed whole
    const int64_t u = (int64_t)w * step;
    if (u >= all) return;
    const int pair = pair_of(p.many_starts, pairs, 0, (int)u), b = pair / p.many_tiles, tile = pair - b * p.many_tiles;
    const Entry e = entry_of(c, p, b);
    const int each = many_pages(p, e, group, tile), in = (int)u - p.many_starts[pair], h = in / each, at = (int)u - (in - h * each);       // at: the rows' first unit
    const int row = tile * kManyRows + threadIdx.x, i = row / group, head = h * group + row - i * group;
    if (at == u || at < (w - 1) * step || row >= e.n * group) return;
    const int last = (at + each - 1) / step;                     // blocks w - 1 .. last
    auto slot = [&](int k) { return (size_t)(2 * k + (k == w - 1 ? 1 : 0)); };
    const float2* stats = p.many_stats + threadIdx.x;
    float top = -INFINITY, sum = 0.f;
    for (int k = w - 1; k <= last; ++k) top = fmaxf(top, stats[slot(k) * kManyRows].x);
    float v[16];
#pragma unroll
    for (int d = 0; d < 16; ++d) v[d] = 0.f;
    const float4* part = reinterpret_cast<const float4*>(p.many_part) + (size_t)blockIdx.y * 4 * kManyRows + threadIdx.x;
    for (int k = w - 1; k <= last; ++k) {
        const float2 s = stats[slot(k) * kManyRows];
        const float f = s.x == -INFINITY && s.y == s.y ? 0.f : at::ex2(s.x - top);           // a sum that is no number stays one
        const float4* from = part + slot(k) * (D / 4) * kManyRows;
        sum = fmaf(s.y, f, sum);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 y = from[q * kManyRows];
            v[4 * q] = fmaf(y.x, f, v[4 * q]);
            v[4 * q + 1] = fmaf(y.y, f, v[4 * q + 1]);
            v[4 * q + 2] = fmaf(y.z, f, v[4 * q + 2]);
            v[4 * q + 3] = fmaf(y.w, f, v[4 * q + 3]);
        }
    }
    const float inv = sum > 0.f ? 1.0f / sum : sum != sum ? sum : 0.f;
    uint32_t z[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) z[d] = within2<T>(v[2 * d] * inv, v[2 * d + 1] * inv);
    uint4* out = reinterpret_cast<uint4*>((T*)p.out + ((size_t)(e.row0 + i) * c.q_heads + head) * D + blockIdx.y * 16);
    out[0] = make_uint4(z[0], z[1], z[2], z[3]);
    out[1] = make_uint4(z[4], z[5], z[6], z[7]);
    if (blockIdx.y == 0 && p.stats != nullptr) p.stats[stat_row(c, p, e, b, i, head)] = make_float2(top == -INFINITY ? top : top - kLift, sum);
}

template <int D>
struct WeightsCfg {
    static constexpr int G = D / 64, KEYS = 128, ROWS = 128, K_PART = Tile<D>::V_CODES;       // keys of a block, packed rows of a step; codes and parameters of a page's keys
    static constexpr int K_BYTES = KEYS * 128 * G, Q_BYTES = ROWS * 128 * G;                 // K: of its high and of its low half
    static constexpr int K_AT = 0, Q_AT = 2 * K_BYTES, PAR_AT = Q_AT + 2 * Q_BYTES, SUM_AT = PAR_AT + 2 * 3 * ROWS * 4, RAW_AT = SUM_AT + KEYS * 4, BARS = RAW_AT + 2 * K_PART;
    static constexpr size_t SMEM = BARS + 112 + 1024;
};
constexpr int kWeightThreads = 13 * 32;

// Summed weights where scores were not kept: S^T = K Q^T once more, 128 keys against 128 packed rows at a time, keys as a pair high + low of
// fp16 so that scores have 32-bit accuracy.  A key is a lane of tensor memory and two threads of warps 0-7, each of which adds up its weights
// 2^(s - m - log2 l) over half the rows of a step, in order: no atomics, no shuffles.  Warps 8-11 bring the rows' operand and (unit, m + log2 l),
// warp 12 issues the products.
// grid (blocks of 128 cached rows, kv heads, batch).  Bound: exponentials and tensor pipe alike (1024 cycles a step each, of 1500 - 1600), and
// 4 us of a block's life before its first step.  16 sequences of 1 .. 256 rows on up to 2056, 16 heads on 2 of 128: 43 us.  Two blocks an SM
// with one buffer for the rows: 54.
template <typename T, int D, int POLLS = kPolls>
__global__ void __launch_bounds__(kWeightThreads, 1) attend_weights_kernel(const Cache c, const AttnParams p) {
    using C = WeightsCfg<D>;
    using L = Tile<D>;
    constexpr int G = C::G;
    extern __shared__ unsigned char weights_smem[];
    const uint32_t raw_base = tc::smem_u32(weights_smem), base = (raw_base + 1023u) & ~1023u;
    unsigned char* sm = weights_smem + (base - raw_base);
    const uint32_t bars = base + C::BARS, raw_full = bars, q_full = bars + 8, q_empty = bars + 24, s_full = bars + 40, s_empty = bars + 56, drain = bars + 72, k_full = bars + 80;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::BARS + 88);
    volatile int *abort_s = reinterpret_cast<volatile int*>(tmem_slot + 1), *brought_s = abort_s + 1;      // brought_s: steps that warps 8-11 have brought
    const int tid = threadIdx.x, warp = tid >> 5, h = blockIdx.y, b = blockIdx.z, group = c.q_heads / c.kv_heads, key0 = blockIdx.x * C::KEYS;

    pdl_wait();                                                  // lengths, pages and keys are what earlier launches wrote
    const Entry e = entry_of(c, p, b);
    if (key0 >= e.len) return;
    bool lost = false;
    for (int i = tid; i < p.n_lost && tid < 256; i += 256) lost = lost || p.lost[i] != 0;
    int page[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) page[i] = key0 + i * kRows < e.len ? page_of(c, b, key0 / kRows + i) : -1;
    if (tid == 0) {
        tc::mbar_init(raw_full, 1);
        tc::mbar_init(k_full, 8);
        tc::mbar_init(drain, 1);
        for (int i = 0; i < 2; ++i) { tc::mbar_init(q_full + 8 * i, 5); tc::mbar_init(q_empty + 8 * i, 1); tc::mbar_init(s_full + 8 * i, 1); tc::mbar_init(s_empty + 8 * i, 8); }
        *abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        const int there = (page[0] >= 0) + (page[1] >= 0);
        if (there > 0) tc::mbar_expect_tx(raw_full, there * C::K_PART); else mbar_arrive(raw_full);
        for (int i = 0; i < 2; ++i)
            if (page[i] >= 0) bulk_copy(base + C::RAW_AT + i * C::K_PART, tile_of<D>(c, page[i], h), C::K_PART, raw_full);
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(tmem_slot)), "r"(256) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();                                     // not before this block has its tensor memory
    if (warp < 8) {                                              // the keys, while the other warps fetch rows
        const bool came = warp_wait<POLLS>(raw_full, 0, abort_s);
        if (!came) *abort_s = 1;
        __half2 par[2][G];
        bool wide = false;
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int r = it * 64 + (tid >> 2);              // row of the block
                const bool have = came && page[it] >= 0 && key0 + r < e.len;
                par[it][g] = have ? reinterpret_cast<const __half2*>(sm + C::RAW_AT + it * C::K_PART + L::K_PARAMS)[r % kRows * G + g] : __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
                wide = wide || wide_range(par[it][g]);
            }
        auto words = [&](auto by_fp32) {
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                const int r = it * 64 + (tid >> 2), x = tid & 3;                 // quarter of its groups
                uint32_t w[G][2];
                quarter_words<D, false>(reinterpret_cast<const uint32_t*>(sm + C::RAW_AT + it * C::K_PART + L::K_CODES), r % kRows, x, w);
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint4* dst = reinterpret_cast<uint4*>(sm + C::K_AT + g * (C::KEYS * 128) + r * 128 + (((2 * x + i) ^ (r & 7)) << 4));
                        uint4 high, low;
                        if constexpr (decltype(by_fp32)::value) wide_values(w[g][i], par[it][g], high, low);
                        else half_pairs(w[g][i], par[it][g], high, low);
                        dst[0] = high;
                        dst[C::K_BYTES / 16] = low;
                    }
            }
        };
        if (!__any_sync(0xffffffffu, wide)) words(std::false_type());
        else words(std::true_type());
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        warp_arrive(k_full);
    }

    const int rows = e.n * group, first_row = max(0, key0 - (e.len - e.n)) * group / C::ROWS * C::ROWS;       // rows before do not see the block
    const int n = rows > first_row ? (rows - first_row + C::ROWS - 1) / C::ROWS : 0;
    auto wait = [&](uint32_t bar, uint32_t parity) { return warp_wait<POLLS>(bar, parity, abort_s); };
    if (warp < 8) {
        const int key = key0 + (tid & 127), half = warp >> 2;         // which half of a step's rows
        uint64_t sum[2] = {0, 0};
        int i = 0;
        for (; i < n; ++i) {
            const int st = i & 1, r0 = first_row + i * C::ROWS;
            if (!wait(s_full + 8 * st, (uint32_t)(i >> 1) & 1u)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float* par = reinterpret_cast<const float*>(sm + C::PAR_AT) + st * 3 * C::ROWS;      // [unit | -m - log2 l | rows seen][row]
            const bool interior = e.len - e.n + r0 / group >= key0 + C::KEYS - 1;          // the step's first row sees every key
            {
                const int q = half * 64;
                float s[64];
                tmem_ld64(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(st * C::ROWS + q), s);
                if (!interior) {
#pragma unroll
                    for (int k = 0; k < 64; ++k) if (key >= reinterpret_cast<const int*>(par)[2 * C::ROWS + q + k]) s[k] = -INFINITY;
                }
#pragma unroll
                for (int k = 0; k < 64; k += 4) {
                    const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(par + q + k), m = *reinterpret_cast<const ulonglong2*>(par + C::ROWS + q + k);
                    const uint64_t x = fma2(pair_of_floats(s[k], s[k + 1]), u.x, m.x), y = fma2(pair_of_floats(s[k + 2], s[k + 3]), u.y, m.y);
                    sum[0] = add2(sum[0], pair_of_floats(at::ex2(low_of(x)), at::ex2(high_of(x))));
                    sum[1] = add2(sum[1], pair_of_floats(at::ex2(low_of(y)), at::ex2(high_of(y))));
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            warp_arrive(s_empty + 8 * st);
        }
        if (i < n || lost) *abort_s = 1;                         // lost: not all rows' sums were there
        float* other = reinterpret_cast<float*>(sm + C::SUM_AT);
        const float mine = (low_of(sum[0]) + high_of(sum[0])) + (low_of(sum[1]) + high_of(sum[1]));
        if (half == 1) other[tid & 127] = mine;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const int pg = page[(tid & 127) >> 6];
        if (half == 0 && *abort_s == 0 && key < e.len && pg >= 0) {              // both halves, and the keys, were there
            const size_t at = row_slot(c, pg, h, key % kRows);
            p.mass_out[at] = p.mass_in[at] + (mine + other[tid]);
        }
    } else if (warp < 12) {
        const int tr = tid - 256;
        struct Row { float2 s; float unit; int seen; };
        auto look = [&](int i) {                                 // a row's parameters, a step ahead of their use
            const int row = first_row + i * C::ROWS + tr;
            const bool have = i < n && row < rows;
            const int qr = have ? row / group : 0, head = h * group + (have ? row - qr * group : 0);
            Row x;
            x.s = have ? p.stats[stat_row(c, p, e, b, qr, head)] : make_float2(-INFINITY, 0.f);
            x.unit = have ? p.units[row_tile(c, p, e, b, h, first_row / C::ROWS + i) * kTileRows + tr] : 1.0f;         // not 0: times -inf
            x.seen = min(e.len, e.len - e.n + qr + 1);
            return x;
        };
        Row x = look(0);
        int i = 0;
        for (; i < n; ++i) {
            const int st = i & 1;
            const Row now = x;
            x = look(i + 1);
            // the products and the sums of two steps before have read this place
            if (i >= 2 && !(wait(q_empty + 8 * st, (uint32_t)(i / 2 - 1) & 1u) && wait(s_empty + 8 * st, (uint32_t)(i / 2 - 1) & 1u))) break;
            if (tr == 0) {                                       // the operand as it is, the rows' parameters by these four warps
                tc::mbar_expect_tx(q_full + 8 * st, C::Q_BYTES);
                bulk_copy(base + C::Q_AT + st * C::Q_BYTES, p.images + row_tile(c, p, e, b, h, first_row / C::ROWS + i) * C::Q_BYTES, C::Q_BYTES, q_full + 8 * st);
            }
            const bool sees = now.s.x != -INFINITY;              // a row that sees nothing: weights of 0
            float* par = reinterpret_cast<float*>(sm + C::PAR_AT) + st * 3 * C::ROWS + tr;
            par[0] = now.unit;
            par[C::ROWS] = sees ? -now.s.x - log2f(now.s.y) : -INFINITY;
            reinterpret_cast<int*>(par)[2 * C::ROWS] = sees ? now.seen : 0;
            warp_arrive(q_full + 8 * st);
        }
        if (i < n) *abort_s = 1;
        if ((tid & 31) == 0) brought_s[warp - 8] = i;
    } else {
        constexpr uint32_t kDesc = at::instr_desc_f16(C::KEYS, C::ROWS);
        const uint32_t lead = elect_one(), tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t kd = tc::umma_desc(base + C::K_AT), qd = tc::umma_desc(base + C::Q_AT);
        bool ok = n == 0 || wait(k_full, 0);
        for (int i = 0; i < n && ok; ++i) {
            const int st = i & 1;
            ok = (i < 2 || wait(s_empty + 8 * st, (uint32_t)(i / 2 - 1) & 1u)) && wait(q_full + 8 * st, (uint32_t)(i >> 1) & 1u);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (lead) {
                const uint64_t qt = qd + (uint64_t)(st * (C::Q_BYTES >> 4));
#pragma unroll
                for (int k = 0; k < 2 * (D / 16); ++k) {
                    const int kk = k % (D / 16), low = k / (D / 16);
                    at::umma_d(tm + (uint32_t)(st * C::ROWS), kd + (uint64_t)((low * C::K_BYTES + (kk >> 2) * (C::KEYS * 128)) / 16 + (kk & 3) * 2), qt + (uint64_t)((kk >> 2) * (C::ROWS * 128 >> 4) + (kk & 3) * 2),
                               kDesc, k != 0 ? 1u : 0u);
                }
                tc::umma_commit(s_full + 8 * st);
                tc::umma_commit(q_empty + 8 * st);
            }
            __syncwarp();
        }
        if (!ok) *abort_s = 1;
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*abort_s != 0) {                                         // given up: products and copies on their way end before the block leaves (bounded)
        volatile int go_on = 0;
        const int brought = brought_s[0];                        // warp 8 asked for the rows; the other three arrive for the steps that they did not come to
        if (warp > 8 && warp < 12 && (tid & 31) == 0)
            for (int i = brought_s[warp - 8]; i < brought; ++i) mbar_arrive(q_full + 8 * (i & 1));
        if (warp == 8)
            for (int i = max(0, brought - 2); i < brought; ++i) (void)tc::mbar_wait(q_full + 8 * (i & 1), (uint32_t)(i >> 1) & 1u, &go_on);
        if (warp == 12) {
            if (elect_one()) tc::umma_commit(drain);             // the lane that issued the products
            __syncwarp();
            (void)tc::mbar_wait(drain, 0, &go_on);
        }
        if (tid == 0) {
            (void)tc::mbar_wait(raw_full, 0, &go_on);
            raise(c, kWait);
        }
    }
    __syncthreads();
    if (warp == 12) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
    }
}

}  // namespace kv4
}  // namespace efm
