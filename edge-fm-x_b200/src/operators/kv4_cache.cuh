// A key/value cache in 4 bits (include/efm_b200_kv4.h has the layout): appending rows and reading them back.
//
// append: y = x r w with r = 1 / sqrt(mean(x^2) + eps), channels turned by their position's angle, q rounded once, k and v snapped to
// min + scale * code.  Codes are whole numbers, so what is done to x before them is fixed operation by operation (squares summed in
// 64 bits, every other product and sum rounded to 32 bits on its own, angles and their sine and cosine in 64 bits): the same input
// gives the same cache whatever the launch shape.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace efm {
namespace kv4 {

constexpr int kRows = 64, kGroup = 64;
constexpr int kBadPage = 1, kFull = 2, kBadCount = 4, kWait = 8;      // EFM_KV4_*

template <int D>
struct Tile {
    static constexpr int G = D / kGroup;                     // groups of a row
    static constexpr int CODES = kRows * D / 2, PARAMS = kRows * G * 4;
    static constexpr int K_CODES = 0, K_PARAMS = CODES, V_CODES = CODES + PARAMS, V_PARAMS = 2 * CODES + PARAMS;
    static constexpr int BYTES = 2 * (CODES + PARAMS);
    static constexpr int WORDS = D / 8;                      // 32-bit words of a row's codes
};

struct Cache {
    int q_heads, kv_heads, n_pages, batch, max_pages;
    uint8_t* pool;
    const int32_t* page_table;
    int32_t* status;
};

__device__ __forceinline__ void raise(const Cache& c, int bit) {
    if (c.status != nullptr) atomicOr(c.status, bit);
}
// Page that holds cache rows [64 k, 64 k + 64) of sequence b, -1 where its number is not one of the pool's.
__device__ __forceinline__ int page_of(const Cache& c, int b, int k) {
    const int p = c.page_table[(size_t)b * c.max_pages + k];
    if ((unsigned)p < (unsigned)c.n_pages) return p;
    raise(c, kBadPage);
    return -1;
}
template <int D>
__device__ __forceinline__ uint8_t* tile_of(const Cache& c, int page, int head) {
    return c.pool + ((size_t)page * c.kv_heads + head) * Tile<D>::BYTES;
}
__device__ __forceinline__ size_t row_slot(const Cache& c, int page, int head, int r) { return ((size_t)page * c.kv_heads + head) * kRows + r; }
__device__ __forceinline__ int held(const Cache& c, const int32_t* lens, int b, int most) {
    const int n = lens[b];
    if ((unsigned)n <= (unsigned)most) return n;
    raise(c, kBadCount);
    return n < 0 ? 0 : most;
}

// nibble of channel i of a word's eight
__host__ __device__ constexpr int nibble(int i) { return (i >> 1) + 4 * (i & 1); }
// word of a key row that holds channels 8 w .. 8 w + 7
template <int D>
__host__ __device__ constexpr int key_word(int w) { return (w & 7) / 2 * (2 * Tile<D>::G) + (w >> 3) * 2 + (w & 1); }

template <typename T> struct Num;
template <> struct Num<__nv_bfloat16> {
    static __device__ __forceinline__ float2 two(uint32_t v) { return make_float2(bf16lo(v), bf16hi(v)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
};
template <> struct Num<__half> {
    static __device__ __forceinline__ float2 two(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        __half2 p = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&p);
    }
};

// A held value as T: fp16 ends at 65504, which the rounding of minimum and scale may take a value 80 beyond.
template <typename T>
__device__ __forceinline__ float within(float x) {
    if constexpr (std::is_same<T, __half>::value) asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(65504.0f));
    return x;
}

template <typename T>
__device__ __forceinline__ uint32_t within2(float a, float b) { return Num<T>::pack(within<T>(a), within<T>(b)); }

struct AppendParams {
    int max_rows;
    const int32_t *cu_rows, *lens_in;
    int32_t* lens_out;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    int norm;
    float eps;
    const void *q_norm, *k_norm;
    int rot_dims, neighbours, axes, section0, section1;
    const double* inv_freq;
    const int32_t *positions, *token_index;
    void *q_out, *k_held, *v_held;
    int32_t* index;
    float* mass;
};

constexpr int kAppendThreads = 128;

// Channels turned: (a, b) -> (a cos - b sin, b cos + a sin), three roundings each.
__device__ __forceinline__ float turn(float a, float c, float b, float s, bool plus) {
    const float x = __fmul_rn(a, c), y = __fmul_rn(b, s);
    return plus ? __fadd_rn(x, y) : __fsub_rn(x, y);
}

// Codes of eight channels, rint((x - m) / s) in 0 .. 15, and the word they make.  By the reciprocal unless a quotient lies within its error
// of a border (product and reciprocal are off by 2^-22 together: 4e-6 at 16), where the divisions decide: IEEE divisions for all of them
// were half of the kernel's instructions.  Rounding by adding 1.5 * 2^23 leaves the code in the sum's low bits.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float m, float s, float (&code)[8]) {
    constexpr float kMagic = 12582912.0f;
    const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
    float near = 1.0f, r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        r[e] = fminf(fmaxf(__fmul_rn(__fsub_rn(x[e], m), inv), 0.0f), 15.25f);
        const float t = __fadd_rn(r[e], kMagic);
        code[e] = __fsub_rn(t, kMagic);
        near = fminf(near, fabsf(fabsf(__fsub_rn(r[e], code[e])) - 0.5f));
    }
    if (near < 1e-5f && s > 0.0f)
#pragma unroll
        for (int e = 0; e < 8; ++e) code[e] = rintf(fminf(fmaxf(__fdiv_rn(__fsub_rn(x[e], m), s), 0.0f), 15.25f));
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) word |= (__float_as_uint(__fadd_rn(code[e], kMagic)) & 15u) << (4 * nibble(e));
    return word;
}

// grid (rows, parts of the row's heads); a lane has eight neighbouring channels of a head (one word of codes), a warp 32 / (D / 8) heads
// of one kind at a time.
// Bound: instruction issue (77 % of the slots; 330 a warp and 32 / (D / 8) heads, most of them products and sums of single numbers), not bytes.  3117 rows
// of 32 + 16 heads of 128 fp16, normed and turned: 30 us, 2.7 TB/s of what has to move.  One row: latency, some 4 us.
template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const Cache c, const AppendParams p, int tasks_per_block) {
    constexpr int LANES = D / 8, HEADS = 32 / LANES;         // lanes of a head, heads of a warp
    using L = Tile<D>;
    __shared__ float2 rot[D / 2];
    __shared__ int place_s, page_s, falls_s;                 // cache row and page of the row; place -1: nobody's row; row counts fall somewhere
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane % LANES, c0 = sub * 8;
    const int cap = c.max_pages * kRows;
    const int tq = p.q != nullptr ? (c.q_heads + HEADS - 1) / HEADS : 0, tk = (c.kv_heads + HEADS - 1) / HEADS;
    const int last = min(tq + 2 * tk, ((int)blockIdx.y + 1) * tasks_per_block);
    auto kind_of = [&](int task) { return task < tq ? 0 : task < tq + tk ? 1 : 2; };      // q, k, v
    auto head_of = [&](int task) { return (task < tq ? task : task < tq + tk ? task - tq : task - tq - tk) * HEADS + lane / LANES; };
    auto fetch = [&](int task) {
        const int kind = kind_of(task), h = head_of(task);
        if (task >= last || h >= (kind == 0 ? c.q_heads : c.kv_heads)) return make_uint4(0u, 0u, 0u, 0u);
        const T* src = kind == 0 ? (const T*)p.q + row * p.q_stride : kind == 1 ? (const T*)p.k + row * p.k_stride : (const T*)p.v + row * p.v_stride;
        return *reinterpret_cast<const uint4*>(src + (size_t)h * D + c0);
    };
    if (tid == 0) { place_s = -1; falls_s = 0; }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    int task = blockIdx.y * tasks_per_block + warp;
    uint4 next = row < p.max_rows ? fetch(task) : make_uint4(0u, 0u, 0u, 0u);             // on its way while the row's place is looked up
    const bool tells = row == 0 && blockIdx.y == 0;
    bool full = false;
    auto look = [&](int b, int lo, int hi) {                 // rows [lo, hi) are sequence b's
        const bool mine = row >= lo && row < hi;
        if (!mine && !tells) return;
        const int have = held(c, p.lens_in, b, cap);
        if (tells) {
            p.lens_out[b] = min(cap - have, hi - lo) + have;
            full = full || hi - lo > cap - have;
        }
        if (mine) {
            const int64_t behind = have + ((int64_t)row - lo);
            place_s = behind < cap ? (int)behind : cap;
            page_s = behind < cap ? page_of(c, b, (int)behind / kRows) : -1;
        }
    };
    auto cut = [&](int at) { return min(max(at, 0), p.max_rows); };
    for (int b = tid; b < c.batch; b += kAppendThreads) {
        const int lo = p.cu_rows[b], hi = p.cu_rows[b + 1];
        if (hi < lo) falls_s = 1;
        if (tells && (lo < 0 || hi < lo || hi > p.max_rows)) raise(c, kBadCount);
        look(b, cut(lo), cut(hi));
    }
    const int half = p.rot_dims / 2;
    if (half > 0 && row < p.max_rows)
        for (int i = kAppendThreads - 1 - tid; i < half; i += kAppendThreads) {      // by the warps that do not look for the owner
            const int axis = p.axes == 1 || i < p.section0 ? 0 : i < p.section0 + p.section1 ? 1 : 2;
            double s, co;
            sincos((double)p.positions[(size_t)axis * p.max_rows + row] * p.inv_freq[i], &s, &co);
            rot[i] = make_float2((float)co, (float)s);
        }
    __syncthreads();
    if (falls_s) {                                           // counts that fall would give a row to several sequences: their running maximum counts
        full = false;
        if (tid == 0) {
            place_s = -1;
            for (int b = 0, lo = 0; b < c.batch; ++b) {
                lo = max(lo, cut(p.cu_rows[b]));
                const int hi = max(lo, cut(p.cu_rows[b + 1]));
                look(b, lo, hi);
                lo = hi;
            }
        }
        __syncthreads();
    }
    if (full) raise(c, kFull);
    if (place_s < 0) return;
    const int place = place_s, page = page_s, r = place % kRows;
    const bool turns = c0 < p.rot_dims, second = c0 >= half;
    const int partner = (lane & ~(LANES - 1)) + ((second ? sub - half / 8 : sub + half / 8) & (LANES - 1));
    for (; task < last; task += kAppendThreads / 32) {
        const int kind = kind_of(task), h = head_of(task), n_heads = kind == 0 ? c.q_heads : c.kv_heads;
        const bool have = h < n_heads;
        float x[8];
        {
            const uint32_t v[4] = {next.x, next.y, next.z, next.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) { const float2 f = Num<T>::two(v[k]); x[2 * k] = f.x; x[2 * k + 1] = f.y; }
        }
        next = fetch(task + kAppendThreads / 32);
        if (kind < 2 && p.norm) {
            double sq = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) sq += (double)x[e] * (double)x[e];
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
            const float f = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn((float)(sq / D), p.eps)));
            const T* w = (const T*)(kind == 0 ? p.q_norm : p.k_norm);
            uint4 ww = make_uint4(0u, 0u, 0u, 0u);
            if (w != nullptr) ww = *reinterpret_cast<const uint4*>(w + c0);
            const uint32_t v[4] = {ww.x, ww.y, ww.z, ww.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 g = Num<T>::two(v[k]);
                x[2 * k] = __fmul_rn(x[2 * k], f);
                x[2 * k + 1] = __fmul_rn(x[2 * k + 1], f);
                if (w != nullptr) { x[2 * k] = __fmul_rn(x[2 * k], g.x); x[2 * k + 1] = __fmul_rn(x[2 * k + 1], g.y); }
            }
        }
        if (kind < 2 && half > 0) {
            if (p.neighbours) {
                if (turns) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float2 cs = rot[(c0 + e) / 2];
                        const float u = x[e], w = x[e + 1];
                        x[e] = turn(u, cs.x, w, cs.y, false);
                        x[e + 1] = turn(w, cs.x, u, cs.y, true);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float o = __shfl_sync(0xffffffffu, x[e], partner);
                    if (turns) {
                        const float2 cs = rot[(second ? c0 - half : c0) + e];
                        x[e] = turn(x[e], cs.x, o, cs.y, second);
                    }
                }
            }
        }
        auto put = [&](void* out) {
            if (have)
                *reinterpret_cast<uint4*>((T*)out + ((size_t)row * n_heads + h) * D + c0) =
                    make_uint4(Num<T>::pack(x[0], x[1]), Num<T>::pack(x[2], x[3]), Num<T>::pack(x[4], x[5]), Num<T>::pack(x[6], x[7]));
        };
        if (kind == 0) { put(p.q_out); continue; }
        float lo = INFINITY, hi = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = x[e] != x[e] ? 0.0f : fminf(fmaxf(x[e], -65504.0f), 65504.0f);
            lo = fminf(lo, x[e]);
            hi = fmaxf(hi, x[e]);
        }
#pragma unroll
        for (int o = kGroup / 16; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const __half sh = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f)), mh = __float2half_rn(lo);
        const float s = __half2float(sh), m = __half2float(mh);
        float code[8];
        const uint32_t word = codes_of(x, m, s, code);
        void* want = kind == 1 ? p.k_held : p.v_held;
        if (want != nullptr) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = within<T>(__fadd_rn(m, __fmul_rn(s, code[e])));
            put(want);
        }
        if (page < 0 || !have) continue;
        uint8_t* tile = tile_of<D>(c, page, h);
        reinterpret_cast<uint32_t*>(tile + (kind == 1 ? L::K_CODES : L::V_CODES))[r * L::WORDS + (kind == 1 ? key_word<D>(sub) : sub)] = word;
        if (sub % 8 == 0) reinterpret_cast<__half2*>(tile + (kind == 1 ? L::K_PARAMS : L::V_PARAMS))[r * L::G + sub / 8] = __halves2half2(sh, mh);
        if (kind == 1 && sub == 0) {
            if (p.index != nullptr) p.index[row_slot(c, page, h, r)] = p.token_index != nullptr ? p.token_index[row] : place;
            if (p.mass != nullptr) p.mass[row_slot(c, page, h, r)] = 0.0f;
        }
    }
}

// What a word of codes stands for: eight channels, rounded once.
template <typename T>
__device__ __forceinline__ uint4 word_values(uint32_t w, __half2 par) {
    const float s = __low2float(par), m = __high2float(par);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = within<T>(__fadd_rn(m, __fmul_rn(s, (float)((w >> (4 * nibble(i))) & 15u))));
    return make_uint4(Num<T>::pack(x[0], x[1]), Num<T>::pack(x[2], x[3]), Num<T>::pack(x[4], x[5]), Num<T>::pack(x[6], x[7]));
}

constexpr int kReadThreads = 256;

// grid (pages of the range x kv heads, batch); a thread has one word of keys or values at a time, in the order of the output.
// Bound: bytes written.  64 sequences of 1024 rows, 4 kv heads of 128: 32 us, 5.4 TB/s; 8 of 1000 .. 1452, 2 heads, 8.1 us, 3.3 TB/s.
template <typename T, int D>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const Cache c, const int32_t* lens, int first, int rows, T* k_out, T* v_out) {
    using L = Tile<D>;
    constexpr int PER = kRows * L::WORDS / kReadThreads;
    const int b = blockIdx.y, h = blockIdx.x % c.kv_heads, k = first / kRows + blockIdx.x / c.kv_heads;
    pdl_wait();
    pdl_launch_dependents();
    const int n = min(held(c, lens, b, c.max_pages * kRows), first + rows);
    if (k * kRows >= n) return;
    const int page = page_of(c, b, k);
    if (page < 0) return;
    const uint8_t* tile = tile_of<D>(c, page, h);
    const uint32_t *kc = reinterpret_cast<const uint32_t*>(tile + L::K_CODES), *vc = reinterpret_cast<const uint32_t*>(tile + L::V_CODES);
    const __half2 *kp = reinterpret_cast<const __half2*>(tile + L::K_PARAMS), *vp = reinterpret_cast<const __half2*>(tile + L::V_PARAMS);
    uint32_t kw[PER], vw[PER];
    __half2 ks[PER], vs[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = i * kReadThreads + threadIdx.x, r = at / L::WORDS, w = at % L::WORDS;
        if (k_out != nullptr) { kw[i] = kc[r * L::WORDS + key_word<D>(w)]; ks[i] = kp[r * L::G + w / 8]; }
        if (v_out != nullptr) { vw[i] = vc[r * L::WORDS + w]; vs[i] = vp[r * L::G + w / 8]; }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = i * kReadThreads + threadIdx.x, r = at / L::WORDS, w = at % L::WORDS, row = k * kRows + r;
        if (row < first || row >= n) continue;
        const size_t dst = (((size_t)b * rows + (row - first)) * c.kv_heads + h) * D + w * 8;
        if (k_out != nullptr) *reinterpret_cast<uint4*>(k_out + dst) = word_values<T>(kw[i], ks[i]);
        if (v_out != nullptr) *reinterpret_cast<uint4*>(v_out + dst) = word_values<T>(vw[i], vs[i]);
    }
}

}  // namespace kv4
}  // namespace efm
