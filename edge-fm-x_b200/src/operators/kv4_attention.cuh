// Attention over a 4-bit cache (kv4_cache.cuh).
#pragma once
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
    float2* stats;            // [max_rows, q_heads] (maximum, 1 / sum) of a row's weights
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

template <typename T>
__device__ __forceinline__ float value_at(uint32_t w, int i, __half2 par) {
    return fmaf(__low2float(par), (float)((w >> (4 * nibble(i))) & 15u), __high2float(par));
}

// A block per (new row, q head): one warp takes every fourth key.
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_plain_kernel(const Cache c, const AttnParams p) {
    using L = Tile<D>;
    constexpr int E = D / 32;
    __shared__ float part[4][D + 2];
    const int i = blockIdx.x, hq = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Entry e = entry_of(c, p, b);
    if (i >= e.n) return;
    const int h = hq / (c.q_heads / c.kv_heads), see = min(e.len, e.len - e.n + i + 1);
    const T* q = (const T*)p.q + ((size_t)(e.row0 + i) * c.q_heads + hq) * D + lane * E;
    float x[E], o[E];
#pragma unroll
    for (int k = 0; k < E; ++k) { x[k] = (float)q[k] * p.scale_log2; o[k] = 0.f; }
    float m = -INFINITY, l = 0.f;
    const int w = lane * E / 8, i0 = lane * E & 7, g = lane * E / kGroup;
    for (int row = warp; row < see; row += 4) {
        const int page = page_of(c, b, row / kRows), r = row % kRows;
        if (page < 0) continue;
        const uint8_t* tile = tile_of<D>(c, page, h);
        const uint32_t kw = reinterpret_cast<const uint32_t*>(tile + L::K_CODES)[r * L::WORDS + key_word<D>(w)];
        const uint32_t vw = reinterpret_cast<const uint32_t*>(tile + L::V_CODES)[r * L::WORDS + w];
        const __half2 kp = reinterpret_cast<const __half2*>(tile + L::K_PARAMS)[r * L::G + g], vp = reinterpret_cast<const __half2*>(tile + L::V_PARAMS)[r * L::G + g];
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < E; ++k) s = fmaf(x[k], value_at<T>(kw, i0 + k, kp), s);
        s = warp_sum(s);
        const float mn = fmaxf(m, s), a = exp2f(m - mn), pr = exp2f(s - mn);
        l = l * a + pr;
#pragma unroll
        for (int k = 0; k < E; ++k) o[k] = fmaf(o[k], a, pr * value_at<T>(vw, i0 + k, vp));
        m = mn;
    }
#pragma unroll
    for (int k = 0; k < E; ++k) part[warp][lane * E + k] = o[k];
    if (lane == 0) { part[warp][D] = m; part[warp][D + 1] = l; }
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int k = 0; k < 4; ++k) top = fmaxf(top, part[k][D]);
    const float safe = top == -INFINITY ? 0.f : top;
    for (int k = 0; k < 4; ++k) sum += part[k][D + 1] * exp2f(part[k][D] - safe);
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    for (int d = threadIdx.x; d < D; d += 128) {
        float v = 0.f;
        for (int k = 0; k < 4; ++k) v += part[k][d] * exp2f(part[k][D] - safe);
        ((T*)p.out)[((size_t)(e.row0 + i) * c.q_heads + hq) * D + d] = (T)(v * inv);
    }
    if (p.stats != nullptr && threadIdx.x == 0) p.stats[(size_t)(e.row0 + i) * c.q_heads + hq] = make_float2(safe, inv);
}

// A warp per cached row: its weights of all new rows and of the q heads of its kv head.
template <typename T, int D>
__global__ void __launch_bounds__(256) mass_plain_kernel(const Cache c, const AttnParams p) {
    using L = Tile<D>;
    constexpr int E = D / 32;
    const int h = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = c.q_heads / c.kv_heads;
    const Entry e = entry_of(c, p, b);
    const int row = blockIdx.x * 8 + warp;
    if (row >= e.len) return;
    const int page = page_of(c, b, row / kRows), r = row % kRows;
    if (page < 0) return;
    const uint8_t* tile = tile_of<D>(c, page, h);
    const int w = lane * E / 8, i0 = lane * E & 7, g = lane * E / kGroup;
    const uint32_t kw = reinterpret_cast<const uint32_t*>(tile + L::K_CODES)[r * L::WORDS + key_word<D>(w)];
    const __half2 kp = reinterpret_cast<const __half2*>(tile + L::K_PARAMS)[r * L::G + g];
    float k[E], sum = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) k[j] = value_at<T>(kw, i0 + j, kp) * p.scale_log2;
    for (int i = max(0, row - (e.len - e.n)); i < e.n; ++i)
        for (int j = 0; j < group; ++j) {
            const size_t at = (size_t)(e.row0 + i) * c.q_heads + h * group + j;
            const T* q = (const T*)p.q + at * D + lane * E;
            float s = 0.f;
#pragma unroll
            for (int d = 0; d < E; ++d) s = fmaf((float)q[d], k[d], s);
            const float2 st = p.stats[at];
            sum += exp2f(warp_sum(s) - st.x) * st.y;
        }
    if (lane == 0) p.mass_out[row_slot(c, page, h, r)] = p.mass_in[row_slot(c, page, h, r)] + sum;
}

}  // namespace kv4
}  // namespace efm
