// Operators of the 4-bit key/value cache (include/efm_b200_kv4.h): checks of arguments, sizes, launches on the caller's stream.
#include <efm_b200_kv4.h>

#include <atomic>
#include <cstdlib>
#include <exception>

#include "../../operators/kv4_attention.cuh"
#include "../../operators/kv4_attention_tc.cuh"
#include "../../operators/kv4_cache.cuh"
#include "../../operators/kv4_evict.cuh"
#include "ctx_util.h"

namespace efm {
namespace {

using kv4::kRows;

efm_status bad(const char* call, const char* what) { return fail(nullptr, EFM_ERR_INVALID_ARGUMENT, std::string(call) + ": " + what); }
bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

efm_status check_cache(const char* call, const efm_kv4_cache* c) {
    if (c == nullptr || c->struct_size != (int32_t)sizeof(efm_kv4_cache)) return bad(call, "cache: struct_size does not match this header");
    if (c->dtype != EFM_BF16 && c->dtype != EFM_F16) return fail(nullptr, EFM_ERR_UNSUPPORTED, std::string(call) + ": dtype bf16 or fp16");
    if (c->head_dim != 64 && c->head_dim != 128) return fail(nullptr, EFM_ERR_UNSUPPORTED, std::string(call) + ": head_dim 64 or 128");
    if (c->kv_heads < 1 || c->q_heads < 1 || c->q_heads > 1024 || c->q_heads % c->kv_heads != 0) return bad(call, "q_heads a multiple of kv_heads, at most 1024");
    if (c->n_pages < 1 || c->n_pages > (1 << 24) || c->batch < 1 || c->batch > 65535 || c->max_pages < 1 || c->max_pages >= (1 << 24)) return bad(call, "n_pages, batch or max_pages out of range");
    return EFM_OK;
}
efm_status check_buffers(const char* call, const efm_kv4_cache* c) {
    if (c->pool == nullptr || c->page_table == nullptr || !aligned(c->pool, 16) || !aligned(c->page_table, 4) || !aligned(c->status, 4))
        return bad(call, "pool (16-byte aligned) and page_table are needed");
    return EFM_OK;
}

// The pool's GPU for the length of a call; what the thread had current comes back with it.
class OnDevice {
public:
    efm_status enter(const char* call, const void* pool) {
        cudaPointerAttributes at{};
        cudaError_t e = cudaPointerGetAttributes(&at, pool);
        if (e != cudaSuccess) { (void)cudaGetLastError(); return cuda_fail(nullptr, e, call); }
        if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) return bad(call, "pool is not device memory");
        e = cudaGetDevice(&before_);
        if (e == cudaSuccess && before_ != at.device) { e = cudaSetDevice(at.device); moved_ = e == cudaSuccess; }
        if (e != cudaSuccess) return cuda_fail(nullptr, e, call);
        device = at.device;
        return EFM_OK;
    }
    ~OnDevice() { if (moved_) (void)cudaSetDevice(before_); }
    int device = 0;

private:
    int before_ = 0;
    bool moved_ = false;
};

struct DeviceInfo { int sms = 0, smem = 0; };
constexpr int kEvictSmemReserve = 12 * 1024;          // static shared memory of the ordering kernel, rounded up

// Kernels whose waits give up after a few polls, for tests of what a call does then: EFM_B200_KV4_HASTY, a sum of 1 (attend_few), 2
// (attend_many) and 4 (attend_weights), looked at if it was there at the first call.
int hasty() {
    static const bool set = std::getenv("EFM_B200_KV4_HASTY") != nullptr;
    const char* e = set ? std::getenv("EFM_B200_KV4_HASTY") : nullptr;
    return e != nullptr ? std::atoi(e) : 0;
}
// Kernels of attention that wait inside.
template <typename T, int D>
struct AttendKernels {
    using Kernel = void (*)(const kv4::Cache, const kv4::AttnParams);
    static constexpr int X = std::is_same<T, __half>::value ? 2 : 0, XM = X == 0 ? 1 : 2;      // of attend_many without and with mass
    Kernel few1, few2, many, many_mass, weights;
    template <int POLLS>
    static AttendKernels of() {
        return {kv4::attend_few_kernel<T, D, 1, POLLS>, kv4::attend_few_kernel<T, D, 2, POLLS>, kv4::attend_many_kernel<T, D, X, POLLS>, kv4::attend_many_kernel<T, D, XM, POLLS>,
                kv4::attend_weights_kernel<T, D, POLLS>};
    }
    static AttendKernels now() {
        AttendKernels k = of<kv4::kPolls>();
        if constexpr (kHasHasty) {
            const AttendKernels h = of<kv4::kHasty>();
            const int which = hasty();
            if (which & 1) { k.few1 = h.few1; k.few2 = h.few2; }
            if (which & 2) { k.many = h.many; k.many_mass = h.many_mass; }
            if (which & 4) k.weights = h.weights;
        }
        return k;
    }
    cudaError_t more_smem() const {
        auto set = [](Kernel kernel, size_t bytes) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes); };
        cudaError_t e = set(few1, kv4::FewCfg<D, 1>::SMEM);
        if (e == cudaSuccess) e = set(few2, kv4::FewCfg<D, 2>::SMEM);
        if (e == cudaSuccess) e = set(weights, kv4::WeightsCfg<D>::SMEM);
        if (e == cudaSuccess) e = set(many, kv4::ManyCfg<D, X>::SMEM);
        if (e == cudaSuccess) e = set(many_mass, kv4::ManyCfg<D, XM>::SMEM);
        return e;
    }
    static constexpr bool kHasHasty = (X == 0 && D == 128) || (X == 2 && D == 64);             // forms that are enough for those tests
};
template <typename T, int D>
cudaError_t more_smem() {
    using K = AttendKernels<T, D>;
    cudaError_t e = K::template of<kv4::kPolls>().more_smem();
    if constexpr (K::kHasHasty) { if (e == cudaSuccess) e = K::template of<kv4::kHasty>().more_smem(); }
    return e;
}

// Once per device: architecture, sizes, shared memory beyond the default.
efm_status device_info(const char* call, int device, DeviceInfo& info) {
    static std::atomic<int64_t> known[64];
    if (device < 0 || device >= 64) return fail(nullptr, EFM_ERR_UNSUPPORTED, "device index above 63");
    int64_t k = known[device].load(std::memory_order_acquire);
    if (k == 0) {
        int major = 0, minor = 0, sms = 0, smem = 0;
        cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, device);
        if (e != cudaSuccess) return cuda_fail(nullptr, e, call);
        if (major != 10 || minor != 0) return fail(nullptr, EFM_ERR_CUDA, std::string(call) + ": needs an sm_100 device");
        e = cudaFuncSetAttribute(kv4::evict_select_kernel<kv4::kKeepMany>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem - kEvictSmemReserve);
        if (e == cudaSuccess) e = more_smem<__nv_bfloat16, 64>();
        if (e == cudaSuccess) e = more_smem<__nv_bfloat16, 128>();
        if (e == cudaSuccess) e = more_smem<__half, 64>();
        if (e == cudaSuccess) e = more_smem<__half, 128>();
        if (e != cudaSuccess) return cuda_fail(nullptr, e, call);
        k = ((int64_t)sms << 32) | smem;
        known[device].store(k, std::memory_order_release);
    }
    info.sms = (int)(k >> 32);
    info.smem = (int)(k & 0xffffffff);
    return EFM_OK;
}

kv4::Cache device_cache(const efm_kv4_cache* c) {
    return kv4::Cache{c->q_heads, c->kv_heads, c->n_pages, c->batch, c->max_pages, (uint8_t*)c->pool, c->page_table, c->status};
}

template <typename F>
void by_type(const efm_kv4_cache* c, F&& f) {
    if (c->dtype == EFM_BF16) { if (c->head_dim == 64) f(__nv_bfloat16(), std::integral_constant<int, 64>()); else f(__nv_bfloat16(), std::integral_constant<int, 128>()); }
    else { if (c->head_dim == 64) f(__half(), std::integral_constant<int, 64>()); else f(__half(), std::integral_constant<int, 128>()); }
}

// Every kernel of this file waits for its predecessor before it touches anything an earlier launch may have written, so all of them start
// ahead of the predecessor's end (a kernel lets its successor start once its own wait is over, so that all but the predecessor has ended by
// then): append, attention and weights of one token on 1450 rows take 14.4 us with and 14.9 without, in a replayed graph.
Launcher on_stream(void* stream) {
    Launcher L;
    L.stream = (cudaStream_t)stream;
    L.pdl = true;
    return L;
}
efm_status launched(const char* call, const Launcher& L) { return L.err == cudaSuccess ? EFM_OK : cuda_fail(nullptr, L.err, call); }

template <typename F>
efm_status guarded(F&& f) {
    try { return f(); } catch (const std::exception&) { return EFM_ERR_OUT_OF_MEMORY; } catch (...) { return EFM_ERR_STATE; }
}

int64_t capacity(const efm_kv4_cache* c) { return (int64_t)c->max_pages * kRows; }
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

efm_status check_attention(const char* call, const efm_kv4_cache* c, const efm_kv4_attention* a) {
    if (a == nullptr || a->struct_size != (int32_t)sizeof(efm_kv4_attention)) return bad(call, "struct_size does not match this header");
    if (a->max_rows < 0 || a->max_rows > (1 << 30) || a->max_new < 0 || a->max_len < 0 || a->max_len > capacity(c)) return bad(call, "max_rows, max_new or max_len out of range");
    if ((a->mass_in == nullptr) != (a->mass_out == nullptr)) return bad(call, "mass_in and mass_out: both or neither");
    if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return bad(call, "scale: positive and finite");
    return EFM_OK;
}

// What a call needs: tiles of 8 nt packed query rows, and the parts of its workspace, in floats.
struct AttnPlan {
    int max_new, max_len, nt, blocks, unit_shift, few_rows;
    int many_tiles, many_blocks;                      // blocks of 256 packed rows a sequence may have; blocks that deal with them
    int64_t many_units, many_starts, many_stats, many_part;
    int64_t lost;                                     // a word a block of either kernel
    bool joined;                                      // pieces of a row may lie in several blocks
    bool scores;                                      // attend_few leaves its scores for the summed weights
    int64_t units, stats, part_stats, part, score, image, image_units, starts;
    bool by_rows;                                     // stats and operands in the order of the call's rows, not so many a sequence
    int score_pages;                                  // scores: pages a sequence; 0: by the pool's pages
    int row_tiles;                                    // tiles of 128 packed rows a sequence may have as operands; 0: nobody asks for them
    int64_t bytes() const { return 4 * (stats + part_stats + part + score + image + image_units + starts + many_starts + many_stats + many_part + lost); }
};
constexpr int kSms = 148;                              // of the GPU these kernels are built for
constexpr int kWholeShift = 2;
// Packed rows of a sequence up to which attend_few takes it, in tiles of 16.  A page costs attend_few 3.7 ns a tile of 128 channels (half
// of it with 64; fp16 a quarter more) once the tiles fill the GPU; attend_many has three launches more and some 8.6 ns a block of 256 rows,
// however few rows are in it (fp16, with its products in three parts: 14).  Equal at some 90 tiles of all sequences and kv heads (fp16: 140), and
// where those are many, at 2 (fp16: 3) of each.  Measured (attend_few / attend_many, us): 28 query heads on 4 kv heads of 128, 4000 tokens, 32 rows
// (56 tiles) 26 / 33, 64 rows (112) 39 / 33, fp16 42 / 44, 96 rows (168) fp16 51 / 48; 8 sequences of 2000 tokens with 32 on 4, 6 rows (96) 27 / 31,
// 12 rows (192, 3 each) 36 / 33, fp16 42 / 42; 64 such, 4 rows (2 tiles each) 72 / 82, 6 rows (3 each) 100 / 84, fp16 127 / 157; 64 channels, 14 on 2,
// 256 rows (224) 25 / 28, fp16 39 / 36.
int few_rows_of(const efm_kv4_cache* c) {
    const bool bf16 = c->dtype == EFM_BF16;
    const int64_t each = (int64_t)c->batch * c->kv_heads, all = (bf16 ? 90 : 140) * (128 / c->head_dim);
    return (int)(16 * std::max<int64_t>(bf16 ? 2 : 3, all / each));
}

AttnPlan plan_attention(const efm_kv4_cache* c, const efm_kv4_attention* a) {
    AttnPlan p{};
    p.max_new = std::min(a->max_new, a->max_rows);
    p.max_len = a->max_len > 0 ? a->max_len : (int)capacity(c);
    const int64_t rows = (int64_t)p.max_new * (c->q_heads / c->kv_heads);
    p.nt = rows <= 8 ? 1 : 2;
    p.few_rows = few_rows_of(c);
    p.many_tiles = rows > p.few_rows ? (int)((rows + kv4::kManyRows - 1) / kv4::kManyRows) : 0;
    const int64_t R = 8 * p.nt, tiles = (std::min<int64_t>(rows, p.few_rows) + R - 1) / R, pages = std::max(1, (p.max_len + kRows - 1) / kRows);
    // A page at a time, or caches of up to four pages whole: nothing is left to join then, which saves the smallest calls a launch.  Append and
    // attention of a token, 14/2 heads of 64: 8.2 us whole, 9.6 by pages on two pages; 10.3 and 10.2 on four; 11.2 and 10.3 on five.
    p.unit_shift = pages <= 1 << kWholeShift ? kWholeShift : 0;
    p.units = (pages + (1 << p.unit_shift) - 1 >> p.unit_shift) * tiles * c->kv_heads * c->batch;
    p.blocks = (int)std::max<int64_t>(1, std::min<int64_t>(kSms * (p.nt == 1 ? 3 : 2), (p.units + kv4::kWarps - 1) / kv4::kWarps));
    p.joined = pages > 1 << p.unit_shift;
    p.scores = a->mass_out != nullptr && rows <= R;
    // Whatever a batch could have if every sequence were its longest is more than the call's buffers and the pool can hold: 64 sequences of
    // 28 query heads of 128 with 2048 rows or one, 2111 in all, would have 954 MB of operands (by rows: 23), and 64 tokens with weights on up to
    // 131072 rows 1074 MB of scores, where a pool of 147 MB has 33 MB of them (with mass no page is two sequences').
    p.by_rows = a->max_rows < (int64_t)c->batch * p.max_new;
    p.stats = a->mass_out != nullptr ? round_up(2 * (p.by_rows ? (int64_t)a->max_rows : (int64_t)c->batch * p.max_new) * c->q_heads, 4) : 0;
    const int64_t pieces = p.joined ? 2 * (int64_t)p.blocks * kv4::kWarps * R : 0;      // two a warp: the one it begins in and the one it ends in
    p.part_stats = 2 * pieces;
    p.part = pieces * c->head_dim;
    p.starts = round_up(c->batch + 1, 4);
    p.row_tiles = p.many_tiles > 0 || (a->mass_out != nullptr && !p.scores) ? (int)((rows + kv4::kTileRows - 1) / kv4::kTileRows) : 0;
    if (p.row_tiles > 0) {                            // every part a multiple of 16 bytes
        const int64_t tiles_of_rows = (int64_t)a->max_rows * (c->q_heads / c->kv_heads) / kv4::kTileRows + c->batch;
        p.image_units = (p.by_rows ? tiles_of_rows : (int64_t)c->batch * p.row_tiles) * c->kv_heads * kv4::kTileRows;
    }
    p.image = p.image_units * c->head_dim / 2;
    if (p.many_tiles > 0) {                           // no more blocks of rows than one a sequence and those that all rows fill
        const int64_t tiles_all = std::min<int64_t>((int64_t)c->batch * p.many_tiles, c->batch + (int64_t)a->max_rows * (c->q_heads / c->kv_heads) / kv4::kManyRows);
        p.many_units = tiles_all * c->kv_heads * pages;
        p.many_blocks = (int)std::min<int64_t>(kSms, (p.many_units + kv4::kManyStep - 1) / kv4::kManyStep);
        p.many_starts = round_up((int64_t)c->batch * p.many_tiles + 2, 4);
        p.many_stats = 2 * 2 * (int64_t)p.many_blocks * kv4::kManyRows;
        p.many_part = 2 * (int64_t)p.many_blocks * kv4::kManyRows * c->head_dim;
    }
    p.lost = rows > 0 ? round_up(p.blocks + p.many_blocks, 4) : 0;
    p.score_pages = c->batch * pages <= c->n_pages ? (int)pages : 0;
    p.score = p.scores ? (p.score_pages > 0 ? c->batch * pages : c->n_pages) * c->kv_heads * R * kRows : 0;
    return p;
}

template <typename T, int D>
void launch_attention(Launcher& L, const efm_kv4_cache* cache, const AttnPlan& plan, const kv4::AttnParams& p) {
    using K = AttendKernels<T, D>;
    const K k = K::now();
    const dim3 block(kv4::kWarps * 32);
    const kv4::Cache c = device_cache(cache);
    const int64_t rows = (int64_t)plan.max_new * (cache->q_heads / cache->kv_heads);
    // as many merging blocks as find room at once
    const int64_t jobs = std::min<int64_t>(rows, plan.few_rows) * (D / 32), room = std::max<int64_t>(1, 8 * kSms / ((int64_t)cache->batch * cache->kv_heads));
    const int merges = plan.joined ? (int)std::min(jobs, room) : 0, masses = plan.scores ? (plan.max_len + kv4::kMassTokens - 1) / kv4::kMassTokens : 0;
    const dim3 join(merges + masses, cache->kv_heads, cache->batch);
    if (rows > 0 && plan.nt == 1) L.launch(k.few1, dim3(plan.blocks), block, kv4::FewCfg<D, 1>::SMEM, c, p);
    if (rows > 0 && plan.nt == 2) L.launch(k.few2, dim3(plan.blocks), block, kv4::FewCfg<D, 2>::SMEM, c, p);
    if (plan.row_tiles > 0) L.launch(kv4::attend_query_kernel<T, D>, dim3(plan.row_tiles + 1, cache->kv_heads, cache->batch), dim3(kv4::kTileRows), 0, c, p);
    if (plan.many_tiles > 0) {
        const dim3 many(plan.many_blocks), threads(kv4::kManyThreads);
        if (p.mass_out != nullptr) L.launch(k.many_mass, many, threads, kv4::ManyCfg<D, K::XM>::SMEM, c, p);
        else L.launch(k.many, many, threads, kv4::ManyCfg<D, K::X>::SMEM, c, p);
        if (plan.many_blocks > 1) L.launch(kv4::attend_join_kernel<T, D>, dim3(plan.many_blocks - 1, D / 16), dim3(kv4::kManyRows), 0, c, p);
    }
    if (join.x > 0 && plan.nt == 1) L.launch(kv4::attend_merge_kernel<T, D, 8>, join, block, 0, c, p, masses);
    if (join.x > 0 && plan.nt == 2) L.launch(kv4::attend_merge_kernel<T, D, 16>, join, block, 0, c, p, masses);
    if (p.mass_out != nullptr && !plan.scores)
        L.launch(k.weights, dim3((plan.max_len + kv4::WeightsCfg<D>::KEYS - 1) / kv4::WeightsCfg<D>::KEYS, cache->kv_heads, cache->batch), dim3(kv4::kWeightThreads),
                 kv4::WeightsCfg<D>::SMEM, c, p);
}

efm_status check_evict(const char* call, const efm_kv4_evict* a) {
    if (a == nullptr || a->struct_size != (int32_t)sizeof(efm_kv4_evict)) return bad(call, "struct_size does not match this header");
    if (a->budget < 1 || a->limit < a->budget || a->keep_first < 0 || a->keep_last < 0) return bad(call, "budget >= 1, limit >= budget, keep_first and keep_last >= 0");
    return EFM_OK;
}
int64_t most_moves(const efm_kv4_cache* c, const efm_kv4_evict* a) {
    return std::max<int64_t>(0, std::min<int64_t>(a->budget, capacity(c) - a->budget));
}
int64_t evict_counts(const efm_kv4_cache* c) { return round_up((int64_t)c->batch * c->kv_heads * 4, 16); }
int64_t evict_bytes(const efm_kv4_cache* c, const efm_kv4_evict* a) {
    return evict_counts(c) + (int64_t)c->batch * c->kv_heads * most_moves(c, a) * (int64_t)sizeof(int2);
}

}  // namespace
}  // namespace efm

using namespace efm;

extern "C" {

efm_status efm_b200_kv4_tile_bytes(int32_t head_dim, int64_t* bytes) {
    return guarded([&] {
        if (bytes == nullptr || (head_dim != 64 && head_dim != 128)) return bad("kv4_tile_bytes", "head_dim 64 or 128");
        *bytes = head_dim == 64 ? kv4::Tile<64>::BYTES : kv4::Tile<128>::BYTES;
        return (efm_status)EFM_OK;
    });
}

efm_status efm_b200_kv4_attention_workspace(const efm_kv4_cache* cache, const efm_kv4_attention* a, int64_t* bytes) {
    return guarded([&] {
        const char* call = "kv4_attention_workspace";
        efm_status st = check_cache(call, cache);
        if (st == EFM_OK) st = check_attention(call, cache, a);
        if (st == EFM_OK && bytes == nullptr) st = bad(call, "bytes is null");
        if (st == EFM_OK) *bytes = plan_attention(cache, a).bytes();
        return st;
    });
}

efm_status efm_b200_kv4_evict_workspace(const efm_kv4_cache* cache, const efm_kv4_evict* a, int64_t* bytes) {
    return guarded([&] {
        const char* call = "kv4_evict_workspace";
        efm_status st = check_cache(call, cache);
        if (st == EFM_OK) st = check_evict(call, a);
        if (st == EFM_OK && bytes == nullptr) st = bad(call, "bytes is null");
        if (st == EFM_OK) *bytes = evict_bytes(cache, a);
        return st;
    });
}

efm_status efm_b200_op_kv4_append(const efm_kv4_cache* cache, const efm_kv4_append* a, void* stream) {
    return guarded([&]() -> efm_status {
        const char* call = "op_kv4_append";
        efm_status st = check_cache(call, cache);
        if (st == EFM_OK) st = check_buffers(call, cache);
        if (st != EFM_OK) return st;
        if (a == nullptr || a->struct_size != (int32_t)sizeof(efm_kv4_append)) return bad(call, "struct_size does not match this header");
        const int64_t D = cache->head_dim, qd = cache->q_heads * D, kd = cache->kv_heads * D;
        if (a->max_rows < 0 || a->max_rows > (1 << 30)) return bad(call, "max_rows out of range");
        if (a->cu_rows == nullptr || a->lens_in == nullptr || a->lens_out == nullptr || a->lens_in == a->lens_out)
            return bad(call, "cu_rows, lens_in and lens_out (two buffers) are needed");
        if (a->max_rows > 0) {
            if (a->k == nullptr || a->v == nullptr || (a->q == nullptr) != (a->q_out == nullptr)) return bad(call, "k and v are needed, q and q_out together");
            if (a->k_stride < kd || a->v_stride < kd || a->k_stride % 8 || a->v_stride % 8 || (a->q != nullptr && (a->q_stride < qd || a->q_stride % 8)))
                return bad(call, "strides: multiples of 8 elements, at least heads x head_dim");
            for (const void* p : {a->q, a->k, a->v, a->q_norm, a->k_norm, (const void*)a->q_out, (const void*)a->k_held, (const void*)a->v_held})
                if (!aligned(p, 16)) return bad(call, "q, k, v, norm weights and their outputs: 16-byte aligned");
            for (const void* p : {(const void*)a->cu_rows, (const void*)a->lens_in, (const void*)a->lens_out, (const void*)a->positions, (const void*)a->token_index,
                                  (const void*)a->index, (const void*)a->mass})
                if (!aligned(p, 4)) return bad(call, "numbers: aligned to their size");
            if (a->norm != 0 && a->norm != 1) return bad(call, "norm: 0 or 1");
            if (a->norm == 1 && !(a->norm_eps >= 0.f)) return bad(call, "norm_eps: not negative");
            if (a->rot_dims < 0 || a->rot_dims > D || a->rot_dims % 16) return bad(call, "rot_dims: a multiple of 16, at most head_dim");
            if (a->rot_dims > 0) {
                if (a->rot_kind != EFM_KV4_ROT_HALVES && a->rot_kind != EFM_KV4_ROT_NEIGHBOURS) return bad(call, "rot_kind");
                if (a->axes != 1 && a->axes != 3) return bad(call, "axes: 1 or 3");
                if (a->axes == 3) {
                    int64_t sum = 0;
                    for (int i = 0; i < 3; ++i) { if (a->sections[i] < 0) return bad(call, "sections: not negative"); sum += a->sections[i]; }
                    if (sum != a->rot_dims / 2) return bad(call, "sections: their sum is rot_dims / 2");
                }
                if (a->inv_freq == nullptr || a->positions == nullptr || !aligned(a->inv_freq, 8)) return bad(call, "inv_freq and positions are needed to rotate");
            }
        }
        OnDevice on;
        DeviceInfo info;
        if ((st = on.enter(call, cache->pool)) != EFM_OK || (st = device_info(call, on.device, info)) != EFM_OK) return st;
        kv4::AppendParams p{};
        p.max_rows = a->max_rows;
        p.cu_rows = a->cu_rows; p.lens_in = a->lens_in; p.lens_out = a->lens_out;
        p.q = a->q; p.k = a->k; p.v = a->v;
        p.q_stride = a->q_stride; p.k_stride = a->k_stride; p.v_stride = a->v_stride;
        p.norm = a->norm; p.eps = a->norm_eps; p.q_norm = a->q_norm; p.k_norm = a->k_norm;
        p.rot_dims = a->rot_dims; p.neighbours = a->rot_kind == EFM_KV4_ROT_NEIGHBOURS; p.axes = a->axes;
        p.section0 = a->sections[0]; p.section1 = a->sections[1];
        p.inv_freq = a->inv_freq; p.positions = a->positions; p.token_index = a->token_index;
        p.q_out = a->q_out; p.k_held = a->k_held; p.v_held = a->v_held;
        p.index = a->index; p.mass = a->mass;
        const int per = 256 / cache->head_dim, kv = (cache->kv_heads + per - 1) / per, tasks = (a->q != nullptr ? (cache->q_heads + per - 1) / per : 0) + 2 * kv, warps = kv4::kAppendThreads / 32;
        // few rows: a task (the heads a warp has at a time) per warp, so that a row's heads are on as many SMs as there are; many rows: a
        // block per row, one table of angles
        const int per_block = (int64_t)a->max_rows * ((tasks + warps - 1) / warps) <= 2 * info.sms ? warps : tasks;
        Launcher L = on_stream(stream);
        by_type(cache, [&](auto t, auto d) {
            L.launch(kv4::append_kernel<decltype(t), decltype(d)::value>, dim3(std::max(a->max_rows, 1), (tasks + per_block - 1) / per_block), dim3(kv4::kAppendThreads), 0,
                     device_cache(cache), p, per_block);
        });
        return launched(call, L);
    });
}

efm_status efm_b200_op_kv4_attention(const efm_kv4_cache* cache, const efm_kv4_attention* a, void* stream) {
    return guarded([&]() -> efm_status {
        const char* call = "op_kv4_attention";
        efm_status st = check_cache(call, cache);
        if (st == EFM_OK) st = check_buffers(call, cache);
        if (st == EFM_OK) st = check_attention(call, cache, a);
        if (st != EFM_OK) return st;
        if (a->cu_rows == nullptr || a->lens == nullptr || !aligned(a->cu_rows, 4) || !aligned(a->lens, 4)) return bad(call, "cu_rows and lens are needed");
        if (a->max_rows > 0 && (a->q == nullptr || a->out == nullptr || !aligned(a->q, 16) || !aligned(a->out, 16))) return bad(call, "q and out are needed, 16-byte aligned");
        if (!aligned(a->mass_in, 4) || !aligned(a->mass_out, 4)) return bad(call, "mass: aligned to 4 bytes");
        const AttnPlan plan = plan_attention(cache, a);
        if (plan.bytes() > 0 && (a->workspace == nullptr || a->workspace_bytes < plan.bytes() || !aligned(a->workspace, 16)))
            return bad(call, "workspace: 16-byte aligned, as large as efm_b200_kv4_attention_workspace says");
        if (plan.units > (1 << 30) || plan.many_units > (1 << 30) || plan.many_starts > (1 << 30)) return fail(nullptr, EFM_ERR_UNSUPPORTED, std::string(call) + ": more than 2^30 pages x kv heads x row tiles");
        OnDevice on;
        DeviceInfo info;
        if ((st = on.enter(call, cache->pool)) != EFM_OK || (st = device_info(call, on.device, info)) != EFM_OK) return st;
        const uint32_t group = cache->q_heads / cache->kv_heads;
        kv4::AttnParams p{};
        p.max_rows = a->max_rows; p.max_new = plan.max_new; p.max_len = plan.max_len;
        p.cu_rows = a->cu_rows; p.lens = a->lens; p.q = a->q; p.out = a->out;
        p.scale_log2 = a->scale * 1.4426950408889634f;
        p.mass_in = a->mass_in; p.mass_out = a->mass_out;
        p.few_rows = plan.few_rows; p.warps = plan.blocks * kv4::kWarps; p.unit_shift = plan.unit_shift; p.group_inv = group == 1 ? 0u : (uint32_t)(((1ull << 32) + group - 1) / group); p.rows = plan.by_rows ? 0 : plan.max_new;
        float* ws = (float*)a->workspace;
        p.stats = plan.stats > 0 ? (float2*)ws : nullptr;
        p.part_stats = (float2*)(ws + plan.stats);
        p.part = ws + plan.stats + plan.part_stats;
        p.scores = plan.scores ? p.part + plan.part : nullptr;
        p.score_pages = plan.score_pages;
        p.row_tiles = plan.row_tiles;
        p.images = (uint8_t*)(ws + plan.stats + plan.part_stats + plan.part + plan.score);
        p.units = (float*)p.images + plan.image;
        p.starts = (int32_t*)(p.units + plan.image_units);
        p.many_tiles = plan.many_tiles; p.many_blocks = plan.many_blocks;
        p.many_starts = p.starts + plan.starts;
        p.many_stats = (float2*)(p.many_starts + plan.many_starts);
        p.many_part = (float*)p.many_stats + plan.many_stats;
        p.lost = (int32_t*)(p.many_part + plan.many_part);
        p.few_blocks = plan.blocks; p.n_lost = plan.lost > 0 ? plan.blocks + plan.many_blocks : 0;
        Launcher L = on_stream(stream);
        by_type(cache, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int D = decltype(d)::value;
            launch_attention<T, D>(L, cache, plan, p);
        });
        return launched(call, L);
    });
}

efm_status efm_b200_op_kv4_evict(const efm_kv4_cache* cache, const efm_kv4_evict* a, void* stream) {
    return guarded([&]() -> efm_status {
        const char* call = "op_kv4_evict";
        efm_status st = check_cache(call, cache);
        if (st == EFM_OK) st = check_buffers(call, cache);
        if (st == EFM_OK) st = check_evict(call, a);
        if (st != EFM_OK) return st;
        if (a->lens_in == nullptr || a->lens_out == nullptr || a->lens_in == a->lens_out) return bad(call, "lens_in and lens_out (two buffers) are needed");
        for (const void* p : {(const void*)a->index_in, (const void*)a->index_out, (const void*)a->mass_in, (const void*)a->mass_out})
            if (p == nullptr || !aligned(p, 4)) return bad(call, "index and mass, in and out, are needed");
        if (!aligned(a->lens_in, 4) || !aligned(a->lens_out, 4)) return bad(call, "lens: aligned to 4 bytes");
        if (a->workspace == nullptr || a->workspace_bytes < evict_bytes(cache, a) || !aligned(a->workspace, 16))
            return bad(call, "workspace: 16-byte aligned, as large as efm_b200_kv4_evict_workspace says");
        OnDevice on;
        DeviceInfo info;
        if ((st = on.enter(call, cache->pool)) != EFM_OK || (st = device_info(call, on.device, info)) != EFM_OK) return st;
        kv4::EvictParams p{};
        p.budget = a->budget; p.limit = a->limit; p.keep_first = a->keep_first; p.keep_last = a->keep_last;
        p.lens_in = a->lens_in; p.lens_out = a->lens_out; p.index_in = a->index_in; p.index_out = a->index_out; p.mass_in = a->mass_in; p.mass_out = a->mass_out;
        p.n_moves = (int32_t*)a->workspace;
        p.moves = (int2*)((char*)a->workspace + evict_counts(cache));
        p.most_moves = (int)most_moves(cache, a);
        p.head_dim = cache->head_dim;
        p.inline_moves = p.most_moves <= kv4::kInlineMoves;
        p.keys_cap = (int)std::min<int64_t>(capacity(cache), (info.smem - kEvictSmemReserve) / 4);
        Launcher L = on_stream(stream);
        const kv4::Cache c = device_cache(cache);
        const dim3 heads(cache->kv_heads, cache->batch);
        if (capacity(cache) <= kv4::kKeepFew * kv4::kEvictThreads) L.launch(kv4::evict_select_kernel<kv4::kKeepFew>, heads, dim3(kv4::kEvictThreads), (size_t)p.keys_cap * 4, c, p);
        else L.launch(kv4::evict_select_kernel<kv4::kKeepMany>, heads, dim3(kv4::kEvictThreads), (size_t)p.keys_cap * 4, c, p);
        if (!p.inline_moves) {
            const int per = kv4::kMoveThreads / 16, all = (p.most_moves + per - 1) / per;
            const int parts = (int)std::min<int64_t>(all, std::max<int64_t>(1, (int64_t)8 * info.sms / ((int64_t)cache->batch * cache->kv_heads)));
            if (cache->head_dim == 64) L.launch(kv4::evict_move_kernel<64>, dim3(parts, cache->kv_heads, cache->batch), dim3(kv4::kMoveThreads), 0, c, p);
            else L.launch(kv4::evict_move_kernel<128>, dim3(parts, cache->kv_heads, cache->batch), dim3(kv4::kMoveThreads), 0, c, p);
        }
        return launched(call, L);
    });
}

efm_status efm_b200_op_kv4_read(const efm_kv4_cache* cache, const efm_kv4_read* a, void* stream) {
    return guarded([&]() -> efm_status {
        const char* call = "op_kv4_read";
        efm_status st = check_cache(call, cache);
        if (st == EFM_OK) st = check_buffers(call, cache);
        if (st != EFM_OK) return st;
        if (a == nullptr || a->struct_size != (int32_t)sizeof(efm_kv4_read)) return bad(call, "struct_size does not match this header");
        if (a->first < 0 || a->rows < 0 || (int64_t)a->first + a->rows > (1 << 30)) return bad(call, "first and rows out of range");
        if (a->lens == nullptr || !aligned(a->lens, 4) || (a->k_out == nullptr && a->v_out == nullptr) || !aligned(a->k_out, 16) || !aligned(a->v_out, 16))
            return bad(call, "lens and k_out or v_out (16-byte aligned) are needed");
        OnDevice on;
        DeviceInfo info;
        if ((st = on.enter(call, cache->pool)) != EFM_OK || (st = device_info(call, on.device, info)) != EFM_OK) return st;
        const int64_t end = std::min<int64_t>(capacity(cache), (int64_t)a->first + a->rows);
        const int64_t pages = end > a->first ? (end + kRows - 1) / kRows - a->first / kRows : 0;
        if (pages == 0) return EFM_OK;
        if (pages * cache->kv_heads > 0x7fffffff) return bad(call, "too many rows");
        Launcher L = on_stream(stream);
        by_type(cache, [&](auto t, auto d) {
            using T = decltype(t);
            L.launch(kv4::read_kernel<T, decltype(d)::value>, dim3((unsigned)(pages * cache->kv_heads), cache->batch), dim3(kv4::kReadThreads), 0, device_cache(cache),
                     a->lens, a->first, a->rows, (T*)a->k_out, (T*)a->v_out);
        });
        return launched(call, L);
    });
}

}  // extern "C"
