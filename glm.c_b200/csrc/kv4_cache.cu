// Rows of the 4-bit latent cache (layout: kv4.cuh): glm_cuda_kv4_store_async
// quantises new rows into their slots, glm_cuda_kv4_load_async reads rows
// back. glm.c caches the same rows in fp32 (infer.c:1003-1016).
//
// A group of values with largest magnitude a gets the scale s = bf16(a / 7),
// and x the code v + 8, v = rint(x / s) clamped to [-7, 7], all in 32-bit
// arithmetic as written (the division rounds correctly: the codes are those of
// the formula, bit for bit). A group with a NaN or an infinity gets the scale
// NaN, so that whatever reads it comes out NaN, as a product with that row
// would; a group whose scale rounds to zero holds zeros.
//
// Both are bound by memory traffic. Eight lanes share a group: 16-byte
// loads (stores) of consecutive lanes touch consecutive addresses, three
// shuffles give the group's largest magnitude, and a warp has four groups in
// flight.
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "glm_internal.h"
#include "kv4.cuh"
#include "q80_common.cuh"
#include "serve_common.h"

namespace glmq {
namespace {

constexpr int kRowThreads = 256;
constexpr int kGroupLanes = 8;

struct RowArgs {
    Kv4Shape sh;
    unsigned char* pages;
    long long n_slots;
    const int64_t* slots;
    long long units;  // rows * groups
    void *latent, *rope;
    long long latent_stride, rope_stride;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// kN consecutive values; kVec: p is aligned to their size.
template <typename T, int kN, bool kVec>
__device__ __forceinline__ void get(const T* p, float (&v)[kN]) {
    alignas(16) T t[kN];
    if constexpr (kVec) {
        static_assert(sizeof t == 16);
        *reinterpret_cast<int4*>(t) = __ldg(reinterpret_cast<const int4*>(p));
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) t[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = to_f(t[i]);
}

template <typename T, int kN, bool kVec>
__device__ __forceinline__ void put(T* p, const float (&v)[kN]) {
    alignas(16) T t[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) t[i] = from_f<T>(v[i]);
    if constexpr (kVec) {
        static_assert(sizeof t == 16);
        *reinterpret_cast<int4*>(p) = *reinterpret_cast<const int4*>(t);
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) p[i] = t[i];
    }
}

// rint(x / s) with the quotient rounded to fp32 first, for |x / s| < 8. The
// product with the rounded reciprocal is within 1.3e-6 of the quotient, so
// only quotients that close to a half need the division itself.
__device__ __forceinline__ int code_of(float x, float s, float inv, bool slow) {
    const float q = x * inv, k = rintf(q);
    int v = (int)k;
    if (slow || fabsf(fabsf(q - k) - 0.5f) < 4e-6f) v = (int)rintf(__fdiv_rn(x, s));
    return min(max(v, -7), 7) + 8;
}

// Where unit (row, group) lies: its first value, how many there are, its codes and its scale.
struct Unit {
    bool ok;
    int n;
    const unsigned char* page;
    size_t codes, scale;
    size_t latent, rope;  // element offsets of the values (one of them is used)
    bool is_rope;
};

__device__ __forceinline__ Unit unit_of(const RowArgs& a, long long unit) {
    const int groups = a.sh.groups();
    const long long row = unit / groups;
    const int g = (int)(unit - row * groups);
    Unit u;
    const long long slot = a.slots[row];
    u.ok = slot >= 0 && slot < a.n_slots;
    u.is_rope = g == groups - 1;
    u.n = u.is_rope ? a.sh.rope : kKv4Group;
    const long long page = u.ok ? slot / a.sh.page : 0;
    const int at = u.ok ? (int)(slot - page * a.sh.page) : 0;
    u.page = a.pages + (size_t)page * a.sh.page_bytes();
    u.codes = (size_t)at * a.sh.row_bytes() + (size_t)g * (kKv4Group / 2);
    u.scale = (size_t)a.sh.page * a.sh.row_bytes() + ((size_t)g * a.sh.page + at) * 2;
    u.latent = (size_t)row * a.latent_stride + (size_t)g * kKv4Group;
    u.rope = (size_t)row * a.rope_stride;
    return u;
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kRowThreads) kv4_store_kernel(RowArgs a) {
    constexpr int kN = 16 / sizeof(T), kChunks = kKv4Group / (kGroupLanes * kN);  // chunks of a 128-value group
    pdl_enter();
    const int l = threadIdx.x % kGroupLanes;
    const long long per = (long long)gridDim.x * (kRowThreads / kGroupLanes);
    // every lane of a warp runs the same number of rounds, for the shuffles
    const long long base = ((long long)blockIdx.x * kRowThreads + (threadIdx.x & ~31)) / kGroupLanes;
    for (long long u0 = base; u0 < a.units; u0 += per) {
        const long long unit = u0 + (threadIdx.x & 31) / kGroupLanes;
        const bool live = unit < a.units;
        const Unit u = unit_of(a, live ? unit : 0);
        const T* src = u.is_rope ? static_cast<const T*>(a.rope) + u.rope : static_cast<const T*>(a.latent) + u.latent;
        float x[kChunks][kN];
        unsigned top = 0u;  // largest magnitude as bits: NaN lies above infinity
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int e = (c * kGroupLanes + l) * kN;
#pragma unroll
            for (int i = 0; i < kN; ++i) x[c][i] = 0.f;
            if (live && u.ok && e < u.n) get<T, kN, kVec>(src + e, x[c]);
#pragma unroll
            for (int i = 0; i < kN; ++i) top = max(top, __float_as_uint(x[c][i]) & 0x7fffffffu);
        }
#pragma unroll
        for (int off = 1; off < kGroupLanes; off <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
        if (!live || !u.ok) continue;
        const bool bad = top >= 0x7f800000u;
        const __nv_bfloat16 sb = bad ? __ushort_as_bfloat16(0x7fc0) : __float2bfloat16_rn(__fdiv_rn(__uint_as_float(top), 7.f));
        const float s = __bfloat162float(sb);
        const bool zero = bad || s == 0.f;
        const bool slow = s < 1e-37f;  // the reciprocal could overflow
        const float inv = zero ? 0.f : __frcp_rn(s);
        unsigned char* page = const_cast<unsigned char*>(u.page);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int e = (c * kGroupLanes + l) * kN;
            if (e >= u.n) continue;
            unsigned w = 0u;
#pragma unroll
            for (int i = 0; i < kN; ++i) w |= (unsigned)(zero ? 8 : code_of(x[c][i], s, inv, slow)) << (4 * i);
            unsigned char* d = page + u.codes + e / 2;
            if constexpr (kN == 8)
                *reinterpret_cast<uint32_t*>(d) = w;
            else
                *reinterpret_cast<uint16_t*>(d) = (uint16_t)w;
        }
        if (l == 0) *reinterpret_cast<__nv_bfloat16*>(page + u.scale) = sb;
    }
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kRowThreads) kv4_load_kernel(RowArgs a) {
    constexpr int kN = 16 / sizeof(T), kChunks = kKv4Group / (kGroupLanes * kN);
    pdl_enter();
    const int l = threadIdx.x % kGroupLanes;
    const long long per = (long long)gridDim.x * (kRowThreads / kGroupLanes);
    for (long long unit = ((long long)blockIdx.x * kRowThreads + threadIdx.x) / kGroupLanes; unit < a.units; unit += per) {
        const Unit u = unit_of(a, unit);
        T* dst = u.is_rope ? static_cast<T*>(a.rope) + u.rope : static_cast<T*>(a.latent) + u.latent;
        const float s = u.ok ? __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(u.page + u.scale)) : 0.f;
        unsigned w[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int e = (c * kGroupLanes + l) * kN;
            w[c] = 0x88888888u;
            if (!u.ok || e >= u.n) continue;
            const unsigned char* p = u.page + u.codes + e / 2;
            if constexpr (kN == 8)
                w[c] = *reinterpret_cast<const uint32_t*>(p);
            else
                w[c] = *reinterpret_cast<const uint16_t*>(p);
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int e = (c * kGroupLanes + l) * kN;
            if (e >= u.n) continue;
            float v[kN];
#pragma unroll
            for (int i = 0; i < kN; ++i) v[i] = (float)((int)((w[c] >> (4 * i)) & 15u) - 8) * s;
            put<T, kN, kVec>(dst + e, v);
        }
    }
}

enum class Way { kStore, kLoad };

template <typename T>
cudaError_t launch_rows(Way way, bool vec, const RowArgs& a, int sms, cudaStream_t st) {
    const long long per = kRowThreads / kGroupLanes;
    long long grid = (a.units + per - 1) / per;
    const long long most = (long long)sms * (2048 / kRowThreads);
    if (grid > most) grid = most;
    auto kernel = way == Way::kStore ? (vec ? kv4_store_kernel<T, true> : kv4_store_kernel<T, false>)
                                     : (vec ? kv4_load_kernel<T, true> : kv4_load_kernel<T, false>);
    return launch_pdl(kernel, (unsigned)grid, kRowThreads, 0, st, a);
}

int rows_entry(const char* fn, Way way, const GlmCudaKv4Cache* cache, const int64_t* slots, int n_rows, int type,
               void* latent, int64_t latent_stride, void* rope, int64_t rope_stride, void* stream) {
    if (int rc = check_kv4_cache(fn, cache)) return rc;
    if (!known_type(type)) return op_fail(GLM_CUDA_ERR_ARG, fn, "unknown type %d", type);
    if (n_rows < 0) return op_fail(GLM_CUDA_ERR_ARG, fn, "n_rows=%d", n_rows);
    if (n_rows == 0) return 0;
    if (!slots || !latent || !rope) return op_fail(GLM_CUDA_ERR_ARG, fn, "a required pointer is NULL");
    if (latent_stride < cache->kv_lora_rank || rope_stride < cache->rope_dim)
        return op_fail(GLM_CUDA_ERR_ARG, fn, "row strides %lld, %lld are shorter than the rows", (long long)latent_stride,
                       (long long)rope_stride);
    const size_t tb = type_bytes(type);
    if (!aligned(latent, tb) || !aligned(rope, tb) || !aligned(slots, 8))
        return op_fail(GLM_CUDA_ERR_ARG, fn, "a pointer is not aligned to its type");
    int sms = 0;
    if (cudaError_t e = current_sms(&sms)) return launch_failed(fn, e);
    RowArgs a;
    a.sh = Kv4Shape{cache->kv_lora_rank, cache->rope_dim, cache->page_size};
    a.pages = static_cast<unsigned char*>(cache->pages);
    a.n_slots = (long long)cache->n_pages * cache->page_size;
    a.slots = slots;
    a.units = (long long)n_rows * a.sh.groups();
    a.latent = latent;
    a.rope = rope;
    a.latent_stride = latent_stride;
    a.rope_stride = rope_stride;
    // 16-byte accesses where every row starts on a 16-byte boundary, one value at a time elsewhere
    const bool vec = aligned(latent, 16) && aligned(rope, 16) && latent_stride * tb % 16 == 0 && rope_stride * tb % 16 == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = type == GLM_CUDA_F32    ? launch_rows<float>(way, vec, a, sms, st)
                    : type == GLM_CUDA_BF16 ? launch_rows<__nv_bfloat16>(way, vec, a, sms, st)
                                            : launch_rows<__half>(way, vec, a, sms, st);
    if (e) return launch_failed(fn, e);
    count_launches(1);
    return 0;
}

}  // namespace
}  // namespace glmq

extern "C" int glm_cuda_kv4_store_async(const GlmCudaKv4Cache* cache, const void* latent_dev, int64_t latent_stride,
                                        const void* rope_dev, int64_t rope_stride, int type, const int64_t* slots_dev,
                                        int n_rows, void* stream) {
    return glmq::rows_entry("glm_cuda_kv4_store_async", glmq::Way::kStore, cache, slots_dev, n_rows, type,
                            const_cast<void*>(latent_dev), latent_stride, const_cast<void*>(rope_dev), rope_stride, stream);
}

extern "C" int glm_cuda_kv4_load_async(const GlmCudaKv4Cache* cache, const int64_t* slots_dev, int n_rows,
                                       void* latent_dev, int64_t latent_stride, void* rope_dev, int64_t rope_stride,
                                       int type, void* stream) {
    return glmq::rows_entry("glm_cuda_kv4_load_async", glmq::Way::kLoad, cache, slots_dev, n_rows, type, latent_dev,
                            latent_stride, rope_dev, rope_stride, stream);
}
