// Log probability of a given token, entropy and the most likely tokens of
// every row of logits, in one pass: glm_cuda_logprobs_async. glm.c answers
// with the argmax or a sample alone (infer.c:1218-1290).
//
//   m = max_i x_i,  l = sum_i e^(x_i - m),  s = sum_i e^(x_i - m) (x_i - m)
//   log p_i = x_i - m - ln l,   entropy = ln l - s / l
//
// The logits are read once (620 KB a row for GLM-4.7-Flash's vocabulary in
// fp32) and that traffic is the bound. Each thread keeps running (m, l, s):
// raising m by d multiplies l by e^-d and turns s into e^-d (s - d l).
//
// The most likely tokens: every warp keeps the best 32 (value, index) pairs
// it has seen, sorted, one to a lane, as 64-bit keys (ordered value bits, then
// the complement of the index, so that ties go to the lowest index). A value
// has to beat the k-th of them to be looked at; those that do collect in a
// shared-memory buffer and enter 32 at a time by a bitonic sort and merge, so
// that an ascending row, where every value is a new best, costs a bounded
// amount per value too. Warps share their bounds: what is below any warp's
// k-th best is not among the row's.
//
// A row is one CTA's, or a thread-block cluster's when there are fewer rows
// than SMs; the CTAs of a cluster meet in distributed shared memory. No
// workspace, no second launch.
#include <cfloat>
#include <cmath>
#include <climits>
#include <cstdint>
#include <type_traits>

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "glm_internal.h"
#include "q80_common.cuh"
#include "serve_common.h"

namespace glmq {
namespace {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;   // one sorted pair to a lane
constexpr int kLpMaxCluster = 8;

struct LpArgs {
    const void* logits;
    long long stride;
    int vocab, top;
    const int32_t* target;
    float *logprob, *entropy;
    int32_t* top_ids;
    float* top_logprobs;
};

// Running sums of a part of a row, in units of ln.
struct Part {
    float m, l, s;
};

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp_fast(float d) { return exp2f(d * kLog2e); }

__device__ __forceinline__ Part join(const Part& a, const Part& b) {
    const float m = fmaxf(a.m, b.m);
    // a part without weight (nothing seen, or all of it -inf) adds nothing
    const float da = a.m == -INFINITY ? 0.f : a.m - m, db = b.m == -INFINITY ? 0.f : b.m - m;
    const float wa = exp_fast(da), wb = exp_fast(db);
    // a weight of zero may stand beside a difference of -inf
    const float sa = wa > 0.f ? wa * (a.s + a.l * da) : 0.f, sb = wb > 0.f ? wb * (b.s + b.l * db) : 0.f;
    return Part{m, a.l * wa + b.l * wb, sa + sb};
}

// Value and index as one key: larger value first, then the lower index. Zero is below every key.
__device__ __forceinline__ uint64_t key_of(float x, int i) {
    const unsigned b = __float_as_uint(x + 0.f);  // -0 ties with +0
    const unsigned o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((uint64_t)o << 32) | (unsigned)~i;
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const unsigned o = (unsigned)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(unsigned)k; }

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int off) { return __shfl_xor_sync(0xffffffffu, v, off); }

__device__ __forceinline__ uint64_t keep(uint64_t v, int off, bool larger) {
    const uint64_t o = shfl_xor64(v, off);
    return (v > o) == larger ? v : o;
}

// The warp's 32 keys in descending order.
__device__ __forceinline__ uint64_t sort32(uint64_t v, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int off = size >> 1; off > 0; off >>= 1)
            v = keep(v, off, ((lane & off) == 0) == ((lane & size) == 0 || size == 32));
    return v;
}

// The 32 largest of two descending lists, in descending order.
__device__ __forceinline__ uint64_t merge32(uint64_t a, uint64_t b, int lane) {
    const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
    uint64_t v = a > r ? a : r;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v = keep(v, off, (lane & off) == 0);
    return v;
}

// Largest float below x (x itself for -inf).
__device__ __forceinline__ float below(float x) {
    if (x == -INFINITY) return x;
    const int b = __float_as_int(x + 0.f);
    return b == 0 ? -FLT_MIN * FLT_EPSILON : __int_as_float(b > 0 ? b - 1 : b + 1);
}

template <typename T>
struct Vec {
    static constexpr int n = 16 / sizeof(T);
    int4 raw;
    __device__ __forceinline__ void load(const T* p) {
        asm volatile("ld.global.nc.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];\n"
                     : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w)
                     : "l"(p));
    }
    __device__ __forceinline__ float get(int i) const {
        const int w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (sizeof(T) == 4) return __int_as_float(w[i]);
        else if constexpr (std::is_same<T, __half>::value)
            return __half2float(__ushort_as_half((unsigned short)((unsigned)w[i >> 1] >> (16 * (i & 1)))));
        else
            return __int_as_float(i & 1 ? w[i >> 1] & 0xffff0000 : w[i >> 1] << 16);
    }
};

template <typename T>
__device__ __forceinline__ float value_of(const T* p, long long i) {
    if constexpr (sizeof(T) == 4) return p[i];
    else if constexpr (std::is_same<T, __half>::value) return __half2float(p[i]);
    else return __bfloat162float(p[i]);
}

// 16-byte loads in flight per thread: 16 values where candidates are
// collected, so that two CTAs' buffers fit an SM at either width.
template <typename T, bool kTop>
constexpr int kLpVecs = kTop ? 16 / Vec<T>::n : 4;

// One warp's candidates: an iteration adds at most 32 lanes x 16 values to
// fewer than 32 left from before.
constexpr int kLpBuffer = 32 * 16 + 32;

template <bool kTop>
constexpr size_t lp_smem() {
    return kTop ? (size_t)kLpWarps * (kLpBuffer + 32) * 8 : 0;
}

template <typename T, bool kTop>
__global__ void __launch_bounds__(kLpThreads, 2) logprobs_kernel(LpArgs a, int cluster) {
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    constexpr int V = Vec<T>::n, U = kLpVecs<T, kTop>;
    extern __shared__ __align__(16) uint64_t lp_sm[];
    __shared__ Part parts[kLpWarps];
    __shared__ Part cta_part;
    __shared__ int shared_bound;     // ordered bits of the largest bound any warp has published
    __shared__ int counts[kLpWarps];
    const int rank = (int)cl.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.x / cluster;
    uint64_t* lists = lp_sm;                                             // [kLpWarps][32] sorted
    uint64_t* buffer = lp_sm + kLpWarps * 32 + warp * (kTop ? kLpBuffer : 0);
    if (kTop && tid < kLpWarps) counts[tid] = 0;
    if (tid == 0) shared_bound = INT_MIN;
    pdl_enter();
    __syncthreads();

    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    // the 16-byte vectors of the row; what lies before and after them goes value by value
    const int head = min(a.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    const int nvec = (a.vocab - head) / V, tail = head + nvec * V;
    const int v_lo = (int)((long long)rank * nvec / cluster), v_hi = (int)((long long)(rank + 1) * nvec / cluster);

    Part p{-INFINITY, 0.f, 0.f};
    uint64_t list = 0;          // this lane's entry of the warp's sorted best
    float bound = -INFINITY;    // a value has to be above it

    // the warp's candidates, 32 at a time, into its list
    auto take = [&](bool all) {
        __syncwarp();
        int n = counts[warp];
        while (n >= 32 || (all && n > 0)) {
            const int got = min(n, 32);
            n -= got;
            const uint64_t c = lane < got ? buffer[n + lane] : 0;
            list = merge32(list, sort32(c, lane), lane);
        }
        __syncwarp();
        if (lane == 0) counts[warp] = n;
        const uint64_t kth = __shfl_sync(0xffffffffu, list, a.top - 1);
        if (kth) {
            bound = fmaxf(bound, key_value(kth));
            if (lane == 0) {
                const int b = __float_as_int(below(key_value(kth)));
                atomicMax(&shared_bound, b >= 0 ? b : b ^ 0x7fffffff);  // float order as int order
            }
        }
        __syncwarp();
    };
    auto push = [&](float v, int i) {
        if (v > bound) buffer[atomicAdd(&counts[warp], 1)] = key_of(v, i);
    };
    auto add = [&](float v) {
        if (v > p.m) {
            const Part q = join(p, Part{v, 0.f, 0.f});
            p = q;
        }
        const float d = v - (p.m == -INFINITY ? 0.f : p.m), e = exp_fast(d);
        p.l += e;
        p.s += e * fmaxf(d, -200.f);  // e is zero there: no 0 * inf
    };

    // values before the first vector: the first warp of the first CTA, before all higher indices
    if (rank == 0 && warp == 0 && head > 0) {
        if (lane < head) {
            const float v = value_of(x, lane);
            add(v);
            if constexpr (kTop) push(v, lane);
        }
        if constexpr (kTop) take(false);
    }
    const T* xv = x + head;
    constexpr int kStep = 32 * U;  // vectors a warp takes at a time, consecutive ones
    for (int v0 = v_lo + warp * kStep; v0 < v_hi; v0 += kLpWarps * kStep) {
        Vec<T> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = v0 + u * 32 + lane;
            if (v < v_hi) r[u].load(xv + (long long)v * V);
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v0 + u * 32 + lane < v_hi)
#pragma unroll
                for (int i = 0; i < V; ++i) top = fmaxf(top, r[u].get(i));
        if (top > p.m) p = join(p, Part{top, 0.f, 0.f});
        const float m = p.m == -INFINITY ? 0.f : p.m;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v0 + u * 32 + lane < v_hi)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = r[u].get(i) - m, e = exp_fast(d);
                    p.l += e;
                    p.s += e * fmaxf(d, -200.f);
                }
        if constexpr (kTop) {
            const int sb = *reinterpret_cast<volatile int*>(&shared_bound);
            if (sb != INT_MIN) bound = fmaxf(bound, __int_as_float(sb >= 0 ? sb : sb ^ 0x7fffffff));
            if (bound == -INFINITY) {
                // nothing to compare with yet: the k-th largest of the lanes'
                // own largest values is no larger than the k-th of them all
                const uint64_t k = sort32(key_of(top, lane), lane);
                bound = fmaxf(bound, below(key_value(__shfl_sync(0xffffffffu, k, a.top - 1))));
            }
            if (__any_sync(0xffffffffu, top > bound)) {
                if (top > bound) {
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (v0 + u * 32 + lane < v_hi)
#pragma unroll
                            for (int i = 0; i < V; ++i) push(r[u].get(i), head + (v0 + u * 32 + lane) * V + i);
                }
                take(false);
            }
        }
    }
    // values past the last vector: the last warp of the last CTA
    if (rank == cluster - 1 && warp == kLpWarps - 1 && tail < a.vocab) {
        if (tail + lane < a.vocab) {
            const float v = value_of(x, tail + lane);
            add(v);
            if constexpr (kTop) push(v, tail + lane);
        }
    }

#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
        p = join(p, Part{__shfl_xor_sync(0xffffffffu, p.m, off), __shfl_xor_sync(0xffffffffu, p.l, off),
                         __shfl_xor_sync(0xffffffffu, p.s, off)});
    if (lane == 0) parts[warp] = p;
    if constexpr (kTop) {
        take(true);
        lists[warp * 32 + lane] = list;
    }
    __syncthreads();
    if constexpr (kTop) {
        for (int half = kLpWarps / 2; half > 0; half >>= 1) {
            if (warp < half) {
                list = merge32(lists[warp * 32 + lane], lists[(warp + half) * 32 + lane], lane);
                lists[warp * 32 + lane] = list;
            }
            __syncthreads();
        }
    }
    if (warp == 0) {
        p = parts[lane % kLpWarps];  // both halves of the warp form the same sum
#pragma unroll
        for (int off = kLpWarps / 2; off > 0; off >>= 1)
            p = join(p, Part{__shfl_xor_sync(0xffffffffu, p.m, off), __shfl_xor_sync(0xffffffffu, p.l, off),
                             __shfl_xor_sync(0xffffffffu, p.s, off)});
        if (lane == 0) cta_part = p;
    }
    if (cluster > 1) {
        cl.sync();
        if (rank == 0 && warp == 0) {
            for (int r = 1; r < cluster; ++r) {
                p = join(p, *cl.map_shared_rank(&cta_part, r));
                if constexpr (kTop) list = merge32(list, *cl.map_shared_rank(lists + lane, r), lane);
            }
        }
        cl.sync();  // no CTA leaves while its memory may still be read
    }
    if (rank != 0 || warp != 0) return;
    const float log_l = logf(p.l);
    if (lane == 0) {
        // a row with nothing but -inf has no distribution: probability zero, no entropy
        const bool empty = p.m == -INFINITY && p.l == 0.f;
        if (a.entropy) a.entropy[row] = empty ? 0.f : log_l - p.s / p.l;
        if (a.logprob) {
            const int t = a.target[row];
            const bool ok = t >= 0 && t < a.vocab;
            a.logprob[row] = !ok || empty ? -INFINITY : value_of(x, t) - p.m - log_l;
        }
    }
    if constexpr (kTop) {
        if (lane < a.top) {
            const long long o = row * a.top + lane;
            const float v = key_value(list);
            a.top_ids[o] = list ? key_index(list) : -1;
            a.top_logprobs[o] = list ? v - p.m - log_l : -INFINITY;
        }
    }
}

template <typename T, bool kTop>
cudaError_t launch_logprobs(const LpArgs& a, int n_rows, int cluster, cudaStream_t st) {
    auto kernel = logprobs_kernel<T, kTop>;
    const size_t smem = lp_smem<kTop>();
    if (cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), (int)smem)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n_rows * (unsigned)cluster);
    cfg.blockDim = dim3(kLpThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a, cluster);
}

}  // namespace
}  // namespace glmq

extern "C" int glm_cuda_logprobs_async(const void* logits_dev, int type, int64_t row_stride, int n_rows, int vocab,
                                       const int32_t* target_dev, float* logprob_dev, float* entropy_dev, int top_k,
                                       int32_t* top_ids_dev, float* top_logprobs_dev, void* stream) {
    using namespace glmq;
    const char* fn = "glm_cuda_logprobs_async";
    if (!known_type(type)) return op_fail(GLM_CUDA_ERR_ARG, fn, "unknown type %d", type);
    if (n_rows < 0 || n_rows > 1 << 24 || vocab < 1 || vocab > 1 << 30 || row_stride < vocab)
        return op_fail(GLM_CUDA_ERR_ARG, fn, "n_rows=%d vocab=%d row_stride=%lld", n_rows, vocab, (long long)row_stride);
    if (top_k < 0 || top_k > kLpMaxTop) return op_fail(GLM_CUDA_ERR_ARG, fn, "top_k=%d (need 0..%d)", top_k, kLpMaxTop);
    if (n_rows == 0) return 0;
    if (!logits_dev || !aligned(logits_dev, type_bytes(type))) return op_fail(GLM_CUDA_ERR_ARG, fn, "logits NULL or not aligned to their type");
    if ((target_dev != nullptr) != (logprob_dev != nullptr)) return op_fail(GLM_CUDA_ERR_ARG, fn, "target and logprob go together");
    if (top_k > 0 && (!top_ids_dev || !top_logprobs_dev)) return op_fail(GLM_CUDA_ERR_ARG, fn, "top_k=%d without its outputs", top_k);
    int sms = 0;
    if (cudaError_t e = current_sms(&sms)) return launch_failed(fn, e);
    // CTAs to a row: the most that leave no more CTAs than SMs, up to the
    // portable cluster size
    int cluster = 1;
    while (cluster < kLpMaxCluster && (long long)n_rows * cluster * 2 <= sms) cluster *= 2;
    LpArgs a{logits_dev, row_stride, vocab, top_k, target_dev, logprob_dev, entropy_dev, top_ids_dev, top_logprobs_dev};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    try {
        cudaError_t e;
        if (type == GLM_CUDA_F32)
            e = top_k ? launch_logprobs<float, true>(a, n_rows, cluster, st) : launch_logprobs<float, false>(a, n_rows, cluster, st);
        else if (type == GLM_CUDA_BF16)
            e = top_k ? launch_logprobs<__nv_bfloat16, true>(a, n_rows, cluster, st)
                      : launch_logprobs<__nv_bfloat16, false>(a, n_rows, cluster, st);
        else
            e = top_k ? launch_logprobs<__half, true>(a, n_rows, cluster, st) : launch_logprobs<__half, false>(a, n_rows, cluster, st);
        if (e) return launch_failed(fn, e);
        count_launches(1);
    } catch (...) {
        return op_fail(GLM_CUDA_ERR_NOMEM, fn, "host allocation failed");
    }
    return 0;
}
