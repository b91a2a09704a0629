// MLA attention of single tokens over the paged 4-bit latent cache:
// glm_cuda_mla4_attention_async. glm.c runs the same attention for its one
// sequence over fp32 rows (infer.c:1003-1058).
//
// Row r is one query token: request row_req[r], position row_pos[r]; it sees
// the positions 0 .. row_pos[r] of its request. With the absorbed query
// q = (k_b_h q_nope, roped q_pe) of head h and the cached row k_t
//   x_t = scale * q . k_t,   p = softmax(x),   out[h] = sum_t p_t k_t[0 .. kv_lora)
//   lse[h] = ln sum_t e^(x_t)
// A position whose page is not in the pool is not seen. A row that sees
// nothing gives zeros and lse = -inf.
//
// Simple form: one CTA per (row, head), a warp per position with the running
// maximum and sum of the softmax, the warps joined at the end.
#include <cfloat>
#include <cmath>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "glm_internal.h"
#include "kv4.cuh"
#include "q80_common.cuh"
#include "serve_common.h"

namespace glmq {
namespace {

constexpr int kAtWarps = 8, kAtThreads = kAtWarps * 32;

struct Mla4Args {
    Kv4Shape sh;
    const unsigned char* pages;
    long long n_pages;
    const void* q;
    long long q_row, q_head;
    const int32_t* table;
    int table_stride, n_req;
    const int32_t *row_req, *row_pos;
    int n_heads;
    float scale;
    void* out;
    long long out_row, out_head;
    float* lse;
};

__device__ __forceinline__ float load_q(const void* q, long long i, int type) {
    if (type == GLM_CUDA_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(q)[i]);
    return __half2float(static_cast<const __half*>(q)[i]);
}

__global__ void __launch_bounds__(kAtThreads) mla4_attention_kernel(Mla4Args a, int type) {
    __shared__ float q[640], acc_s[kAtWarps][512], m_s[kAtWarps], l_s[kAtWarps];
    pdl_enter();
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int dim = a.sh.kv_lora + a.sh.rope;
    for (int i = threadIdx.x; i < dim; i += kAtThreads) q[i] = load_q(a.q, row * a.q_row + h * a.q_head + i, type);
    __syncthreads();
    const int req = a.row_req[row];
    long long len = req >= 0 && req < a.n_req ? (long long)a.row_pos[row] + 1 : 0;
    len = min(len, (long long)a.table_stride * a.sh.page);
    float m = -INFINITY, l = 0.f, acc[16] = {};
    for (long long t = warp; t < len; t += kAtWarps) {
        const int page = a.table[(size_t)req * a.table_stride + t / a.sh.page], at = (int)(t % a.sh.page);
        if (page < 0 || page >= a.n_pages) continue;
        const unsigned char* p = a.pages + (size_t)page * a.sh.page_bytes();
        const __nv_bfloat16* sc = reinterpret_cast<const __nv_bfloat16*>(p + (size_t)a.sh.page * a.sh.row_bytes());
        float x = 0.f, v[20];
#pragma unroll
        for (int i = 0; i < 20; ++i) {
            const int e = i * 32 + lane;
            v[i] = 0.f;
            if (e >= dim) continue;
            const unsigned b = p[(size_t)at * a.sh.row_bytes() + e / 2];
            const int g = min(e / kKv4Group, a.sh.groups() - 1);
            v[i] = (float)((int)((e & 1 ? b >> 4 : b) & 15u) - 8) * __bfloat162float(sc[g * a.sh.page + at]);
            x += q[e] * v[i];
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
        x *= a.scale;
        const float mn = fmaxf(m, x), w = m == -INFINITY ? 0.f : expf(m - mn), e = expf(x - mn);
        m = mn;
        l = l * w + e;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = acc[i] * w + e * v[i];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) acc_s[warp][i * 32 + lane] = acc[i];
    if (lane == 0) {
        m_s[warp] = m;
        l_s[warp] = l;
    }
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < kAtWarps; ++w) M = fmaxf(M, m_s[w]);
    for (int w = 0; w < kAtWarps; ++w) L += m_s[w] == -INFINITY ? l_s[w] : l_s[w] * expf(m_s[w] - M);
    for (int i = threadIdx.x; i < a.sh.kv_lora; i += kAtThreads) {
        float o = 0.f;
        for (int w = 0; w < kAtWarps; ++w) o += m_s[w] == -INFINITY ? acc_s[w][i] : acc_s[w][i] * expf(m_s[w] - M);
        if (L != 0.f) o /= L;
        const long long at = row * a.out_row + h * a.out_head + i;
        if (type == GLM_CUDA_BF16)
            static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(o);
        else
            static_cast<__half*>(a.out)[at] = __float2half_rn(o);
    }
    if (a.lse && threadIdx.x == 0) a.lse[(size_t)row * a.n_heads + h] = M + logf(L);
}

}  // namespace
}  // namespace glmq

extern "C" size_t glm_cuda_mla4_workspace_bytes(int n_rows, int n_heads, int kv_lora_rank) {
    if (n_rows < 1 || n_heads < 1 || kv_lora_rank < 1) return 0;
    return 16;
}

extern "C" int glm_cuda_mla4_attention_async(const GlmCudaKv4Cache* cache, const void* q_dev, int type,
                                             int64_t q_row_stride, int64_t q_head_stride, const int32_t* block_table_dev,
                                             int table_stride, int n_req, const int32_t* row_req_dev,
                                             const int32_t* row_pos_dev, int n_rows, int n_heads, float scale,
                                             void* out_dev, int64_t out_row_stride, int64_t out_head_stride,
                                             float* lse_dev, void* ws_dev, size_t ws_bytes, void* stream) {
    using namespace glmq;
    const char* fn = "glm_cuda_mla4_attention_async";
    if (int rc = check_kv4_cache(fn, cache)) return rc;
    if (type != GLM_CUDA_BF16 && type != GLM_CUDA_F16) return op_fail(GLM_CUDA_ERR_ARG, fn, "type %d (need bf16 or f16)", type);
    if (n_rows < 0 || n_rows > 16384 || n_heads < 1 || n_heads > 256 || n_req < 1 || table_stride < 1)
        return op_fail(GLM_CUDA_ERR_ARG, fn, "n_rows=%d n_heads=%d n_req=%d table_stride=%d", n_rows, n_heads, n_req, table_stride);
    if (n_rows == 0) return 0;
    if (!q_dev || !block_table_dev || !row_req_dev || !row_pos_dev || !out_dev || !ws_dev)
        return op_fail(GLM_CUDA_ERR_ARG, fn, "a required pointer is NULL");
    if (!aligned(q_dev, 2) || !aligned(out_dev, 2) || !aligned(ws_dev, 16))
        return op_fail(GLM_CUDA_ERR_ARG, fn, "a pointer is not aligned (16 bytes for the workspace)");
    if (ws_bytes < glm_cuda_mla4_workspace_bytes(n_rows, n_heads, cache->kv_lora_rank))
        return op_fail(GLM_CUDA_ERR_ARG, fn, "workspace of %zu bytes (need %zu)", ws_bytes,
                       glm_cuda_mla4_workspace_bytes(n_rows, n_heads, cache->kv_lora_rank));
    Mla4Args a{Kv4Shape{cache->kv_lora_rank, cache->rope_dim, cache->page_size},
               static_cast<const unsigned char*>(cache->pages), cache->n_pages, q_dev, q_row_stride, q_head_stride,
               block_table_dev, table_stride, n_req, row_req_dev, row_pos_dev, n_heads, scale, out_dev,
               out_row_stride, out_head_stride, lse_dev};
    cudaError_t e = launch_pdl(mla4_attention_kernel, dim3(n_rows, n_heads), kAtThreads, 0,
                               static_cast<cudaStream_t>(stream), a, type);
    if (e) return launch_failed(fn, e);
    count_launches(1);
    return 0;
}
