// Host-side helpers shared by the entry points that serve many requests over
// the 4-bit latent cache (kv_plan.cu, kv4_cache.cu, mla4_attention.cu,
// logprobs.cu). These calls keep no state of their own: they need no
// glm_cuda_init, use the current device and allocate nothing.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

#include "glm_cuda.h"

namespace glmq {

// Record and print "<fn>: <message>" as glm_cuda_last_error() reports it; returns `code`.
int op_fail(int code, const char* fn, const char* fmt, ...);

// The current device's SM count (asked for once per device).
cudaError_t current_sms(int* sms);

// Add to glm_cuda_launch_count().
void count_launches(int n);

// GLM_CUDA_ERR_* of a failed launch, with its message.
int launch_failed(const char* fn, cudaError_t e);

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

inline size_t type_bytes(int type) { return type == GLM_CUDA_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == GLM_CUDA_F32 || type == GLM_CUDA_BF16 || type == GLM_CUDA_F16; }

// 0, or the error of a cache description that no call takes.
int check_kv4_cache(const char* fn, const GlmCudaKv4Cache* c);

}  // namespace glmq
