// Layout of the 4-bit latent cache.
//
// A position's row is its compressed key (kv_lora latents) followed by the
// rope part of its key, as mla_cluster_kernel caches them in fp32 (model.h's
// k_cache_comp and k_cache_pe). An element is stored as the code v + 8 with v
// in [-7, 7] and is worth v * s, with one bf16 scale s for every 128 latents
// and one for the rope part. A page holds `page` positions:
//   codes  [page][(kv_lora + rope) / 2]   element 2b in the low, 2b + 1 in the high half of byte b
//   scales [kv_lora / 128 + 1][page]      bf16
// 298 bytes a position at 512 + 64, against 2304 in fp32.
//
// Why 128 latents to a scale: the attention's second product sums over
// positions, so the scale has to be multiplied into the probabilities, once
// for every group of latents; 4 groups cost a tenth of that kernel's
// arithmetic, 16 groups of 32 would cost more than its products. For normal
// data a group of 128 costs 1.9 dB of signal to noise against one of 32 (19.7
// against 21.6 dB) and 7.5 % fewer bytes.
//
// Why the code is v + 8: put into the low mantissa bits of the f16 number 1024
// it is 1024 + v + 8 exactly, so that one packed subtraction turns two codes
// into tensor-core operands, without a sign to extend.
#pragma once

#include <cstddef>
#include <cstdint>

namespace glmq {

constexpr int kKv4Group = 128;       // latents to a scale
constexpr int kKv4MaxGroups = 5;     // 4 of 128 latents and the rope part's

struct Kv4Shape {
    int kv_lora, rope, page;
    __host__ __device__ constexpr int row_bytes() const { return (kv_lora + rope) / 2; }
    __host__ __device__ constexpr int groups() const { return kv_lora / kKv4Group + 1; }
    __host__ __device__ constexpr size_t page_bytes() const {
        return (size_t)page * (size_t)(row_bytes() + 2 * groups());
    }
};

// Row bytes are a multiple of 32 and a page of 16 positions a multiple of 16
// bytes, so that every page starts on a 16-byte boundary.
inline bool kv4_shape_ok(int kv_lora, int rope, int page) {
    return kv_lora > 0 && kv_lora <= 512 && kv_lora % kKv4Group == 0 && (rope == 64 || rope == 128) &&
           (page == 16 || page == 32 || page == 64 || page == 128 || page == 256);
}

}  // namespace glmq
