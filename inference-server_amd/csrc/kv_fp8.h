// The 8-bit KV pages that the writers (kv_fp8.hip) fill and the attention (attn_fp8.hip) reads: e4m3 codes,
// 2 KB per (page of 16 tokens, kv head) for K and as much for V, each with one fp32 scale that is a power of two.
//   K block [dim / 16][token 16][dim % 16]: the 16 bytes of 16 consecutive lanes are 16 tokens' codes of 16
//     dims, an MFMA operand's rows as they lie, and a wave's 16-byte loads cover 1 KB in a row.
//   V block [dim / 64][token / 4][dim % 64][token % 4]: a lane's 16 bytes are 4 dims of 4 tokens, which is how
//     the softmax's probabilities come out of the score MFMA (4 keys per lane), so they need no transpose.
// A scale that is a power of two loses nothing against amax / 448 (e4m3 is a floating-point format: only where its
// subnormals begin moves, by less than one binade), v_cvt_scalef32_pk_bf16_fp8 applies it in the conversion
// itself and exactly, and a page whose scale grows as it fills is re-coded without a second rounding of its
// normal values.
#pragma once

#include "common.h"

constexpr int kKvHead = 128;                    // head dim
constexpr int kKvBlock = 16 * kKvHead;          // bytes per (page, kv head) of K or V
constexpr uint32_t kKvMinScale = 27u << 23;     // 2^-100

// The smallest power of two s with amax / s <= 448 = 1.75 * 2^8, at least 2^-100.
__device__ __forceinline__ float kv_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(max(e, (int)(kKvMinScale >> 23)) << 23);
}

// 4 e4m3 codes of x / s, saturated; NaN stays NaN (the clamp alone would make it -448).
__device__ __forceinline__ uint32_t kv_pack4(float a, float b, float c, float d, float inv) {
  const float x[4] = {a * inv, b * inv, c * inv, d * inv};
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = x[i] == x[i] ? clamp_fp8(x[i]) : x[i];
  return pack4_e4m3(y[0], y[1], y[2], y[3]);
}

// 4 codes under scale s to codes under the scale s / ratio.
__device__ __forceinline__ uint32_t kv_recode4(uint32_t codes, float ratio) {
  return kv_pack4(__builtin_amdgcn_cvt_f32_fp8(codes, 0), __builtin_amdgcn_cvt_f32_fp8(codes, 1),
                  __builtin_amdgcn_cvt_f32_fp8(codes, 2), __builtin_amdgcn_cvt_f32_fp8(codes, 3), ratio);
}
