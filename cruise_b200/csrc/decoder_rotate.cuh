// decoder_rotate.cuh -- norms of queries and keys for each head, the position
// rotation and the write into the paged cache, in one pass.
//
// For a head vector x of q or k (norm weights given):
//   y = x * rsqrt(mean(x^2) + eps) * w,
//   z_i = y_i cos_i - y_{i+h} sin_i,  z_{i+h} = y_{i+h} cos_{i+h} + y_i sin_{i+h}   (i < h = rotary / 2)
// and z = y beyond `rotary`.  q goes to q_out, k and v to the token's cache
// slot.  Sums, norms and the rotation are in fp32, rounded once to the stored type.
#pragma once

#include "decoder_common.cuh"
#include "decoder_ops.h"

namespace cruise {
namespace ops {

constexpr int kRotateThreads = 256;

// 16 bytes (8 elements) per lane: D / 8 lanes share a head, so a warp moves
// 32 * 8 / D heads of one token per round and takes `rounds` rounds; the
// token's table row stays in registers over them.
template <typename T, int D>
__global__ void __launch_bounds__(kRotateThreads) rotate_store_kernel(const RotateArgs a, int rounds, int warps_per_token) {
  constexpr int kLanes = D / 8;
  constexpr int kHeads = 32 / kLanes;
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * kRotateThreads + threadIdx.x) >> 5;
  const int64_t t = warp / warps_per_token;
  if (t >= a.tokens) return;   // uniform over the warp
  const int first = static_cast<int>(warp - t * warps_per_token) * rounds;
  const int lane = threadIdx.x & 31;
  const int chunk = lane % kLanes, sub = lane / kLanes;
  const int64_t pos = a.position[t];
  const int32_t slot = a.slot[t];
  const bool known = pos >= 0 && pos < a.rope_rows;
  const bool stored = known && slot >= 0 && slot < a.num_blocks * a.block_size;
  const int half = a.rotary / 16;   // chunks in half the rotated part
  const bool turns = chunk < 2 * half;
  const int partner = (lane & ~(kLanes - 1)) | (turns ? (chunk < half ? chunk + half : chunk - half) : chunk);
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) cs[i] = 1.f, sn[i] = 0.f;
  if (known && turns) {
    const int64_t at = pos * a.rotary + chunk * 8;
    if (a.rope_dtype == kFp32) {
      const float4 *c = reinterpret_cast<const float4 *>(static_cast<const float *>(a.rope_cos) + at);
      const float4 *s = reinterpret_cast<const float4 *>(static_cast<const float *>(a.rope_sin) + at);
      const float4 c0 = c[0], c1 = c[1], s0 = s[0], s1 = s[1];
      cs[0] = c0.x; cs[1] = c0.y; cs[2] = c0.z; cs[3] = c0.w; cs[4] = c1.x; cs[5] = c1.y; cs[6] = c1.z; cs[7] = c1.w;
      sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w; sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
    } else {
      unpack8<__nv_bfloat16>(*reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(a.rope_cos) + at), cs);
      unpack8<__nv_bfloat16>(*reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(a.rope_sin) + at), sn);
    }
    if (chunk < half) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sn[i] = -sn[i];
    }
  }
  const bool norm = a.q_norm != nullptr;
  uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
  if (norm) {
    wq = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q_norm) + chunk * 8);
    wk = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.k_norm) + chunk * 8);
  }
  const T *src = static_cast<const T *>(a.qkv) + t * a.qkv_stride + chunk * 8;
  T *q_dst = static_cast<T *>(a.q_out) + t * a.q_stride + chunk * 8;
  const int64_t cell = stored ? (slot / a.block_size) * a.block_stride +
                                    static_cast<int64_t>(slot % a.block_size) * a.nkv * D + chunk * 8
                              : 0;
  T *k_dst = static_cast<T *>(a.key_cache) + cell;
  T *v_dst = static_cast<T *>(a.value_cache) + cell;
  const int heads = a.nq + 2 * a.nkv;
  const int last = min(heads, (first + rounds) * kHeads);
#pragma unroll 4
  for (int base = first * kHeads; base < last; base += kHeads) {
    const int head = base + sub;
    const bool live = head < heads;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live) raw = *reinterpret_cast<const uint4 *>(src + static_cast<int64_t>(head) * D);
    if (base >= a.nq + a.nkv) {   // v heads only: copied as they are
      if (live && stored)
        *reinterpret_cast<uint4 *>(v_dst + static_cast<int64_t>(head - a.nq - a.nkv) * D) = raw;
      continue;
    }
    float y[8];
    unpack8<T>(raw, y);
    if (norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(ss * (1.f / D) + a.eps);
      float w[8];
      unpack8<T>(head < a.nq ? wq : wk, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * inv * w[i];
    }
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_sync(0xffffffffu, y[i], partner);
      z[i] = turns ? fmaf(other, sn[i], y[i] * cs[i]) : y[i];
    }
    if (!live) continue;
    if (head < a.nq) {
      *reinterpret_cast<uint4 *>(q_dst + static_cast<int64_t>(head) * D) = known ? pack8<T>(z) : make_uint4(0, 0, 0, 0);
    } else if (stored) {
      if (head < a.nq + a.nkv)
        *reinterpret_cast<uint4 *>(k_dst + static_cast<int64_t>(head - a.nq) * D) = pack8<T>(z);
      else
        *reinterpret_cast<uint4 *>(v_dst + static_cast<int64_t>(head - a.nq - a.nkv) * D) = raw;
    }
  }
}

}  // namespace ops
}  // namespace cruise
