// decoder_rotate.cuh -- norms of queries and keys for each head, the position
// rotation and the write into the paged cache, in one pass.
//
// For a head vector x of q or k (norm weights given):
//   y = x * rsqrt(mean(x^2) + eps) * w,
//   z_i = y_i cos_i - y_{i+h} sin_i,  z_{i+h} = y_{i+h} cos_{i+h} + y_i sin_{i+h}   (i < h = rotary / 2)
// and z = y beyond `rotary`.  q goes to q_out, k and v to the token's cache
// slot.  Sums, norms and the rotation are in fp32, rounded once to the stored type.
//
// What bounds it is bytes, each read and written once: 8192 tokens of 28 + 2 x 4
// heads of 128 with norms take 31.0 us, 77% of the copy bandwidth.  What is left
// is the fp32 work between: the SMs issue in 53% of their cycles and wait for
// loads in the rest.  Few tokens are bounded by the start and one round trip
// (4 tokens: 2.1 us).
#pragma once

#include "decoder_common.cuh"
#include "decoder_ops.h"

namespace cruise {
namespace ops {

// 8192 tokens: 31.0 us with five CTAs per SM, 35.2 with four (six would leave 85
// registers for the 96 in use); 31.0 with three rounds of loads in flight, 35.9 with two.
constexpr int kRotateThreads = 128;
constexpr int kRotateCtas = 5;    // CTAs per SM
constexpr int kRotateBatch = 3;

// Two fp32 operations in one instruction (8192 tokens: 35.1 us with single ones, 31.0 so).
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<uint64_t *>(&r))
      : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<uint64_t *>(&r))
      : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)), "l"(*reinterpret_cast<uint64_t *>(&c)));
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack2(const uint4 &u, float2 (&v)[4]) {
  v[0] = Element<T>::unpack(u.x);
  v[1] = Element<T>::unpack(u.y);
  v[2] = Element<T>::unpack(u.z);
  v[3] = Element<T>::unpack(u.w);
}

template <typename T>
__device__ __forceinline__ uint4 pack2(const float2 (&v)[4]) {
  return make_uint4(Element<T>::pack(v[0].x, v[0].y), Element<T>::pack(v[1].x, v[1].y), Element<T>::pack(v[2].x, v[2].y),
                    Element<T>::pack(v[3].x, v[3].y));
}

// Eight table entries.
__device__ __forceinline__ void table8(const void *table, int32_t type, int64_t at, float2 (&v)[4]) {
  if (type == kFp32) {
    const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(table) + at);
    const float4 a = p[0], b = p[1];
    v[0] = make_float2(a.x, a.y);
    v[1] = make_float2(a.z, a.w);
    v[2] = make_float2(b.x, b.y);
    v[3] = make_float2(b.z, b.w);
  } else {
    unpack2<__nv_bfloat16>(*reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(table) + at), v);
  }
}

// A lane holds two 16-byte chunks of a head: a chunk of the rotated part's
// first half and its partner half a rotation further (or two neighbours behind
// the rotated part), so the rotation needs no exchange between lanes.  D / 16
// lanes share a head, a warp moves 512 / D heads of one token and one kind (q,
// k or v) per round and takes `rounds` rounds of the token's.  Norm weights and
// table entries become one factor per element, z_lo = inv (x_lo c_lo + x_hi s_lo),
// kept in registers over the token's heads.  kRotateBatch rounds of loads are in
// flight before their first use.  Where the whole head is rotated no lane asks
// whether its chunks are (8192 tokens: 33 us asking, 31.0 not).
template <typename T, int D, bool Norm, bool Full>
__global__ void __launch_bounds__(kRotateThreads, kRotateCtas) rotate_store_kernel(const RotateArgs a, int rounds, int warps_per_token) {
  constexpr int kLanes = D / 16;
  constexpr int kHeads = 32 / kLanes;
  follow_predecessor();
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * kRotateThreads + threadIdx.x) >> 5;
  const int64_t t = warp / warps_per_token;
  if (t >= a.tokens) return;   // uniform over the warp
  const int lane = threadIdx.x & 31;
  const int j = lane % kLanes, sub = lane / kLanes;
  const int half = a.rotary / 16;   // chunks in half the rotated part
  const bool turns = Full || j < half;   // Full: the whole head is rotated
  const int lo = (turns ? j : 2 * j) * 8, step = (turns ? half : 1) * 8;   // this lane's elements of a head: lo, lo + step
  const int q_rounds = (a.nq + kHeads - 1) / kHeads, k_rounds = (a.nkv + kHeads - 1) / kHeads;
  const int first = static_cast<int>(warp - t * warps_per_token) * rounds;
  const int last = min(q_rounds + 2 * k_rounds, first + rounds);
  const T *src = static_cast<const T *>(a.qkv) + t * a.qkv_stride + lo;
  // of round r: its kind (0 q, 1 k, 2 v) and this lane's head of that kind
  auto kind_of = [&](int r) { return r < q_rounds ? 0 : r < q_rounds + k_rounds ? 1 : 2; };
  auto head_of = [&](int r, int kind) { return (r - (kind == 0 ? 0 : kind == 1 ? q_rounds : q_rounds + k_rounds)) * kHeads + sub; };
  uint4 raw[kRotateBatch][2];
  auto load = [&](int r0) {
#pragma unroll
    for (int b = 0; b < kRotateBatch; ++b) {
      const int r = r0 + b, kind = kind_of(r), head = head_of(r, kind);
      raw[b][0] = raw[b][1] = make_uint4(0, 0, 0, 0);
      if (r < last && head < (kind == 0 ? a.nq : a.nkv)) {
        const T *x = src + ((kind == 0 ? 0 : kind == 1 ? a.nq : a.nq + a.nkv) + head) * D;
        raw[b][0] = *reinterpret_cast<const uint4 *>(x);
        raw[b][1] = *reinterpret_cast<const uint4 *>(x + step);
      }
    }
  };
  load(first);
  const int64_t pos = a.position[t];
  const int32_t slot = a.slot[t];
  const bool known = pos >= 0 && pos < a.rope_rows;
  const bool stored = slot >= 0 && slot < a.num_blocks * a.block_size;
  T *q_dst = static_cast<T *>(a.q_out) + t * a.q_stride + lo;
  if (!known) {   // uniform over the warp: zeros, nothing stored
    for (int head = first * kHeads + sub; head < min(a.nq, last * kHeads); head += kHeads)
      *reinterpret_cast<uint4 *>(q_dst + head * D) = *reinterpret_cast<uint4 *>(q_dst + head * D + step) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int64_t cell =
      (stored ? (slot / a.block_size) * a.block_stride + static_cast<int64_t>(slot % a.block_size) * a.nkv * D : 0) + lo;
  // z_lo = x_lo c_lo + x_hi s_lo, z_hi = x_hi c_hi + x_lo s_hi (times the head's inverse norm)
  float2 c_lo[4], c_hi[4], s_lo[4], s_hi[4];
  auto factors = [&](const void *weights) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c_lo[i] = c_hi[i] = make_float2(1.f, 1.f);
      s_lo[i] = s_hi[i] = make_float2(0.f, 0.f);
    }
    if (turns) {
      const int64_t at = pos * a.rotary + lo;
      table8(a.rope_cos, a.rope_dtype, at, c_lo);
      table8(a.rope_cos, a.rope_dtype, at + step, c_hi);
      table8(a.rope_sin, a.rope_dtype, at, s_lo);
      table8(a.rope_sin, a.rope_dtype, at + step, s_hi);
    }
    if (Norm) {
      float2 w_lo[4], w_hi[4];
      unpack2<T>(*reinterpret_cast<const uint4 *>(static_cast<const T *>(weights) + lo), w_lo);
      unpack2<T>(*reinterpret_cast<const uint4 *>(static_cast<const T *>(weights) + lo + step), w_hi);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c_lo[i] = mul2(c_lo[i], w_lo[i]);
        c_hi[i] = mul2(c_hi[i], w_hi[i]);
        s_lo[i] = mul2(s_lo[i], w_hi[i]);
        s_hi[i] = mul2(s_hi[i], w_lo[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s_lo[i] = make_float2(-s_lo[i].x, -s_lo[i].y);
  };
  int built = kind_of(first);
  if (built < 2) factors(built == 0 ? a.q_norm : a.k_norm);
  for (int r0 = first; r0 < last; r0 += kRotateBatch) {
    if (r0 > first) load(r0);
#pragma unroll
    for (int b = 0; b < kRotateBatch; ++b) {
      const int r = r0 + b;
      if (r >= last) break;
      const int kind = kind_of(r), head = head_of(r, kind);   // the kind is uniform over the warp
      if (kind < 2) {
        if (Norm && kind != built) factors(a.k_norm);
        built = kind;
        float2 x_lo[4], x_hi[4], z_lo[4], z_hi[4];
        unpack2<T>(raw[b][0], x_lo);
        unpack2<T>(raw[b][1], x_hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          z_lo[i] = mul2(x_lo[i], c_lo[i]);
          z_hi[i] = mul2(x_hi[i], c_hi[i]);
          if (turns) {
            z_lo[i] = fma2(x_hi[i], s_lo[i], z_lo[i]);
            z_hi[i] = fma2(x_lo[i], s_hi[i], z_hi[i]);
          }
        }
        if (Norm) {
          float2 s0 = mul2(x_lo[0], x_lo[0]), s1 = mul2(x_hi[0], x_hi[0]);
#pragma unroll
          for (int i = 1; i < 4; ++i) {
            s0 = fma2(x_lo[i], x_lo[i], s0);
            s1 = fma2(x_hi[i], x_hi[i], s1);
          }
          float sum = (s0.x + s0.y) + (s1.x + s1.y);
#pragma unroll
          for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float inv = rsqrtf(sum * (1.f / D) + a.eps);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            z_lo[i] = mul2(z_lo[i], make_float2(inv, inv));
            z_hi[i] = mul2(z_hi[i], make_float2(inv, inv));
          }
        }
        raw[b][0] = pack2<T>(z_lo);
        raw[b][1] = pack2<T>(z_hi);
      }
      if (kind == 0) {
        if (head < a.nq) {
          T *dst = q_dst + head * D;
          *reinterpret_cast<uint4 *>(dst) = raw[b][0];
          *reinterpret_cast<uint4 *>(dst + step) = raw[b][1];
        }
      } else if (stored && head < a.nkv) {
        T *dst = static_cast<T *>(kind == 1 ? a.key_cache : a.value_cache) + cell + head * D;
        *reinterpret_cast<uint4 *>(dst) = raw[b][0];
        *reinterpret_cast<uint4 *>(dst + step) = raw[b][1];
      }
    }
  }
}

}  // namespace ops
}  // namespace cruise
