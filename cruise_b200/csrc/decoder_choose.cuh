// decoder_choose.cuh -- rules on the logits and the greedy choice, in one pass.
//
// Per row, for every token n of the vocabulary, in fp32 and in this order:
//   x = logit (+ the token's bias);
//   in the row's history (prompt or output): x = x > 0 ? x / repetition : x * repetition;
//   x = x - frequency * count, x = x - presence * [count > 0], count its occurrences in the output;
//   not allowed by the row's bit mask: x = -inf.
// The choice is the first maximum above -inf: -1 where there is none, -2 where
// an x is NaN or +inf.  Each step is one rounded fp32 operation, so the choice
// equals that of the same steps done one by one.
//
// A cluster of CTAs shares a row.  Each CTA keeps a 32-bit word per token of
// its slice in shared memory (occurrences, "in the prompt", "has a bias"),
// filled from the row's history; the slices' maxima meet in the first CTA's
// shared memory, so a call is one launch and keeps no state.
#pragma once

#include <climits>

#include "decoder_common.cuh"
#include "decoder_ops.h"

namespace cruise {
namespace ops {

constexpr int kChooseThreads = 512;
constexpr int kChooseMaxCluster = 16;
constexpr uint32_t kInPrompt = 0x80000000u, kHasBias = 0x40000000u, kCount = 0x3fffffffu;

struct ChooseBest {
  float value;
  int32_t index;
  int32_t bad;
};

__device__ __forceinline__ void better(ChooseBest &a, float value, int32_t index) {
  if (value > a.value || (value == a.value && index < a.index)) {
    a.value = value;
    a.index = index;
  }
}

__device__ __forceinline__ ChooseBest warp_best(ChooseBest b) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, b.value, o);
    const int32_t i = __shfl_xor_sync(0xffffffffu, b.index, o);
    b.bad |= __shfl_xor_sync(0xffffffffu, b.bad, o);
    better(b, v, i);
  }
  return b;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Stores a word into the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ void store_cluster(void *local, uint32_t rank, uint32_t v) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Tokens of a CTA's slice: a multiple of 32, so that slices share no mask word.
__host__ __device__ inline int32_t choose_slice(int32_t vocab, int32_t ctas) {
  return static_cast<int32_t>(((static_cast<int64_t>(vocab) + ctas - 1) / ctas + 31) / 32 * 32);
}

template <typename T>
struct Logit;
template <>
struct Logit<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ void load(const float *p, float (&v)[4]) {
    const float4 f = __ldcs(reinterpret_cast<const float4 *>(p));
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  }
  static __device__ __forceinline__ float one(const float *p) { return *p; }
};
template <typename H>
struct LogitHalf {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ void load(const H *p, float (&v)[8]) {
    unpack8<H>(__ldcs(reinterpret_cast<const uint4 *>(p)), v);
  }
  static __device__ __forceinline__ float one(const H *p) { return Element<H>::load(*p); }
};
template <>
struct Logit<__nv_bfloat16> : LogitHalf<__nv_bfloat16> {};
template <>
struct Logit<__half> : LogitHalf<__half> {};

template <typename T>
__global__ void __launch_bounds__(kChooseThreads) choose_kernel(const ChooseArgs a) {
  extern __shared__ __align__(16) uint32_t marks[];   // [slice]
  __shared__ ChooseBest warp_part[kChooseThreads / 32];
  __shared__ ChooseBest parts[kChooseMaxCluster];
  constexpr int kVec = Logit<T>::kVec;
  const int tid = threadIdx.x, row = blockIdx.y;
  const int rank = static_cast<int>(cluster_rank()), ctas = static_cast<int>(cluster_size());
  cluster_arrive();   // every CTA of the cluster runs before its shared memory is written
  const bool active = a.active == nullptr || a.active[row] != 0;
  const int32_t slice = choose_slice(a.vocab, ctas);
  const int64_t v0 = min(static_cast<int64_t>(rank) * slice, static_cast<int64_t>(a.vocab));
  const int32_t width = static_cast<int32_t>(min(static_cast<int64_t>(slice), a.vocab - v0));
  const int32_t length = a.history != nullptr ? min(max(a.history_len[row], 0), a.history_width) : 0;
  const float rep = a.repetition != nullptr ? a.repetition[row] : 1.f;
  const float freq = a.frequency != nullptr ? a.frequency[row] : 0.f;
  const float pres = a.presence != nullptr ? a.presence[row] : 0.f;
  const bool penal = length > 0 && (rep != 1.f || freq != 0.f || pres != 0.f);
  const int32_t biases = a.bias_token != nullptr ? min(max(a.bias_len[row], 0), a.bias_width) : 0;
  const int32_t *bias_token = a.bias_token + (a.bias_token != nullptr ? row * a.bias_stride : 0);
  const float *bias_value = a.bias_value + (a.bias_token != nullptr ? row * a.bias_stride : 0);
  const bool marked = penal || biases > 0;
  ChooseBest best{-INFINITY, INT_MAX, 0};

  if (active) {
    if (marked) {
      for (int i = tid; i < slice / 4; i += kChooseThreads)
        reinterpret_cast<uint4 *>(marks)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      if (penal) {
        const int32_t prompt = min(max(a.prompt_len[row], 0), length);
        const int32_t *history = a.history + row * a.history_stride;
        for (int i = tid; i < length; i += kChooseThreads) {
          const int64_t n = history[i] - v0;
          if (n >= 0 && n < width) {
            if (i < prompt)
              atomicOr(&marks[n], kInPrompt);
            else
              atomicAdd(&marks[n], 1u);
          }
        }
      }
      for (int i = tid; i < biases; i += kChooseThreads) {
        const int64_t n = bias_token[i] - v0;
        if (n >= 0 && n < width) atomicOr(&marks[n], kHasBias);
      }
      __syncthreads();
    }
    const T *logits = static_cast<const T *>(a.logits) + row * a.logits_stride + v0;
    float *out = a.processed != nullptr ? a.processed + row * a.processed_stride + v0 : nullptr;
    const uint32_t *allowed = a.allowed != nullptr ? a.allowed + row * a.allowed_stride + v0 / 32 : nullptr;

    // the rules on token v0 + n; `mark` its word, `open` whether the mask allows it
    auto rules = [&](float x, int32_t n, uint32_t mark, bool open) {
      if (mark != 0) {
        if (mark & kHasBias) {
          const int32_t want = static_cast<int32_t>(v0 + n);
          int32_t lo = 0, hi = biases;   // the first entry not below the token
          while (lo < hi) {
            const int32_t mid = (lo + hi) >> 1;
            if (bias_token[mid] < want) lo = mid + 1;
            else hi = mid;
          }
          if (lo < biases && bias_token[lo] == want) x = __fadd_rn(x, bias_value[lo]);
        }
        const uint32_t count = mark & kCount;
        if (mark & (kInPrompt | kCount)) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        if (count != 0) {
          x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(count)));
          x = __fsub_rn(x, pres);
        }
      }
      x = open ? x : -INFINITY;
      if (!(x < INFINITY)) best.bad = 1;   // NaN or +inf
      better(best, x, x > -INFINITY ? static_cast<int32_t>(v0 + n) : INT_MAX);
      return x;
    };
    auto one = [&](int32_t n) {
      const bool open = allowed == nullptr || ((allowed[n >> 5] >> (n & 31)) & 1u);
      const float x = rules(Logit<T>::one(logits + n), n, marked ? marks[n] : 0u, open);
      if (out != nullptr) out[n] = x;
    };
    // the row need not begin on a 16-byte boundary: single tokens up to the first one
    const int32_t lead = min(width, static_cast<int32_t>(((16 - (reinterpret_cast<uintptr_t>(logits) & 15)) & 15) / sizeof(T)));
    const int32_t vectors = (width - lead) / kVec;
    const int32_t rest = lead + vectors * kVec;
    const bool out16 = (reinterpret_cast<uintptr_t>(out + lead) & 15) == 0;
    if (tid < lead) one(tid);
    for (int32_t i = tid; i < vectors; i += kChooseThreads) {
      const int32_t n = lead + i * kVec;
      float x[kVec];
      Logit<T>::load(logits + n, x);
      uint32_t open = 0xffffffffu;
      if (allowed != nullptr) {
        const int32_t w = n >> 5, s = n & 31;
        open = allowed[w] >> s;
        if (s > 32 - kVec) open |= allowed[w + 1] << (32 - s);
      }
#pragma unroll
      for (int k = 0; k < kVec; ++k) x[k] = rules(x[k], n + k, marked ? marks[n + k] : 0u, (open >> k) & 1u);
      if (out != nullptr) {
        if (out16) {
#pragma unroll
          for (int k = 0; k < kVec; k += 4)
            __stcs(reinterpret_cast<float4 *>(out + n + k), make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]));
        } else {
#pragma unroll
          for (int k = 0; k < kVec; ++k) out[n + k] = x[k];
        }
      }
    }
    if (tid < width - rest) one(rest + tid);
  }

  best = warp_best(best);
  if ((tid & 31) == 0) warp_part[tid >> 5] = best;
  __syncthreads();
  cluster_wait();
  if (tid < 32) {
    best = tid < kChooseThreads / 32 ? warp_part[tid] : ChooseBest{-INFINITY, INT_MAX, 0};
    best = warp_best(best);
    if (tid == 0) {
      store_cluster(&parts[rank].value, 0, __float_as_uint(best.value));
      store_cluster(&parts[rank].index, 0, static_cast<uint32_t>(best.index));
      store_cluster(&parts[rank].bad, 0, static_cast<uint32_t>(best.bad));
    }
  }
  cluster_arrive();
  cluster_wait();
  if (rank == 0 && tid == 0) {
    best = parts[0];
    for (int c = 1; c < ctas; ++c) {
      better(best, parts[c].value, parts[c].index);
      best.bad |= parts[c].bad;
    }
    const int64_t token = !active ? -1 : best.bad ? -2 : best.index == INT_MAX ? -1 : best.index;
    a.token[row] = token;
    if (a.append && a.history != nullptr && token >= 0) {
      const int32_t end = a.history_len[row];
      if (end >= 0 && end < a.history_width) a.history[row * a.history_stride + end] = static_cast<int32_t>(token);
    }
  }
}

}  // namespace ops
}  // namespace cruise
