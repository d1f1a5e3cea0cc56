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
// A cluster of CTAs shares a row, a slice of the vocabulary each; the slices'
// maxima meet in the first CTA's shared memory, so a call is one launch and
// keeps no state.  Few tokens of a slice are in the history or the bias list: a
// bit map in shared memory marks them, their rank in it (a scan of the words'
// bit counts) is their place in a table of occurrences and a list.  The stream
// over the slice masks the logits and takes the maximum of the unmarked tokens,
// a few operations an element; the marked tokens follow, one a thread.
#pragma once

#include <climits>

#include "decoder_common.cuh"
#include "decoder_ops.h"

namespace cruise {
namespace ops {

constexpr int kChooseThreads = 512;
constexpr int kChooseCtas = 2;           // CTAs per SM
constexpr int kChooseMaxCluster = 16;
constexpr int kChooseAhead = 4;          // vectors a thread has in flight
constexpr int kChooseWindow = kChooseAhead * kChooseThreads;
constexpr int kChooseBatch = 4;          // history entries a thread has in flight
constexpr int32_t kChooseMaxVocab = 393216;
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

// The best of a warp, with integer reductions: fp32 values as integers of the
// same order (-0 as 0, which it equals; NaN is never a best value).
__device__ __forceinline__ ChooseBest warp_best(ChooseBest b) {
  const int32_t bits = __float_as_int(__fadd_rn(b.value, 0.f));
  const int32_t key = bits >= 0 ? bits : bits ^ 0x7fffffff;
  const int32_t top = __reduce_max_sync(0xffffffffu, key);
  b.index = __reduce_min_sync(0xffffffffu, key == top ? b.index : INT_MAX);
  b.value = __int_as_float(top >= 0 ? top : top ^ 0x7fffffff);
  b.bad = __any_sync(0xffffffffu, b.bad) ? 1 : 0;
  return b;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
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

template <typename T>
struct Logit;
template <>
struct Logit<float> {
  static constexpr int kVec = 4;   // of 16 bytes
  static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x);
    v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z);
    v[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float one(const float *p) { return *p; }
};
template <typename H>
struct LogitHalf {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[8]) { unpack8<H>(u, v); }
  static __device__ __forceinline__ float one(const H *p) { return Element<H>::load(*p); }
};
template <>
struct Logit<__nv_bfloat16> : LogitHalf<__nv_bfloat16> {};
template <>
struct Logit<__half> : LogitHalf<__half> {};

// The larger value; NaN when either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// `count` <= 32 bits from bit n of a bit array.
__device__ __forceinline__ uint32_t bits_at(const uint32_t *words, int32_t n, int count) {
  const int32_t w = n >> 5, s = n & 31;
  uint32_t bits = words[w] >> s;
  if (s + count > 32) bits |= words[w + 1] << (32 - s);
  return bits;
}

// Tokens of a CTA's slice: a multiple of 32, so that slices share no mask word.
inline int32_t choose_slice(int32_t vocab, int32_t ctas) { return ((vocab + ctas - 1) / ctas + 31) / 32 * 32; }

// Shared memory of a slice with up to `entries` history and bias entries:
// marks and their ranks per word, occurrences and the list per marked token.
__host__ __device__ inline int32_t choose_listed(int32_t slice, int64_t entries) {
  return static_cast<int32_t>(entries < slice ? entries : slice);
}

inline size_t choose_shared(int32_t slice, int64_t entries) {
  return static_cast<size_t>(slice) / 32 * 8 + static_cast<size_t>(choose_listed(slice, entries)) * 8;
}

template <typename T>
__global__ void __launch_bounds__(kChooseThreads, kChooseCtas) choose_kernel(const ChooseArgs a, const int32_t slice) {
  extern __shared__ __align__(16) uint32_t shared[];
  __shared__ ChooseBest warp_part[kChooseThreads / 32];
  __shared__ ChooseBest parts[kChooseMaxCluster];
  __shared__ int32_t scan[kChooseThreads / 32];
  constexpr int kVec = Logit<T>::kVec;
  const int tid = threadIdx.x, row = blockIdx.y, ctas = gridDim.x;
  const int part = static_cast<int>(cluster_rank());
  cluster_arrive();   // every CTA of the cluster runs before its shared memory is written
  const int32_t words = slice / 32;
  uint32_t *const marks = shared, *const ranks = marks + words, *const counts = ranks + words;
  const int32_t v0 = min(part * slice, a.vocab);
  const int32_t width = min(slice, a.vocab - v0);
  const T *logits = static_cast<const T *>(a.logits) + row * a.logits_stride + v0;
  const uint32_t *allowed = a.allowed != nullptr ? a.allowed + row * a.allowed_stride + v0 / 32 : nullptr;
  // the row need not begin on a 16-byte boundary: single tokens up to the first one
  const int32_t lead = min(width, static_cast<int32_t>(((16 - (reinterpret_cast<uintptr_t>(logits) & 15)) & 15) / sizeof(T)));
  const int32_t vectors = (width - lead) / kVec;
  const int32_t rest = lead + vectors * kVec;
  uint4 ahead[kChooseAhead];
  uint32_t open[kChooseAhead], open_next[kChooseAhead];   // their mask words, as loaded
  auto fetch = [&](int k, int32_t i) {   // nothing here waits for a load
    if (i < vectors) {
      ahead[k] = __ldcs(reinterpret_cast<const uint4 *>(logits + lead) + i);
      if (allowed != nullptr) {
        const int32_t n = lead + i * kVec;
        open[k] = allowed[n >> 5];
        if ((n & 31) > 32 - kVec) open_next[k] = allowed[(n >> 5) + 1];
      }
    }
  };
  auto ahead_l2 = [&](int32_t first) {
    if (first < vectors)
      prefetch_l2(reinterpret_cast<const uint4 *>(logits + lead) + first, min(kChooseWindow, vectors - first) * 16);
  };
  const bool active = a.active == nullptr || a.active[row] != 0;
  ChooseBest best{-INFINITY, INT_MAX, 0};

  if (active) {
#pragma unroll
    for (int k = 0; k < kChooseAhead; ++k) fetch(k, k * kChooseThreads + tid);
    // the two windows of the stream after the one in registers, into L2
    if (tid == 0) {
      ahead_l2(kChooseWindow);
      ahead_l2(2 * kChooseWindow);
    }
    // the thread's first history and bias entries are fetched with the lengths
    // that say which of them count
    const int32_t *history = a.history + (a.history != nullptr ? row * a.history_stride : 0);
    const int32_t *bias_token = a.bias_token + (a.bias_token != nullptr ? row * a.bias_stride : 0);
    const float *bias_value = a.bias_value + (a.bias_token != nullptr ? row * a.bias_stride : 0);
    int32_t kept[kChooseBatch];
#pragma unroll
    for (int k = 0; k < kChooseBatch; ++k) {
      const int32_t i = k * kChooseThreads + tid;
      kept[k] = a.history != nullptr && i < a.history_width ? history[i] : -1;
    }
    const bool has_bias = a.bias_token != nullptr && tid < a.bias_width;
    int32_t bias_id = has_bias ? bias_token[tid] : -1;
    const int32_t bias_before = has_bias && tid > 0 ? bias_token[tid - 1] : -1;
    const int32_t length = a.history != nullptr ? min(max(a.history_len[row], 0), a.history_width) : 0;
    const int32_t prompt = a.history != nullptr ? min(max(a.prompt_len[row], 0), length) : 0;
    const float rep = a.repetition != nullptr ? a.repetition[row] : 1.f;
    const float freq = a.frequency != nullptr ? a.frequency[row] : 0.f;
    const float pres = a.presence != nullptr ? a.presence[row] : 0.f;
    const int32_t counted = rep != 1.f || freq != 0.f || pres != 0.f ? length : 0;
    const int32_t biases = a.bias_token != nullptr ? min(max(a.bias_len[row], 0), a.bias_width) : 0;
    const int32_t entries = counted + biases;
    if (tid >= biases) bias_id = -1;
    uint32_t *const list = counts + choose_listed(slice, static_cast<int64_t>(a.history != nullptr ? a.history_width : 0) +
                                                             (a.bias_token != nullptr ? a.bias_width : 0));
    int32_t listed = 0;
    // this thread's first marked token and bias entry are fetched before the
    // stream and used after it
    T bias_x{}, listed_x{};
    // a vocabulary id as a token of this slice (-1: of another)
    auto here = [&](int32_t id) {
      const int64_t n = static_cast<int64_t>(id) - v0;
      return n >= 0 && n < width ? static_cast<int32_t>(n) : -1;
    };
    // f(entry, token) for the entries of this slice: the history's, a batch of
    // loads in flight, then the bias list's
    auto each = [&](auto &&f) {
#pragma unroll
      for (int k = 0; k < kChooseBatch; ++k) {
        const int32_t i = k * kChooseThreads + tid, n = here(kept[k]);
        if (i < counted && n >= 0) f(i, n);
      }
      for (int32_t i0 = kChooseBatch * kChooseThreads + tid; i0 < counted; i0 += kChooseBatch * kChooseThreads) {
        int32_t id[kChooseBatch];
#pragma unroll
        for (int k = 0; k < kChooseBatch; ++k) id[k] = i0 + k * kChooseThreads < counted ? history[i0 + k * kChooseThreads] : -1;
#pragma unroll
        for (int k = 0; k < kChooseBatch; ++k) {
          const int32_t n = here(id[k]);
          if (n >= 0) f(i0 + k * kChooseThreads, n);
        }
      }
      if (here(bias_id) >= 0) f(counted, here(bias_id));
      for (int32_t i = kChooseThreads + tid; i < biases; i += kChooseThreads) {
        const int32_t n = here(bias_token[i]);
        if (n >= 0) f(counted + i, n);
      }
    };
    auto rank = [&](int32_t n) { return ranks[n >> 5] + __popc(marks[n >> 5] & ((1u << (n & 31)) - 1)); };
    if (entries > 0) {
      for (int i = tid; i < words; i += kChooseThreads) marks[i] = 0;
      for (int i = tid; i < min(entries, slice); i += kChooseThreads) counts[i] = 0;
      __syncthreads();
      each([&](int32_t, int32_t n) { atomicOr(&marks[n >> 5], 1u << (n & 31)); });
      __syncthreads();
      // ranks: every thread its run of words
      const int32_t per = (words + kChooseThreads - 1) / kChooseThreads;
      const int32_t w0 = min(tid * per, words), w1 = min(w0 + per, words);
      int32_t mine = 0;
      for (int32_t w = w0; w < w1; ++w) mine += __popc(marks[w]);
      int32_t incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if ((tid & 31) >= o) incl += v;
      }
      if ((tid & 31) == 31) scan[tid >> 5] = incl;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kChooseThreads / 32; ++w) {
        if (w < (tid >> 5)) incl += scan[w];
        listed += scan[w];
      }
      int32_t at = incl - mine;
      for (int32_t w = w0; w < w1; ++w) {
        ranks[w] = at;
        at += __popc(marks[w]);
      }
      __syncthreads();
      each([&](int32_t i, int32_t n) {
        const int32_t r = rank(n);
        list[r] = n;   // the token's entries agree
        if (i >= counted)
          atomicOr(&counts[r], kHasBias);
        else if (i < prompt)
          atomicOr(&counts[r], kInPrompt);
        else
          atomicAdd(&counts[r], 1u);
      });
      __syncthreads();
      if (tid < listed) listed_x = logits[list[tid]];
      if (here(bias_id) >= 0) bias_x = logits[here(bias_id)];
    }
    float *out = a.processed != nullptr ? a.processed + row * a.processed_stride + v0 : nullptr;
    const bool out16 = (reinterpret_cast<uintptr_t>(out + lead) & 15) == 0;

    auto one = [&](int32_t n) {   // a single token
      const bool allow = allowed == nullptr || bits_at(allowed, n, 1) & 1u;
      const bool marked = entries > 0 && (bits_at(marks, n, 1) & 1u);
      const float x = allow ? Logit<T>::one(logits + n) : -INFINITY;
      if (out != nullptr) out[n] = x;
      if (marked) return;
      if (!(x < INFINITY)) best.bad = 1;   // NaN or +inf
      if (x > -INFINITY) better(best, x, v0 + n);
    };
    if (tid < lead) one(tid);
    for (int32_t first = 0; first < vectors; first += kChooseWindow) {
      if (tid == 0) ahead_l2(first + 3 * kChooseWindow);
#pragma unroll
      for (int k = 0; k < kChooseAhead; ++k) {
        const int32_t i = first + k * kChooseThreads + tid;
        if (i >= vectors) break;
        const int32_t n = lead + i * kVec;
        float x[kVec];
        Logit<T>::unpack(ahead[k], x);
        if (allowed != nullptr) {
          const uint32_t bits = __funnelshift_r(open[k], open_next[k], n & 31);
#pragma unroll
          for (int j = 0; j < kVec; ++j) x[j] = (bits >> j) & 1u ? x[j] : -INFINITY;
        }
        fetch(k, i + kChooseWindow);
        if (out != nullptr) {
          if (out16) {
#pragma unroll
            for (int j = 0; j < kVec; j += 4)
              __stcs(reinterpret_cast<float4 *>(out + n + j), make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]));
          } else {
#pragma unroll
            for (int j = 0; j < kVec; ++j) out[n + j] = x[j];
          }
        }
        if (entries > 0) {
          const uint32_t marked = bits_at(marks, n, kVec) & ((1u << kVec) - 1);
          if (marked != 0) {
#pragma unroll
            for (int j = 0; j < kVec; ++j) x[j] = (marked >> j) & 1u ? -INFINITY : x[j];
          }
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < kVec; ++j) top = max_nan(top, x[j]);
        if (!(top < INFINITY)) best.bad = 1;
        if (top > best.value) {   // the thread's tokens come in order: a later equal one loses
          best.value = top;
#pragma unroll
          for (int j = kVec - 1; j >= 0; --j)
            if (x[j] == top) best.index = v0 + n + j;
        }
      }
    }
    if (tid < width - rest) one(rest + tid);

    if (entries > 0) {
      __syncthreads();
      // a marked token, its bias added
      auto rules = [&](int32_t n, uint32_t word, float x) {
        const uint32_t times = word & kCount;
        if (word & (kInPrompt | kCount)) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        if (times != 0) {
          x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(times)));
          x = __fsub_rn(x, pres);
        }
        if (allowed != nullptr && (bits_at(allowed, n, 1) & 1u) == 0) x = -INFINITY;
        if (out != nullptr) out[n] = x;
        if (!(x < INFINITY)) best.bad = 1;
        if (x > -INFINITY) better(best, x, v0 + n);
      };
      for (int32_t i = tid; i < listed; i += kChooseThreads) {
        const int32_t n = static_cast<int32_t>(list[i]);
        if ((counts[i] & kHasBias) == 0) rules(n, counts[i], Logit<T>::one(i == tid ? &listed_x : logits + n));
      }
      for (int32_t i = tid; i < biases; i += kChooseThreads) {
        const int32_t id = i == tid ? bias_id : bias_token[i], n = here(id);
        if (n < 0 || (i > 0 && (i == tid ? bias_before : bias_token[i - 1]) == id)) continue;
        float x = Logit<T>::one(i == tid ? &bias_x : logits + n);
        for (int32_t j = i; j < biases && bias_token[j] == id; ++j) x = __fadd_rn(x, bias_value[j]);
        rules(n, counts[rank(n)], x);
      }
    }
  }

  best = warp_best(best);
  if ((tid & 31) == 0) warp_part[tid >> 5] = best;
  __syncthreads();
  cluster_wait();
  if (tid < 32) {
    best = tid < kChooseThreads / 32 ? warp_part[tid] : ChooseBest{-INFINITY, INT_MAX, 0};
    best = warp_best(best);
    if (tid == 0) {
      store_cluster(&parts[part].value, 0, __float_as_uint(best.value));
      store_cluster(&parts[part].index, 0, static_cast<uint32_t>(best.index));
      store_cluster(&parts[part].bad, 0, static_cast<uint32_t>(best.bad));
    }
  }
  cluster_arrive();
  cluster_wait();
  if (part == 0 && tid == 0) {
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
