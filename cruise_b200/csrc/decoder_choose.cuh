// decoder_choose.cuh -- rules on the logits and the greedy choice, in one pass.
//
// Per row, for every token n of the vocabulary, in fp32 and in this order:
//   x = logit (+ the token's bias);
//   in the row's history (prompt or output): x = x > 0 ? x / repetition : x * repetition;
//   count > 0, its occurrences in the output: x = x - frequency * count, x = x - presence;
//   not allowed by the row's bit mask: x = -inf.
// The choice is the first maximum above -inf: -1 where there is none, -2 where
// an x is NaN or +inf.  Each step is one rounded fp32 operation, so the choice
// equals that of the same steps done one by one.
//
// A cluster of CTAs shares a row, a slice of the vocabulary each; the slices'
// maxima meet in the first CTA's shared memory, so a call is one launch and
// keeps no state.  Few tokens of a slice are in the history or the bias list.  Four or eight
// warps deal with them: a bit map in shared memory marks them, their rank in it
// is their place in a table of occurrences, and from that come their processed
// values.  Meanwhile the other warps stream over the slice and know nothing of
// it: they mask the logits and keep each thread's maximum, a few operations an
// element.  After the barrier between the two, a thread whose maximum is a marked
// token has its elements gone over again without them, by a warp together, and
// the marked tokens' values are written over the stream's.
//
// What bounds it: for many rows the logits' bytes.  256 rows of 152064 with every
// rule and the processed logits written take 74 us, 66% of the copy bandwidth (the
// stream alone 57; then the marked tokens' values and second looks, while little
// is in flight).  For few rows the chain of the marked tokens' steps (clear, mark,
// rank, count, value, compare): 4.2 us for one row of 4096, 5.6 for 4 of 152064,
// 8.1 for 64 of 50257 with 1000 entries each.  Two kernels, one for the marked
// tokens, took 126 us for the 256 rows; one CTA's warps doing first the one and
// then the other 82.
#pragma once

#include <climits>
#include <type_traits>

#include "decoder_common.cuh"
#include "decoder_ops.h"

namespace cruise {
namespace ops {

constexpr int kChooseThreads = 512;
constexpr int kChooseFewThreads = 128;     // of them, those of the marked tokens,
constexpr int kChooseManyThreads = 256;    // and where these are many for the slice
constexpr int kChooseCtas = 2;             // CTAs per SM
constexpr int kChooseMaxCluster = 16;
constexpr int kChooseAhead = 4;            // vectors a thread has in flight (256 rows of 152064: 74 us; two 78, six 79)
constexpr int kChooseBatch = 8;            // history entries a thread has in flight (four: 78)
constexpr size_t kChooseShared = 200 * 1024;
constexpr size_t kChooseAlone = 118 * 1024;   // shared memory that leaves an SM no second CTA
constexpr int32_t kChooseMaxVocab = 1 << 20;
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

// Tokens of a CTA's slice: a multiple of 32, so that slices share no mask word.
inline int32_t choose_slice(int32_t vocab, int32_t ctas) { return ((vocab + ctas - 1) / ctas + 31) / 32 * 32; }

// Marked tokens of a slice at most.
__host__ __device__ inline int32_t choose_listed(int32_t slice, int64_t entries) {
  return static_cast<int32_t>(entries < slice ? entries : slice);
}

// Words of a slice's marks, a multiple of 4.
__host__ __device__ inline int32_t choose_words(int32_t slice) { return (slice / 32 + 3) / 4 * 4; }

// Shared memory of a slice: marks and ranks per word, occurrences and tokens listed.
inline size_t choose_shared(int32_t slice, int64_t entries) {
  return static_cast<size_t>(choose_words(slice)) * 8 + static_cast<size_t>(choose_listed(slice, entries)) * 8;
}

// The larger value; NaN when either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
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

template <typename T, int Table>
__global__ void __launch_bounds__(kChooseThreads, kChooseCtas) choose_kernel(const ChooseArgs a, const int32_t slice) {
  extern __shared__ __align__(16) uint32_t shared[];
  constexpr int kStream = kChooseThreads - Table;   // threads of the stream
  __shared__ ChooseBest warp_part[kChooseThreads / 32];
  __shared__ ChooseBest parts[kChooseMaxCluster];
  __shared__ int32_t scan[Table / 32];
  __shared__ uint32_t spare[32];      // where entries of other slices leave what they would mark
  __shared__ int32_t shared_listed;   // marked tokens of the slice
  __shared__ int32_t retakes;         // stream threads whose maximum is one of them
  __shared__ uint16_t retake_list[kStream];
  constexpr int kVec = Logit<T>::kVec;
  const int tid = threadIdx.x, row = blockIdx.y, ctas = gridDim.x;
  const int part = ctas > 1 ? static_cast<int>(cluster_rank()) : 0;
  if (ctas > 1) cluster_arrive();   // every CTA of the cluster runs before its shared memory is written
  follow_predecessor();
  const int32_t v0 = min(part * slice, a.vocab);
  const int32_t width = min(slice, a.vocab - v0);
  const T *const logits = static_cast<const T *>(a.logits) + row * a.logits_stride + v0;
  const uint32_t *const allowed = a.allowed != nullptr ? a.allowed + row * a.allowed_stride + v0 / 32 : nullptr;
  float *const out = a.processed != nullptr ? a.processed + row * a.processed_stride + v0 : nullptr;
  const int32_t *const bias_token = a.bias_token != nullptr ? a.bias_token + row * a.bias_stride : nullptr;
  // the row need not begin on a 16-byte boundary: single tokens up to the first one
  const int32_t lead = min(width, static_cast<int32_t>(((16 - (reinterpret_cast<uintptr_t>(logits) & 15)) & 15) / sizeof(T)));
  const int32_t vectors = (width - lead) / kVec;
  const int32_t rest = lead + vectors * kVec;
  const int32_t steps = (vectors + kStream - 1) / kStream;
  const int32_t last_word = (width - 1) >> 5;
  const bool split = lead % kVec != 0;   // a vector's mask bits may go on in the next word
  const uint4 *const stream = reinterpret_cast<const uint4 *>(logits + lead);
  const bool active = a.active == nullptr || a.active[row] != 0;
  ChooseBest best{-INFINITY, INT_MAX, 0};
  const int32_t words = choose_words(slice);
  uint32_t *const marks = shared, *const ranks = marks + words, *const counts = ranks + words;
  uint32_t *const list = counts + choose_listed(slice, static_cast<int64_t>(a.history != nullptr ? a.history_width : 0) +
                                                           (bias_token != nullptr ? a.bias_width : 0));
  auto masked = [&](float (&x)[kVec], uint32_t bits) {   // -inf where a bit is 0
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[j] = bits & (1u << j) ? x[j] : -INFINITY;
  };
  auto open_at = [&](int32_t n) { return allowed == nullptr || ((allowed[n >> 5] >> (n & 31)) & 1u); };
  float top = -INFINITY;
  int32_t top_at = -1;
  bool broken = false;   // NaN or +inf among the thread's tokens
  if (tid == 0) retakes = 0;

  if (active && tid < Table) {
    // -- the marked tokens.  What a thread does for an entry it does without
    // branches (an entry of another slice marks nothing and counts nothing), so
    // that a batch's entries overlap; the first history entries are fetched with
    // the lengths that say which of them count --
    const int32_t *const history = a.history != nullptr ? a.history + row * a.history_stride : nullptr;
    const int32_t history_width = history != nullptr ? a.history_width : 0;
    const bool has_bias = bias_token != nullptr && tid < a.bias_width;
    int32_t id[kChooseBatch];
    auto fetch = [&](int32_t i0, int32_t end) {
#pragma unroll
      for (int k = 0; k < kChooseBatch; ++k) {
        const int32_t i = i0 + k * Table;
        id[k] = i < end ? history[i] : -1;
      }
    };
    fetch(tid, history_width);
    const int32_t bias_id = has_bias ? bias_token[tid] : -1;
    int32_t length = 0, prompt = 0, biases = 0;
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if (history != nullptr) {
      length = a.history_len[row];
      prompt = a.prompt_len[row];
    }
    if (bias_token != nullptr) biases = min(max(a.bias_len[row], 0), a.bias_width);
    if (a.repetition != nullptr) rep = a.repetition[row];
    if (a.frequency != nullptr) freq = a.frequency[row];
    if (a.presence != nullptr) pres = a.presence[row];
    const int32_t counted = rep != 1.f || freq != 0.f || pres != 0.f ? min(max(length, 0), history_width) : 0;
    constexpr int32_t kStride = kChooseBatch * Table;
    int32_t listed = 0;
    if (counted + biases > 0) {
      // a vocabulary id as a token of this slice; others are at least `width`
      auto here = [&](int32_t v) { return static_cast<uint32_t>(v) - static_cast<uint32_t>(v0); };
      auto mark = [&](uint32_t n) { atomicOr(&marks[n >> 5], 1u << (n & 31)); };
      auto rank = [&](uint32_t n) { return ranks[n >> 5] + __popc(marks[n >> 5] & ((1u << (n & 31)) - 1)); };
      for (int32_t i = tid; i < words / 4; i += Table) reinterpret_cast<uint4 *>(marks)[i] = make_uint4(0, 0, 0, 0);
      const int32_t most = min(counted + biases, width);
      for (int32_t i = tid; i < most; i += Table) counts[i] = 0;
      named_sync(1, Table);
      for (int32_t i0 = tid; i0 - tid < counted; i0 += kStride) {
        if (i0 != tid) fetch(i0, counted);
#pragma unroll
        for (int k = 0; k < kChooseBatch; ++k) {
          if (i0 - tid + k * Table >= counted) break;   // uniform: short histories run little code
          const uint32_t n = here(id[k]);
          const bool mine = i0 + k * Table < counted && n < static_cast<uint32_t>(width);
          atomicOr(mine ? &marks[n >> 5] : &spare[tid & 31], mine ? 1u << (n & 31) : 0u);
        }
      }
      if (here(bias_id) < static_cast<uint32_t>(width) && tid < biases) mark(here(bias_id));
      for (int32_t i = tid + Table; i < biases; i += Table)
        if (here(bias_token[i]) < static_cast<uint32_t>(width)) mark(here(bias_token[i]));
      named_sync(1, Table);
      // ranks: every thread its run of words
      const int32_t per = (words / 4 + Table - 1) / Table * 4;
      const int32_t w0 = min(tid * per, words), w1 = min(w0 + per, words);
      int32_t mine = 0;
      for (int32_t w = w0; w < w1; w += 4) {
        const uint4 m = *reinterpret_cast<const uint4 *>(marks + w);
        mine += __popc(m.x) + __popc(m.y) + __popc(m.z) + __popc(m.w);
      }
      int32_t incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if ((tid & 31) >= o) incl += v;
      }
      if ((tid & 31) == 31) scan[tid >> 5] = incl;
      named_sync(1, Table);
#pragma unroll
      for (int w = 0; w < Table / 32; ++w) {
        if (w < (tid >> 5)) incl += scan[w];
        listed += scan[w];
      }
      uint32_t at = incl - mine;
      for (int32_t w = w0; w < w1; w += 4) {
        const uint4 m = *reinterpret_cast<const uint4 *>(marks + w);
        const uint32_t b = at + __popc(m.x), c = b + __popc(m.y), d = c + __popc(m.z);
        *reinterpret_cast<uint4 *>(ranks + w) = make_uint4(at, b, c, d);
        at = d + __popc(m.w);
      }
      named_sync(1, Table);
      for (int32_t i0 = tid; i0 - tid < counted; i0 += kStride) {
        if (counted > kStride) fetch(i0, counted);
#pragma unroll
        for (int k = 0; k < kChooseBatch; ++k) {
          if (i0 - tid + k * Table >= counted) break;
          const int32_t i = i0 + k * Table;
          const bool mine = i < counted && here(id[k]) < static_cast<uint32_t>(width);
          const uint32_t n = mine ? here(id[k]) : 0, r = mine ? rank(n) : 0;   // (slot 0 exists)
          if (mine) list[r] = n;   // the token's entries agree
          uint32_t *const count = mine ? &counts[r] : &spare[tid & 31];
          atomicOr(count, i < prompt ? kInPrompt : 0u);
          atomicAdd(count, i >= prompt ? 1u : 0u);
        }
      }
      auto mark_bias = [&](uint32_t n) {
        if (n < static_cast<uint32_t>(width)) {
          const uint32_t r = rank(n);
          list[r] = n;
          atomicOr(&counts[r], kHasBias);
        }
      };
      if (tid < biases) mark_bias(here(bias_id));
      for (int32_t i = tid + Table; i < biases; i += Table) mark_bias(here(bias_token[i]));
      named_sync(1, Table);
      // the processed value takes the place of the occurrences
      auto rules = [&](uint32_t n, uint32_t r, float x) {
        const uint32_t word = counts[r], times = word & kCount;
        if (word & (kInPrompt | kCount)) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        if (times != 0) {
          x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(times)));
          x = __fsub_rn(x, pres);
        }
        if (!open_at(n)) x = -INFINITY;
        counts[r] = __float_as_uint(x);
        if (!(x < INFINITY)) best.bad = 1;   // NaN or +inf
        if (x > -INFINITY) better(best, x, v0 + static_cast<int32_t>(n));
      };
      // (in place, the stream may have masked a logit already: -inf then, as here)
      constexpr int kTogether = 4;
      for (int32_t i0 = tid; i0 < listed; i0 += kTogether * Table) {
        T raw[kTogether];
#pragma unroll
        for (int k = 0; k < kTogether; ++k) raw[k] = logits[list[min(i0 + k * Table, listed - 1)]];
#pragma unroll 1
        for (int k = 0; k < kTogether && i0 - tid + k * Table < listed; ++k) {
          const int32_t i = i0 + k * Table;
          if (i < listed && (counts[i] & kHasBias) == 0) rules(list[i], i, Logit<T>::one(&raw[0]));
#pragma unroll
          for (int q = 0; q + 1 < kTogether; ++q) raw[q] = raw[q + 1];
        }
      }
      if (biases > 0) named_sync(1, Table);
      for (int32_t i = tid; i < biases; i += Table) {   // entries of one token add up
        const int32_t v = bias_token[i];
        const uint32_t n = here(v);
        if (n >= static_cast<uint32_t>(width) || (i > 0 && bias_token[i - 1] == v)) continue;
        const float *const value = a.bias_value + row * a.bias_stride;
        float x = Logit<T>::one(logits + n);
        for (int32_t q = i; q < biases && bias_token[q] == v; ++q) x = __fadd_rn(x, value[q]);
        rules(n, rank(n), x);
      }
    }
    if (tid == 0) shared_listed = listed;
  } else if (active) {
    // -- the stream: every token as if the rules left it --
    const int32_t me = tid - Table;
    float worst = -INFINITY;   // NaN and +inf stay in it
    if (vectors > 0) {
      uint4 ahead[kChooseAhead];
      uint32_t open[kChooseAhead], open_next[kChooseAhead];   // their mask words, as loaded
      auto run = [&](auto mask_flag, auto out_flag) {
        constexpr bool kMask = decltype(mask_flag)::value, kOut = decltype(out_flag)::value;
        // Nothing here waits for a load; a step past the end fetches the slice's last
        // vector again, for a load under a condition would be waited for.
        auto fetch = [&](int k, int32_t step) {
          const int32_t i = min(step * kStream + me, vectors - 1);
          ahead[k] = stream[i];
          if (kMask) {
            const int32_t w = (lead + i * kVec) >> 5;
            open[k] = allowed[w];
            if (split) open_next[k] = allowed[min(w + 1, last_word)];
          }
        };
        const bool out16 = (reinterpret_cast<uintptr_t>(out + lead) & 15) == 0;
        const int shift = (lead + me * kVec) & 31;   // a step is a whole number of mask words
#pragma unroll
        for (int k = 0; k < kChooseAhead; ++k) fetch(k, k);
        for (int32_t step0 = 0; step0 < steps; step0 += kChooseAhead) {
#pragma unroll
          for (int k = 0; k < kChooseAhead; ++k) {
            const int32_t step = step0 + k, vector = step * kStream + me;
            float x[kVec];
            Logit<T>::unpack(ahead[k], x);
            if (kMask) masked(x, split ? __funnelshift_r(open[k], open_next[k], shift) : open[k] >> shift);
            fetch(k, step + kChooseAhead);
            if (vector < vectors) {
              if (kOut) {
                float *const to = out + lead + vector * kVec;
                if (out16) {
#pragma unroll
                  for (int j = 0; j < kVec; j += 4)
                    __stcs(reinterpret_cast<float4 *>(to + j), make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]));
                } else {
#pragma unroll
                  for (int j = 0; j < kVec; ++j) to[j] = x[j];
                }
              }
              float here_top = x[0];
#pragma unroll
              for (int j = 1; j < kVec; ++j) here_top = max_nan(here_top, x[j]);
              worst = max_nan(worst, here_top);
              if (here_top > top) {   // a later equal one loses
                top = here_top;
#pragma unroll
                for (int j = kVec - 1; j >= 0; --j)   // the first of the vector's equal ones
                  if (x[j] == here_top) top_at = lead + vector * kVec + j;
              }
            }
          }
        }
      };
      using Yes = std::true_type;
      using No = std::false_type;
      static_assert(kStream * kVec % 32 == 0, "a step is a whole number of mask words");
      if (allowed != nullptr)
        out != nullptr ? run(Yes{}, Yes{}) : run(Yes{}, No{});
      else
        out != nullptr ? run(No{}, Yes{}) : run(No{}, No{});
    }
    broken = !(worst < INFINITY);
  }
  // the tokens outside the vectors, a thread each
  const int32_t single = tid < lead ? tid : tid - lead < width - rest ? rest + tid - lead : -1;
  float single_x = -INFINITY;
  if (active && single >= 0) {
    single_x = open_at(single) ? Logit<T>::one(logits + single) : -INFINITY;
    if (out != nullptr) out[single] = single_x;
    broken |= !(single_x < INFINITY);
  }
  __syncthreads();

  if (active) {
    const int32_t listed = shared_listed;
    auto ruled = [&](int32_t n) { return listed > 0 && ((marks[n >> 5] >> (n & 31)) & 1u); };
    // raises (value, at) to the first maximum of a vector's tokens that no rule is for
    auto look = [&](int32_t vector, float &value, int32_t &at) {
      float x[kVec];
      Logit<T>::unpack(stream[vector], x);
      const int32_t n = lead + vector * kVec;
      if (allowed != nullptr)
        masked(x, __funnelshift_r(allowed[n >> 5], allowed[min((n >> 5) + 1, last_word)], n & 31));
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        if (x[j] > value && !ruled(n + j)) {
          value = x[j];
          at = n + j;
        }
      }
    };
    // No rule takes NaN or +inf away, but a negative repetition, which makes +inf of a
    // token in the history -inf: there the marked tokens, who answer for themselves,
    // are left out of the question.  (One at a time: the rare branch's length is paid
    // by every call.  One row of 4096: 4.1 us without it, 4.2 so, 4.3 a vector at a time.)
    if (__builtin_expect(broken, 0)) {
      if (a.repetition == nullptr || !signbit(a.repetition[row])) {
        best.bad = 1;
      } else {
        if (!(single_x < INFINITY) && !ruled(single)) best.bad = 1;
#pragma unroll 1
        for (int32_t vector = tid - Table; vector >= 0 && vector < vectors; vector += kStream) {
#pragma unroll 1
          for (int32_t n = lead + vector * kVec; n < lead + (vector + 1) * kVec; ++n)
            if (open_at(n) && !(Logit<T>::one(logits + n) < INFINITY) && !ruled(n)) best.bad = 1;
        }
      }
    }
    const bool retake = top_at >= 0 && ruled(top_at);
    if (retake) {
      top = -INFINITY;
      retake_list[atomicAdd(&retakes, 1)] = static_cast<uint16_t>(tid - Table);
    }
    if (__syncthreads_or(retake)) {
      const int32_t again = retakes;
      constexpr int kWarps = kChooseThreads / 32;
      if ((again + kWarps - 1) / kWarps * ((steps + 31) / 32) <= steps) {   // few: a warp takes a thread's elements together
        for (int32_t q = tid >> 5; q < again; q += kWarps) {
          float value = -INFINITY;
          int32_t at = 0;
          for (int32_t vector = (tid & 31) * kStream + retake_list[q]; vector < vectors; vector += 32 * kStream)
            look(vector, value, at);
          if (value > -INFINITY) better(best, value, v0 + at);
        }
      } else if (retake) {
        for (int32_t vector = tid - Table; vector < vectors; vector += kStream) look(vector, top, top_at);
      }
    }
    if (top > -INFINITY) better(best, top, v0 + top_at);
    if (single_x > -INFINITY && !ruled(single)) better(best, single_x, v0 + single);

    if (out != nullptr && listed > 0) {
      // in place, the second look above has to end before a value replaces a logit
      if (static_cast<const void *>(a.processed) == a.logits) __syncthreads();
      for (int32_t i = tid; i < listed; i += kChooseThreads) out[list[i]] = __uint_as_float(counts[i]);
    }
  }

  best = warp_best(best);
  if ((tid & 31) == 0) warp_part[tid >> 5] = best;
  __syncthreads();
  if (ctas > 1) cluster_wait();
  if (tid < 32) {
    best = tid < kChooseThreads / 32 ? warp_part[tid] : ChooseBest{-INFINITY, INT_MAX, 0};
    best = warp_best(best);
    if (tid == 0 && ctas > 1) {
      store_cluster(&parts[part].value, 0, __float_as_uint(best.value));
      store_cluster(&parts[part].index, 0, static_cast<uint32_t>(best.index));
      store_cluster(&parts[part].bad, 0, static_cast<uint32_t>(best.bad));
    }
  }
  if (ctas > 1) {
    cluster_arrive();
    cluster_wait();
    if (part == 0 && tid < 32) best = warp_best(tid < ctas ? parts[tid] : ChooseBest{-INFINITY, INT_MAX, 0});
  }
  if (part == 0 && tid == 0) {
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
