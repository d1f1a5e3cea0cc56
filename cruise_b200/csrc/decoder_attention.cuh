// decoder_attention.cuh -- attention of one new token per row over the paged
// cache, split over the length and joined.
//
// For every row and query head: o = sum_t softmax_t(scale q.k_t) v_t over the
// row's positions t < seq_len, lse = log sum_t exp(scale q.k_t).  One pass over
// K and V with the running maximum m and sum l of the softmax; pieces
// (m_i, l_i, O_i) join as m = max m_i, l = sum l_i 2^(m_i - m),
// O = sum O_i 2^(m_i - m), o = O / l (scores carry a factor log2 e).
//
// The query heads of a KV head share its keys: S^T = K Q^T and O^T = V^T P^T as
// m16n8k16 products with 16 keys (16 dimensions) as the rows and 8 heads as
// the columns, so a group of up to 8 heads reads its keys once.  Probabilities
// are rounded to the cache's type for the second product (relative 2^-9 in
// bf16, 2^-12 in fp16, as the values they weight); m, l and O are fp32.
#pragma once

#include "decoder_common.cuh"
#include "decoder_ops.h"

namespace cruise {
namespace ops {

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kAttendKeys = 16;                          // keys of a warp's step
constexpr int kAttendTile = kAttendWarps * kAttendKeys;  // keys of a CTA's step
constexpr int kAttendStages = 3;
constexpr int kAttendCtas = 2;                           // CTAs per SM
constexpr int kAttendMinShare = 2;                       // fewest tiles worth a CTA of their own
constexpr int kJoinThreads = 128;

// Pieces of split units: CTA c leaves its first piece (of a unit that began
// before c) in slot 2c and its last (of a unit that goes on after c) in 2c + 1.
struct AttentionPlan {
  AttentionArgs a;
  int32_t groups;      // query heads per KV head
  int32_t chunk;       // of them, heads of one unit
  int32_t chunks;      // units per KV head
  int32_t units;       // units per row: nkv * chunks
  int32_t block_shift; // log2(block_size), -1 when not a power of two
  int32_t capacity;    // table_width * block_size
  int32_t whole;       // 1: one CTA per unit, nothing to join
  float scale_log2;    // scale * log2(e)
  float *piece_o;      // [2 grid][heads][d]
  float *piece_ml;     // [2 grid][heads][2]
  int4 *piece_of;      // [grid]: row, unit, pieces of the unit that begins in the CTA's slot 1 (0: none)
};

template <int D>
struct AttendShared {
  static constexpr int kRowBytes = D * 2;
  static constexpr int kStageBytes = 2 * kAttendKeys * kRowBytes;   // K then V
  static constexpr int kRingBytes = kAttendWarps * kAttendStages * kStageBytes;
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// The transpose of an 8 x 8 matrix of 16-bit elements held as one fragment register.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// 16 bytes global -> shared; with `bytes` 0 it reads nothing and writes zeros.
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ int row_length(const AttentionPlan &p, int row) {
  return min(max(p.a.seq_len[row], 0), p.capacity);
}

// A row without keys still takes one tile: its zeros have to be written.
__device__ __forceinline__ int row_tiles(int length) {
  return max(1, (length + kAttendTile - 1) / kAttendTile);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kAttendThreads, kAttendCtas) attention_kernel(const AttentionPlan p) {
  using S = AttendShared<D>;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint32_t live_mask[kAttendWarps][kAttendStages];
  __shared__ float merge_ml[kAttendWarps][NT * 8][2];
  __shared__ int scan[kAttendThreads / 32 + 1];
  __shared__ int found[3];
  constexpr int kChunks = D / 8;   // 16-byte chunks of a row
  const AttentionArgs &a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, q2 = (lane & 3) * 2;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // -- this CTA's share of the tiles (row-major, units of a row, tiles of a unit) --
  int row, off, left;
  if (p.whole) {
    row = blockIdx.x / p.units;
    const int n = row_tiles(row_length(p, row));
    off = (blockIdx.x - row * p.units) * n;
    left = n;
  } else {
    const int per = (a.rows + kAttendThreads - 1) / kAttendThreads;
    const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
    int mine = 0;
    for (int r = r0; r < r1; ++r) mine += row_tiles(row_length(p, r));
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < kAttendWarps; ++w) {
      if (w < warp) incl += scan[w];
      total += scan[w];
    }
    total *= p.units;
    const int share = max(kAttendMinShare, (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
    const int64_t begin64 = static_cast<int64_t>(blockIdx.x) * share;
    if (begin64 >= total) {
      if (tid == 0) p.piece_of[blockIdx.x] = make_int4(0, 0, 0, 0);
      return;
    }
    const int begin = static_cast<int>(begin64);
    int before = incl - mine;   // tiles (of one unit per row) before this thread's rows
    if (before * p.units <= begin && begin < incl * p.units) {
      for (int r = r0; r < r1; ++r) {
        const int n = row_tiles(row_length(p, r));
        if (begin < (before + n) * p.units) {
          found[0] = r;
          found[1] = begin - before * p.units;
          found[2] = min(share, total - begin);
          break;
        }
        before += n;
      }
    }
    __syncthreads();
    row = found[0];
    off = found[1];
    left = found[2];
  }
  const int share_tiles = left;   // the full share wherever a unit goes on after this CTA
  int4 tail = make_int4(0, 0, 0, 0);

  uint8_t *const my_ring = ring + warp * kAttendStages * S::kStageBytes;
  const uint32_t ring_addr = smem_u32(my_ring);

  while (left > 0) {
    const int length = row_length(p, row);
    const int n = row_tiles(length);
    const int unit = off / n, t0 = off - unit * n;
    const int count = min(n - t0, left);
    const int kvh = unit / p.chunks, head0 = kvh * p.groups + (unit - kvh * p.chunks) * p.chunk;
    const int heads = min(p.chunk, (kvh + 1) * p.groups - head0);
    const int32_t *table = a.block_table + row * a.table_stride;
    const T *kbase = static_cast<const T *>(a.key_cache) + kvh * D;
    const T *vbase = static_cast<const T *>(a.value_cache) + kvh * D;

    // Q fragments: column n of the product is head head0 + 8 nt + n
    uint32_t qf[NT][D / 16][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + g;
      const T *qrow = static_cast<const T *>(a.q) + row * a.q_stride + static_cast<int64_t>(head0 + h) * D;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[nt][kk][0] = h < heads ? *reinterpret_cast<const uint32_t *>(qrow + kk * 16 + q2) : 0u;
        qf[nt][kk][1] = h < heads ? *reinterpret_cast<const uint32_t *>(qrow + kk * 16 + 8 + q2) : 0u;
      }
    }

    auto load = [&](int i, int stage) {
      const int base = (t0 + i) * kAttendTile + warp * kAttendKeys;
      int64_t at = 0;
      bool live = false;
      if (i < count && lane < kAttendKeys && base + lane < length) {
        const int t = base + lane;
        const int blk = p.block_shift >= 0 ? t >> p.block_shift : t / a.block_size;
        const int in = t - blk * a.block_size;
        const int id = table[blk];
        live = id >= 0 && id < a.num_blocks;
        if (live) at = id * a.block_stride + static_cast<int64_t>(in) * a.nkv * D;
      }
      const uint32_t mask = __ballot_sync(0xffffffffu, live);
      if (lane == 0) live_mask[warp][stage] = mask;
      const uint32_t kdst = ring_addr + stage * S::kStageBytes, vdst = kdst + kAttendKeys * S::kRowBytes;
      if (i < count) {
#pragma unroll
        for (int j = 0; j < kAttendKeys * kChunks / 32; ++j) {
          const int idx = j * 32 + lane, key = idx / kChunks, c = idx % kChunks;
          const int64_t src = __shfl_sync(0xffffffffu, at, key) + c * 8;
          const int bytes = (mask >> key) & 1 ? 16 : 0;
          const uint32_t dst = key * S::kRowBytes + ((c ^ (key & 7)) << 4);
          cp_async16_zfill(kdst + dst, kbase + src, bytes);
          cp_async16_zfill(vdst + dst, vbase + src, bytes);
        }
      }
      cp_async_commit();
    };

    float acc[NT][D / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) acc[nt][dt][0] = acc[nt][dt][1] = acc[nt][dt][2] = acc[nt][dt][3] = 0.f;
    }

#pragma unroll
    for (int i = 0; i < kAttendStages - 1; ++i) load(i, i);
    int stage = 0, fill = kAttendStages - 1;
    for (int i = 0; i < count; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAttendStages - 2) : "memory");
      __syncwarp();
      const uint32_t mask = live_mask[warp][stage];
      load(i + kAttendStages - 1, fill);   // the stage every lane left before the barrier above
      if (mask != 0) {
        const uint32_t kaddr = ring_addr + stage * S::kStageBytes, vaddr = kaddr + kAttendKeys * S::kRowBytes;
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
        const int krow = lane & 15;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t ka[4];
          ldmatrix_x4(ka, kaddr + krow * S::kRowBytes + (((2 * kk + (lane >> 4)) ^ (krow & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) Element<T>::mma(s[nt], ka, qf[nt][kk][0], qf[nt][kk][1]);
        }
        const bool live0 = (mask >> g) & 1, live1 = (mask >> (g + 8)) & 1;
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float alpha[2], e[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float s0 = live0 ? s[nt][j] * p.scale_log2 : -INFINITY;
            const float s1 = live1 ? s[nt][2 + j] * p.scale_log2 : -INFINITY;
            float top = fmaxf(s0, s1);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(top, m[nt][j]);
            const float base = top == -INFINITY ? 0.f : top;   // no finite score yet
            alpha[j] = exp2f(m[nt][j] - base);
            m[nt][j] = top;
            e[j] = exp2f(s0 - base);
            e[2 + j] = exp2f(s1 - base);
            l[nt][j] = l[nt][j] * alpha[j] + (e[j] + e[2 + j]);
          }
          pb[nt][0] = transpose8x8(Element<T>::pack(e[0], e[1]));
          pb[nt][1] = transpose8x8(Element<T>::pack(e[2], e[3]));
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            acc[nt][dt][0] *= alpha[0];
            acc[nt][dt][1] *= alpha[1];
            acc[nt][dt][2] *= alpha[0];
            acc[nt][dt][3] *= alpha[1];
          }
        }
        const int vrow = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          uint32_t va[4];
          ldmatrix_x4_trans(va, vaddr + vrow * S::kRowBytes + (((2 * dt + ((lane >> 3) & 1)) ^ (vrow & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) Element<T>::mma(acc[nt][dt], va, pb[nt][0], pb[nt][1]);
        }
      }
      stage = stage + 1 == kAttendStages ? 0 : stage + 1;
      fill = fill + 1 == kAttendStages ? 0 : fill + 1;
    }
    cp_async_wait_all();

    // -- the warps' parts of the segment meet in shared memory --
    constexpr int kStride = D + 4;   // fp32 row stride: no bank conflicts for the fragment stores
    float *const merge = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], o);
        if (g == 0) {
          merge_ml[warp][nt * 8 + q2 + j][0] = m[nt][j];
          merge_ml[warp][nt * 8 + q2 + j][1] = l[nt][j];
        }
      }
    }
    __syncthreads();   // every warp is done with its ring
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float *const h0 = merge + (warp * NT * 8 + nt * 8 + q2) * kStride + g;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        h0[dt * 16] = acc[nt][dt][0];
        h0[dt * 16 + kStride] = acc[nt][dt][1];
        h0[dt * 16 + 8] = acc[nt][dt][2];
        h0[dt * 16 + 8 + kStride] = acc[nt][dt][3];
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && count == n;
    const int64_t piece = 2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0 ? 1 : 0);
    for (int i = tid; i < heads * D; i += kAttendThreads) {
      const int h = i / D, c = i % D;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kAttendWarps; ++w) top = fmaxf(top, merge_ml[w][h][0]);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < kAttendWarps; ++w) {
        const float f = exp2f(merge_ml[w][h][0] - base);
        sum = fmaf(merge_ml[w][h][1], f, sum);
        o = fmaf(merge[(w * NT * 8 + h) * kStride + c], f, o);
      }
      if (whole) {
        // no key with a weight: zeros and log 0
        static_cast<T *>(a.out)[row * a.out_stride + static_cast<int64_t>(head0) * D + i] =
            Element<T>::round(sum == 0.f ? 0.f : o / sum);
        if (c == 0 && a.lse != nullptr)
          a.lse[static_cast<int64_t>(row) * a.nq + head0 + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
      } else {
        p.piece_o[piece * (NT * 8 * D) + i] = o;
        if (c == 0) {
          p.piece_ml[(piece * (NT * 8) + h) * 2] = top;
          p.piece_ml[(piece * (NT * 8) + h) * 2 + 1] = sum;
        }
      }
    }
    __syncthreads();   // the ring is free for the next segment
    if (!whole && t0 == 0) tail = make_int4(row, unit, 1 + (n - count + share_tiles - 1) / share_tiles, 0);
    off += count;
    left -= count;
    if (off == n * p.units) {
      off = 0;
      ++row;
    }
  }
  if (!p.whole && tid == 0) p.piece_of[blockIdx.x] = tail;
}

// Joins the pieces of the unit that begins in CTA blockIdx.x of the attention
// and goes on after it; one CTA per (attention CTA, head of the unit).
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(const AttentionPlan p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 of = p.piece_of[blockIdx.x];
  const int pieces = of.z;
  if (pieces == 0) return;
  const AttentionArgs &a = p.a;
  const int row = of.x, kvh = of.y / p.chunks;
  const int head0 = kvh * p.groups + (of.y - kvh * p.chunks) * p.chunk;
  const int heads = min(p.chunk, (kvh + 1) * p.groups - head0);
  const int h = blockIdx.y;
  if (h >= heads) return;
  constexpr int kLanes = D / 4;                       // 4 dimensions a thread
  constexpr int kParts = kJoinThreads / kLanes;       // pieces taken in turn
  __shared__ __align__(16) float red[kParts][D];
  __shared__ float red_ml[kParts][2];
  const int c = threadIdx.x % kLanes, part = threadIdx.x / kLanes;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = part; i < pieces; i += kParts) {
    // the first piece lies in slot 1 of its CTA, the others in slot 0 of the CTAs after it
    const int64_t piece = i == 0 ? 2 * static_cast<int64_t>(blockIdx.x) + 1 : 2 * (static_cast<int64_t>(blockIdx.x) + i);
    const float2 ml = *reinterpret_cast<const float2 *>(p.piece_ml + (piece * (NT * 8) + h) * 2);
    const float4 v = *reinterpret_cast<const float4 *>(p.piece_o + piece * (NT * 8 * D) + h * D + c * 4);
    const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.f : top;
    const float fa = exp2f(m - base), fb = exp2f(ml.x - base);
    o.x = o.x * fa + v.x * fb;
    o.y = o.y * fa + v.y * fb;
    o.z = o.z * fa + v.z * fb;
    o.w = o.w * fa + v.w * fb;
    l = l * fa + ml.y * fb;
    m = top;
  }
  *reinterpret_cast<float4 *>(&red[part][c * 4]) = o;
  if (c == 0) {
    red_ml[part][0] = m;
    red_ml[part][1] = l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += kJoinThreads) {
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kParts; ++k) top = fmaxf(top, red_ml[k][0]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, v = 0.f;
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const float f = exp2f(red_ml[k][0] - base);
      sum = fmaf(red_ml[k][1], f, sum);
      v = fmaf(red[k][i], f, v);
    }
    static_cast<T *>(a.out)[row * a.out_stride + static_cast<int64_t>(head0 + h) * D + i] =
        Element<T>::round(sum == 0.f ? 0.f : v / sum);
    if (i == 0 && a.lse != nullptr)
      a.lse[static_cast<int64_t>(row) * a.nq + head0 + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
  }
}

}  // namespace ops
}  // namespace cruise
