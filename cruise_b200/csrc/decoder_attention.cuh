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
// the columns, so a group of up to 8 heads reads its keys once.  m, l and O are
// fp32.  The second product takes a probability p as two terms of the cache's
// type, hi = round(c p (1 - 2 u)) and lo = round(c p - hi), where u is half a step of
// the type (2^-8 in bf16, 2^-11 in fp16): together at most 3 u^2 p off, far below
// the output's own rounding u.  c = 2^15 in fp16, whose range ends at 2^-24: weights
// down to 2^-40 of a warp's largest count.  hi stays below c p, so lo is positive and an
// infinite value gives an infinite output, not inf - inf.  The second term costs 0.1 us
// where latency counts (4 rows of 256: 4.3 to 4.4; 22 rows of 1576 8.5 to 8.8) and 0 to
// 1% of the long cases.
//
// What bounds it is the cache's bytes: a key and its value, 4 d bytes, take 4 d
// operations for each of the group's heads, far below the tensor pipe (13% of
// its cycles at 64 ragged rows).  So the products are the warp-wide ones, whose
// operands a warp takes from its own ring as they arrive, 16 keys a step, with
// no barrier between warps until the unit's end; larger tiles would only wait
// for more bytes.  256 rows of up to 4096 (28 heads over 4 of 128) take 212 us,
// 98% of the copy bandwidth; one row of 131071 47 us (87%: 3 us to start, 3 for
// the join); 64 ragged rows of up to 16384 in pages of 16, head size 64, 46 us
// (75%: units of a few steps, and two steps of copies in flight per warp).  Few
// and short units are bounded by the chain of start, first loads, products and
// merge: 4 rows of 256 4.4 us, 4 of 16 2.6.
//
// Which CTAs take a unit (a row and a KV head, at most 16 query heads):
//   split:   all CTAs share all tiles evenly, whatever the rows' lengths, and a
//            second kernel joins the pieces of the units that were cut;
//   whole:   a CTA of one, four or eight warps takes a unit;
//   cluster: up to 16 CTAs of eight warps take a unit, every n-th tile each,
//            and join over their shared memory.
// The launch chooses by rows, units and capacity, and has the times.
#pragma once

#include "decoder_common.cuh"
#include "decoder_ops.h"

namespace cruise {
namespace ops {

constexpr int kAttendKeys = 16;      // keys of a warp's step
constexpr int kAttendWarps = 4;      // warps of a CTA that shares the work with the others
constexpr int kAttendWholeWarps = 8; // warps of a CTA of a cluster that takes one unit
constexpr int kAttendRanks = 16;     // CTAs of such a cluster, at most
constexpr int kJoinThreads = 512;
constexpr int kJoinBatch = 6;        // pieces a thread has in flight

// CTAs per SM that share the work: what shared memory (head size 128) or
// registers (64, for 16 heads a unit) allow.  (64 ragged rows of head size 64:
// 45.8 us with three, 59.1 with four.)
__host__ __device__ constexpr int attend_ctas(int d) { return d == 128 ? 2 : 3; }

// What starting a unit costs, in tiles: the pipeline fills and the warps' parts
// meet once per unit, whatever its length.  (Shares of tiles alone: 64 ragged rows
// 68 us instead of 46, 128 rows of 100 to 500 23.9 instead of 21.3.)  A share is at
// least one tile and its setup: with two setups 22 rows of 1576 took 12.1 us, not 10.9.
__host__ __device__ constexpr int attend_setup(int d) { return d == 128 ? 2 : 4; }

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
  uint32_t block_chunks, slot_chunks;   // 16-byte chunks between blocks and between slots
  float scale_log2;    // scale * log2(e)
  float *piece_o;      // [2 grid][heads][d]
  float *piece_ml;     // [2 grid][heads][2]
  // Where the join finds a split unit: row, unit, pieces (0: not split), the CTA of
  // its first piece.  By unit [rows * units], written by the CTA that begins it, or
  // where units outnumber the CTAs by CTA [grid], for the unit in its slot 1.
  int4 *piece_of;
  int32_t by_unit;
  int32_t ranks;       // CTAs of a cluster that takes one unit
};

// How the work meets the CTAs: units split over all of them, a unit for each, or
// a unit for a cluster of them.
enum class AttendForm { kSplit, kWhole, kCluster };

template <int D, int Warps>
struct AttendShared {
  // Steps of a warp's ring.  Two steps of copies in flight keep an SM's copy path
  // busy with 8 warps of head size 128, or 12 of 64; with one (two stages) 64 ragged
  // rows took 52.7 us, not 45.8.  Eight warps of head size 64 have room for five: 4 rows
  // x 8 heads of 3000 7.9 us, with two 9.4.
  static constexpr int kStages = Warps == kAttendWholeWarps && D == 64 ? 6 : 3;
  static constexpr int kRowBytes = D * 2;
  static constexpr int kStageBytes = 2 * kAttendKeys * kRowBytes;   // K then V
  static constexpr int kRingBytes = Warps * kStages * kStageBytes;
  static constexpr int kMergeStride = D + 4;                        // fp32; no bank conflicts for the fragment stores
  static constexpr int kMergeBytes = Warps * 8 * kMergeStride * 4;  // 8 heads of every warp
  // what a cluster's CTAs send one another: m and l of every rank and head, and of O the slice this CTA joins
  static constexpr int kInboxBytes(int heads) { return kAttendRanks * heads * 8 + (heads * (D / 4) + kAttendRanks) * 16; }
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

// A tile is a step of all warps of a CTA.  A row without keys still takes one:
// its zeros have to be written.
template <int Warps>
__host__ __device__ __forceinline__ int row_tiles(int length) {
  constexpr int kTile = Warps * kAttendKeys;
  return length <= kTile ? 1 : (length + kTile - 1) / kTile;
}

template <typename T, int D, int NT, int Warps, AttendForm Form>
__global__ void __launch_bounds__(Warps * 32, Form == AttendForm::kSplit ? attend_ctas(D) : Warps == 8 ? 1 : Warps == 4 ? 2 : 8)
attention_kernel(const AttentionPlan p) {
  using S = AttendShared<D, Warps>;
  constexpr bool kOneUnit = Form != AttendForm::kSplit, kCluster = Form == AttendForm::kCluster;
  constexpr int kAttendStages = S::kStages;
  constexpr int kAttendThreads = Warps * 32, kAttendTile = Warps * kAttendKeys;
  // The ring, then the merge's room (a whole unit's CTA merges in the ring).  Two
  // CTAs of head size 128 take the SM's shared memory to the last byte, so the
  // few words beside them lie in the padding of the merge's rows.
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float merge_ml[Warps][NT * 8][2];
  __shared__ float merge_f_room[NT == 1 ? Warps * 8 : 1];   // (16 heads: the factor replaces the maximum)
  auto factor = [&](int w, int h) -> float & { return NT == 1 ? merge_f_room[w * 8 + h] : merge_ml[w][h][0]; };
  uint32_t *const words = reinterpret_cast<uint32_t *>(ring + S::kRingBytes);
  auto word = [&](int line, int i) -> uint32_t & {   // word i < 4 (8) of 8 * Warps lines
    return kOneUnit ? words[line * 8 + i] : words[line * S::kMergeStride + D + i];
  };
  static_assert(kAttendStages <= (kOneUnit ? 8 : 4), "a line holds a warp's masks");
  constexpr int kChunks = D / 8;   // 16-byte chunks of a row
  const AttentionArgs &a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, q2 = (lane & 3) * 2;
  follow_predecessor();

  // -- this CTA's share of the work (row-major, units of a row; a unit is its
  // set-up, then its tiles) --
  constexpr int kSetup = attend_setup(D);
  int row, off = 0, left = 1, length0;
  const int ranks = kCluster ? p.ranks : 1, rank = kCluster ? static_cast<int>(blockIdx.x) : 0;
  if constexpr (kOneUnit) {
    // grid: (CTAs of the cluster, units, rows), or (units, rows in y and z)
    row = kCluster ? blockIdx.z : blockIdx.z * gridDim.y + blockIdx.y;
    if (row >= a.rows) return;
    length0 = row_length(p, row);
    if constexpr (kCluster) cluster_arrive();   // every CTA of the cluster runs before its shared memory is written
  } else {
    const int per = (a.rows + kAttendThreads - 1) / kAttendThreads;
    const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
    int mine = 0;
    for (int r = r0; r < r1; ++r) mine += row_tiles<Warps>(row_length(p, r)) + kSetup;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) word(Warps + warp, 0) = incl;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < Warps; ++w) {
      const int sum = static_cast<int>(word(Warps + w, 0));
      if (w < warp) incl += sum;
      total += sum;
    }
    total *= p.units;
    const int share = max(kSetup + 1, (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
    const int64_t begin64 = static_cast<int64_t>(blockIdx.x) * share;
    if (begin64 >= total) {
      if (!p.by_unit && tid == 0) p.piece_of[blockIdx.x] = make_int4(0, 0, 0, 0);
      return;
    }
    const int begin = static_cast<int>(begin64);
    int before = incl - mine;   // work (of one unit per row) before this thread's rows
    if (before * p.units <= begin && begin < incl * p.units) {
      for (int r = r0; r < r1; ++r) {
        const int n = row_tiles<Warps>(row_length(p, r)) + kSetup;
        if (begin < (before + n) * p.units) {
          word(2 * Warps, 0) = r;
          word(2 * Warps, 1) = begin - before * p.units;
          word(2 * Warps, 2) = min(share, total - begin);
          word(2 * Warps, 3) = row_length(p, r);
          break;
        }
        before += n;
      }
    }
    __syncthreads();
    row = word(2 * Warps, 0);
    off = word(2 * Warps, 1);
    left = word(2 * Warps, 2);
    length0 = word(2 * Warps, 3);
  }
  const int share_work = left;   // the full share wherever a unit goes on after this CTA
  int4 tail = make_int4(0, 0, 0, 0);

  // The CTA's work as segments, tiles of one unit each.  The copies run
  // kAttendStages - 1 steps ahead of the products, over the segments' ends: the
  // next unit's keys arrive while the last one's parts meet.
  struct Segment {
    int row, unit, n, t0, count, length;
  };
  struct Cursor {
    int row, off, left, length, length_ahead;   // lengths of the row and the next
  };
  auto begin_at = [&]() {
    Cursor c{row, off, left, length0, 0};
    if (!kOneUnit && row + 1 < a.rows) c.length_ahead = row_length(p, row + 1);
    return c;
  };
  auto next_segment = [&](Cursor &c, Segment &s) {
    while (c.left > 0) {
      s.row = c.row;
      s.length = c.length;
      s.n = row_tiles<Warps>(s.length);
      if constexpr (kOneUnit) {
        s.unit = kCluster ? blockIdx.y : blockIdx.x;
        s.t0 = rank;   // and every `ranks`-th tile from there, so that the first is known before the length
        s.count = s.n > rank ? (s.n - rank + ranks - 1) / ranks : 0;
        c.left = 0;
        return true;
      } else {
        const int cost = s.n + kSetup;
        s.unit = c.off / cost;
        const int at0 = c.off - s.unit * cost, take = min(cost - at0, c.left);
        s.t0 = max(0, at0 - kSetup);
        s.count = max(0, at0 + take - kSetup) - s.t0;
        c.off += take;
        c.left -= take;
        if (c.off == cost * p.units) {
          c.off = 0;
          ++c.row;
          c.length = c.length_ahead;
          if (c.row + 1 < a.rows) c.length_ahead = row_length(p, c.row + 1);
        }
        if (s.count > 0) return true;   // else only the set-up of a unit that the next CTA takes
      }
    }
    return false;
  };

  uint8_t *const my_ring = ring + warp * kAttendStages * S::kStageBytes;
  const uint32_t ring_addr = smem_u32(my_ring);
  Cursor load_cursor = begin_at();
  Segment from{};
  int load_tile = 0, next_block = -1;
  bool loading = true;
  const int32_t *table = nullptr;
  const uint4 *ksrc = nullptr, *vsrc = nullptr;
  // the block of this lane's key of a tile, fetched a step before its use (the
  // copies of a step do not wait for the table) and without the row's length
  // (the first step waits for one load, not two)
  auto block_of = [&](int i) {
    const int t = (from.t0 + i * ranks) * kAttendTile + warp * kAttendKeys + lane;
    if (lane >= kAttendKeys || t >= p.capacity) return -1;
    return table[p.block_shift >= 0 ? t >> p.block_shift : t / a.block_size];
  };
  auto load = [&](int stage) {
    if (loading && load_tile == from.count) {
      loading = next_segment(load_cursor, from);
      if (loading) {
        const int kvh = from.unit / p.chunks;
        table = a.block_table + from.row * a.table_stride;
        ksrc = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.key_cache) + kvh * D) + lane % kChunks;
        vsrc = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.value_cache) + kvh * D) + lane % kChunks;
        load_tile = 0;
        next_block = block_of(0);
        if constexpr (kOneUnit) loading = from.count > 0;
      }
    }
    uint32_t mask = 0;
    if (loading) {
      const int id = next_block;
      next_block = block_of(load_tile + 1);
      const int t = (from.t0 + load_tile * ranks) * kAttendTile + warp * kAttendKeys + lane;
      const bool live = t < from.length && id >= 0 && id < a.num_blocks;
      uint32_t at = 0;   // the key's row, in 16-byte chunks of the cache
      if (live) {
        const int in = p.block_shift >= 0 ? t & (a.block_size - 1) : t % a.block_size;
        at = static_cast<uint32_t>(id) * p.block_chunks + static_cast<uint32_t>(in) * p.slot_chunks;
      }
      mask = __ballot_sync(0xffffffffu, live);
      if (mask != 0) {
        // lane l copies chunk l % kChunks of the keys kKeys j + l / kChunks; a row's
        // chunks lie permuted by chunk ^ (key & 7) against bank conflicts
        constexpr int kKeys = 32 / kChunks;
        const int c = lane % kChunks, k0 = lane / kChunks;
        const uint32_t kdst = ring_addr + stage * S::kStageBytes + k0 * S::kRowBytes, swizzle = (c ^ k0) << 4;
#pragma unroll
        for (int j = 0; j < kAttendKeys / kKeys; ++j) {
          const uint32_t row_at = __shfl_sync(0xffffffffu, at, j * kKeys + k0);
          const int bytes = (mask >> (j * kKeys + k0)) & 1 ? 16 : 0;
          const uint32_t dst = kdst + j * kKeys * S::kRowBytes + (swizzle ^ (((j * kKeys) & 7) << 4));
          cp_async16_zfill(dst, ksrc + row_at, bytes);
          cp_async16_zfill(dst + kAttendKeys * S::kRowBytes, vsrc + row_at, bytes);
        }
      }
      ++load_tile;
    }
    if (lane == 0) word(warp, stage) = mask;
    cp_async_commit();
  };

  Cursor cursor = load_cursor;
  Segment now{};
#pragma unroll
  for (int i = 0; i < kAttendStages - 1; ++i) load(i);
  int stage = 0, fill = kAttendStages - 1;
  while (next_segment(cursor, now)) {
    const int unit = now.unit, t0 = now.t0, count = now.count, n = now.n, row_now = now.row;
    const int kvh = unit / p.chunks, head0 = kvh * p.groups + (unit - kvh * p.chunks) * p.chunk;
    const int heads = min(p.chunk, (kvh + 1) * p.groups - head0);

    // Q fragments: column n of the product is head head0 + 8 nt + n
    uint32_t qf[NT][D / 16][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + g;
      const T *qrow = static_cast<const T *>(a.q) + row_now * a.q_stride + static_cast<int64_t>(head0 + h) * D;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[nt][kk][0] = h < heads ? *reinterpret_cast<const uint32_t *>(qrow + kk * 16 + q2) : 0u;
        qf[nt][kk][1] = h < heads ? *reinterpret_cast<const uint32_t *>(qrow + kk * 16 + 8 + q2) : 0u;
      }
    }

    float acc[NT][D / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) acc[nt][dt][0] = acc[nt][dt][1] = acc[nt][dt][2] = acc[nt][dt][3] = 0.f;
    }

    for (int i = 0; i < count; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAttendStages - 2) : "memory");
      __syncwarp();
      const uint32_t mask = word(warp, stage);
      load(fill);   // the stage every lane left before the barrier above
      if (mask != 0) {
        const uint32_t kaddr = ring_addr + stage * S::kStageBytes, vaddr = kaddr + kAttendKeys * S::kRowBytes;
        float s[NT][4], s2[NT][4];   // two chains: a product waits for the one before the last
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[nt][j] = s2[nt][j] = 0.f;
        const int krow = lane & 15;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t ka[4];
          ldmatrix_x4(ka, kaddr + krow * S::kRowBytes + (((2 * kk + (lane >> 4)) ^ (krow & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) Element<T>::mma(kk & 1 ? s2[nt] : s[nt], ka, qf[nt][kk][0], qf[nt][kk][1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[nt][j] += s2[nt][j];
        const bool live0 = (mask >> g) & 1, live1 = (mask >> (g + 8)) & 1;
        uint32_t pb[NT][2], pl[NT][2];   // the probabilities' two terms
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
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            constexpr float kLift = Element<T>::kLift, kBelow = kLift * (1.f - 2.f * Element<T>::kHalfStep);
            const uint32_t top = Element<T>::pack(e[2 * j] * kBelow, e[2 * j + 1] * kBelow);
            const float2 taken = Element<T>::unpack(top);
            pb[nt][j] = transpose8x8(top);
            pl[nt][j] = transpose8x8(Element<T>::pack(fmaf(e[2 * j], kLift, -taken.x), fmaf(e[2 * j + 1], kLift, -taken.y)));
          }
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
          for (int nt = 0; nt < NT; ++nt) {
            Element<T>::mma(acc[nt][dt], va, pb[nt][0], pb[nt][1]);
            Element<T>::mma(acc[nt][dt], va, pl[nt][0], pl[nt][1]);
          }
        }
      }
      stage = stage + 1 == kAttendStages ? 0 : stage + 1;
      fill = fill + 1 == kAttendStages ? 0 : fill + 1;
    }
    // -- the warps' parts of the segment meet in shared memory --
    if constexpr (kOneUnit) cp_async_wait_all();   // the ring, done with, is the room for it
    float *const merge = reinterpret_cast<float *>(kOneUnit ? ring : ring + S::kRingBytes);
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
    __syncthreads();   // every warp is done with its products, and with the merge before this one
    const bool whole = kOneUnit ? !kCluster : t0 == 0 && count == n;
    // the cluster's inbox: [rank][head] (m, l), then [rank][join_each] four dimensions of O
    float2 *const inbox_ml = reinterpret_cast<float2 *>(words + Warps * 8);
    float4 *const inbox_o = reinterpret_cast<float4 *>(inbox_ml + kAttendRanks * NT * 8);
    const int join_each = kOneUnit ? (heads * (D / 4) + ranks - 1) / ranks : 0;
    if constexpr (kCluster) cluster_wait();
    const int64_t piece = 2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0 ? 1 : 0);
    if (tid < (heads * Warps + 31) / 32 * 32) {   // whole warps: a lane per (head, warp)
      // the head's maximum and sum over the warps, each warp's factor, lse
      const int h = tid / Warps, w = tid % Warps;
      const bool live = h < heads;
      const float m_w = live ? merge_ml[w][h][0] : -INFINITY, l_w = live ? merge_ml[w][h][1] : 0.f;
      float top = m_w;
#pragma unroll
      for (int o = 1; o < Warps; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float f = exp2f(m_w - (top == -INFINITY ? 0.f : top));
      float sum = l_w * f;
#pragma unroll
      for (int o = 1; o < Warps; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (live) {
        // a whole unit is divided here; no key with a weight gives zeros and log 0
        factor(w, h) = (!whole ? f : sum == 0.f ? 0.f : f / sum) * (1.f / Element<T>::kLift);
        if constexpr (kCluster) {
          for (int r = w; r < ranks; r += Warps) store_cluster(inbox_ml + rank * (NT * 8) + h, r, make_float2(top, sum));
        } else if (w == 0) {
          if (!whole) {
            *reinterpret_cast<float2 *>(p.piece_ml + (piece * (NT * 8) + h) * 2) = make_float2(top, sum);
          } else if (a.lse != nullptr) {
            a.lse[static_cast<int64_t>(row_now) * a.nq + head0 + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
          }
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {   // 8 heads at a time
      if (nt > 0) __syncthreads();
      float *const h0 = merge + (warp * 8 + q2) * S::kMergeStride + g;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        h0[dt * 16] = acc[nt][dt][0];
        h0[dt * 16 + S::kMergeStride] = acc[nt][dt][1];
        h0[dt * 16 + 8] = acc[nt][dt][2];
        h0[dt * 16 + 8 + S::kMergeStride] = acc[nt][dt][3];
      }
      __syncthreads();
      for (int i = tid; i < min(8, heads - nt * 8) * (D / 4); i += kAttendThreads) {   // four dimensions a thread
        const int h = i / (D / 4), c = i % (D / 4) * 4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < Warps; ++w) {
          const float f = factor(w, nt * 8 + h);
          const float4 v = *reinterpret_cast<const float4 *>(merge + (w * 8 + h) * S::kMergeStride + c);
          o.x = fmaf(v.x, f, o.x);
          o.y = fmaf(v.y, f, o.y);
          o.z = fmaf(v.z, f, o.z);
          o.w = fmaf(v.w, f, o.w);
        }
        if (whole) {
          *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + row_now * a.out_stride + static_cast<int64_t>(head0 + nt * 8 + h) * D + c) =
              make_uint2(Element<T>::pack(o.x, o.y), Element<T>::pack(o.z, o.w));
        } else if constexpr (kCluster) {
          const int to = (nt * (8 * D / 4) + i) / join_each;
          store_cluster(inbox_o + rank * join_each + (nt * (8 * D / 4) + i - to * join_each), to, o);
        } else {
          *reinterpret_cast<float4 *>(p.piece_o + piece * (NT * 8 * D) + (nt * 8 + h) * D + c) = o;
        }
      }
    }
    if constexpr (kCluster) {   // every CTA joins its slice of the heads' dimensions
      cluster_arrive();
      cluster_wait();
      const int i = rank * join_each + tid, h = i / (D / 4), c = i % (D / 4) * 4;
      if (tid < join_each && h < heads) {
        float top = -INFINITY;
        for (int r = 0; r < ranks; ++r) top = fmaxf(top, inbox_ml[r * (NT * 8) + h].x);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < ranks; ++r) {
          const float2 ml = inbox_ml[r * (NT * 8) + h];
          const float4 v = inbox_o[r * join_each + tid];
          const float f = exp2f(ml.x - base);
          sum = fmaf(ml.y, f, sum);
          o.x = fmaf(v.x, f, o.x);
          o.y = fmaf(v.y, f, o.y);
          o.z = fmaf(v.z, f, o.z);
          o.w = fmaf(v.w, f, o.w);
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + row_now * a.out_stride + static_cast<int64_t>(head0 + h) * D + c) =
            make_uint2(Element<T>::pack(o.x * inv, o.y * inv), Element<T>::pack(o.z * inv, o.w * inv));
        if (c == 0 && a.lse != nullptr)
          a.lse[static_cast<int64_t>(row_now) * a.nq + head0 + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
      }
    }
    if (NT > 1 && !kOneUnit) __syncthreads();   // the factors have been read
    if (!kOneUnit && t0 == 0) {
      const int4 of = make_int4(row_now, unit, whole ? 0 : 1 + (n - count + share_work - 1) / share_work, blockIdx.x);
      if (p.by_unit) {
        if (tid == 0) p.piece_of[row_now * p.units + unit] = of;
      } else if (!whole) {
        tail = of;
      }
    }
  }
  if (!kOneUnit && !p.by_unit && tid == 0) p.piece_of[blockIdx.x] = tail;
}

// Joins the pieces of a split unit (piece_of), `heads_each` of its heads a CTA.
// D / 4 lanes take a head's row of a piece, four dimensions each; the lanes'
// groups share the heads and their pieces.  The pieces come from L2 and latency
// bounds it: 3 us of 47 for one row of 131071 (4 units of 74 pieces, a CTA for
// each of their heads; with a CTA for each unit 52 us in all).
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinThreads, 1) attention_join_kernel(const AttentionPlan p, const int32_t heads_each) {
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes;
  __shared__ __align__(16) float red[kGroups][D];
  __shared__ float red_ml[kGroups][2];
  follow_predecessor();
  const int4 of = p.piece_of[blockIdx.x];
  const int pieces = of.z;
  if (pieces == 0) return;
  const AttentionArgs &a = p.a;
  const int row = of.x, kvh = of.y / p.chunks;
  const int unit_head0 = kvh * p.groups + (of.y - kvh * p.chunks) * p.chunk;
  const int skip = blockIdx.y * heads_each;   // the unit's heads before this CTA's
  const int head0 = unit_head0 + skip;
  const int heads = min(min(p.chunk, (kvh + 1) * p.groups - unit_head0) - skip, heads_each);
  if (heads <= 0) return;
  const int parts = min(kGroups / heads, pieces);   // groups that share a head
  const int c = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int h = group % heads, part = group / heads;
  if (part < parts) {
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = part; i0 < pieces; i0 += parts * kJoinBatch) {
      float2 ml[kJoinBatch];
      float4 v[kJoinBatch];
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) {
        const int i = i0 + k * parts;
        ml[k] = make_float2(-INFINITY, 0.f);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < pieces) {
          // the first piece lies in slot 1 of its CTA, the others in slot 0 of the CTAs after it
          const int64_t piece = i == 0 ? 2 * static_cast<int64_t>(of.w) + 1 : 2 * (static_cast<int64_t>(of.w) + i);
          ml[k] = *reinterpret_cast<const float2 *>(p.piece_ml + (piece * (NT * 8) + skip + h) * 2);
          v[k] = *reinterpret_cast<const float4 *>(p.piece_o + piece * (NT * 8 * D) + (skip + h) * D + c * 4);
        }
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) top = fmaxf(top, ml[k].x);
      const float base = top == -INFINITY ? 0.f : top;
      const float fa = exp2f(m - base);
      o.x *= fa;
      o.y *= fa;
      o.z *= fa;
      o.w *= fa;
      l *= fa;
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) {
        const float f = exp2f(ml[k].x - base);
        o.x = fmaf(v[k].x, f, o.x);
        o.y = fmaf(v[k].y, f, o.y);
        o.z = fmaf(v[k].z, f, o.z);
        o.w = fmaf(v[k].w, f, o.w);
        l = fmaf(ml[k].y, f, l);
      }
      m = top;
    }
    *reinterpret_cast<float4 *>(&red[group][c * 4]) = o;
    if (c == 0) {
      red_ml[group][0] = m;
      red_ml[group][1] = l;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * D; i += kJoinThreads) {
    const int head = i / D, d = i % D;
    float top = -INFINITY;
    for (int k = 0; k < parts; ++k) top = fmaxf(top, red_ml[k * heads + head][0]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, v = 0.f;
    for (int k = 0; k < parts; ++k) {
      const float f = exp2f(red_ml[k * heads + head][0] - base);
      sum = fmaf(red_ml[k * heads + head][1], f, sum);
      v = fmaf(red[k * heads + head][d], f, v);
    }
    static_cast<T *>(a.out)[row * a.out_stride + static_cast<int64_t>(head0) * D + i] = Element<T>::round(sum == 0.f ? 0.f : v / sum);
    if (d == 0 && a.lse != nullptr)
      a.lse[static_cast<int64_t>(row) * a.nq + head0 + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
  }
}

}  // namespace ops
}  // namespace cruise
