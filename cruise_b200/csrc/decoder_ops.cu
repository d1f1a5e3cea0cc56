// decoder_ops.cu -- launches and C ABI of the decoder operators
// (include/cruise_decoder.h).
#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "../../include/cruise_decoder.h"
#include "decoder_attention.cuh"
#include "decoder_choose.cuh"
#include "decoder_ops.h"
#include "decoder_rotate.cuh"

namespace cruise {
namespace ops {
namespace {

constexpr int kMaxDevices = 64;
constexpr int64_t kMaxIndex = 0x7fffffff;

// Streaming multiprocessors of a device (148 where it cannot be asked: sizes
// are then only planned, not run).
int sm_count(int device) {
  static std::atomic<int> known[kMaxDevices];
  const bool cached = device >= 0 && device < kMaxDevices;
  if (cached) {
    const int n = known[device].load(std::memory_order_relaxed);
    if (n > 0) return n;
  }
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 148;
  }
  if (cached) known[device].store(n, std::memory_order_relaxed);
  return n;
}

// The calling thread's device for the length of a launch.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    error = cudaGetDevice(&before_);
    if (error == cudaSuccess && before_ != device) {
      error = cudaSetDevice(device);
      moved_ = error == cudaSuccess;
    }
  }
  ~DeviceScope() {
    if (moved_) cudaSetDevice(before_);
  }
  cudaError_t error = cudaSuccess;

 private:
  int before_ = 0;
  bool moved_ = false;
};

// Raises a kernel's shared-memory limit once per device.
template <typename Kernel>
cudaError_t allow_shared(Kernel kernel, size_t bytes, int device, std::atomic<uint64_t> &done, bool wide_cluster = false) {
  const uint64_t bit = device >= 0 && device < kMaxDevices ? 1ull << device : 0;
  if (bit != 0 && (done.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (err == cudaSuccess && wide_cluster)
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (err == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return err;
}

// Launches a kernel so that it may come onto the SMs while its predecessor in
// the stream drains; it waits for that inside (follow_predecessor): calls of 4 rows
// of 256 one after the other take 4.8 us each so, 6.3 without.  `cluster` CTAs of x
// share their shared memory.
template <typename... Params, typename... Actual>
cudaError_t launch(void (*kernel)(Params...), dim3 grid, int threads, size_t shared, int cluster, cudaStream_t stream,
                   const Actual &...args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// What an occupancy query takes of such a launch.
cudaLaunchConfig_t cluster_launch(dim3 grid, int threads, size_t shared, int cluster, cudaLaunchAttribute &attr) {
  cudaLaunchConfig_t cfg{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cfg;
}

// ---- rotate_store --------------------------------------------------------------

template <typename T, int D>
cudaError_t rotate_typed(const RotateArgs &a, int device, cudaStream_t stream) {
  constexpr int kHeads = 512 / D;   // heads of a kind a warp moves per round
  const int all = (a.nq + kHeads - 1) / kHeads + 2 * ((a.nkv + kHeads - 1) / kHeads);
  // as many rounds per warp as still leave 16 warps per SM: few tokens spread
  // their heads over the GPU, many keep their table row in registers (4 tokens: 2.1 us
  // with one round, 4.1 with all; 8192 tokens: 65 and 31)
  const int64_t want = static_cast<int64_t>(sm_count(device)) * 16;
  const int rounds = static_cast<int>(std::clamp<int64_t>(static_cast<int64_t>(a.tokens) * all / want, 1, all));
  const int warps_per_token = (all + rounds - 1) / rounds;
  const int64_t warps = static_cast<int64_t>(a.tokens) * warps_per_token;
  const unsigned grid = static_cast<unsigned>((warps * 32 + kRotateThreads - 1) / kRotateThreads);
  const bool full = a.rotary == D;
  auto *kernel = a.q_norm != nullptr ? (full ? rotate_store_kernel<T, D, true, true> : rotate_store_kernel<T, D, true, false>)
                                     : (full ? rotate_store_kernel<T, D, false, true> : rotate_store_kernel<T, D, false, false>);
  return launch(kernel, dim3(grid), kRotateThreads, 0, 1, stream, a, rounds, warps_per_token);
}

// ---- paged_attention -----------------------------------------------------------

// How the heads of a KV head form units of at most 16, and how many CTAs take a
// unit as a cluster (0: the units are split over all CTAs).
struct AttentionShape {
  int32_t groups, chunks, chunk, units;
  int32_t warps;   // of a CTA that takes a unit, 0: units are split over all CTAs
  int32_t ranks;
  int grid;   // CTAs of the split form
};

template <typename T, int D, int NT, int Warps, bool Cluster>
cudaError_t allow_whole(int device, size_t *bytes) {
  using Shared = AttendShared<D, Warps>;
  static_assert(Shared::kMergeBytes <= Shared::kRingBytes, "the merge takes the ring's room");
  static std::atomic<uint64_t> done{0};
  *bytes = Shared::kRingBytes + Warps * 32 + (Cluster ? Shared::kInboxBytes(NT * 8) : 0);
  return allow_shared(attention_kernel<T, D, NT, Warps, Cluster ? AttendForm::kCluster : AttendForm::kWhole>, *bytes, device, done, Cluster);
}

// Clusters of `ranks` CTAs, an SM each, that run at once (the types' kernels do
// not differ in this).
template <int D, int NT>
int attention_fit(int ranks, int device) {
  static std::atomic<int> known[kMaxDevices][kAttendRanks + 1];
  const bool cached = device >= 0 && device < kMaxDevices;
  if (ranks == 1) return sm_count(device);
  if (cached) {
    const int n = known[device][ranks].load(std::memory_order_relaxed);
    if (n > 0) return n;
  }
  DeviceScope scope(device);
  size_t shared = 0;
  int n = 0;
  if (scope.error == cudaSuccess && allow_whole<__nv_bfloat16, D, NT, kAttendWholeWarps, true>(device, &shared) == cudaSuccess) {
    cudaLaunchAttribute attr{};
    const cudaLaunchConfig_t cfg = cluster_launch(dim3(ranks), kAttendWholeWarps * 32, shared, ranks, attr);
    if (cudaOccupancyMaxActiveClusters(&n, attention_kernel<__nv_bfloat16, D, NT, kAttendWholeWarps, AttendForm::kCluster>, &cfg) != cudaSuccess) n = 0;
  }
  if (n <= 0) {
    cudaGetLastError();
    return sm_count(device) / 16 * (16 / ranks);
  }
  if (cached) known[device][ranks].store(n, std::memory_order_relaxed);
  return n;
}

AttentionShape attention_shape(int32_t rows, int32_t nq, int32_t nkv, int32_t d, int64_t capacity, int device) {
  AttentionShape s;
  s.groups = nq / nkv;
  s.chunks = (s.groups + 15) / 16;
  s.chunk = (s.groups + s.chunks - 1) / s.chunks;
  s.units = nkv * s.chunks;
  s.ranks = 1;
  s.warps = 0;
  s.grid = 0;
  const int sms = sm_count(device);
  const int64_t units = std::max<int64_t>(1, static_cast<int64_t>(rows) * s.units);
  // Which form, in us for units x positions of head size 128 (28 heads over 4)
  // where nothing else is said.  A CTA of one warp needs no merge and comes eight
  // times to an SM, one of four twice, but each works through its unit alone:
  //   8 x 16: one warp 2.6, four 2.8, eight 3.6; 8 x 64: 4.3, 2.8, 3.7
  //   300 x 64: one 5.1, four 5.4; 300 x 128: 7.5, 6.4; 1200 x 256: 23.0, 28.6
  //   (head size 64, whose four-warp CTAs are smaller: 600 x 128: 6.7, 5.7; 1200 x 128: 8.2, 9.3)
  // (Short rows in a wide table are taken for long ones: 4 rows of 256 4.5 us, in a table
  // for 131072 positions 8.1; 64 of up to 500 8.5 and 11.2.)
  if (capacity <= kAttendKeys || (units * d >= 512 * capacity && capacity <= 512)) {
    s.warps = 1;
    return s;
  }
  if (units <= sms) {
    //   64 x 64: four 3.2, eight 3.6; 144 x 128: 4.4, 4.2
    if (capacity <= 4 * kAttendKeys || (capacity <= 8 * kAttendKeys && 2 * units <= sms)) {
      s.warps = 4;
      return s;
    }
    // A cluster's join costs 1 us, the split's second kernel 4 and more, but the
    // split also evens out lengths and uses every SM; a CTA takes 0.75 us per
    // 128 positions.  16 x 256: one CTA 4.4, clusters of two 5.1; 32 x 384 of head size 64: 4.0, 4.6;
    // 16 x 512: one 5.9, four 5.1; 16 x 2048: clusters 7.0, split 9.4; 4 x 8192: 8.0, 9.1;
    // 4 x 16384: 12.2, 11.7; head size 64, 8 x 30000: 18.6, 16.4.
    const auto fit = d == 128 ? (s.chunk <= 8 ? attention_fit<128, 1> : attention_fit<128, 2>)
                              : (s.chunk <= 8 ? attention_fit<64, 1> : attention_fit<64, 2>);
    constexpr int kTile = kAttendWholeWarps * kAttendKeys;
    const int64_t tiles = (capacity + kTile - 1) / kTile;
    int ranks = tiles <= 3 ? 1 : static_cast<int>(std::min<int64_t>({sms / units, tiles, kAttendRanks}));
    while (ranks > 1 && fit(ranks, device) < units) --ranks;
    if (tiles <= 8 * ranks) {
      s.warps = kAttendWholeWarps;
      s.ranks = ranks;
      return s;
    }
  } else if (capacity <= std::min<int64_t>(1024, 512 + units)) {
    // 240 x 512: four warps a unit 13.6, split 18.9; 600 x 768: 46.2, 45.9; but the
    // longest unit alone takes 15 ns a position: 240 rows of 1 to 1024: 13.9, split 11.1
    s.warps = 4;
    return s;
  }
  s.grid = sms * attend_ctas(d);
  return s;
}

size_t align16(size_t v) { return (v + 15) / 16 * 16; }

size_t pieces_bytes(int grid, int heads, int d, size_t *ml, size_t *of) {
  size_t bytes = align16(static_cast<size_t>(2) * grid * heads * d * 4);
  if (ml != nullptr) *ml = bytes;
  bytes += align16(static_cast<size_t>(2) * grid * heads * 2 * 4);
  if (of != nullptr) *of = bytes;
  return bytes + static_cast<size_t>(grid) * sizeof(int4);
}

template <typename T, int D, int NT>
cudaError_t attention_typed(const AttentionArgs &a, const AttentionShape &s, int device, cudaStream_t stream) {
  AttentionPlan p{};
  p.a = a;
  p.groups = s.groups;
  p.chunk = s.chunk;
  p.chunks = s.chunks;
  p.units = s.units;
  p.block_shift = -1;
  for (int b = 0; b < 31; ++b)
    if (a.block_size == 1 << b) p.block_shift = b;
  p.capacity = a.table_width * a.block_size;
  p.block_chunks = static_cast<uint32_t>(a.block_stride / 8);
  p.slot_chunks = static_cast<uint32_t>(a.nkv * D / 8);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  static std::atomic<uint64_t> done{0};
  if (s.warps > 0) {
    p.ranks = s.ranks;
    const auto run = [&](auto warps, auto cluster) {
      size_t smem = 0;
      const cudaError_t err = allow_whole<T, D, NT, warps, cluster>(device, &smem);
      if (err != cudaSuccess) return err;
      const unsigned units = s.units, rows = a.rows, most = 65535;
      const dim3 grid = cluster ? dim3(s.ranks, units, rows) : dim3(units, std::min(rows, most), (rows + most - 1) / most);
      return launch(attention_kernel<T, D, NT, warps, cluster ? AttendForm::kCluster : AttendForm::kWhole>, grid, warps * 32, smem,
                    s.ranks, stream, p);
    };
    using Eight = std::integral_constant<int, kAttendWholeWarps>;
    switch (s.warps) {
      case 1: return run(std::integral_constant<int, 1>(), std::false_type());
      case 4: return run(std::integral_constant<int, 4>(), std::false_type());
      default: return s.ranks > 1 ? run(Eight(), std::true_type()) : run(Eight(), std::false_type());
    }
  }
  // where the join looks: at every unit while they are no more than the CTAs (one
  // row of 131071: 47 us; a join per CTA, most with nothing to do, 51)
  p.by_unit = static_cast<int64_t>(a.rows) * s.units <= s.grid ? 1 : 0;
  size_t ml = 0, of = 0;
  pieces_bytes(s.grid, NT * 8, D, &ml, &of);
  uint8_t *w = static_cast<uint8_t *>(a.workspace);
  p.piece_o = reinterpret_cast<float *>(w);
  p.piece_ml = reinterpret_cast<float *>(w + ml);
  p.piece_of = reinterpret_cast<int4 *>(w + of);
  constexpr size_t smem = AttendShared<D, kAttendWarps>::kRingBytes + AttendShared<D, kAttendWarps>::kMergeBytes;
  auto *kernel = attention_kernel<T, D, NT, kAttendWarps, AttendForm::kSplit>;
  cudaError_t err = allow_shared(kernel, smem, device, done);
  if (err != cudaSuccess) return err;
  err = launch(kernel, dim3(s.grid), kAttendWarps * 32, smem, 1, stream, p);
  if (err != cudaSuccess) return err;
  // few units: a CTA for some heads of each, so that the join is spread over the SMs
  // (one row of 131071: 47.1 us, 52.0 with all heads of a unit in one)
  const int64_t units = static_cast<int64_t>(a.rows) * s.units;
  const int entries = p.by_unit ? static_cast<int>(units) : s.grid;
  const int each = std::clamp((s.chunk * entries + sm_count(device) - 1) / sm_count(device), 1, s.chunk);
  return launch(attention_join_kernel<T, D, NT>, dim3(entries, (s.chunk + each - 1) / each), kJoinThreads, 0, 1, stream, p, each);
}

template <typename T>
cudaError_t attention_of(const AttentionArgs &a, const AttentionShape &s, int device, cudaStream_t stream) {
  if (a.d == 128)
    return s.chunk <= 8 ? attention_typed<T, 128, 1>(a, s, device, stream) : attention_typed<T, 128, 2>(a, s, device, stream);
  return s.chunk <= 8 ? attention_typed<T, 64, 1>(a, s, device, stream) : attention_typed<T, 64, 2>(a, s, device, stream);
}

// ---- choose --------------------------------------------------------------------

// Clusters of 2^log CTAs that run at once: `alone` with an SM for each CTA, else
// two to an SM.  Asked once per device (clusters lie within a group of SMs, and
// the groups are not of one size: eight of 16 do not fit 148 SMs).
template <typename T>
int choose_fit(int log, bool alone, int device) {
  static std::atomic<int> known[kMaxDevices][2][5];
  const int ctas = 1 << log;
  const bool cached = device >= 0 && device < kMaxDevices;
  if (cached) {
    const int n = known[device][alone ? 1 : 0][log].load(std::memory_order_relaxed);
    if (n > 0) return n;
  }
  cudaLaunchAttribute attr{};
  const cudaLaunchConfig_t cfg = cluster_launch(dim3(ctas), kChooseThreads, alone ? kChooseAlone : kChooseAlone / 2, ctas, attr);
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, choose_kernel<T, kChooseFewThreads>, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 1;
  }
  if (cached) known[device][alone ? 1 : 0][log].store(n, std::memory_order_relaxed);
  return n;
}

template <typename T>
cudaError_t choose_typed(const ChooseArgs &a, int device, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0}, done_many{0};
  cudaError_t err = allow_shared(choose_kernel<T, kChooseFewThreads>, kChooseShared, device, done, true);
  if (err == cudaSuccess) err = allow_shared(choose_kernel<T, kChooseManyThreads>, kChooseShared, device, done_many, true);
  if (err != cudaSuccess) return err;
  const int64_t entries = (a.history != nullptr ? a.history_width : 0) + static_cast<int64_t>(a.bias_token != nullptr ? a.bias_width : 0);
  // CTAs per row: a CTA takes about 5 us for the chain of its steps and the
  // marked tokens (as long as it streams 32768 fp32 logits), clusters 1 us more;
  // two to an SM, the first takes 1.3 and the stream 1.6 times as long.  One row
  // of 152064 with 1000 entries: 6.0 us with 16 CTAs, 7.6 with four, 14.3 with one;
  // 17 rows: 12.9, 8.0, 16.3; 64 rows: 36 with 16, 12.6 with four, 26 with one.
  // The entries are the tensors' widths, for the lengths are on the device: where
  // these are far smaller, a wide history still costs a cluster's room (64 rows of
  // 152064 with 1000 tokens: 10.8 us in a history of 1024, 13.0 of 8192, 31.9 of 32768).
  int best = 0;
  bool alone = false;
  double least = 0;
  for (int log = 0; log < 5; ++log) {
    const int32_t slice = choose_slice(a.vocab, 1 << log);
    const size_t shared = choose_shared(slice, entries);
    if (shared > (log < 4 ? 100 * 1024 : kChooseShared)) continue;
    const bool one = a.rows <= choose_fit<T>(log, true, device);
    const int two = one ? a.rows : choose_fit<T>(log, false, device);
    const double stream_cost = slice * (sizeof(T) / 4.0), chain = 32768 + (log > 0 ? 7000 : 0);
    const double cost = (one ? chain + stream_cost : 1.3 * chain + 1.6 * stream_cost) * ((a.rows + two - 1) / two);
    if (least == 0 || cost < least) {
      least = cost;
      best = log;
      alone = one;
    }
  }
  const int ctas = 1 << best;
  const int32_t slice = choose_slice(a.vocab, ctas);
  // Where every CTA can have an SM of its own it takes more than half its shared
  // memory: a successor's CTAs, which come while this launch drains, would else
  // settle two on the SMs it left idle (64 rows of 50257: 11.2 us, 8.0 so)
  const size_t shared = choose_shared(slice, entries);
  // The marked tokens and the stream share a CTA's threads: 100 rows of 32000 with
  // 1000 entries 8.0 us with few threads for the former and 6.9 with many, with 30
  // entries and processed logits 7.8 and 9.4; 100 rows of 64000: 9.9 and 13.6,
  // with 4000 entries 17.9 and 13.8; 256 rows of 152064 with 4000: 33 and 41.
  const double streamed = slice * (sizeof(T) / 4.0) * (a.processed != nullptr ? 2 : 1);
  auto *kernel = 36.0 * entries >= streamed ? choose_kernel<T, kChooseManyThreads> : choose_kernel<T, kChooseFewThreads>;
  return launch(kernel, dim3(ctas, a.rows), kChooseThreads, alone ? std::max(shared, kChooseAlone) : shared, ctas,
                stream, a, slice);
}

// ---- errors --------------------------------------------------------------------

thread_local char g_error[256] = "";

int32_t refuse(const char *format, ...) {
  va_list args;
  va_start(args, format);
  std::vsnprintf(g_error, sizeof(g_error), format, args);
  va_end(args);
  return -1;
}

int32_t report(cudaError_t err, const char *what) {
  if (err == cudaSuccess) {
    g_error[0] = 0;
    return 0;
  }
  std::snprintf(g_error, sizeof(g_error), "%s: %s", what, cudaGetErrorString(err));
  return static_cast<int32_t>(err);
}

// An array, from its first byte to its last; whether two meet (one of `a` and one of `b`).
struct Span {
  const void *at;
  int64_t bytes;
};
bool meets(const Span &a, const Span &b) { return overlap(a.at, a.bytes, b.at, b.bytes); }
template <size_t N, size_t M>
bool meets(const Span (&a)[N], const Span (&b)[M]) {
  for (const Span &x : a)
    for (const Span &y : b)
      if (meets(x, y)) return true;
  return false;
}

// Whether a block of `a` overlaps one of `b`: both have n blocks of `bytes`, `stride`
// bytes apart, and may lie between one another (the two caches in one tensor).
bool blocks_overlap(const void *a, const void *b, int64_t n, int64_t stride, int64_t bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  const uint64_t apart = x < y ? y - x : x - y, blocks = apart / stride, rest = apart % stride;
  const uint64_t last = static_cast<uint64_t>(n) - 1;   // block i of the lower one meets block i - blocks (- 1) of the other
  return (blocks <= last && rest < static_cast<uint64_t>(bytes)) ||
         (blocks + 1 <= last && static_cast<uint64_t>(stride) - rest < static_cast<uint64_t>(bytes));
}

bool aligned(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace

cudaError_t launch_rotate_store(const RotateArgs &a, int device, cudaStream_t stream) {
  if (a.tokens == 0) return cudaSuccess;
  if (a.dtype == kBf16)
    return a.d == 128 ? rotate_typed<__nv_bfloat16, 128>(a, device, stream) : rotate_typed<__nv_bfloat16, 64>(a, device, stream);
  return a.d == 128 ? rotate_typed<__half, 128>(a, device, stream) : rotate_typed<__half, 64>(a, device, stream);
}

int64_t attention_workspace(int32_t rows, int32_t nq, int32_t nkv, int32_t d, int64_t capacity, int device) {
  const AttentionShape s = attention_shape(rows, nq, nkv, d, capacity, device);
  if (s.warps > 0) return 0;
  return static_cast<int64_t>(pieces_bytes(s.grid, s.chunk <= 8 ? 8 : 16, d, nullptr, nullptr));
}

cudaError_t launch_paged_attention(const AttentionArgs &a, int device, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  const AttentionShape s =
      attention_shape(a.rows, a.nq, a.nkv, a.d, static_cast<int64_t>(a.table_width) * a.block_size, device);
  return a.dtype == kBf16 ? attention_of<__nv_bfloat16>(a, s, device, stream) : attention_of<__half>(a, s, device, stream);
}

cudaError_t launch_choose(const ChooseArgs &a, int device, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.dtype) {
    case kFp32: return choose_typed<float>(a, device, stream);
    case kBf16: return choose_typed<__nv_bfloat16>(a, device, stream);
    default: return choose_typed<__half>(a, device, stream);
  }
}

}  // namespace ops
}  // namespace cruise

using namespace cruise::ops;

extern "C" {

const char *cruise_decoder_last_error(void) { return g_error; }

int32_t cruise_decoder_rotate_store(const void *qkv, int64_t qkv_stride, int32_t tokens, int32_t num_heads,
                                    int32_t num_kv_heads, int32_t head_dim, int32_t dtype, const int64_t *position,
                                    const int32_t *slot, const void *q_norm, const void *k_norm, float eps,
                                    const void *rope_cos, const void *rope_sin, int32_t rope_dtype, int32_t rope_rows,
                                    int32_t rotary, void *q_out, int64_t q_stride, void *key_cache, void *value_cache,
                                    int64_t num_blocks, int32_t block_size, int64_t block_stride, int32_t device,
                                    void *stream) {
  const char *const op = "cruise_decoder_rotate_store";
  if (tokens < 0 || num_heads < 1 || num_kv_heads < 1 || num_heads > 1024 || num_kv_heads > 1024)
    return refuse("%s: %d tokens of %d query and %d KV heads (tokens >= 0, heads 1 to 1024)", op, tokens, num_heads, num_kv_heads);
  if (head_dim != 64 && head_dim != 128) return refuse("%s: head size %d (64 or 128)", op, head_dim);
  if (dtype != kBf16 && dtype != kFp16) return refuse("%s: dtype %d (0 bf16 or 1 fp16)", op, dtype);
  if (rope_dtype != kBf16 && rope_dtype != kFp32) return refuse("%s: rope dtype %d (0 bf16 or 2 fp32)", op, rope_dtype);
  if (rope_rows < 1 || rotary < 16 || rotary % 16 != 0 || rotary > head_dim)
    return refuse("%s: tables of %d rows x %d (rows >= 1, a multiple of 16 up to the head size)", op, rope_rows, rotary);
  if ((q_norm == nullptr) != (k_norm == nullptr)) return refuse("%s: pass both norm weights or neither", op);
  if (num_blocks < 1 || block_size < 1 || num_blocks > kMaxIndex / block_size)
    return refuse("%s: a cache of %lld blocks of %d slots (at least one, slots below 2^31)", op, static_cast<long long>(num_blocks), block_size);
  const int64_t width = static_cast<int64_t>(num_heads + 2 * num_kv_heads) * head_dim, q_width = static_cast<int64_t>(num_heads) * head_dim;
  const int64_t block_elems = static_cast<int64_t>(block_size) * num_kv_heads * head_dim;
  if (qkv_stride < width || q_stride < q_width || block_stride < block_elems)
    return refuse("%s: a stride is smaller than its row (qkv %lld, q %lld, block %lld)", op, static_cast<long long>(qkv_stride),
                  static_cast<long long>(q_stride), static_cast<long long>(block_stride));
  if (qkv_stride % 8 != 0 || q_stride % 8 != 0 || block_stride % 8 != 0)
    return refuse("%s: strides must be multiples of 8 elements", op);
  if (tokens == 0) return report(cudaSuccess, op);
  if (qkv == nullptr || position == nullptr || slot == nullptr || rope_cos == nullptr || rope_sin == nullptr ||
      q_out == nullptr || key_cache == nullptr || value_cache == nullptr)
    return refuse("%s: a required pointer is NULL", op);
  if (!aligned(qkv, 16) || !aligned(q_norm, 16) || !aligned(k_norm, 16) || !aligned(rope_cos, 16) ||
      !aligned(rope_sin, 16) || !aligned(q_out, 16) || !aligned(key_cache, 16) || !aligned(value_cache, 16) ||
      !aligned(position, 8) || !aligned(slot, 4))
    return refuse("%s: pointers must be 16-byte aligned (position 8, slot 4)", op);
  const int64_t in_bytes = extent(tokens, qkv_stride, width, 2), out_bytes = extent(tokens, q_stride, q_width, 2);
  const int64_t cache_bytes = extent(num_blocks, block_stride, block_elems, 2);
  const int64_t rope_bytes = static_cast<int64_t>(rope_rows) * rotary * (rope_dtype == kFp32 ? 4 : 2);
  const Span written[] = {{q_out, out_bytes}, {key_cache, cache_bytes}, {value_cache, cache_bytes}};
  const Span read[] = {{qkv, in_bytes},         {position, 8ll * tokens},   {slot, 4ll * tokens},
                       {rope_cos, rope_bytes},  {rope_sin, rope_bytes},     {q_norm, q_norm != nullptr ? 2 * head_dim : 0},
                       {k_norm, k_norm != nullptr ? 2 * head_dim : 0}};
  if (meets(written, read) || meets(written[0], written[1]) || meets(written[0], written[2]))
    return refuse("%s: q_out and the caches must not overlap the inputs, nor q_out the caches", op);
  if (key_cache == value_cache) return refuse("%s: the two caches must not be one", op);
  if (blocks_overlap(key_cache, value_cache, num_blocks, 2 * block_stride, 2 * block_elems))
    return refuse("%s: the blocks of the two caches must not overlap", op);
  DeviceScope scope(device);
  if (scope.error != cudaSuccess) return report(scope.error, op);
  RotateArgs a{qkv, qkv_stride, tokens, num_heads, num_kv_heads, head_dim, dtype, position, slot, q_norm, k_norm, eps,
               rope_cos, rope_sin, rope_dtype, rope_rows, rotary, q_out, q_stride, key_cache, value_cache, num_blocks,
               block_stride, block_size};
  return report(launch_rotate_store(a, device, static_cast<cudaStream_t>(stream)), op);
}

static int32_t check_attention_sizes(const char *op, int32_t rows, int32_t num_heads, int32_t num_kv_heads,
                                     int32_t head_dim, int64_t capacity) {
  if (rows < 0 || num_kv_heads < 1 || num_heads < 1 || num_heads % num_kv_heads != 0 || num_heads > 1024)
    return refuse("%s: %d rows of %d query heads over %d KV heads (a multiple, at most 1024)", op, rows, num_heads, num_kv_heads);
  if (head_dim != 64 && head_dim != 128) return refuse("%s: head size %d (64 or 128)", op, head_dim);
  constexpr int kTile = kAttendWarps * kAttendKeys;
  // (the kernels count positions a few tiles past the end, and work up to a CTA's share past it, in 32 bits)
  if (capacity < 0 || capacity > kMaxIndex - 4 * kTile) return refuse("%s: a capacity of %lld positions (below 2^31 - 256)", op, static_cast<long long>(capacity));
  const int64_t units = static_cast<int64_t>(num_kv_heads) * ((num_heads / num_kv_heads + 15) / 16);
  if (rows * units * (std::max<int64_t>(1, (capacity + kTile - 1) / kTile) + attend_setup(head_dim)) > kMaxIndex - 1024)
    return refuse("%s: rows x KV heads x capacity / %d passes 2^31", op, kTile);
  return 0;
}

int64_t cruise_decoder_attention_workspace(int32_t rows, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                           int64_t capacity, int32_t device) {
  const char *const op = "cruise_decoder_attention_workspace";
  if (check_attention_sizes(op, rows, num_heads, num_kv_heads, head_dim, capacity) != 0) return -1;
  report(cudaSuccess, op);
  return attention_workspace(rows, num_heads, num_kv_heads, head_dim, capacity, device);
}

int32_t cruise_decoder_attention(const void *q, int64_t q_stride, int32_t rows, int32_t num_heads, int32_t num_kv_heads,
                                 int32_t head_dim, int32_t dtype, const void *key_cache, const void *value_cache,
                                 int64_t num_blocks, int32_t block_size, int64_t block_stride,
                                 const int32_t *block_table, int64_t table_stride, int32_t table_width,
                                 const int32_t *seq_len, float scale, void *out, int64_t out_stride, float *lse,
                                 void *workspace, int64_t workspace_bytes, int32_t device, void *stream) {
  const char *const op = "cruise_decoder_attention";
  if (dtype != kBf16 && dtype != kFp16) return refuse("%s: dtype %d (0 bf16 or 1 fp16)", op, dtype);
  if (num_blocks < 1 || block_size < 1 || table_width < 0 || num_blocks > kMaxIndex / block_size)
    return refuse("%s: a cache of %lld blocks of %d slots, tables of %d (at least one block, slots below 2^31)", op,
                  static_cast<long long>(num_blocks), block_size, table_width);
  const int64_t capacity = static_cast<int64_t>(table_width) * block_size;
  if (const int32_t bad = check_attention_sizes(op, rows, num_heads, num_kv_heads, head_dim, capacity)) return bad;
  const int64_t width = static_cast<int64_t>(num_heads) * head_dim;
  const int64_t block_elems = static_cast<int64_t>(block_size) * num_kv_heads * head_dim;
  if (q_stride < width || out_stride < width || block_stride < block_elems || table_stride < table_width)
    return refuse("%s: a stride is smaller than its row (q %lld, out %lld, block %lld, table %lld)", op,
                  static_cast<long long>(q_stride), static_cast<long long>(out_stride), static_cast<long long>(block_stride),
                  static_cast<long long>(table_stride));
  if (q_stride % 8 != 0 || out_stride % 8 != 0 || block_stride % 8 != 0)
    return refuse("%s: strides must be multiples of 8 elements", op);
  if (num_blocks > (int64_t(1) << 35) / block_stride)
    return refuse("%s: %lld blocks %lld elements apart pass 2^35 elements", op, static_cast<long long>(num_blocks),
                  static_cast<long long>(block_stride));
  if (!(scale - scale == 0.f)) return refuse("%s: the scale must be finite", op);
  if (rows == 0) return report(cudaSuccess, op);
  if (q == nullptr || key_cache == nullptr || value_cache == nullptr || seq_len == nullptr || out == nullptr ||
      (block_table == nullptr && table_width > 0))
    return refuse("%s: a required pointer is NULL", op);
  if (!aligned(q, 16) || !aligned(key_cache, 16) || !aligned(value_cache, 16) || !aligned(out, 16) ||
      !aligned(workspace, 16) || !aligned(block_table, 4) || !aligned(seq_len, 4) || !aligned(lse, 4))
    return refuse("%s: pointers must be 16-byte aligned (block_table, seq_len, lse 4)", op);
  const int64_t out_bytes = extent(rows, out_stride, width, 2), lse_bytes = lse != nullptr ? 4ll * rows * num_heads : 0;
  const int64_t cache_bytes = extent(num_blocks, block_stride, block_elems, 2), q_bytes = extent(rows, q_stride, width, 2);
  const int64_t table_bytes = extent(rows, table_stride, table_width, 4);
  if (overlap(out, out_bytes, q, q_bytes) || overlap(out, out_bytes, key_cache, cache_bytes) ||
      overlap(out, out_bytes, value_cache, cache_bytes) || overlap(out, out_bytes, block_table, table_bytes) ||
      overlap(out, out_bytes, seq_len, 4ll * rows) || overlap(lse, lse_bytes, out, out_bytes) ||
      overlap(lse, lse_bytes, q, q_bytes) || overlap(lse, lse_bytes, key_cache, cache_bytes) ||
      overlap(lse, lse_bytes, value_cache, cache_bytes) || overlap(lse, lse_bytes, block_table, table_bytes) ||
      overlap(lse, lse_bytes, seq_len, 4ll * rows))
    return refuse("%s: out and lse must not overlap the inputs or each other", op);
  DeviceScope scope(device);
  if (scope.error != cudaSuccess) return report(scope.error, op);
  const int64_t need = attention_workspace(rows, num_heads, num_kv_heads, head_dim, capacity, device);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return refuse("%s: a workspace of %lld bytes, %lld needed", op, static_cast<long long>(workspace != nullptr ? workspace_bytes : 0),
                  static_cast<long long>(need));
  if (need > 0 && (overlap(workspace, need, out, out_bytes) || overlap(workspace, need, lse, lse_bytes) ||
                   overlap(workspace, need, q, q_bytes) || overlap(workspace, need, key_cache, cache_bytes) ||
                   overlap(workspace, need, value_cache, cache_bytes) || overlap(workspace, need, block_table, table_bytes) ||
                   overlap(workspace, need, seq_len, 4ll * rows)))
    return refuse("%s: the workspace must not overlap the tensors", op);
  AttentionArgs a{q, q_stride, rows, num_heads, num_kv_heads, head_dim, dtype, key_cache, value_cache, num_blocks,
                  block_stride, block_size, block_table, table_stride, table_width, seq_len, scale, out, out_stride, lse,
                  workspace};
  return report(launch_paged_attention(a, device, static_cast<cudaStream_t>(stream)), op);
}

int32_t cruise_decoder_choose(const void *logits, int64_t logits_stride, int32_t rows, int32_t vocab, int32_t dtype,
                              const int32_t *active, int32_t *history, int64_t history_stride, int32_t history_width,
                              const int32_t *prompt_len, const int32_t *history_len, const float *repetition,
                              const float *frequency, const float *presence, const int32_t *bias_token,
                              const float *bias_value, int64_t bias_stride, int32_t bias_width, const int32_t *bias_len,
                              const uint32_t *allowed, int64_t allowed_stride, float *processed,
                              int64_t processed_stride, int64_t *token, int32_t append, int32_t device, void *stream) {
  const char *const op = "cruise_decoder_choose";
  if (rows < 0 || rows > 65535 || vocab < 1 || vocab > kChooseMaxVocab)
    return refuse("%s: %d rows of %d logits (at most 65535 rows of 1 to %d)", op, rows, vocab, kChooseMaxVocab);
  const int64_t entries = (history != nullptr ? history_width : 0) + static_cast<int64_t>(bias_token != nullptr ? bias_width : 0);
  if (entries >= (1 << 30)) return refuse("%s: a history and bias list of %lld entries (below 2^30)", op, static_cast<long long>(entries));
  if (choose_shared(choose_slice(vocab, kChooseMaxCluster), entries) > kChooseShared)
    return refuse("%s: a history and bias list of %lld entries with %d logits (at most 20000 beyond 390000 logits)", op,
                  static_cast<long long>(entries), vocab);
  if (dtype < kBf16 || dtype > kFp32) return refuse("%s: dtype %d (0 bf16, 1 fp16 or 2 fp32)", op, dtype);
  if (logits_stride < vocab || (processed != nullptr && processed_stride < vocab) ||
      (allowed != nullptr && allowed_stride < (vocab + 31) / 32))
    return refuse("%s: a stride is smaller than its row", op);
  if (history != nullptr && (history_width < 1 || history_stride < history_width || prompt_len == nullptr || history_len == nullptr))
    return refuse("%s: a history needs a width (at most its stride), prompt_len and history_len", op);
  if (history == nullptr && (append != 0 || repetition != nullptr || frequency != nullptr || presence != nullptr))
    return refuse("%s: penalties and append need a history", op);
  if (bias_token != nullptr && (bias_width < 1 || bias_stride < bias_width || bias_value == nullptr || bias_len == nullptr))
    return refuse("%s: a bias list needs a width (at most its stride), bias_value and bias_len", op);
  if (rows == 0) return report(cudaSuccess, op);
  if (logits == nullptr || token == nullptr) return refuse("%s: a required pointer is NULL", op);
  const int size = dtype == kFp32 ? 4 : 2;
  if (!aligned(logits, size) || !aligned(token, 8) || !aligned(active, 4) || !aligned(history, 4) ||
      !aligned(prompt_len, 4) || !aligned(history_len, 4) || !aligned(repetition, 4) || !aligned(frequency, 4) ||
      !aligned(presence, 4) || !aligned(bias_token, 4) || !aligned(bias_value, 4) || !aligned(bias_len, 4) ||
      !aligned(allowed, 4) || !aligned(processed, 4))
    return refuse("%s: a pointer is not aligned to its element", op);
  const int64_t per_row = 4ll * rows;   // bytes of a vector of 32-bit values
  auto span = [](const void *p, int64_t bytes) { return Span{p, p != nullptr ? bytes : 0}; };
  auto rows_of = [&](const void *p, int64_t stride, int64_t width, int64_t bytes) { return span(p, extent(rows, stride, width, bytes)); };
  const Span logits_span = rows_of(logits, logits_stride, vocab, size), history_span = rows_of(history, history_stride, history_width, 4);
  const Span processed_span = rows_of(processed, processed_stride, vocab, 4), token_span = span(token, 8ll * rows);
  const bool has_bias = bias_token != nullptr;
  const Span rules[] = {rows_of(allowed, allowed_stride, (vocab + 31) / 32, 4),
                        rows_of(bias_token, bias_stride, bias_width, 4),
                        has_bias ? rows_of(bias_value, bias_stride, bias_width, 4) : Span{},
                        has_bias ? span(bias_len, per_row) : Span{},
                        history != nullptr ? span(prompt_len, per_row) : Span{},
                        history != nullptr ? span(history_len, per_row) : Span{},
                        span(repetition, per_row),
                        span(frequency, per_row),
                        span(presence, per_row),
                        span(active, per_row)};
  const bool in_place = static_cast<const void *>(processed) == logits && dtype == kFp32 && processed_stride == logits_stride;
  if (!in_place && meets(processed_span, logits_span))
    return refuse("%s: processed must be the fp32 logits themselves or not overlap them", op);
  // rows write while others read: every output apart from every input
  const Span outputs[] = {token_span, processed_span}, appended[] = {append != 0 ? history_span : Span{}};
  if (meets(outputs, rules) || meets(appended, rules) || meets(appended[0], logits_span) || meets(token_span, logits_span) ||
      meets(token_span, history_span) || meets(processed_span, history_span) || meets(token_span, processed_span))
    return refuse("%s: token, processed and the history must not overlap the inputs", op);
  DeviceScope scope(device);
  if (scope.error != cudaSuccess) return report(scope.error, op);
  ChooseArgs a{logits, logits_stride, rows, vocab, dtype, active, history, history_stride, history_width, prompt_len,
               history_len, repetition, frequency, presence, bias_token, bias_value, bias_stride, bias_width, bias_len,
               allowed, allowed_stride, processed, processed_stride, token, append != 0 ? 1 : 0};
  return report(launch_choose(a, device, static_cast<cudaStream_t>(stream)), op);
}

}  // extern "C"
