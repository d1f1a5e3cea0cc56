// decoder_common.cuh -- element types and small warp helpers of the decoder operators.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "ptx.cuh"

namespace cruise {
namespace ops {

// The first thing every kernel of the operators does.  They are launched as
// programmatic dependents: a kernel may come onto the SMs while its predecessor
// in the stream drains, lets its own successor do so, and waits for the
// predecessor's completion (and its memory) before it reads or writes anything.
// Calls one after the other then follow without a launch's latency between them.
__device__ __forceinline__ void follow_predecessor() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The CTAs of a cluster: a barrier in two halves, and their shared memory.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The address in CTA `rank`'s shared memory of what `local` is in this one's.
__device__ __forceinline__ uint32_t cluster_address(const void *local, uint32_t rank) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(local)), "r"(rank));
  return addr;
}
__device__ __forceinline__ void store_cluster(void *local, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_address(local, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void store_cluster(void *local, uint32_t rank, float2 v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(cluster_address(local, rank)), "f"(v.x), "f"(v.y) : "memory");
}
__device__ __forceinline__ void store_cluster(void *local, uint32_t rank, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_address(local, rank)), "f"(v.x), "f"(v.y),
               "f"(v.z), "f"(v.w)
               : "memory");
}

template <typename T>
struct Element;

template <>
struct Element<__nv_bfloat16> {
  static constexpr float kHalfStep = 0x1p-8f;   // half a step relative to the value: a rounding is off by at most this
  static constexpr float kLift = 1.f;           // brings values of at most 1 to the top of the range (fp32's here)
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <>
struct Element<__half> {
  static constexpr float kHalfStep = 0x1p-11f;
  static constexpr float kLift = 0x1p15f;
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ float load(const __half v) { return __half2float(v); }
  static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = Element<T>::unpack(w[k]);
    v[2 * k] = f.x;
    v[2 * k + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(Element<T>::pack(v[0], v[1]), Element<T>::pack(v[2], v[3]), Element<T>::pack(v[4], v[5]),
                    Element<T>::pack(v[6], v[7]));
}

}  // namespace ops
}  // namespace cruise
