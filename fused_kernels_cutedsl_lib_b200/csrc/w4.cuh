// What the two forms of the 4-bit linear layer share: the packed weight's constants and
// expansion, element conversions, bulk copies, and the hand-over of partial sums within a
// cluster.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace fk {
namespace w4 {

constexpr int kBlockK = 128;    // inputs per packed block
constexpr int kSlab = 2;        // blocks per slab

// A checked call of the layer.
struct Call {
  const void* x;
  long long ldx;
  const uint8_t* packed;
  const void* residual;
  void* y;
  int* err;
  bool bf16;
  int M, N, K, group;
  int withhold;  // test hook: the slab whose copy the first CTA leaves out (-1: none)
};
// The form of w4_tc.cu.
int linear_tc(const Call& c, cudaStream_t st);

// (a & MASK) | c in one logic instruction. It has room for one immediate only: with both constants known the
// compiler takes two, so c is kept in a register (`in_register`).
template <uint32_t MASK>
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "n"(MASK), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t in_register(uint32_t v) {
  uint32_t d;
  asm volatile("mov.b32 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
// A word's eight nibbles as fp16 pairs of inputs (0,1) (2,3) (4,5) (6,7), offset by 256, 16, 256, 16.
struct ExpandConsts {
  uint32_t c256 = in_register(0x5C005C00u), c16 = in_register(0x4C004C00u);
};
__device__ __forceinline__ void expand(uint32_t w, uint32_t (&p)[4], const ExpandConsts& k) {
  const uint32_t t = __funnelshift_r(w, w, 8);
  p[0] = and_or<0x003C003Cu>(w, k.c256);
  p[1] = and_or<0x03C003C0u>(w, k.c16);
  p[2] = and_or<0x003C003Cu>(t, k.c256);
  p[3] = and_or<0x03C003C0u>(t, k.c16);
}

template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
  static __device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
  static __device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
  static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Half<__half> {
  static __device__ __forceinline__ float lo(uint32_t v) {
    return __half2float(__ushort_as_half((unsigned short)(v & 0xFFFFu)));
  }
  static __device__ __forceinline__ float hi(uint32_t v) {
    return __half2float(__ushort_as_half((unsigned short)(v >> 16)));
  }
  static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t pol) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(pol)
      : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Shared-memory address of the same place in another CTA of the cluster.
__device__ __forceinline__ uint32_t map_to(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void ld_cluster(uint32_t addr, float& a, float& b) {
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(a), "=f"(b) : "r"(addr) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float a, float b) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}
__device__ __forceinline__ void st_cluster4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
// One arrival on another CTA's mbarrier, after everything this thread has seen (its CTA's stores
// into the cluster, ordered before it by a CTA barrier).
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Bounded wait for a phase. The bound itself lies in global memory and is looked at only when a
// wait has lasted some time: its latency would be paid after every wait that does not succeed at once.
constexpr uint64_t kPatienceNs = 50000;
__device__ __forceinline__ bool try_wait_at(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_at(uint32_t bar, uint32_t parity, int* err, int code) {
  if (try_wait_at(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (!try_wait_at(bar, parity)) {
    const uint64_t t = global_timer_ns() - t0;
    if (t > kPatienceNs && t > wait_limit_ns(err)) {
      record_device_error(err, code);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  return wait_at(smem_u32(bar), parity, err, code);
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The same for arrivals from the cluster, with acquire at its scope.
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, int* err) {
  const uint64_t t0 = global_timer_ns();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    const uint64_t t = global_timer_ns() - t0;
    if (t > kPatienceNs && t > wait_limit_ns(err)) break;
  }
  record_device_error(err, kDevErrFlagWait);
  return false;
}
// A thread whose wait for the cluster ran out keeps its CTA in place for another four bounds before it leaves:
// others of the cluster may still store into the CTA's shared memory. They stop at the latest when a wait
// of their own for this CTA has run out. (A second phase of the cluster's barrier would not do: it has
// no bound, and a CTA that has ended without arriving is waited for.)
__device__ __forceinline__ void linger(const int* err) {
  const uint64_t t0 = global_timer_ns(), lim = 4 * wait_limit_ns(err);
  while (global_timer_ns() - t0 < lim) __nanosleep(1000);
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

template <int GROUP>
__host__ __device__ constexpr int block_bytes() { return 1024 + (kBlockK / GROUP) * 64; }
}  // namespace w4
}  // namespace fk
