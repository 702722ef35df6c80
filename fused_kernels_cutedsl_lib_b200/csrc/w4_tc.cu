// Linear layer with 4-bit weights and group scales for more than 8 or 16 tokens, on tcgen05:
//   y[m, n] = sum_k x[m, k] * (q[n, k] - z[n, k / g]) * s[n, k / g]  (+ residual[m, n])
// (the layout of the weight, the form for fewer tokens and the choice are in w4_linear.cu).
//
// Up to 64 tokens share one pass over the weight, 32 with groups of 32 (the accumulators of a block's four
// groups fill the columns). What bounds it is the latency of its stages: 0.45 instructions per cycle and
// scheduler, tcgen05 16 % busy, DRAM 16 % (64 tokens, groups of 64, 4096 x 14336); past one wave of tiles also
// the part-filled last one. Measured on weights that do not lie in L2, groups of 128: 4096 outputs of 14336
// inputs 14.1 us for 16 tokens, 14.4 for 32, 17.5 for 64 (mma.sync, with 32 products and 16 shared-memory reads
// per KB of weight at 32 tokens: 61 us for 64); 28672 of 4096: 30.6 and 38.4 us for 32 and 64. This
// package's 16-bit linear (skinny_gemm) takes 24.0, 25.2 and 26.8 us for 32, 64 and 128 tokens on 4096 x 14336:
// from 65 tokens on, two passes, this form saves memory, not time.
//
// One CTA: 128 output rows, a slice of the inputs, N tokens (32 or 64). Per slab of 256
// inputs
//   * warp 24 copies the rows' packed blocks (one bulk copy, contiguous) and x (TMA,
//     128B-swizzled boxes of 64 inputs x N tokens) into two rings: x comes from L2 and is
//     released by the products, the weight comes from memory and is held longer (one ring
//     of three stages for both: 18.5 us at 64 tokens);
//   * of warps 0-15, four take each block of 128 inputs of every second slab. Thread = row =
//     TMEM lane: it expands its row's 16 words to the exact integers q - z (bf16: 32 + q
//     from a rotation and a logic instruction per pair, minus 32 + z; fp16: 256 + q and
//     16 + q) and stores them to TMEM as the A operand (two buffers). With eight warps, one
//     slab at a time: 15.7 instead of 13.6 us at 32 tokens;
//   * warp 25 issues D = A x^T, one accumulator per group of g inputs, and commits;
//   * warps 16-23 (thread = row and half of the tokens) read D and add s * D to their fp32
//     sums. Integers and x are exact, so the only roundings are those of fp32 sums and
//     the output.
// Earlier steps, 64 tokens on 4096 x 14336, part of the weight from L2: 27.5 us with the expanding warps adding up too,
// 20.4 with warps of their own for it, 19.0 with addresses carried along, 17.9 with one
// logic instruction per pair. CTAs that go on to the next tile of rows instead of leaving:
// 15.6 for 32 tokens instead of 13.3, no gain elsewhere.
// The inputs are split over the CS CTAs of a cluster; their sums go to the shared memory
// of the CTA that owns the rows (mbarrier with one arrival per CTA), which adds them in a
// fixed order: no workspace, no atomic.
//
// Waits for copies, products and other CTAs are bounded, that for the preceding kernel of the stream
// (programmatic dependent launch) is not: each warp waits for it before its first bounded wait for
// anything that follows from x, so that a long predecessor is not taken for a fault.
#include <cuda_fp16.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "fk_b200.h"
#include "w4.cuh"

namespace fk {
namespace w4tc {

using w4::kBlockK;
using w4::kSlab;

constexpr int kRows = 128;     // output rows per CTA (UMMA M, TMEM lanes)
constexpr int kRowBlocks = 8;  // of 16 rows
// Warps: 0-15 expand, 16-23 add up, 24 loads, 25 issues the products.
constexpr int kAddWarp = 16, kLoadWarp = 24, kMmaWarp = 25, kThreads = 26 * 32;
constexpr int kSmem = 227 * 1024;
constexpr int kTmemBar = 2, kTmemThreads = 25 * 32;  // named barrier: all but the loading warp are done with TMEM
constexpr uint32_t kACol = 256;  // TMEM: D of warp group w at 128 w, its A buffers at 256 + 128 w + 64 buf

struct Params {
  const uint8_t* packed;
  const void* residual;
  void* y;
  int* err;
  int M, N;
  int nrb, nkb, nslab;
  int cs_log;
  int withhold;  // test hook: the slab of x that the first CTA does not load (-1: none)
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// K-major operand, 128B swizzle, 8-row groups 1024 B apart.
__device__ __forceinline__ uint64_t desc_k_sw128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16, A and B both bf16 or both fp16, D fp32, M = 128, N = n.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int n) {
  constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
// D (+)= A . B with A (M = 128 x K = 16, 16-bit pairs packed per 32-bit column) in TMEM.
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(db), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// One lane of the warp, in a form that the compiler knows to be a single one: the operands of the
// products stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
// 32 consecutive TMEM columns of this thread's lane (no wait).
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
      "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
      "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One row's word as the exact 16-bit integers q - z, four pairs of neighbouring inputs.
template <typename T>
struct Expand;
template <>
struct Expand<__nv_bfloat16> {
  __nv_bfloat162 c;  // 32 + z, twice
  __device__ __forceinline__ void zero(uint32_t sz) {
    const float z = __uint_as_float(sz & 0xFFFF0000u);
    c = __float2bfloat162_rn(32.f + z);
  }
  struct Consts {
    uint32_t one = w4::in_register(0x42004200u);
  };
  __device__ __forceinline__ void word(uint32_t w, uint32_t* p, const Consts& k) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = w4::and_or<0x003C003Cu>(__funnelshift_r(w, w, 4 * i), k.one);
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), c);
      p[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
};
template <>
struct Expand<__half> {
  __half2 c256, c16;
  __device__ __forceinline__ void zero(uint32_t sz) {
    const float z = __half2float(__ushort_as_half((unsigned short)(sz >> 16)));
    c256 = __float2half2_rn(256.f + z);
    c16 = __float2half2_rn(16.f + z);
  }
  using Consts = w4::ExpandConsts;
  __device__ __forceinline__ void word(uint32_t w, uint32_t* p, const Consts& k) const {
    uint32_t v[4];
    w4::expand(w, v, k);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v[i]), i & 1 ? c16 : c256);
      p[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
};

template <int GROUP>
__host__ __device__ constexpr int weight_bytes() { return kRowBlocks * kSlab * w4::block_bytes<GROUP>(); }
template <int NTOK>
__host__ __device__ constexpr int x_bytes() { return kSlab * 2 * NTOK * 128; }
// Partial sums of the rows a CTA owns, from every CTA of the cluster; 4 floats of padding per row keep a warp's
// 16-byte stores on distinct banks.
template <int NTOK>
__host__ __device__ constexpr int part_bytes() { return kRows * (NTOK + 4) * 4; }
// Slabs of x (from L2) and of the weight (from memory, released later) in shared memory.
template <int NTOK>
__host__ __device__ constexpr int x_stages() { return NTOK > 32 ? 3 : 4; }
template <int NTOK, int GROUP>
__host__ __device__ constexpr int w_stages() {
  constexpr int s = (kSmem - 2048 - part_bytes<NTOK>() - x_stages<NTOK>() * x_bytes<NTOK>()) / weight_bytes<GROUP>();
  return s > 8 ? 8 : s;
}
template <int NTOK, int GROUP>
__host__ __device__ constexpr int ring_bytes() {
  return x_stages<NTOK>() * x_bytes<NTOK>() + w_stages<NTOK, GROUP>() * weight_bytes<GROUP>();
}

template <typename T, int NTOK, int GROUP>
__global__ void __launch_bounds__(kThreads, 1)
    w4_tc_kernel(const __grid_constant__ CUtensorMap tmX, const Params p) {
  constexpr int S = w_stages<NTOK, GROUP>(), SX = x_stages<NTOK>();
  static_assert(S >= 3, "a slab each for the two halves of the expanding warps, and one on its way");
  constexpr int GPB = kBlockK / GROUP;
  static_assert(GPB * NTOK <= 128, "the accumulators of a slab's first and second blocks have 128 columns each");
  constexpr int DB = GPB * NTOK <= 64 ? 2 : 1;  // accumulator buffers
  constexpr int BB = w4::block_bytes<GROUP>();
  constexpr int STAGE = weight_bytes<GROUP>(), XSTAGE = x_bytes<NTOK>();
  constexpr int PR = NTOK + 4;  // floats per row of partial sums
  extern __shared__ uint8_t smem_raw[];
  // Aligned by the shared-window address: the same in every CTA of the cluster.
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* wring = smem + SX * XSTAGE;
  float* part_buf = reinterpret_cast<float*>(smem + ring_bytes<NTOK, GROUP>());  // [cs][128 / cs][PR]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ring_bytes<NTOK, GROUP>() + part_bytes<NTOK>());  // of the weight
  uint64_t* empty = full + S;      // 8 warps have read its codes, 8 its scales
  uint64_t* x_full = empty + S;
  uint64_t* x_empty = x_full + SX;  // the slab's products are done: x and A's buffer are free
  uint64_t* a_full = x_empty + SX;  // [slab & 1]
  uint64_t* d_full = a_full + 2;    // [slab & 1], with one accumulator buffer: [block of the slab]
  uint64_t* d_empty = d_full + 2;   // same
  uint64_t* done = d_empty + 2;  // one arrival per CTA: its partial sums are stored
  uint64_t* idle = done + 1;     // every product that was issued is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(idle + 1);

  using Half = w4::Half<T>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cs = 1 << p.cs_log, rank = blockIdx.x & (cs - 1), tile = blockIdx.x >> p.cs_log;
  const int tok0 = blockIdx.y * NTOK;
  const int nsl = (p.nslab - rank + cs - 1) >> p.cs_log;  // slabs rank, rank + cs, ..
  auto slab_blocks = [&](int s) { return min(kSlab, p.nkb - s * kSlab); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 16);
    }
    for (int i = 0; i < SX; ++i) {
      mbar_init(&x_full[i], 1);
      mbar_init(&x_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&a_full[i], 8);
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 8);
    }
    mbar_init(done, cs);
    mbar_init(idle, 1);
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The other CTAs must have started, their barriers included, before anything is stored into their
  // shared memory. The only phase of the cluster's own barrier.
  w4::cluster_arrive();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == kLoadWarp) {
    // ------------------------------ loads ------------------------------
    const uint64_t pol_w = l2_policy_evict_first(), pol_x = l2_policy_evict_last();
    const int rows = min(kRowBlocks, p.nrb - tile * kRowBlocks);
    int nw = 0, nx = 0;  // slabs of the weight and of x whose copies have been issued
    auto load_w = [&](int i) {
      const int st = i % S, s = rank + i * cs, nb = slab_blocks(s);
      nw = i + 1;
      const uint32_t bytes = (uint32_t)(rows * nb) * BB;
      mbar_arrive_expect_tx(&full[st], bytes);
      w4::bulk_load(smem_u32(wring + st * STAGE),
                    p.packed + ((size_t)s * kSlab * p.nrb + (size_t)tile * kRowBlocks * nb) * BB, bytes, &full[st], pol_w);
    };
    auto load_x = [&](int i) {
      const int st = i % SX, s = rank + i * cs, nb = slab_blocks(s);
      nx = i + 1;
      if (i == p.withhold && blockIdx.x == 0 && blockIdx.y == 0) return;
      mbar_arrive_expect_tx(&x_full[st], nb * 2 * NTOK * 128);
      for (int q = 0; q < nb * 2; ++q)
        tma_load_2d(smem + st * XSTAGE + q * (NTOK * 128), &tmX, &x_full[st], s * kSlab * kBlockK + q * 64, tok0, pol_x);
    };
    // The weights' first copies do not wait for the preceding kernel, x does.
    if (lane == 0) {
      tma_prefetch_desc(&tmX);
      for (int i = 0; i < min(S, nsl); ++i) load_w(i);
      asm volatile("griddepcontrol.wait;" ::: "memory");
      for (int i = 0; i < min(SX, nsl); ++i) load_x(i);
      for (int i = 0; i + min(S, SX) < nsl; ++i) {
        if (i + SX < nsl) {
          if (!w4::wait(&x_empty[i % SX], (i / SX) & 1, p.err, kDevErrEmptyWait)) break;
          load_x(i + SX);
        }
        if (i + S < nsl) {
          if (!w4::wait(&empty[i % S], (i / S) & 1, p.err, kDevErrEmptyWait)) break;
          load_w(i + S);
        }
      }
      // No copy may be in flight when the CTA ends, also when the warps that wait for them gave up.
      for (int i = max(0, nw - S); i < nw; ++i) w4::wait(&full[i % S], (i / S) & 1, p.err, kDevErrFullWait);
      for (int i = max(0, nx - SX); i < nx; ++i) w4::wait(&x_full[i % SX], (i / SX) & 1, p.err, kDevErrFullWait);
    }
    __syncwarp();
    w4::cluster_wait();
    return;
  }
  w4::cluster_wait();  // the other warps have something to wait for in any case

  if (warp == kMmaWarp) {
    // ------------------------------ products ------------------------------
    constexpr uint32_t ID = idesc<T>(NTOK);
    const bool leader = elect_one();
    const uint64_t x0 = desc_k_sw128(smem_u32(smem));
    const uint32_t x_full0 = smem_u32(x_full), a_full0 = smem_u32(a_full), d_empty0 = smem_u32(d_empty);
    uint32_t st = 0, ph = 0;
    bool ok = true;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = 0; i < nsl && ok; ++i) {
      const int b = i & 1, nb = slab_blocks(rank + i * cs);
      ok = w4::wait_at(x_full0 + st * 8, ph, p.err, kDevErrFullWait) &&
           (DB == 1 || i < 2 || w4::wait_at(d_empty0 + b * 8, ((i >> 1) & 1) ^ 1, p.err, kDevErrMmaWait)) &&
           w4::wait_at(a_full0 + b * 8, (i >> 1) & 1, p.err, kDevErrMmaWait);
      const uint64_t xd = x0 + (st * XSTAGE >> 4);
      const uint32_t a = tmem + kACol + b * 64, d = tmem + (DB == 2 ? b * 64 : 0);
#pragma unroll
      for (int w = 0; w < kSlab; ++w) {
        if (w >= nb) break;
        if (DB == 1 && i > 0) ok = ok && w4::wait_at(d_empty0 + w * 8, (i - 1) & 1, p.err, kDevErrMmaWait);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ts(d + w * 128 + kk * 16 / GROUP * NTOK, a + w * 128 + kk * 8,
                    xd + (((w * 2 + (kk >> 2)) * (NTOK * 128) + (kk & 3) * 32) >> 4), ID, kk * 16 % GROUP ? 1u : 0u);
          if (DB == 1) umma_commit(&d_full[w]);
          if (w == nb - 1) {
            if (DB == 2) umma_commit(&d_full[b]);
            umma_commit(&x_empty[st]);
          }
        }
        __syncwarp();
      }
      if (++st == SX) st = 0, ph ^= 1;
    }
    __syncwarp();
    // TMEM is given back when all products are done and all warps are through with it, those that gave up
    // among them: their waits are bounded, so the barrier fills.
    if (leader) umma_commit(idle);
    __syncwarp();
    w4::wait(idle, 0, p.err, kDevErrMmaWait);
    named_bar_sync(kTmemBar, kTmemThreads);
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    return;
  }

  // In the loops below every instruction counts (a block's expansion is some 180): stage, parities and
  // addresses are carried along, not derived from the slab's index.
  const int quarter = warp & 3, r = 32 * quarter + lane;  // this thread's row of the tile, its TMEM lane
  const uint32_t tlane = tmem + ((uint32_t)(32 * quarter) << 16);
  const uint32_t smem0 = smem_u32(wring), full0 = smem_u32(full), empty0 = smem_u32(empty);
  const bool short_tail = nsl > 0 && slab_blocks(rank + (nsl - 1) * cs) < kSlab;  // the last slab has one block
  uint32_t st = 0;  // stage
  if (warp < kAddWarp) {
    // ------------------------------ expand ------------------------------
    const int w = (warp >> 2) & 1;    // block of the slab
    const int parity = warp >> 3;     // of this warp's slabs, and A's buffer
    const uint32_t a_full0 = smem_u32(a_full), x_empty0 = smem_u32(x_empty);
    const uint32_t a0 = tlane + kACol + w * 128;
    const uint32_t b8 = parity * 8;
    uint32_t ph = 0;  // parity of the stage's phase
    st = parity;
    uint32_t xst = parity, xph = 0;  // x's stage of the slab two before, its phase
    const typename Expand<T>::Consts consts;
    for (int i = parity; i < nsl; i += 2) {
      const bool tail = short_tail && i == nsl - 1;
      // The products of the buffer's last slab are done, and with them the phase of a_full that this warp's
      // next arrival must not count for.
      auto buffer_free = [&] {
        if (i < 2) return true;
        if (i < 4) asm volatile("griddepcontrol.wait;" ::: "memory");  // this warp's first wait for products
        const bool done = __all_sync(~0u, w4::wait_at(x_empty0 + xst * 8, xph, p.err, kDevErrMmaWait));
        xst += 2;
        if (xst >= SX) xst -= SX, xph ^= 1;
        return done;
      };
      if (w == 1 && tail) {
        if (buffer_free() && lane == 0) w4::arrive_at(a_full0 + b8);
        break;
      }
      if (!__all_sync(~0u, w4::wait_at(full0 + st * 8, ph, p.err, kDevErrFullWait))) break;
      const uint32_t ba = smem0 + st * STAGE + (tail ? (r >> 4) * BB : ((r >> 4) * kSlab + w) * BB) + (r & 15) * 64;
      const uint32_t sa = ba - (r & 15) * 60 + 1024;
      uint32_t words[4][4];  // [c][j]: inputs 32 j + 8 c
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint4 v = w4::lds128(ba + c * 16);
        words[c][0] = v.x, words[c][1] = v.y, words[c][2] = v.z, words[c][3] = v.w;
      }
      Expand<T> ex[GPB];
#pragma unroll
      for (int gi = 0; gi < GPB; ++gi) ex[gi].zero(w4::lds32(sa + gi * 64));
      if (!buffer_free()) break;
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // 64 inputs: 32 columns
        uint32_t a[32];
#pragma unroll
        for (int jj = 0; jj < 2; ++jj)
#pragma unroll
          for (int c = 0; c < 4; ++c) ex[(2 * h + jj) * 32 / GROUP].word(words[c][2 * h + jj], a + jj * 16 + c * 4, consts);
        tmem_st32(a0 + b8 * 8 + h * 32, a);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        w4::arrive_at(a_full0 + b8);
        w4::arrive_at(empty0 + st * 8);
      }
      st += 2;
      if (st >= S) st -= S, ph ^= 1;
    }
    tc_fence_before();
    __syncwarp();
    named_bar_arrive(kTmemBar, kTmemThreads);
    return;
  }

  // ------------------------------ add up ------------------------------
  constexpr int HT = NTOK / 2;  // tokens of this warp: the first four warps take the first half
  const int half = (warp >> 2) & 1;
  const uint32_t d_full0 = smem_u32(d_full), d_empty0 = smem_u32(d_empty);
  float acc[HT];
#pragma unroll
  for (int n = 0; n < HT; ++n) acc[n] = 0.f;
  bool ok = true;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int i = 0; i < nsl && ok; ++i) {
    const bool tail = short_tail && i == nsl - 1;
    const uint32_t b8 = (i & 1) * 8, db8 = DB == 2 ? b8 : 0;
    if (DB == 2) {
      ok = __all_sync(~0u, w4::wait_at(d_full0 + b8, (i >> 1) & 1, p.err, kDevErrMmaWait));
      if (!ok) break;
      tc_fence_after();
    }
    const uint32_t sa = smem0 + st * STAGE + (r >> 4) * (tail ? BB : kSlab * BB) + (r & 15) * 4 + 1024;
#pragma unroll
    for (int w = 0; w < kSlab; ++w) {
      if (w == 1 && tail) break;
      if (DB == 1) {
        ok = __all_sync(~0u, w4::wait_at(d_full0 + w * 8, i & 1, p.err, kDevErrMmaWait));
        if (!ok) break;
        tc_fence_after();
      }
#pragma unroll
      for (int gi = 0; gi < GPB; ++gi) {
        const float scale = w4::Half<T>::lo(w4::lds32(sa + w * BB + gi * 64));
#pragma unroll
        for (int c = 0; c < HT; c += 16) {
          uint32_t d[16];
          tmem_ld16(tlane + w * 128 + db8 * 8 + gi * NTOK + half * HT + c, d);
          tmem_ld_wait();
#pragma unroll
          for (int n = 0; n < 16; ++n) acc[c + n] = fmaf(scale, __uint_as_float(d[n]), acc[c + n]);
        }
      }
      if (DB == 1) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) w4::arrive_at(d_empty0 + w * 8);
      }
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) {
      if (DB == 2) w4::arrive_at(d_empty0 + db8);
      w4::arrive_at(empty0 + st * 8);  // the scales have been read
    }
    if (++st == S) st = 0;
  }
  tc_fence_before();
  __syncwarp();
  named_bar_arrive(kTmemBar, kTmemThreads);

  // ---- the sums go to the CTAs that own the rows, 128 / cs each ----
  {
    const int tid = threadIdx.x - kAddWarp * 32;
    const int rows_log = 7 - p.cs_log, owner = r >> rows_log, slot = r & ((1 << rows_log) - 1);
    const uint32_t to =
        w4::map_to(smem_u32(part_buf + ((size_t)(rank << rows_log) + slot) * PR + half * HT), owner);
#pragma unroll
    for (int n = 0; n < HT; n += 4) w4::st_cluster4(to + n * 4, acc[n], acc[n + 1], acc[n + 2], acc[n + 3]);
    // Element e of this CTA's part of the output: four tokens of a row, lanes along the rows, so that a
    // token's outputs are contiguous.
    const int rows = 1 << rows_log, plane = rows * PR, elems = rows * (NTOK / 4);
    auto locate = [&](int e, int& row, int& n) {
      row = tile * kRows + rank * rows + (e & (rows - 1));
      n = (e >> rows_log) * 4;
      return e < elems && row < p.N && tok0 + n < p.M;
    };
    auto load_residual = [&](int e, T (&res)[4]) {
      int row, n;
      const bool in = locate(e, row, n) && p.residual;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (in && tok0 + n + i < p.M) res[i] = static_cast<const T*>(p.residual)[(size_t)(tok0 + n + i) * p.N + row];
    };
    // The first two elements' residuals arrive during the exchange.
    T res[2][4] = {};
    load_residual(tid, res[0]);
    load_residual(tid + 256, res[1]);
    named_bar_sync(1, 256);
    if (warp == kAddWarp && lane < cs) w4::arrive_cluster(w4::map_to(smem_u32(done), lane));
    if (!__all_sync(~0u, w4::wait_cluster(done, 0, p.err))) {
      w4::linger(p.err);
      return;
    }
    for (int e0 = tid; e0 < elems; e0 += 512) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        int row, n;
        if (!locate(e0 + u * 256, row, n)) continue;
        const float* from = part_buf + (row & (rows - 1)) * PR + n;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int q = 0; q < cs; ++q) {
          const float4 f = *reinterpret_cast<const float4*>(from + q * plane);
          v.x += f.x, v.y += f.y, v.z += f.z, v.w += f.w;
        }
        const float out[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (tok0 + n + i < p.M)
            static_cast<T*>(p.y)[(size_t)(tok0 + n + i) * p.N + row] =
                Half::round(p.residual ? out[i] + Half::to_float(res[u][i]) : out[i]);
      }
      load_residual(e0 + 512, res[0]);
      load_residual(e0 + 768, res[1]);
    }
  }
}

// Clusters of 1, 2, 4 and 8 CTAs that can be resident at once, asked once per kernel and device.
template <typename T, int NTOK, int GROUP>
static int resident_clusters(int smem, int (&out)[4]) {
  constexpr int kDevices = 64;
  static std::mutex mu;
  static int known[kDevices][4] = {};
  auto kern = w4_tc_kernel<T, NTOK, GROUP>;
  int dev = 0;
  FK_CHECK_CUDA(cudaGetDevice(&dev));
  FK_CHECK_ARG(dev >= 0 && dev < kDevices, "device index too large");
  std::lock_guard<std::mutex> lock(mu);
  int* k = known[dev];
  if (k[3] == 0) {
    FK_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    for (int i = 0; i < 4; ++i) {
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1 << i;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1u << i, 1, 1);
      cfg.blockDim = dim3(kThreads, 1, 1);
      cfg.dynamicSmemBytes = smem;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      FK_CHECK_CUDA(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
      k[i] = n < 1 ? 1 : n;
    }
  }
  for (int i = 0; i < 4; ++i) out[i] = k[i];
  return kOk;
}

template <typename T, int NTOK, int GROUP>
static int launch(const w4::Call& c, cudaStream_t st) {
  constexpr int smem = 1024 + ring_bytes<NTOK, GROUP>() + part_bytes<NTOK>() + 512;
  static_assert(smem <= kSmem, "shared memory budget");
  int resident[4];
  int rc = resident_clusters<T, NTOK, GROUP>(smem, resident);
  if (rc) return rc;
  Params p;
  p.packed = c.packed;
  p.residual = c.residual;
  p.y = c.y;
  p.err = c.err;
  p.M = c.M;
  p.N = c.N;
  p.withhold = c.withhold;
  p.nrb = (c.N + 15) / 16;
  p.nkb = (c.K + kBlockK - 1) / kBlockK;
  p.nslab = (p.nkb + kSlab - 1) / kSlab;
  const long long row_tiles = (c.N + kRows - 1) / kRows, tok_tiles = (c.M + NTOK - 1) / NTOK;
  // CTAs per cluster: the least waves x (slabs of the busiest CTA + what a CTA costs besides, as much as
  // six slabs).
  long long best = -1;
  for (int l = 0; l < 4 && (1 << l) <= p.nslab; ++l) {
    const long long waves = (row_tiles * tok_tiles + resident[l] - 1) / resident[l];
    const long long cost = waves * ((p.nslab + (1 << l) - 1) / (1 << l) + 6);
    if (best < 0 || cost < best) {
      best = cost;
      p.cs_log = l;
    }
  }
  FK_CHECK_ARG(row_tiles << p.cs_log < (1LL << 31), "N too large");
  CUtensorMap tmX;
  const uint64_t dims[2] = {(uint64_t)c.K, (uint64_t)c.M};
  const uint64_t strides[1] = {(uint64_t)c.ldx * 2};
  const uint32_t box[2] = {64, NTOK};
  rc = encode_tma(&tmX,
                  std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  2, const_cast<void*>(c.x), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1 << p.cs_log;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(row_tiles << p.cs_log), (unsigned)tok_tiles, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, w4_tc_kernel<T, NTOK, GROUP>, tmX, p));
  return kOk;
}

template <typename T>
static int by_group(const w4::Call& c, cudaStream_t st) {
  // Tokens per pass: 64, or 32 where that is enough or the groups' accumulators need the columns.
  if (c.group == 32) return launch<T, 32, 32>(c, st);
  if (c.M <= 32) return c.group == 64 ? launch<T, 32, 64>(c, st) : launch<T, 32, 128>(c, st);
  return c.group == 64 ? launch<T, 64, 64>(c, st) : launch<T, 64, 128>(c, st);
}

}  // namespace w4tc

int w4::linear_tc(const Call& c, cudaStream_t st) {
  return c.bf16 ? w4tc::by_group<__nv_bfloat16>(c, st) : w4tc::by_group<__half>(c, st);
}

}  // namespace fk
