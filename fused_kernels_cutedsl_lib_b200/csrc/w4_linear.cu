// Linear layer with 4-bit weights and group scales for a few tokens:
//   y[m, n] = sum_k x[m, k] * (q[n, k] - z[n, k / g]) * s[n, k / g]  (+ residual[m, n])
// with q, z in [0, 15], g in {32, 64, 128} and x, s, y bf16 or fp16.
//
// Bound: the 4-bit weights are read once (N*K/2 bytes); everything else is small.
//
// Arithmetic. The weights never become rounded 16-bit products q*s. A nibble q
// is or-ed into the mantissa of 16.0 (bf16: bit 3, fp16: bit 6), which is the
// exact 16-bit number 16 + q: one shift and one logic instruction per pair.
// Those integers go to the tensor cores as they are; per group of g inputs
//   sum_k x (q - z) = sum_k x (16 + q) - (16 + z) * sum_k x,
// so the zero point costs one fused multiply-add per output and group, with
// sum_k x computed once per CTA, and the scale another, both in fp32. The
// offset 16 (rather than the 128 or 1024 of a nibble in the lowest mantissa
// bits) keeps the cancelled part within about 4x of the result, a relative
// error of a few 2^-22, far below the output's rounding.
//
// Layout (made once by the caller, `pack_w4`): rows in blocks of 16, inputs in
// blocks of 128 and slabs of 4 blocks (the last slab may have fewer). A block is
// its codes, [2][32][4] words: half h, lane l = 4*g + c, word j holds the eight
// nibbles of row 8*h + g, inputs 32*j + 8*c + 0..7; nibble i < 4 is input 2i, nibble
// i >= 4 input 2(i - 4) + 1, so that the pair (i, i + 4) a shift exposes is a pair
// of neighbouring inputs; then its scales and zero points, [groups][16] words. Lane
// l of a warp therefore reads its mma.sync A operands of both row halves as two
// 16-byte words, the B operands are 16 bytes of x as they lie in memory, and a group
// of 32 inputs is one word j across the four lanes of a row, so every group size is
// a whole number of mma steps. Memory order is slab, row block, block: the rows of a
// slab are one contiguous stream.
//
// Work split. Slabs go to the CS CTAs of a cluster, row blocks to the clusters, one
// persistent grid. A CTA stages its slabs of x in shared memory once, in operand
// order, with the group sums. A producer thread streams W / KW row blocks of a slab
// at a time (up to 70 KB in one bulk copy; a copy per KB block reached 1.5 TB/s only)
// into a ring of two stages; each of the W warps multiplies one row block (or one
// of KW parts of it). A finished row block's partial sums are stored into the shared
// memory of the CTA of the cluster that owns the rows; after one cluster barrier
// every owner adds what it got in a fixed order: no workspace, no atomic, and
// results do not depend on timing. The first weight copies are issued before the
// wait for the preceding kernel (programmatic dependent launch).
#include <cuda_fp16.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "fk_b200.h"

namespace fk {
namespace w4 {

constexpr int kBlockK = 128;    // inputs per packed block
constexpr int kSlab = 4;        // blocks per slab
constexpr int kStages = 2;
constexpr int kSmem = 227 * 1024;

struct Params {
  const void* x;
  long long ldx;
  const uint8_t* packed;
  const void* residual;      // [M, N] or null
  void* y;                   // [M, N]
  int* err;
  int M, N, K;
  int nrb, nkb, nslab;       // row blocks of 16, input blocks of 128, slabs
  int cs_log;                // log2 of the CTAs per cluster
  int rb_each, rb_more;      // row blocks per cluster; the first rb_more clusters have one more
  int kw_log;                // log2 of the warps that share a row block
  int chunk;                 // slabs of a CTA whose x is staged at a time
  int tile;                  // row blocks per cluster whose partial sums are held at a time
};

template <typename T>
struct Half;

template <>
struct Half<__nv_bfloat16> {
  static __device__ __forceinline__ void expand(uint32_t w, uint32_t (&p)[4]) {
    constexpr uint32_t kMask = 0x00780078u, kSixteen = 0x41804180u;
    p[0] = ((w << 3) & kMask) | kSixteen;
    p[1] = ((w >> 1) & kMask) | kSixteen;
    p[2] = ((w >> 5) & kMask) | kSixteen;
    p[3] = ((w >> 9) & kMask) | kSixteen;
  }
  static __device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
  static __device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
  static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16_16816(d, a, b0, b1);
  }
};

template <>
struct Half<__half> {
  static __device__ __forceinline__ void expand(uint32_t w, uint32_t (&p)[4]) {
    constexpr uint32_t kMask = 0x03C003C0u, kSixteen = 0x4C004C00u;
    p[0] = ((w << 6) & kMask) | kSixteen;
    p[1] = ((w << 2) & kMask) | kSixteen;
    p[2] = ((w >> 2) & kMask) | kSixteen;
    p[3] = ((w >> 6) & kMask) | kSixteen;
  }
  static __device__ __forceinline__ float lo(uint32_t v) {
    return __half2float(__ushort_as_half((unsigned short)(v & 0xFFFFu)));
  }
  static __device__ __forceinline__ float hi(uint32_t v) {
    return __half2float(__ushort_as_half((unsigned short)(v >> 16)));
  }
  static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_f16_16816(d, a, b0, b1);
  }
};

// D = A * B: the first step of a group starts from nothing.
template <typename T>
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

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

template <int GROUP>
__host__ __device__ constexpr int block_bytes() { return 1024 + (kBlockK / GROUP) * 64; }
// Warps that multiply: 16 where the registers of one CTA per SM allow it.
template <int NT>
__host__ __device__ constexpr int warps() { return NT <= 2 ? 16 : 8; }
// Bytes of shared memory: the ring with its barriers, one slab of x with its group sums, one row
// block's partial sums from one warp.
template <int NT, int GROUP>
__host__ __device__ constexpr int stage_bytes() { return warps<NT>() * kSlab * block_bytes<GROUP>(); }
template <int NT, int GROUP>
__host__ __device__ constexpr int ring_bytes() { return kStages * stage_bytes<NT, GROUP>() + 128; }
template <int NT, int GROUP>
__host__ __device__ constexpr int x_bytes() { return kSlab * (4 * NT * 32 * 16 + (kBlockK / GROUP) * NT * 8 * 4); }
template <int NT>
__host__ __device__ constexpr int part_bytes() { return 16 * NT * 8 * 4; }

// NT: tiles of 8 tokens; GROUP: inputs per scale.
template <typename T, int NT, int GROUP>
__global__ void __launch_bounds__(warps<NT>() * 32 + 32, 1) w4_linear_kernel(const Params p) {
  using H = Half<T>;
  constexpr int W = warps<NT>();
  constexpr int GPB = kBlockK / GROUP;  // groups per input block
  constexpr int WPG = 4 / GPB;          // words of a lane per group
  constexpr int TOK = NT * 8;
  constexpr int BB = block_bytes<GROUP>();
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // The host did the divisions: emulated ones in every warp cost a small call 1.4 us.
  const int cs = 1 << p.cs_log, rank = blockIdx.x & (cs - 1), cid = blockIdx.x >> p.cs_log;
  const int tok0 = blockIdx.y * TOK;
  const int ntok = min(TOK, p.M - tok0);
  // This cluster's row blocks; this CTA's slabs are rank, rank + cs, ...
  const int rb0 = cid * p.rb_each + min(cid, p.rb_more), rb1 = rb0 + p.rb_each + (cid < p.rb_more);
  const int nsl = (p.nslab - rank + cs - 1) >> p.cs_log;
  const int max_sl = (p.nslab + cs - 1) >> p.cs_log;  // of any CTA of the cluster
  const int rows_stage = W >> p.kw_log;               // row blocks per stage

  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * stage_bytes<NT, GROUP>());
  uint64_t* empty = full + kStages;
  uint4* xs = reinterpret_cast<uint4*>(smem + ring_bytes<NT, GROUP>());               // [chunk][slab blocks][4 words j][NT][32 lanes]
  float* xsum = reinterpret_cast<float*>(xs + (size_t)p.chunk * kSlab * 4 * NT * 32);  // [chunk][slab blocks][GPB][TOK]
  float* part_buf = xsum + (size_t)p.chunk * kSlab * GPB * TOK;                        // [cs * kw][own][16][TOK]
  const int own_max = (p.tile + cs - 1) >> p.cs_log;  // row blocks of a tile that one CTA owns

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], W);
    }
    fence_barrier_init();
  }
  __syncthreads();
  // The other CTAs must have started before anything is stored into their shared memory.
  cluster_arrive();

  auto slab_blocks = [&](int s) { return min(kSlab, p.nkb - s * kSlab); };

  if (warp == W) {
    // ------------------------------ producer ------------------------------
    const uint64_t pol = l2_policy_evict_first();
    int stage = 0, filled = 0;
    uint32_t phase = 0;
    cluster_wait();
    for (int r0 = rb0; r0 < rb1; r0 += p.tile) {
      const int nr = min(p.tile, rb1 - r0);
      if (lane == 0) {
        for (int c0 = 0; c0 < max_sl; c0 += p.chunk) {
          const int c1 = min(c0 + p.chunk, nsl);
          for (int rg = 0; rg < nr; rg += rows_stage) {
            for (int sl = c0; sl < c1; ++sl) {
              const int s = rank + sl * cs, nb = slab_blocks(s);
              const uint32_t bytes = (uint32_t)min(rows_stage, nr - rg) * nb * BB;
              if (filled >= kStages) mbar_wait(&empty[stage], phase ^ 1, p.err, kDevErrEmptyWait);
              mbar_arrive_expect_tx(&full[stage], bytes);
              bulk_load(smem_u32(smem + stage * stage_bytes<NT, GROUP>()),
                        p.packed + ((size_t)s * kSlab * p.nrb + (size_t)(r0 + rg) * nb) * BB, bytes, &full[stage], pol);
              ++filled;
              if (++stage == kStages) {
                stage = 0;
                phase ^= 1;
              }
            }
          }
        }
      }
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      if (r0 + p.tile < rb1) {
        cluster_arrive();
        cluster_wait();
      }
    }
    // No copy may be in flight when the CTA ends, also when a multiplying warp gave up waiting for one.
    if (lane == 0) {
      for (int f = max(0, filled - kStages); f < filled; ++f)
        mbar_wait(&full[f % kStages], (f / kStages) & 1, p.err, kDevErrFullWait);
    }
    return;
  }

  // ------------------------------ multiply ------------------------------
  const int g = lane >> 2, c = lane & 3;
  const int wrow = warp & (rows_stage - 1), wk = warp >> (__ffs(W) - 1 - p.kw_log);  // row block of a stage, part of its slab
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;

  for (int r0 = rb0; r0 < rb1; r0 += p.tile) {
    const int nr = min(p.tile, rb1 - r0);
    for (int c0 = 0; c0 < max_sl; c0 += p.chunk) {
      const int c1 = min(c0 + p.chunk, nsl);  // c0 >= c1 in a CTA with one slab less
      // ---- stage x of these slabs: 8 inputs of a token per thread and iteration. Columns past the
      // last token stay whatever they are: they reach only sums that nobody reads. ----
      if (r0 == rb0 || p.chunk < max_sl) {
        if (c0 > 0 || r0 > rb0) named_bar_sync(1, W * 32);  // the previous chunk has been used
        constexpr int kPieces = kSlab * 16;  // of a token and slab; whole warps share a token (shuffles below)
        const int q = threadIdx.x % kPieces;
        const int kb = q >> 4, j = (q >> 2) & 3, cc = q & 3;
        for (int sl = 0; sl < c1 - c0; ++sl) {
          const int k = (rank + (c0 + sl) * cs) * (kSlab * kBlockK) + q * 8;
          for (int n = threadIdx.x / kPieces; n < ntok; n += W * 32 / kPieces) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (k < p.K)
              v = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + (size_t)(tok0 + n) * p.ldx + k);
            float sum = ((H::lo(v.x) + H::hi(v.x)) + (H::lo(v.y) + H::hi(v.y))) +
                        ((H::lo(v.z) + H::hi(v.z)) + (H::lo(v.w) + H::hi(v.w)));
#pragma unroll
            for (int off = 1; off < GROUP / 8; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            xs[(((sl * kSlab + kb) * 4 + j) * NT + (n >> 3)) * 32 + (n & 7) * 4 + cc] = v;
            if (q % (GROUP / 8) == 0) xsum[(sl * (kPieces * 8 / GROUP) + q / (GROUP / 8)) * TOK + n] = sum;
          }
        }
        named_bar_sync(1, W * 32);
      }
      if (r0 == rb0 && c0 == 0) cluster_wait();

      for (int rg = 0; rg < nr; rg += rows_stage) {
        const int lr = rg + wrow;  // this warp's row block of the tile
        float acc[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
        for (int sl = c0; sl < c1; ++sl) {
          if (ok && !mbar_wait(&full[stage], phase, p.err, kDevErrFullWait)) ok = false;
          if (lr < nr) {
            const int nb = slab_blocks(rank + sl * cs);
            const uint8_t* sb = smem + stage * stage_bytes<NT, GROUP>() + (size_t)wrow * nb * BB;
            const int b_end = min(nb, (wk + 1) * (kSlab >> p.kw_log));
#pragma unroll 1
            for (int bl = wk * (kSlab >> p.kw_log); bl < b_end; ++bl) {
              const uint8_t* bb = sb + bl * BB;
              const uint4 lo4 = *reinterpret_cast<const uint4*>(bb + lane * 16);
              const uint4 hi4 = *reinterpret_cast<const uint4*>(bb + 512 + lane * 16);
              const uint32_t* sz = reinterpret_cast<const uint32_t*>(bb + 1024) + g;
              const int lb = (sl - c0) * kSlab + bl;
              const uint4* xb = xs + (size_t)lb * 4 * NT * 32 + lane;
              const float* xg = xsum + lb * GPB * TOK + 2 * c;
              const uint32_t wlo[4] = {lo4.x, lo4.y, lo4.z, lo4.w};
              const uint32_t whi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
#pragma unroll
              for (int i = 0; i < GPB; ++i) {
                float part[NT][4];
#pragma unroll
                for (int jj = 0; jj < WPG; ++jj) {
                  const int j = i * WPG + jj;
                  uint32_t pl[4], ph[4];
                  H::expand(wlo[j], pl);
                  H::expand(whi[j], ph);
                  const uint32_t a0[4] = {pl[0], ph[0], pl[1], ph[1]};
                  const uint32_t a1[4] = {pl[2], ph[2], pl[3], ph[3]};
#pragma unroll
                  for (int t = 0; t < NT; ++t) {
                    const uint4 b = xb[(j * NT + t) * 32];
                    if (jj == 0)
                      mma_first<T>(part[t], a0, b.x, b.y);
                    else
                      H::mma(part[t], a0, b.x, b.y);
                    H::mma(part[t], a1, b.z, b.w);
                  }
                }
                const uint32_t z0 = sz[i * 16], z1 = sz[i * 16 + 8];
                const float s_lo = H::lo(z0), z_lo = H::hi(z0);
                const float s_hi = H::lo(z1), z_hi = H::hi(z1);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                  const float2 xx = *reinterpret_cast<const float2*>(xg + i * TOK + t * 8);
                  acc[t][0] = fmaf(s_lo, fmaf(-z_lo, xx.x, part[t][0]), acc[t][0]);
                  acc[t][1] = fmaf(s_lo, fmaf(-z_lo, xx.y, part[t][1]), acc[t][1]);
                  acc[t][2] = fmaf(s_hi, fmaf(-z_hi, xx.x, part[t][2]), acc[t][2]);
                  acc[t][3] = fmaf(s_hi, fmaf(-z_hi, xx.y, part[t][3]), acc[t][3]);
                }
              }
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[stage]);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        // The row block's partial sums go to the CTA that owns the rows. A warp whose CTA has no
        // slab in the first chunk leaves zeros; a later chunk adds to what this lane stored before.
        if (lr < nr && (c0 == 0 || c0 < c1)) {
          const int owner = lr & (cs - 1), slot = lr >> p.cs_log;
          float* mine = part_buf + (size_t)((((rank << p.kw_log) + wk) * own_max + slot) * 16 + g) * TOK + 2 * c;
          const uint32_t to = map_to(smem_u32(mine), owner);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (t * 8 + 2 * c < ntok) {
              const uint32_t at = to + t * 32;
              if (c0 > 0) {
                float a0, a1, a2, a3;
                ld_cluster(at, a0, a1);
                ld_cluster(at + 8 * TOK * 4, a2, a3);
                acc[t][0] += a0, acc[t][1] += a1, acc[t][2] += a2, acc[t][3] += a3;
              }
              st_cluster(at, acc[t][0], acc[t][1]);
              st_cluster(at + 8 * TOK * 4, acc[t][2], acc[t][3]);
            }
          }
        }
      }
    }

    // ---- every owner adds up its rows' partial sums, in order ----
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    {
      // Row block lr of the tile belongs to CTA lr mod cs; 16 lanes take its rows, for one token.
      const int n_own = (nr - rank + cs - 1) >> p.cs_log, parts = cs << p.kw_log;
      const int plane = own_max * 16 * TOK;
      const int r = lane & 15;
      for (int i = warp * 2 + (lane >> 4); i < n_own * TOK; i += W * 2) {
        const int slot = i / TOK, n = i % TOK;  // TOK is a power of two
        const int row = (r0 + (slot << p.cs_log) + rank) * 16 + r;
        if (n >= ntok || row >= p.N) continue;
        const float* from = part_buf + (slot * 16 + r) * TOK + n;
        float v = 0.f;
#pragma unroll 8
        for (int q = 0; q < parts; ++q) v += from[q * plane];
        const size_t off = (size_t)(tok0 + n) * p.N + row;
        if (p.residual) v += H::to_float(static_cast<const T*>(p.residual)[off]);
        static_cast<T*>(p.y)[off] = H::round(v);
      }
    }
    if (r0 + p.tile < rb1) {  // the next tile's partial sums overwrite these
      __syncwarp();
      cluster_arrive();
      cluster_wait();
    }
  }
}

// Clusters of 1, 2, 4 and 8 CTAs that can be resident at once, one CTA per SM; asked once per
// kernel and device (asking takes longer than a launch).
template <typename T, int NT, int GROUP>
static int resident_clusters(int (&out)[4]) {
  constexpr int kDevices = 64;
  static std::mutex mu;
  static int known[kDevices][4] = {};
  auto kern = w4_linear_kernel<T, NT, GROUP>;
  int dev = 0;
  FK_CHECK_CUDA(cudaGetDevice(&dev));
  FK_CHECK_ARG(dev >= 0 && dev < kDevices, "device index too large");
  std::lock_guard<std::mutex> lock(mu);
  int* k = known[dev];
  if (k[3] == 0) {
    FK_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    for (int i = 0; i < 4; ++i) {
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1 << i;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1u << i, 1, 1);
      cfg.blockDim = dim3(warps<NT>() * 32 + 32, 1, 1);
      cfg.dynamicSmemBytes = kSmem;
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

template <typename T, int NT, int GROUP>
static int launch(Params p, cudaStream_t st) {
  constexpr int W = warps<NT>();
  constexpr int kBudget = kSmem - ring_bytes<NT, GROUP>();  // for x and the partial sums
  constexpr int kX = x_bytes<NT, GROUP>();
  int resident[4];
  int rc = resident_clusters<T, NT, GROUP>(resident);
  if (rc) return rc;
  const int tiles = (p.M + NT * 8 - 1) / (NT * 8);
  // CTAs per cluster: the fewest that hold all of their x and partial sums at once, and whose
  // clusters have a row block for three quarters of the warps; at most 8 (the portable
  // size), and no more than there are slabs. With 8, x and rows may go in several rounds.
  int kw = 1, ncl = 0, own_bytes = 0, rows = 0, slabs = 0;
  for (p.cs_log = 0;; ++p.cs_log) {
    const int cs = 1 << p.cs_log;
    ncl = resident[p.cs_log] / tiles > 0 ? resident[p.cs_log] / tiles : 1;
    if (ncl > p.nrb) ncl = p.nrb;
    rows = (p.nrb + ncl - 1) / ncl;
    slabs = (p.nslab + cs - 1) / cs;
    // Few rows per cluster: 2 or 4 warps share a row block. Each part costs a plane of partial sums.
    for (kw = 1; kw < kSlab && W / kw >= 2 * rows;) kw *= 2;
    own_bytes = part_bytes<NT>() * cs * kw;  // one owned row block
    if (cs == 8 || 2 * cs > p.nslab) break;
    if ((long long)slabs * kX + (long long)((rows + cs - 1) / cs) * own_bytes <= kBudget && 4 * rows >= 3 * W) break;
  }
  const int cs = 1 << p.cs_log;
  // x takes what is left by one round of row blocks, the partial sums what is left by x.
  int own = (W / kw + cs - 1) / cs;
  if (own > (rows + cs - 1) / cs) own = (rows + cs - 1) / cs;
  p.chunk = (kBudget - own * own_bytes) / kX;
  if (p.chunk < 1) return fail(kErrUnsupported, "w4 linear: x does not fit into shared memory");
  if (p.chunk > slabs) p.chunk = slabs;
  own = (kBudget - p.chunk * kX) / own_bytes;
  const int rounds = (rows + own * cs - 1) / (own * cs);  // of equal size
  p.tile = (rows + rounds - 1) / rounds;
  own = (p.tile + cs - 1) / cs;
  const int smem = ring_bytes<NT, GROUP>() + p.chunk * kX + own * own_bytes;
  p.kw_log = kw == 4 ? 2 : kw == 2 ? 1 : 0;
  p.rb_each = p.nrb / ncl;
  p.rb_more = p.nrb % ncl;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cs;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ncl * cs), (unsigned)tiles, 1);
  cfg.blockDim = dim3(W * 32 + 32, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, w4_linear_kernel<T, NT, GROUP>, p));
  return kOk;
}

template <typename T, int NT>
static int by_group(const Params& p, int group, cudaStream_t st) {
  if (group == 32) return launch<T, NT, 32>(p, st);
  if (group == 64) return launch<T, NT, 64>(p, st);
  return launch<T, NT, 128>(p, st);
}

// 8, 16 or 32 tokens share one pass over the weight; more go in passes of 32, side by side.
template <typename T>
static int by_tokens(const Params& p, int group, cudaStream_t st) {
  if (p.M <= 8) return by_group<T, 1>(p, group, st);
  if (p.M <= 16) return by_group<T, 2>(p, group, st);
  return by_group<T, 4>(p, group, st);
}

}  // namespace w4
}  // namespace fk

using namespace fk;

extern "C" int fk_w4_linear(const void* x, long long ldx, const void* packed, const void* residual, void* y, int dtype,
                            int M, int N, int K, int group_size, void* stream) {
  FK_CHECK_ARG(x && packed && y, "null tensor pointer");
  FK_CHECK_ARG(dtype == FK_BF16 || dtype == FK_FP16, "dtype must be FK_BF16 or FK_FP16");
  FK_CHECK_ARG(M >= 1 && N >= 1 && K >= 1, "M, N and K must be >= 1");
  FK_CHECK_ARG(M <= 65535 * 32, "M too large");
  FK_CHECK_ARG(N <= (1 << 24) && K <= (1 << 24), "N and K must be <= 2^24");
  FK_CHECK_ARG(group_size == 32 || group_size == 64 || group_size == 128, "group_size must be 32, 64 or 128");
  FK_CHECK_ARG(K % group_size == 0, "K must be a multiple of group_size");
  FK_CHECK_ARG(ldx >= K && ldx % 8 == 0, "x row stride must be >= K and a multiple of 8 elements");
  FK_CHECK_ARG(((uintptr_t)x & 15) == 0 && ((uintptr_t)packed & 15) == 0,
               "x and packed must be 16-byte aligned");
  FK_CHECK_ARG(((uintptr_t)y & 1) == 0 && ((uintptr_t)residual & 1) == 0, "y and residual must be 2-byte aligned");
  w4::Params p = {};
  p.x = x;
  p.ldx = ldx;
  p.packed = static_cast<const uint8_t*>(packed);
  p.err = device_error_word();
  if (!p.err) return fail(kErrCuda, "device error word unavailable");
  p.residual = residual;
  p.y = y;
  p.M = M;
  p.N = N;
  p.K = K;
  p.nrb = (N + 15) / 16;
  p.nkb = (K + w4::kBlockK - 1) / w4::kBlockK;
  p.nslab = (p.nkb + w4::kSlab - 1) / w4::kSlab;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FK_BF16) return w4::by_tokens<__nv_bfloat16>(p, group_size, st);
  return w4::by_tokens<__half>(p, group_size, st);
}
