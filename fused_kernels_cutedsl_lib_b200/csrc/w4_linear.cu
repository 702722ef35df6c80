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
// blocks of 128. Block (nb, kb) is 1 KB, [2][32][4] words: half h, lane
// l = 4*g + c, word j holds the eight nibbles of row nb*16 + 8*h + g, inputs
// kb*128 + 32*j + 8*c + 0..7. Lane l of a warp therefore loads its mma.sync A
// operands of both row halves as two 16-byte words, the warp 2 x 512 contiguous
// bytes, and a group of 32 inputs is one word j across the four lanes of a row,
// so every group size is a whole number of mma steps. Which input sits at which
// k index of the mma does not matter as long as x uses the same order.
//
// Work split. A CTA is 8 warps = WR row blocks x KW input slices, and a cluster
// of CS CTAs splits the inputs further; the partial sums meet in (distributed)
// shared memory and are added in a fixed order, so there is no workspace, no
// atomic, and results do not depend on timing. Each warp keeps four 1 KB blocks
// in flight in registers; the weights' first loads are issued before the wait
// for the preceding kernel (programmatic dependent launch).
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "fk_b200.h"

namespace fk {
namespace w4 {

namespace cg = cooperative_groups;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kBlockK = 128;  // inputs per packed block
constexpr int kPrefetch = 4;  // packed blocks in flight per warp

struct Params {
  const void* x;
  long long ldx;
  const uint4* packed;       // [nb16][nkb][2][32] x 16 B
  const uint32_t* sz;        // [nb16][nkb * 128 / group][16]: scale (low half) and 16 + z (high half)
  const void* residual;      // [M, N] or null
  void* y;                   // [M, N]
  int M, N, K;
  int nb16, nkb;
  int wr, kw;                // row blocks and input slices per CTA (wr * kw == kWarps)
  int chunk_steps;           // steps (of kw blocks) whose x is staged at a time
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

__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// NT: tiles of 8 tokens; GROUP: inputs per scale.
template <typename T, int NT, int GROUP>
__global__ void __launch_bounds__(kThreads) w4_linear_kernel(const Params p) {
  using H = Half<T>;
  constexpr int GPB = kBlockK / GROUP;  // groups per packed block
  constexpr int WPG = 4 / GPB;          // words of a lane per group
  constexpr int TOK = NT * 8;
  extern __shared__ uint4 smem4[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int wrow = warp % p.wr, wk = warp / p.wr;

  cg::cluster_group cluster = cg::this_cluster();
  const int cs = cluster.num_blocks(), rank = cluster.block_rank();
  const int row_cta = blockIdx.x / cs;
  const int tok0 = blockIdx.y * TOK;
  const int ntok = min(TOK, p.M - tok0);
  // This CTA's slice of the packed input blocks.
  const int kb0 = (int)((long long)p.nkb * rank / cs);
  const int nblk = (int)((long long)p.nkb * (rank + 1) / cs) - kb0;
  const int steps = (nblk + p.kw - 1) / p.kw;
  // The last CTA may hold row blocks past the end: it repeats the last one and stores nothing for it.
  const int nb = min(row_cta * p.wr + wrow, p.nb16 - 1);

  const uint4* wp = p.packed + ((size_t)nb * p.nkb + kb0) * 64 + lane;
  const uint32_t* sp = p.sz + ((size_t)nb * p.nkb + kb0) * (GPB * 16) + g;

  struct Block {
    uint4 lo, hi;
    uint32_t slo[GPB], shi[GPB];
  } blk[kPrefetch];
  auto load = [&](Block& d, int step) {
    const int kb = step * p.kw + wk;
    if (kb < nblk) {
      d.lo = ld_stream(wp + (size_t)kb * 64);
      d.hi = ld_stream(wp + (size_t)kb * 64 + 32);
#pragma unroll
      for (int i = 0; i < GPB; ++i) {
        d.slo[i] = __ldg(sp + (size_t)kb * (GPB * 16) + i * 16);
        d.shi[i] = __ldg(sp + (size_t)kb * (GPB * 16) + i * 16 + 8);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kPrefetch; ++i) load(blk[i], i);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  uint4* xs = smem4;  // [chunk blocks][4 words j][NT][32 lanes]: B operands in lane order
  float* xsum = reinterpret_cast<float*>(xs + (size_t)p.chunk_steps * p.kw * 4 * NT * 32);  // [groups][TOK]

  float acc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;

  for (int s0 = 0; s0 < steps; s0 += p.chunk_steps) {
    // ---- stage x of this chunk: 8 inputs of a token per thread and iteration ----
    const int cblk = min(p.chunk_steps * p.kw, nblk - s0 * p.kw);
    const int pieces = cblk * 16;
    const int kbase = (kb0 + s0 * p.kw) * kBlockK;
    if (s0) __syncthreads();
    for (int it = 0; it < TOK * pieces; it += kThreads) {  // whole warps run every iteration (shuffles below)
      const int i = it + threadIdx.x;
      const int n = i / pieces, q = i - n * pieces;
      const int k = kbase + q * 8;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (n < ntok && k < p.K)
        v = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + (size_t)(tok0 + n) * p.ldx + k);
      float sum = ((H::lo(v.x) + H::hi(v.x)) + (H::lo(v.y) + H::hi(v.y))) +
                  ((H::lo(v.z) + H::hi(v.z)) + (H::lo(v.w) + H::hi(v.w)));
#pragma unroll
      for (int off = 1; off < GROUP / 8; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (n < TOK) {
        // Pairs in the order the nibbles come out of a word: (0,4) (1,5) (2,6) (3,7).
        uint4 o;
        o.x = __byte_perm(v.x, v.z, 0x5410);
        o.y = __byte_perm(v.x, v.z, 0x7632);
        o.z = __byte_perm(v.y, v.w, 0x5410);
        o.w = __byte_perm(v.y, v.w, 0x7632);
        const int kb = q >> 4, j = (q >> 2) & 3, cc = q & 3;
        xs[((kb * 4 + j) * NT + (n >> 3)) * 32 + (n & 7) * 4 + cc] = o;
        if (q % (GROUP / 8) == 0) xsum[(q / (GROUP / 8)) * TOK + n] = sum;
      }
    }
    __syncthreads();

    // ---- multiply: kPrefetch steps at a time so that the register ring is indexed statically ----
    const int s1 = min(s0 + p.chunk_steps, steps);
    for (int sb = s0; sb < s1; sb += kPrefetch) {
#pragma unroll
      for (int u = 0; u < kPrefetch; ++u) {
        const int step = sb + u;
        const int kb = step * p.kw + wk;
        if (step < s1 && kb < nblk) {
          Block& d = blk[u];
          const int lb = kb - s0 * p.kw;  // block within the staged chunk
          const uint32_t wlo[4] = {d.lo.x, d.lo.y, d.lo.z, d.lo.w};
          const uint32_t whi[4] = {d.hi.x, d.hi.y, d.hi.z, d.hi.w};
#pragma unroll
          for (int i = 0; i < GPB; ++i) {
            float part[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) part[t][0] = part[t][1] = part[t][2] = part[t][3] = 0.f;
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
                const uint4 b = xs[((lb * 4 + j) * NT + t) * 32 + lane];
                H::mma(part[t], a0, b.x, b.y);
                H::mma(part[t], a1, b.z, b.w);
              }
            }
            const float s_lo = H::lo(d.slo[i]), z_lo = H::hi(d.slo[i]);
            const float s_hi = H::lo(d.shi[i]), z_hi = H::hi(d.shi[i]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const float2 xx = *reinterpret_cast<const float2*>(xsum + (lb * GPB + i) * TOK + t * 8 + 2 * c);
              acc[t][0] = fmaf(s_lo, fmaf(-z_lo, xx.x, part[t][0]), acc[t][0]);
              acc[t][1] = fmaf(s_lo, fmaf(-z_lo, xx.y, part[t][1]), acc[t][1]);
              acc[t][2] = fmaf(s_hi, fmaf(-z_hi, xx.x, part[t][2]), acc[t][2]);
              acc[t][3] = fmaf(s_hi, fmaf(-z_hi, xx.y, part[t][3]), acc[t][3]);
            }
          }
        }
        // Refill after the use; steps past the end load nothing.
        if (step < s1) load(blk[u], step + kPrefetch);
      }
    }
  }

  // ---- add up the slices: this CTA's kw partials, then the cluster's, in order ----
  __syncthreads();  // xs is free
  float* red = reinterpret_cast<float*>(smem4);  // [kw][TOK][rows]
  const int rows = p.wr * 16;
  {
    float* dst = red + (size_t)wk * TOK * rows + wrow * 16;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int n0 = t * 8 + 2 * c;
      dst[(size_t)n0 * rows + g] = acc[t][0];
      dst[(size_t)(n0 + 1) * rows + g] = acc[t][1];
      dst[(size_t)n0 * rows + g + 8] = acc[t][2];
      dst[(size_t)(n0 + 1) * rows + g + 8] = acc[t][3];
    }
  }
  if (cs > 1) cluster.sync(); else __syncthreads();
  const int total = ntok * rows;
  for (int i = rank * kThreads + threadIdx.x; i < total; i += cs * kThreads) {
    const int n = i / rows, r = i - n * rows;
    const int row = row_cta * rows + r;
    if (row >= p.N) continue;
    float v = 0.f;
    for (int q = 0; q < cs; ++q) {
      const float* src = cs > 1 ? cluster.map_shared_rank(red, q) : red;
      for (int w = 0; w < p.kw; ++w) v += src[((size_t)w * TOK + n) * rows + r];
    }
    const size_t off = (size_t)(tok0 + n) * p.N + row;
    if (p.residual) v += H::to_float(static_cast<const T*>(p.residual)[off]);
    static_cast<T*>(p.y)[off] = H::round(v);
  }
  if (cs > 1) cluster.sync();  // no CTA leaves while another reads its partials
}

template <typename T, int NT, int GROUP>
static int launch(Params p, cudaStream_t st) {
  auto kern = w4_linear_kernel<T, NT, GROUP>;
  // Inputs across a cluster: as many slices as there are blocks, at most 8 (the
  // portable cluster size). Rows per CTA: 128, halved (with the warps moved to
  // more input slices) while the grid does not cover the SMs twice. kw * NT <= 16
  // bounds the staged x to 128 KB.
  int cs = 8;
  while (cs > 1 && cs > p.nkb) cs >>= 1;
  p.wr = 8;
  const long long tiles = (p.M + NT * 8 - 1) / (NT * 8);
  while (p.wr > 1 && 2 * (kWarps / p.wr) * NT <= 16 &&
         (long long)((p.nb16 + p.wr - 1) / p.wr) * cs * tiles < 2 * num_sms())
    p.wr >>= 1;
  p.kw = kWarps / p.wr;
  const int steps = ((p.nkb + cs - 1) / cs + p.kw - 1) / p.kw;
  // x staged per chunk: up to 64 KB of it, in whole rounds of the register ring.
  int max_steps = 32 / (NT * p.kw);
  max_steps = max_steps < kPrefetch ? kPrefetch : max_steps / kPrefetch * kPrefetch;
  p.chunk_steps = steps < max_steps ? steps : max_steps;
  const size_t xbytes = (size_t)p.chunk_steps * p.kw * (4 * NT * 32 * 16 + (kBlockK / GROUP) * NT * 8 * 4);
  const size_t rbytes = (size_t)p.kw * NT * 8 * p.wr * 16 * 4;
  const size_t smem = xbytes > rbytes ? xbytes : rbytes;
  FK_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cs;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.nb16 + p.wr - 1) / p.wr * cs), (unsigned)tiles, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  return kOk;
}

template <typename T, int NT>
static int by_group(const Params& p, int group, cudaStream_t st) {
  if (group == 32) return launch<T, NT, 32>(p, st);
  if (group == 64) return launch<T, NT, 64>(p, st);
  return launch<T, NT, 128>(p, st);
}

template <typename T>
static int by_tokens(const Params& p, int group, cudaStream_t st) {
  if (p.M <= 8) return by_group<T, 1>(p, group, st);
  if (p.M <= 16) return by_group<T, 2>(p, group, st);
  if (p.M <= 32) return by_group<T, 4>(p, group, st);
  return by_group<T, 8>(p, group, st);
}

}  // namespace w4
}  // namespace fk

using namespace fk;

extern "C" int fk_w4_linear(const void* x, long long ldx, const void* packed, const void* scale_zero,
                            const void* residual, void* y, int dtype, int M, int N, int K, int group_size,
                            void* stream) {
  FK_CHECK_ARG(x && packed && scale_zero && y, "null tensor pointer");
  FK_CHECK_ARG(dtype == FK_BF16 || dtype == FK_FP16, "dtype must be FK_BF16 or FK_FP16");
  FK_CHECK_ARG(M >= 1 && N >= 1 && K >= 1, "M, N and K must be >= 1");
  FK_CHECK_ARG(M <= 65535 * 64, "M too large");
  FK_CHECK_ARG(N <= (1 << 24) && K <= (1 << 24), "N and K must be <= 2^24");
  FK_CHECK_ARG(group_size == 32 || group_size == 64 || group_size == 128, "group_size must be 32, 64 or 128");
  FK_CHECK_ARG(K % group_size == 0, "K must be a multiple of group_size");
  FK_CHECK_ARG(ldx >= K && ldx % 8 == 0, "x row stride must be >= K and a multiple of 8 elements");
  FK_CHECK_ARG(((uintptr_t)x & 15) == 0 && ((uintptr_t)packed & 15) == 0 && ((uintptr_t)scale_zero & 3) == 0,
               "x and packed must be 16-byte aligned");
  FK_CHECK_ARG(((uintptr_t)y & 1) == 0 && ((uintptr_t)residual & 1) == 0, "y and residual must be 2-byte aligned");
  w4::Params p = {};
  p.x = x;
  p.ldx = ldx;
  p.packed = static_cast<const uint4*>(packed);
  p.sz = static_cast<const uint32_t*>(scale_zero);
  p.residual = residual;
  p.y = y;
  p.M = M;
  p.N = N;
  p.K = K;
  p.nb16 = (N + 15) / 16;
  p.nkb = (K + w4::kBlockK - 1) / w4::kBlockK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FK_BF16) return w4::by_tokens<__nv_bfloat16>(p, group_size, st);
  return w4::by_tokens<__half>(p, group_size, st);
}
