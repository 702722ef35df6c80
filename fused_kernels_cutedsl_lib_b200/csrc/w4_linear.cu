// Linear layer with 4-bit weights and group scales for up to 16 tokens (more, and some sizes
// from 9 on: w4_tc.cu; the choice is explained in fk_w4_linear):
//   y[m, n] = sum_k x[m, k] * (q[n, k] - z[n, k / g]) * s[n, k / g]  (+ residual[m, n])
// with q, z in [0, 15], g in {32, 64, 128} and x, s, y bf16 or fp16.
//
// The 4-bit weights are read once (N*K/2 bytes). What bounds the kernel is latency within its warps: four
// to a scheduler, each of which waits for a stage, expands a block, multiplies and scales it, one after
// the other. Profiled, 28672 x 4096, groups of 128, weights from memory: for one token 0.52 instructions per
// cycle and scheduler, the tensor pipe 16 % busy, DRAM 34 %; for 16 tokens 0.49 and 25 %. Measured on weights
// that do not lie in L2, bf16, groups of 128: 4096 x 4096 5.7 us for one token, of which some 4 are launch,
// cluster start and join; 28672 x 4096 18.4 us for one token (3.4 TB/s) and 26.5 for 16.
//
// Arithmetic. The weights never become rounded 16-bit products q*s. Nibbles are or-ed
// into the mantissa of fp16 256.0 (bit 2) or 16.0 (bit 6), which gives the exact numbers
// 256 + q and 16 + q, two nibbles of a 16-bit half per rotation of the word: five ALU
// instructions for eight weights (bf16 has too few mantissa bits for a second nibble:
// eight). Those integers go to the tensor cores as they are; per group of g inputs
//   sum x (q - z) = sum x (off + q) - sum x off - z sum x,
// with both sums of x computed once per CTA, so offset and zero point cost an addition
// and a multiply-add per output and group, and the scale another, all in fp32. bf16
// activations become fp16 by a power of two per token and 128 inputs that brings the
// greatest to [2^14, 2^15): exact for everything within 2^-28 of it, off by 2^-39 of it
// below. The offsets cancel: an error of some 2^-22 * 256 / 5 of the result, under a
// quarter of fp16's half step.
//
// Layout (made once by the caller, `pack_w4`): rows in blocks of 16, inputs in
// blocks of 128 and slabs of 2 blocks (the last slab may have one). A block is
// its codes, [2][32][4] words: half h, lane l = 4*g + c, word j holds the eight
// nibbles of row 8*h + g, inputs 32*j + 8*c + 0..7, as the word rotated left by 2 of
// which nibble i < 4 is input 2i and nibble i >= 4 input 2(i - 4) + 1, so that a pair
// (i, i + 4) is a pair of neighbouring inputs; then its scales and zero points,
// [groups][16] words. Lane l of a warp therefore reads its mma.sync A operands of both
// row halves as two 16-byte words, the B operands are 16 bytes of x as they lie in
// memory, and a group of 32 inputs is one word j across the four lanes of a row, so
// every group size is a whole number of mma steps. Memory order is slab, row block,
// block: the rows of a slab are one contiguous stream.
//
// Work split. Slabs go to the CS CTAs of a cluster, row blocks to the clusters, one
// persistent grid. A CTA stages its slabs of x in shared memory once, in operand
// order, with the group sums. A producer thread streams 8 / KW row blocks of a slab per
// bulk copy (17 KB; copies of 1 KB reached 1.5 TB/s only) into a ring of six stages; groups
// of eight warps take turns at row blocks, each warp one row block or one of KW parts
// of its slab. A finished row block's partial sums are stored into the shared memory of
// the CTA of the cluster that owns the rows; when every CTA has told it so (an mbarrier
// with one arrival per CTA), an owner adds what it got in a fixed order: no workspace, no
// atomic, and results do not depend on timing. The first weight copies are issued before the wait for the preceding kernel
// (programmatic dependent launch).
#include <cuda_fp16.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "fk_b200.h"
#include "w4.cuh"

namespace fk {
namespace w4 {

constexpr int kSlabK = kSlab * kBlockK;
constexpr int kGroupWarps = 8;  // warps that share a stage
constexpr int kStages = 6;
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
  int withhold;              // test hook: the fill that the first CTA's producer leaves out (-1: none)
};

// D = A * B: the first step of a group starts from nothing.
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ float4 lds128f(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float2 lds64f(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}
constexpr int kWarps = 16;  // that multiply
template <int GROUP>
__host__ __device__ constexpr int stage_bytes() { return kGroupWarps * kSlab * block_bytes<GROUP>(); }
// Bytes of shared memory: the ring with its barriers; one slab of x with the sums of its groups and the
// scales of its blocks; one row block's partial sums from one warp.
template <int GROUP>
__host__ __device__ constexpr int ring_bytes() { return kStages * stage_bytes<GROUP>() + 128; }
template <int NT>
__host__ __device__ constexpr int xop_bytes() { return kSlab * 4 * NT * 32 * 16; }
template <int NT, int GROUP>
__host__ __device__ constexpr int sum_bytes() { return kSlab * (kBlockK / GROUP) * NT * 8 * 8; }
template <int NT>
__host__ __device__ constexpr int inv_bytes() { return kSlab * NT * 8 * 4; }
template <int NT, int GROUP>
__host__ __device__ constexpr int x_bytes() { return xop_bytes<NT>() + sum_bytes<NT, GROUP>() + inv_bytes<NT>(); }
template <int NT>
__host__ __device__ constexpr int part_bytes() { return 16 * NT * 8 * 4; }

// NT: tiles of 8 tokens; GROUP: inputs per scale.
template <typename T, int NT, int GROUP>
__global__ void __launch_bounds__(kWarps * 32 + 32, 1) w4_linear_kernel(const Params p) {
  using H = Half<T>;
  constexpr bool kScaled = std::is_same<T, __nv_bfloat16>::value;  // x goes in as fp16 times a power of two
  constexpr int W = kWarps;
  constexpr int NG = W / kGroupWarps;
  constexpr int GPB = kBlockK / GROUP;  // groups per input block
  constexpr int WPG = 4 / GPB;          // words of a lane per group
  constexpr int TOK = NT * 8;
  constexpr int BB = block_bytes<GROUP>();
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // The host did the divisions: emulated ones in every warp cost a small call 1.4 us.
  const int cs = 1 << p.cs_log, rank = blockIdx.x & (cs - 1), cid = blockIdx.x >> p.cs_log;
  const int ntok = p.M;  // at most TOK
  // This cluster's row blocks; this CTA's slabs are rank, rank + cs, ...
  const int rb0 = cid * p.rb_each + min(cid, p.rb_more), rb1 = rb0 + p.rb_each + (cid < p.rb_more);
  const int nsl = (p.nslab - rank + cs - 1) >> p.cs_log;
  const int max_sl = (p.nslab + cs - 1) >> p.cs_log;   // of any CTA of the cluster
  const int rows_stage = kGroupWarps >> p.kw_log;      // row blocks per stage

  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * stage_bytes<GROUP>());
  uint64_t* empty = full + kStages;
  uint64_t* done = empty + kStages;  // one arrival per CTA: its partial sums of the tile are stored
  uint64_t* taken = done + 1;        // one arrival per CTA: it has added up the tile's
  volatile int* gave_up = reinterpret_cast<volatile int*>(taken + 1);  // a wait of this CTA has run out
  uint8_t* xmem = smem + ring_bytes<GROUP>();
  uint4* xs = reinterpret_cast<uint4*>(xmem);                                           // [chunk][blocks][4 words j][NT][32 lanes]
  float4* xsum = reinterpret_cast<float4*>(xmem + (size_t)p.chunk * xop_bytes<NT>());   // [chunk][blocks][GPB][TOK / 2]: sums of two tokens, then their offset sums
  float* xinv = reinterpret_cast<float*>(xsum) + (size_t)p.chunk * (sum_bytes<NT, GROUP>() / 4);  // [chunk][blocks][TOK]: 1 / scale
  float* part_buf = xinv + (size_t)p.chunk * (inv_bytes<NT>() / 4);                     // [cs * kw][own][16][TOK]
  const int own_max = (p.tile + cs - 1) >> p.cs_log;  // row blocks of a tile that one CTA owns

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kGroupWarps);
    }
    mbar_init(done, cs);
    mbar_init(taken, cs);
    *gave_up = 0;
    fence_barrier_init();
  }
  __syncthreads();
  // The other CTAs must have started, their barriers included, before anything is stored into their
  // shared memory. The only phase of the cluster's own barrier.
  cluster_arrive();

  auto slab_blocks = [&](int s) { return min(kSlab, p.nkb - s * kSlab); };

  if (warp == W) {
    // ------------------------------ producer ------------------------------
    const uint64_t pol = l2_policy_evict_first();
    int stage = 0, filled = 0;
    uint32_t phase = 0;
    bool live = true;  // until a wait runs out: nothing more is loaded then
    for (int r0 = rb0; r0 < rb1; r0 += p.tile) {
      const int nr = min(p.tile, rb1 - r0);
      if (lane == 0) {
        for (int c0 = 0; c0 < max_sl && live; c0 += p.chunk) {
          const int c1 = min(c0 + p.chunk, nsl);
          for (int rg = 0; rg < nr && live; rg += NG * rows_stage) {
            for (int sl = c0; sl < c1 && live; ++sl) {
              const int s = rank + sl * cs, nb = slab_blocks(s);
              const uint8_t* src = p.packed + ((size_t)s * kSlab * p.nrb + (size_t)(r0 + rg) * nb) * BB;
#pragma unroll
              for (int q = 0; q < NG; ++q) {
                const int n = min(rows_stage, nr - rg - q * rows_stage);
                if (n <= 0) break;
                const uint32_t bytes = (uint32_t)(n * nb) * BB;
                // Stages are emptied by warps that wait for the preceding kernel, however long it takes.
                if (filled == kStages) asm volatile("griddepcontrol.wait;" ::: "memory");
                if (filled >= kStages) live = w4::wait(&empty[stage], phase ^ 1, p.err, kDevErrEmptyWait);
                if (!live) break;
                if (filled != p.withhold || blockIdx.x != 0) {
                  mbar_arrive_expect_tx(&full[stage], bytes);
                  bulk_load(smem_u32(smem + stage * stage_bytes<GROUP>()), src + (size_t)(q * rows_stage * nb) * BB,
                            bytes, &full[stage], pol);
                }
                ++filled;
                if (++stage == kStages) {
                  stage = 0;
                  phase ^= 1;
                }
              }
            }
          }
        }
      }
    }
    __syncwarp();
    cluster_wait();
    // No copy may be in flight when the CTA ends, also when a multiplying warp gave up waiting for one.
    if (lane == 0) {
      for (int f = max(0, filled - kStages); f < filled; ++f)
        w4::wait(&full[f % kStages], (f / kStages) & 1, p.err, kDevErrFullWait);
    }
    return;
  }

  // ------------------------------ multiply ------------------------------
  const int g = lane >> 2, c = lane & 3;
  const int gid = warp / kGroupWarps, gw = warp % kGroupWarps;
  const int wrow = gw & (rows_stage - 1), wk = gw >> (3 - p.kw_log);  // row block of a stage, part of its slab
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // Where a lane reads its tokens' operands: columns past the last token read the last one's, whose
  // bytes the shared memory serves once (one token: a quarter of the wavefronts).
  uint32_t xlane[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) xlane[t] = (min(g, max(0, ntok - 1 - t * 8)) * 4 + c) * 16;
  int stage = 0;  // of the next fill of the current round of row blocks
  uint32_t phase = 0;
  auto advance = [&](int& st, uint32_t& ph, int n) {  // n <= kStages
    st += n;
    if (st >= kStages) {
      st -= kStages;
      ph ^= 1;
    }
  };
  bool ok = true;  // the same in all lanes wherever products depend on it

  uint32_t tile_phase = 0;
  // All of this CTA's multiplying warps have come here, and one of them tells the cluster; no more of that once a
  // wait of any of them has run out. The CTA then goes through the rest without waiting; the cluster's other
  // CTAs, which now wait in vain, do the same.
  auto tell = [&](uint64_t* bar) {
    if (!ok) *gave_up = 1;
    named_bar_sync(1, W * 32);
    if (warp == 0 && lane < cs && *gave_up == 0) arrive_cluster(map_to(smem_u32(bar), lane));
  };
  for (int r0 = rb0; r0 < rb1; r0 += p.tile, tile_phase ^= 1) {
    const int nr = min(p.tile, rb1 - r0);
    for (int c0 = 0; c0 < max_sl; c0 += p.chunk) {
      const int c1 = min(c0 + p.chunk, nsl);  // c0 >= c1 in a CTA with one slab less
      // ---- stage x of these slabs: a warp takes a token's slab, a lane 8 inputs; four such loads in
      // flight. Columns past the last token stay whatever they are: they reach only sums that nobody reads. ----
      if (r0 == rb0 || p.chunk < max_sl) {
        if (c0 > 0 || r0 > rb0) named_bar_sync(1, W * 32);  // the previous chunk has been used
        const int j = (lane >> 2) & 3, cc = lane & 3, kb = lane >> 4;
        constexpr int U = 4;
        int sl = c0, n = warp;  // item (slab, token)
        while (sl < c1 && n >= ntok) n -= ntok, ++sl;
        while (sl < c1) {
          uint4 v[U];
          int isl[U], in[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            isl[u] = sl;
            in[u] = n;
            v[u] = make_uint4(0u, 0u, 0u, 0u);
            if (sl < c1) {
              const int k = (rank + sl * cs) * kSlabK + lane * 8;
              if (k < p.K)
                v[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + (size_t)n * p.ldx + k);
              n += W;
              while (sl < c1 && n >= ntok) n -= ntok, ++sl;
            }
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (isl[u] >= c1) break;
            const int lsl = isl[u] - c0, nn = in[u];
            uint4 w = v[u];
            float inv = 1.f;
            if constexpr (kScaled) {
              // The greatest magnitude of the token's 128 inputs, by the bits without signs.
              uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu),
                                    __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
              m = max(m & 0xFFFFu, m >> 16);
#pragma unroll
              for (int off = 1; off < 16; off <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
              const int e = min(141 - (int)(m >> 7), 126);  // x * 2^e is below 2^15
              const float scale = __uint_as_float((uint32_t)(127 + e) << 23);
              inv = __uint_as_float((uint32_t)(127 - e) << 23);
              uint32_t* wp = &w.x;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const __half2 hh = __floats2half2_rn(H::lo(wp[i]) * scale, H::hi(wp[i]) * scale);
                wp[i] = *reinterpret_cast<const uint32_t*>(&hh);
              }
            }
            xs[(((lsl * kSlab + kb) * 4 + j) * NT + (nn >> 3)) * 32 + (nn & 7) * 4 + cc] = w;
            if (kScaled && (lane & 15) == 0) xinv[(lsl * kSlab + kb) * TOK + nn] = inv;
          }
        }
        named_bar_sync(1, W * 32);
        // The groups' sums, by the tensor cores: a matrix whose row 0 is all ones and whose row 1 has the
        // offsets (256 256 16 16 per lane and step) times the operands just stored. A warp takes
        // a block's 8 tokens; lanes 0..3 end up with the sums of tokens 2c, 2c + 1 and lanes 4..7 with
        // their offset sums.
        const uint32_t one = g == 0 ? 0x3C003C00u : g == 1 ? 0x5C005C00u : 0u;
        const uint32_t two = g == 0 ? 0x3C003C00u : g == 1 ? 0x4C004C00u : 0u;
        const uint32_t af[4] = {one, 0u, two, 0u};
        for (int i = warp; i < (c1 - c0) * kSlab * NT; i += W) {
          const int blk = i / NT, t = i % NT;
#pragma unroll
          for (int gi = 0; gi < GPB; ++gi) {
            float d[4];
#pragma unroll
            for (int jj = 0; jj < WPG; ++jj) {
              const uint4 b = xs[((blk * 4 + gi * WPG + jj) * NT + t) * 32 + lane];
              if (jj == 0)
                mma_first(d, af, b.x, b.y);
              else
                mma_f16_16816(d, af, b.x, b.y);
              mma_f16_16816(d, af, b.z, b.w);
            }
            if (lane < 8)
              reinterpret_cast<float2*>(xsum + (blk * GPB + gi) * (TOK / 2) + t * 4 + c)[g] = make_float2(d[0], d[1]);
          }
        }
        named_bar_sync(1, W * 32);
      }
      if (c0 == 0) {
        if (r0 == rb0)
          cluster_wait();
        else if (ok)  // the owners are done with the tile before
          ok = wait_cluster(taken, tile_phase ^ 1, p.err);
        if (__any_sync(0xffffffffu, !ok)) ok = false;
      }

      const ExpandConsts consts;
      for (int rg = 0; rg < nr; rg += NG * rows_stage) {
        const int lr = rg + gid * rows_stage + wrow;                      // this warp's row block of the tile
        const int groups = min(NG, (nr - rg + rows_stage - 1) >> (3 - p.kw_log));  // warp groups with rows in this round
        bool mine = gid < groups && ok;
        const bool live = lr < nr;
        float acc[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
        int st = stage;
        uint32_t ph = phase;
        if (gid) advance(st, ph, gid);
        for (int sl = c0; sl < c1; ++sl) {
          advance(stage, phase, groups);
          if (!mine) continue;
          if (!__all_sync(0xffffffffu, w4::wait(&full[st], ph, p.err, kDevErrFullWait))) {
            ok = mine = false;  // nor are its stages given back
            continue;
          }
          if (live) {
            const int nb = slab_blocks(rank + sl * cs);
            const int b0 = wk * (kSlab >> p.kw_log), b1 = min(nb, b0 + (kSlab >> p.kw_log));
            const int lb0 = (sl - c0) * kSlab + b0;
            uint32_t wa = smem_u32(smem + st * stage_bytes<GROUP>() + (wrow * nb + b0) * BB) + lane * 16;
            uint32_t xa = smem_u32(xs + (size_t)lb0 * (4 * NT * 32));
            uint32_t sa = smem_u32(xsum + (size_t)lb0 * (GPB * (TOK / 2)) + c);
            uint32_t va = smem_u32(xinv + lb0 * TOK + 2 * c);
#pragma unroll 1
            for (int bl = b0; bl < b1; ++bl) {
              const uint4 lo4 = lds128(wa), hi4 = lds128(wa + 512);
              const uint32_t za = wa - lane * 16 + 1024 + g * 4;
              const uint32_t wlo[4] = {lo4.x, lo4.y, lo4.z, lo4.w};
              const uint32_t whi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
#pragma unroll
              for (int i = 0; i < GPB; ++i) {
                float part[NT][4];
#pragma unroll
                for (int jj = 0; jj < WPG; ++jj) {
                  const int j = i * WPG + jj;
                  uint32_t pl[4], ph4[4];
                  expand(wlo[j], pl, consts);
                  expand(whi[j], ph4, consts);
                  const uint32_t a0[4] = {pl[0], ph4[0], pl[1], ph4[1]};
                  const uint32_t a1[4] = {pl[2], ph4[2], pl[3], ph4[3]};
#pragma unroll
                  for (int t = 0; t < NT; ++t) {
                    const uint4 b = lds128(xa + (j * NT + t) * 512 + xlane[t]);
                    if (jj == 0)
                      mma_first(part[t], a0, b.x, b.y);
                    else
                      mma_f16_16816(part[t], a0, b.x, b.y);
                    mma_f16_16816(part[t], a1, b.z, b.w);
                  }
                }
                const uint32_t z0 = lds32(za + i * 64), z1 = lds32(za + i * 64 + 32);
                const float s_lo = H::lo(z0), z_lo = H::hi(z0);
                const float s_hi = H::lo(z1), z_hi = H::hi(z1);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                  const float4 xx = lds128f(sa + (i * (TOK / 2) + t * 4) * 16);
                  const float2 iv = kScaled ? lds64f(va + t * 32) : make_float2(1.f, 1.f);
                  const float s0 = kScaled ? s_lo * iv.x : s_lo, s1 = kScaled ? s_lo * iv.y : s_lo;
                  const float s2 = kScaled ? s_hi * iv.x : s_hi, s3 = kScaled ? s_hi * iv.y : s_hi;
                  acc[t][0] = fmaf(s0, fmaf(-z_lo, xx.x, part[t][0] - xx.z), acc[t][0]);
                  acc[t][1] = fmaf(s1, fmaf(-z_lo, xx.y, part[t][1] - xx.w), acc[t][1]);
                  acc[t][2] = fmaf(s2, fmaf(-z_hi, xx.x, part[t][2] - xx.z), acc[t][2]);
                  acc[t][3] = fmaf(s3, fmaf(-z_hi, xx.y, part[t][3] - xx.w), acc[t][3]);
                }
              }
              wa += BB;
              xa += 4 * NT * 512;
              sa += GPB * (TOK / 2) * 16;
              va += TOK * 4;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[st]);
          advance(st, ph, groups);
        }
        // The row block's partial sums go to the CTA that owns the rows. A warp whose CTA has no
        // slab in the first chunk leaves zeros; a later chunk adds to what this lane stored before.
        if (live && (c0 == 0 || c0 < c1)) {
          const int owner = lr & (cs - 1), slot = lr >> p.cs_log;
          float* dst = part_buf + (size_t)((((rank << p.kw_log) + wk) * own_max + slot) * 16 + g) * TOK + 2 * c;
          const uint32_t to = map_to(smem_u32(dst), owner);
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
    tell(done);
    {
      // Row block lr of the tile belongs to CTA lr mod cs; 16 lanes take its rows, for four tokens.
      const int n_own = (nr - rank + cs - 1) >> p.cs_log, parts = cs << p.kw_log;
      const int plane = own_max * 16 * TOK;
      const int r = lane & 15;
      auto locate = [&](int i, int& slot, int& n, size_t& off) {
        slot = i / (TOK / 4), n = (i % (TOK / 4)) * 4;  // TOK is a power of two
        const int row = (r0 + (slot << p.cs_log) + rank) * 16 + r;
        off = (size_t)n * p.N + row;
        return i < n_own * (TOK / 4) && n < ntok && row < p.N;
      };
      auto load_residual = [&](int i, T (&res)[4]) {
        int slot, n;
        size_t off;
        const bool in = locate(i, slot, n, off) && p.residual;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (in && n + e < ntok) res[e] = static_cast<const T*>(p.residual)[off + (size_t)e * p.N];
      };
      const int i0 = warp * 2 + (lane >> 4);
      T res[4] = {};
      // Arrives during the wait. (Two tiles of tokens have no registers to spare for it: 26.3 instead of 26.0 us
      // for 16 tokens on 28672 x 4096. One: 5.65 instead of 5.8 for one token on 4096 x 4096.)
      if (NT == 1) load_residual(i0, res);
      if (ok) ok = wait_cluster(done, tile_phase, p.err);
      for (int i = i0; i < n_own * (TOK / 4); i += W * 2) {
        int slot, n;
        size_t off;
        if (NT > 1 || i > i0) load_residual(i, res);
        if (!locate(i, slot, n, off)) continue;
        const float* from = part_buf + (slot * 16 + r) * TOK + n;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int q = 0; q < parts; ++q) {
          const float4 f = *reinterpret_cast<const float4*>(from + q * plane);
          v.x += f.x, v.y += f.y, v.z += f.z, v.w += f.w;
        }
        const float out[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < ntok)
            static_cast<T*>(p.y)[off + (size_t)e * p.N] =
                H::round(p.residual ? out[e] + H::to_float(res[e]) : out[e]);
      }
    }
    if (r0 + p.tile < rb1) tell(taken);  // the next tile's partial sums overwrite these
  }
  if (__any_sync(0xffffffffu, !ok)) linger(p.err);
}

static int g_withhold = -1;  // fk_debug_w4_withhold_slab

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
      cfg.blockDim = dim3(kWarps * 32 + 32, 1, 1);
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
  constexpr int kBudget = kSmem - ring_bytes<GROUP>();  // for x and the partial sums
  constexpr int kX = x_bytes<NT, GROUP>();
  static_assert(kX + 8 * part_bytes<NT>() <= kBudget, "a slab of x and one owned row block must fit");
  int resident[4];
  int rc = resident_clusters<T, NT, GROUP>(resident);
  if (rc) return rc;
  // Four CTAs per cluster where there are slabs for them: measured best or within 2 % of it from one
  // token on 4096 rows to 16 on 28672. Two or one leave too many slabs of x to every CTA, eight
  // leave SMs idle (15 clusters of 8, 36 of 4 are resident on 148 SMs).
  p.cs_log = p.nslab >= 4 ? 2 : p.nslab >= 2 ? 1 : 0;
  const int cs = 1 << p.cs_log;
  const int ncl = resident[p.cs_log] > p.nrb ? p.nrb : resident[p.cs_log];
  const int rows = (p.nrb + ncl - 1) / ncl, slabs = (p.nslab + cs - 1) / cs;
  // Few rows per cluster: two warps share a row block. Each part costs a plane of partial sums.
  p.kw_log = 2 * rows <= kWarps ? 1 : 0;
  const int own_bytes = part_bytes<NT>() * cs << p.kw_log;  // one owned row block
  // All partial sums at once if they leave room for a slab of x, which takes the rest.
  int own = (rows + cs - 1) / cs;
  if ((long long)own * own_bytes > kBudget - kX) own = (kBudget - kX) / own_bytes;
  p.chunk = (kBudget - own * own_bytes) / kX;
  if (p.chunk > slabs) p.chunk = slabs;
  const int rounds = (rows + own * cs - 1) / (own * cs);  // of equal size
  p.tile = (rows + rounds - 1) / rounds;
  own = (p.tile + cs - 1) / cs;
  const int smem = ring_bytes<GROUP>() + p.chunk * kX + own * own_bytes;
  p.rb_each = p.nrb / ncl;
  p.rb_more = p.nrb % ncl;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1 << p.cs_log;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ncl << p.cs_log), 1, 1);
  cfg.blockDim = dim3(kWarps * 32 + 32, 1, 1);
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

template <typename T>
static int by_tokens(const Params& p, int group, cudaStream_t st) {
  return p.M <= 8 ? by_group<T, 1>(p, group, st) : by_group<T, 2>(p, group, st);
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
  const long long y_bytes = 2LL * M * N, block = 1024 + 128 / group_size * 64;
  FK_CHECK_ARG(!bytes_meet(y, y_bytes, x, 2 * ((M - 1) * ldx + K)) &&
                   !bytes_meet(y, y_bytes, packed, (N + 15) / 16 * ((K + 127LL) / 128) * block),
               "y must not overlap x or the weight");
  FK_CHECK_ARG(!residual || residual == y || !bytes_meet(y, y_bytes, residual, y_bytes),
               "residual must be y or other memory");
  int* err = device_error_word();
  if (!err) return fail(kErrCuda, "device error word unavailable");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // The form of w4_tc.cu for more than 16 tokens; for 9 to 16 where its tiles of 128 rows are one wave on the SMs, or
  // so many that this form, which goes through its rows in rounds, is slower than its part-filled last wave.
  // For 16 tokens of 4096 inputs it took, against the form of this file, in us with groups of 128 / 64 / 32 and
  // weights that do not lie in L2:
  //   16384 rows (0.9 tiles per SM)  15.4 : 17.1   16.9 : 18.5   18.0 : 21.6
  //   33024 (1.7)                    30.6 : 28.8   33.4 : 31.4   35.6 : 37.9
  //   37888 (2.0)                    31.4 : 32.6   34.1 : 35.5   36.5 : 47.1
  //   40960 (2.2)                    43.9 : 34.4   48.0 : 37.8   51.3 : 49.6
  //   49152 (2.6)                    45.2 : 44.3   49.5 : 48.2   52.9 : 66.9
  //   53248 (2.8)                    45.9 : 47.9   50.0 : 62.4   53.5 : 85.1
  //   57344 (3.0)                    58.0 : 60.7   63.6 : 75.5   68.2 : 87.3
  // (fp16, groups of 128: 31.9 : 30.0 at 2.0, 45.8 : 41.3 at 2.6, 46.7 : 44.6 at 2.8, 59.9 : 69.6 at 3.2.) For 8 tokens,
  // where this form does half the products: 7.0 : 6.1 on 4096 x 4096, 13.2 : 14.1 on 4096 x 14336, 27.1 : 19.0 on
  // 28672 x 4096.
  const int tiles = (N + 127) / 128, sms = num_sms();
  if (M > 16 || (M > 8 && (tiles <= sms || 5 * tiles > (group_size == 32 ? 8 : 13) * sms))) {
    const w4::Call c{x, ldx, static_cast<const uint8_t*>(packed), residual, y, err, dtype == FK_BF16, M, N, K, group_size,
                    w4::g_withhold};
    return w4::linear_tc(c, st);
  }
  w4::Params p = {};
  p.x = x;
  p.ldx = ldx;
  p.packed = static_cast<const uint8_t*>(packed);
  p.err = err;
  p.residual = residual;
  p.y = y;
  p.M = M;
  p.N = N;
  p.K = K;
  p.nrb = (N + 15) / 16;
  p.nkb = (K + w4::kBlockK - 1) / w4::kBlockK;
  p.nslab = (p.nkb + w4::kSlab - 1) / w4::kSlab;
  p.withhold = w4::g_withhold;
  if (dtype == FK_BF16) return w4::by_tokens<__nv_bfloat16>(p, group_size, st);
  return w4::by_tokens<__half>(p, group_size, st);
}

extern "C" int fk_debug_w4_withhold_slab(int slab) {
  w4::g_withhold = slab < 0 ? -1 : slab;
  return kOk;
}
