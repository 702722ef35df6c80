// Attention of one new token per sequence over a contiguous or paged KV cache,
// optionally adding every cached token's attention weight to its running mass
// (what cache_evict.cu selects by).
//
//   s_j = scale * q . k_j,  w_j = exp(s_j - lse),  lse = log sum_{j < len} exp(s_j)
//   out = sum_j w_j v_j,    mass_out[j] = mass[j] + sum over the group's q heads of w_j
//
// Bound: HBM, 4 * D bytes per (token, kv head), plus 8 bytes of mass and the
// scores' round trip described below.
//
// Pass 1 (`attend_kernel`): units (row b, kv head h, split of `chunk` tokens) are
// dealt round-robin to the warps of a persistent grid. A warp works alone: it
// streams its 16-token tiles through a private ring filled by its own 16-byte
// cp.async copies and writes its unit's partial itself, so there is no barrier
// in the kernel (a merge of four warps per unit, tried first, drained the loads
// for 1.5 us per unit). Each token's address comes from its own page: pages may
// have any size. The load side runs STAGES - 1 tiles ahead of the arithmetic,
// across units. Tokens are the M side of mma.sync m16n8k16 and the group's query
// heads the N side (NT tiles of 8), so a K/V byte is read once for all heads that
// share it. Running maximum and sum are fp32, in the log2 domain. P is multiplied as
// a sum of two 16-bit numbers (its rounding and the rounding of the rest): the products
// cost nothing next to the loads, and the output's error is then that of its own
// rounding instead of sqrt(2) times it. For fp16, whose least number is 2^-24, P is scaled by
// 2^15: weights are held to 2^-40 of the greatest of their unit, not to 2^-25 (behind a
// token that takes nearly all the weight, the others would vanish). With a mass, the raw log2-domain scores go
// to scratch as fp32 (4 bytes per token and q head), because a token's weight is
// known only with the lse of the whole row.
//
// Pass 2 (`finish_kernel`, a programmatic dependent): blocks that merge the
// splits of each (row, q head) into out and lse, and blocks that turn a stretch
// of scores into weights and add them to the mass.
//
// Measured, 8 kv heads of 128 dims, 4 q heads each, caches from memory: 64 ragged rows of up to 32768 tokens
// (4.5 GB) 683 to 690 us without masses, a plain copy's rate, and 767 to 777 with them, 84 of them in pass 2.
// Small calls are two launches and a join: 7.5 us for one row of 1000 tokens, 18 for four of 4096 (pass
// 1 12, pass 2 5).
//
// A row of length 0 gives out = 0, lse = -inf and leaves its mass. A page id
// outside the pool reads as zero rows, as a TMA load outside its tensor does.
#include <cuda_fp16.h>
#include <math.h>

#include <mutex>

#include "common.cuh"
#include "fk_b200.h"

namespace fk {
namespace cattn {

constexpr int T = 16;   // tokens per tile
constexpr int NW = 4;   // warps per CTA
constexpr int kThreads = NW * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

struct Params {
  const void* q;            // row b at q + b * q_stride: [Hq, D]
  long long q_stride;
  const void* k;            // [B, Lmax, Hkv, D] or [num_blocks, block_size, Hkv, D]
  const void* v;
  const int* block_table;   // [B, max_blocks] or null
  int max_blocks, block_size, num_blocks;
  FastDiv page;             // by block_size
  const int* seqlens;
  float* o_part;            // [S, B, Hq, D], normalised per split
  float* lse_part;          // [S, B, Hq], log2 domain
  float* scores;            // [B * Hkv, Lmax, gs] log2-domain scores, or null
  int gs;                   // floats per token in scores
  const float* mass_in;     // [B, Hkv, mass_cap]
  float* mass_out;
  long long mass_cap;
  void* out;                // [B, Hq, D]
  float* lse;               // [B, Hq]
  int B, Lmax, Hq, Hkv, G;
  FastDiv chunk;            // tokens per split, a multiple of 16
  float scale_log2;
};

template <typename E>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr float kShift = 0.f;  // P is 2^kShift times exp2(score - maximum)
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
  static __device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16_16816(d, a, b0, b1);
  }
};
template <>
struct Elem<__half> {
  static constexpr float kShift = 15.f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ float lo(uint32_t v) {
    return __half2float(__ushort_as_half((unsigned short)(v & 0xFFFFu)));
  }
  static __device__ __forceinline__ float hi(uint32_t v) {
    return __half2float(__ushort_as_half((unsigned short)(v >> 16)));
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_f16_16816(d, a, b0, b1);
  }
};

// Both kernels are resident while kernels before them still write what they read: lengths, q, tables and caches, and
// in pass 2 the partial results and scores. So nothing is read through the read-only path (__ldg): such
// loads may be moved ahead of the wait.
__device__ __forceinline__ int seq_len(const Params& p, int b) {
  const int L = p.seqlens[b];
  return min(max(L, 0), p.Lmax);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // 0: the 16 bytes are zero-filled and src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Transposes an 8x8 matrix of 16-bit values held one 2-value row piece per lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ int num_splits(const Params& p, int len) { return p.chunk.div(len + p.chunk.d - 1); }

// The tiles a warp works on, in order: units (b, h, split) dealt round-robin over the
// grid's warps, and the 16-token tiles of each.
struct TileIter {
  long long u, base;  // current unit, first unit of row b
  int b, nb, len;     // row, its splits and length
  int h, s;           // kv head and split of the unit
  int t, t1;          // current tile's first token, end of the unit
  bool valid;
  __device__ __forceinline__ void row(const Params& p) {
    len = seq_len(p, b);
    nb = num_splits(p, len);
  }
  __device__ __forceinline__ void locate(const Params& p) {
    while (true) {
      const long long cnt = (long long)nb * p.Hkv;
      if (u < base + cnt) break;
      base += cnt;
      if (++b >= p.B) {
        valid = false;
        return;
      }
      row(p);
    }
    const int r = (int)(u - base);
    h = r / nb;
    s = r - h * nb;
    t = s * p.chunk.d;
    t1 = min(t + p.chunk.d, len);
  }
  __device__ __forceinline__ void init(const Params& p) {
    u = (long long)blockIdx.x * NW + (threadIdx.x >> 5);
    base = 0;
    b = 0;
    valid = true;
    row(p);
    locate(p);
  }
  __device__ __forceinline__ void next(const Params& p) {
    t += T;
    if (t >= t1) {
      u += (long long)gridDim.x * NW;
      locate(p);
    }
  }
};

template <int D>
__host__ __device__ constexpr int stage_bytes() { return 2 * 16 * D * 2; }  // one warp's K and V of 16 tokens
// Stages of a warp's ring: 96 KB per CTA, two CTAs per SM. At D = 64 more warps with fewer stages
// (4 CTAs of 3, 3 of 4) measured 5-10 % slower on a large batch than 2 of 6.
template <int D>
__host__ __device__ constexpr int stages() { return D == 128 ? 3 : 6; }
constexpr int kCtas = 2;
template <int D>
__host__ __device__ constexpr int attend_smem() { return NW * stages<D>() * stage_bytes<D>(); }

template <typename E, int D, int NT, bool MASS>
__global__ void __launch_bounds__(kThreads, kCtas) attend_kernel(const Params p) {
  using El = Elem<E>;
  constexpr int S = stages<D>();
  constexpr int KS = D / 16;
  constexpr int LPR = D / 8;      // lanes (16-byte pieces) per token row
  constexpr int RPI = 32 / LPR;   // rows per copy instruction
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int j = lane >> 3, r = lane & 7;
  const float NEG_INF = -INFINITY;
  const int G = p.G;
  const uint32_t ring = smem_u32(smem) + warp * S * stage_bytes<D>();

  asm volatile("griddepcontrol.wait;" ::: "memory");
  // After the wait: the second kernel reads lengths and masses, which kernels before this one wrote, before its own.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  TileIter ld, it;
  ld.init(p);
  it = ld;

  // Lanes 0..15 resolve the cache row of "their" token of the next tile to load
  // one tile ahead, so the page lookup's latency is off the copies' path.
  auto resolve = [&]() -> int {
    if (!ld.valid) return -1;
    const int t = ld.t + (lane & 15);
    if (t >= ld.t1) return -1;
    if (p.block_table == nullptr) return ld.b * p.Lmax + t;
    const int pg = p.page.div(t);
    const int page = p.block_table[(size_t)ld.b * p.max_blocks + pg];
    if (page < 0 || page >= p.num_blocks) return -1;
    return page * p.block_size + (t - pg * p.block_size);
  };
  int next_row = resolve();
  int ld_stage = 0;
  auto issue = [&]() {
    if (ld.valid) {
      const int row = next_row, h = ld.h;
      ld.next(p);
      next_row = resolve();
      const uint32_t kd = ring + ld_stage * stage_bytes<D>();
      const uint32_t vd = kd + 16 * D * 2;
      const int piece = lane % LPR;
      const uint32_t half_off = (piece >> 3) * (16 * 128);
#pragma unroll
      for (int i = 0; i < 16 / RPI; ++i) {
        const int tok = i * RPI + lane / LPR;
        const int rr = __shfl_sync(0xffffffffu, row, tok);
        const size_t off = ((size_t)max(rr, 0) * p.Hkv + h) * D + piece * 8;
        const uint32_t so = half_off + tok * 128 + (((piece ^ tok) & 7) << 4);
        cp_async16(kd + so, static_cast<const E*>(p.k) + off, rr >= 0);
        cp_async16(vd + so, static_cast<const E*>(p.v) + off, rr >= 0);
      }
      if (++ld_stage == S) ld_stage = 0;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) issue();

  int stage = 0;
  while (it.valid) {
    const int b = it.b, h = it.h, t1 = it.t1, split = it.s;
    // Q^T as the B operand: column n = query head of the group (zero past the group).
    uint32_t qf[NT][KS][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int hh = nt * 8 + g;
      const E* qrow = static_cast<const E*>(p.q) + (size_t)b * p.q_stride + ((size_t)h * G + hh) * D;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qf[nt][ks][0] = hh < G ? *reinterpret_cast<const uint32_t*>(qrow + 16 * ks + 2 * c) : 0u;
        qf[nt][ks][1] = hh < G ? *reinterpret_cast<const uint32_t*>(qrow + 16 * ks + 8 + 2 * c) : 0u;
      }
    }
    float o[NT][KS][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = NEG_INF;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }

    bool last;
    do {
      const int t = it.t;
      cp_async_wait<S - 2>();
      __syncwarp();  // every lane's copies of this stage are in, and the stage refilled below is free
      issue();
      const uint32_t kb = ring + stage * stage_bytes<D>();
      const uint32_t vb = kb + 16 * D * 2;
      if (++stage == S) stage = 0;

      // S^T[16 tokens x 8 heads] = K[16 x D] . Q^T[D x 8]
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int tok = (j & 1) * 8 + r;
        const int cc = 2 * (ks & 3) + (j >> 1);
        uint32_t a[4];
        ldsm_x4(kb + (ks >> 2) * (16 * 128) + tok * 128 + (((cc ^ tok) & 7) << 4), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) El::mma(sc[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
      }

      const int nv = t1 - t;  // valid tokens among the 16
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float x0 = sc[nt][0] * p.scale_log2, x1 = sc[nt][1] * p.scale_log2;
        const float x2 = sc[nt][2] * p.scale_log2, x3 = sc[nt][3] * p.scale_log2;
        if (MASS) {
          const int h0 = nt * 8 + 2 * c;
          float* dst = p.scores + (((size_t)b * p.Hkv + h) * p.Lmax + (t + g)) * p.gs + h0;
          if (p.gs > 1) {  // gs is even: a pair of heads per store
            if (h0 < p.gs) {
              if (g < nv) *reinterpret_cast<float2*>(dst) = make_float2(x0, x1);
              if (g + 8 < nv) *reinterpret_cast<float2*>(dst + 8 * (size_t)p.gs) = make_float2(x2, x3);
            }
          } else if (h0 == 0) {
            if (g < nv) dst[0] = x0;
            if (g + 8 < nv) dst[8] = x2;
          }
        }
        const float y0 = g < nv ? x0 : NEG_INF, y1 = g < nv ? x1 : NEG_INF;
        const float y2 = g + 8 < nv ? x2 : NEG_INF, y3 = g + 8 < nv ? x3 : NEG_INF;
        float mx0 = fmaxf(y0, y2), mx1 = fmaxf(y1, y3);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
        }
        const float mn0 = fmaxf(m[nt][0], mx0), mn1 = fmaxf(m[nt][1], mx1);
        const float sf0 = mn0 == NEG_INF ? 0.f : mn0;  // nothing but -inf so far
        const float sf1 = mn1 == NEG_INF ? 0.f : mn1;
        const float al0 = exp2f(m[nt][0] - sf0), al1 = exp2f(m[nt][1] - sf1);
        const float pf0 = sf0 - El::kShift, pf1 = sf1 - El::kShift;
        const float p0 = exp2f(y0 - pf0), p1 = exp2f(y1 - pf1);
        const float p2 = exp2f(y2 - pf0), p3 = exp2f(y3 - pf1);
        l[nt][0] = l[nt][0] * al0 + (p0 + p2);
        l[nt][1] = l[nt][1] * al1 + (p1 + p3);
        m[nt][0] = mn0;
        m[nt][1] = mn1;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          o[nt][i][0] *= al0;
          o[nt][i][1] *= al1;
          o[nt][i][2] *= al0;
          o[nt][i][3] *= al1;
        }
        // P^T (rows = tokens) as the B operand (rows = tokens as k): two 8x8 transposes
        // each for the rounded P and for what the rounding left.
        const uint32_t h01 = El::pack(p0, p1), h23 = El::pack(p2, p3);
        ph[nt][0] = transpose8x8(h01);
        ph[nt][1] = transpose8x8(h23);
        pl[nt][0] = transpose8x8(El::pack(p0 - El::lo(h01), p1 - El::hi(h01)));
        pl[nt][1] = transpose8x8(El::pack(p2 - El::lo(h23), p3 - El::hi(h23)));
      }

      // O^T[D x 8 heads] += V^T[D x 16 tokens] . P^T[16 x 8]; rows past the end are zero-filled.
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int tok = (j >> 1) * 8 + r;
        const int cc = 2 * (i & 3) + (j & 1);
        uint32_t a[4];
        ldsm_x4_t(vb + (i >> 2) * (16 * 128) + tok * 128 + (((cc ^ tok) & 7) << 4), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          El::mma(o[nt][i], a, ph[nt][0], ph[nt][1]);
          El::mma(o[nt][i], a, pl[nt][0], pl[nt][1]);
        }
      }
      last = t + T >= t1;
      it.next(p);
    } while (!last);

    // ---- the unit's partial: O normalised, and its lse. A sum of exactly 0 means that every
    // score was -inf; NaN scores give a NaN sum and go on to the output. ----
    const size_t row0 = ((size_t)split * p.B + b) * p.Hq + (size_t)h * G;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[nt][0] += __shfl_xor_sync(0xffffffffu, l[nt][0], off);
        l[nt][1] += __shfl_xor_sync(0xffffffffu, l[nt][1], off);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int hh = nt * 8 + 2 * c + e;
        if (hh >= G) continue;
        const float L = l[nt][e];
        const float inv = L == 0.f ? 0.f : 1.f / L;
        float* dst = p.o_part + (row0 + hh) * D + g;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          dst[16 * i] = o[nt][i][e] * inv;
          dst[16 * i + 8] = o[nt][i][e + 2] * inv;
        }
        if (g == 0) p.lse_part[row0 + hh] = L == 0.f ? NEG_INF : m[nt][e] + (log2f(L) - El::kShift);
      }
    }
  }
  cp_async_wait<0>();
}

// Scores h0 .. h0 + 3 of one token (gs of them, 1 or an even number); 0 past the end.
__device__ __forceinline__ float4 load_scores(const float* sc, int h0, int gs) {
  if ((gs & 3) == 0) return *reinterpret_cast<const float4*>(sc + h0);
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  if (gs == 1) {
    f.x = *sc;
  } else {
    const float2 a = *reinterpret_cast<const float2*>(sc + h0);
    f.x = a.x, f.y = a.y;
    if (h0 + 2 < gs) {
      const float2 c = *reinterpret_cast<const float2*>(sc + h0 + 2);
      f.z = c.x, f.w = c.y;
    }
  }
  return f;
}

constexpr int kFinishThreads = 256;
constexpr int kMassUnroll = 4;                                // tokens of a thread whose loads are in flight together
constexpr int kMassTokens = kFinishThreads * kMassUnroll;     // tokens per mass block

// One (row, q head)'s lse in the log2 domain from the splits'. Whole warps.
__device__ __forceinline__ float merge_lse(const float* src, size_t plane, int n, int lane) {
  float M = -INFINITY, W = 0.f;
  for (int s0 = 0; s0 < n; s0 += 128) {
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + u * 32 + lane;
      x[u] = s < n ? src[s * plane] : -INFINITY;
    }
    // fmaxf passes over NaN, the sum does not.
    const float top = fmaxf(fmaxf(M, fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
    const float ts = top == -INFINITY ? 0.f : top;
    W = W * exp2f(M - ts) + ((exp2f(x[0] - ts) + exp2f(x[1] - ts)) + (exp2f(x[2] - ts) + exp2f(x[3] - ts)));
    M = top;
  }
  float top = M;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  const float ts = top == -INFINITY ? 0.f : top;
  W *= exp2f((M == -INFINITY ? ts : M) - ts);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) W += __shfl_xor_sync(0xffffffffu, W, off);
  return W == 0.f ? -INFINITY : top + log2f(W);
}

// One (row, q head)'s output once more, with each weight as one fp32 number in the splits whose partial is NaN
// although its lse is not. Two 16-bit parts of a weight (`attend_kernel`) are right for every finite v,
// but not for an infinite one: a second part of 0 or below makes NaN of it. Only an output that is NaN
// although its lse is not comes here. A warp, D / 32 dims per lane, one token at a time (0.2 ms per split); n splits, lse of
// the row in the log2 domain.
template <typename E, int D>
__device__ __noinline__ float4 attend_again(const Params& p, int row, int b, int n, int len, float lse) {
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31, head = row - b * p.Hq, h = head / p.G;
  const size_t plane = (size_t)p.B * p.Hq;
  const float z = lse == -INFINITY ? 0.f : lse;
  auto load = [](const void* base, size_t off, float (&f)[PER]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(static_cast<const E*>(base) + off);
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) f[2 * i] = Elem<E>::lo(w[i]), f[2 * i + 1] = Elem<E>::hi(w[i]);
  };
  float qv[PER], acc[4] = {};
  load(p.q, (size_t)b * p.q_stride + (size_t)head * D + PER * lane, qv);
  for (int split = 0; split < n; ++split) {
    const float part_lse = p.lse_part[split * plane + row];
    const float* part = p.o_part + (split * plane + row) * D + PER * lane;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += part[i];
    if (part_lse != part_lse || !__any_sync(0xffffffffu, sum != sum)) {
      const float w = exp2f(part_lse - z);
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] += w * part[i];
      continue;
    }
    for (int t = split * p.chunk.d; t < min((split + 1) * p.chunk.d, len); ++t) {
      long long at = (long long)b * p.Lmax + t;
      if (p.block_table) {
        const int pg = p.page.div(t), page = p.block_table[(size_t)b * p.max_blocks + pg];
        if (page < 0 || page >= p.num_blocks) continue;  // zero rows
        at = (long long)page * p.block_size + (t - pg * p.block_size);
      }
      const size_t off = ((size_t)at * p.Hkv + h) * D + PER * lane;
      float kv[PER], vv[PER], s = 0.f;
      load(p.k, off, kv);
      load(p.v, off, vv);
#pragma unroll
      for (int i = 0; i < PER; ++i) s += qv[i] * kv[i];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      const float w = exp2f(s * p.scale_log2 - z);
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] += w * vv[i];
    }
  }
  return make_float4(acc[0], acc[1], acc[2], acc[3]);
}

// Blocks [0, merge_blocks) merge splits: 8 >> wpr_log (row, q head) pairs each, with
// 1 << wpr_log warps per pair. The others: one stretch of kMassTokens tokens of one (row,
// kv head). Both read what pass 1 left, mostly in L2, and are short: what matters is that
// a thread's loads are issued before the first is used.
template <typename E, int D>
__global__ void __launch_bounds__(kFinishThreads) finish_kernel(const __grid_constant__ Params p, int merge_blocks, int wpr_log,
                                                                FastDiv stretches, FastDiv heads_q, FastDiv heads_kv) {
  // What the first kernel wrote (partial results, scores) is read behind this wait only.
  auto wait_first = [] { asm volatile("griddepcontrol.wait;" ::: "memory"); };
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int kWarps = kFinishThreads / 32;
  __shared__ float s_acc[kWarps][D];
  __shared__ float s_lse[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t plane = (size_t)p.B * p.Hq;
  if ((int)blockIdx.x < merge_blocks) {
    const int wpr = 1 << wpr_log, part = warp & (wpr - 1);
    const int row = blockIdx.x * (kWarps >> wpr_log) + (warp >> wpr_log);
    const bool in_range = row < p.B * p.Hq;
    constexpr int PER = D / 32;  // dims per lane
    constexpr int CH = 8;        // splits whose loads are in flight together
    float acc[PER], lse = -INFINITY;
    int len = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
    if (in_range) {
      len = seq_len(p, heads_q.div(row));
      const int n = num_splits(p, len);
      wait_first();
      float ls[CH], v[CH][PER];
      // Splits part, part + wpr, ..: each warp's in order, then the warps' in order.
      auto load = [&](int s0) {
#pragma unroll
        for (int u = 0; u < CH; ++u) {
          const int s = s0 + u * wpr;
          const bool in = s < n;
          ls[u] = in ? p.lse_part[s * plane + row] : -INFINITY;
          const float* src = p.o_part + (s * plane + row) * D + PER * lane;
          if constexpr (PER == 4) {
            const float4 f = in ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[u][0] = f.x, v[u][1] = f.y, v[u][2] = f.z, v[u][3] = f.w;
          } else {
            const float2 f = in ? *reinterpret_cast<const float2*>(src) : make_float2(0.f, 0.f);
            v[u][0] = f.x, v[u][1] = f.y;
          }
        }
      };
      load(part);
      lse = merge_lse(p.lse_part + row, plane, n, lane);
      // The weights add up to 1: split s has exp2(lse_s - lse).
      const float z = lse == -INFINITY ? 0.f : lse;
      for (int s0 = part; s0 < n; s0 += CH * wpr) {
        if (s0 > part) load(s0);
#pragma unroll
        for (int u = 0; u < CH; ++u) {
          if (s0 + u * wpr < n) {
            const float w = exp2f(ls[u] - z);
#pragma unroll
            for (int i = 0; i < PER; ++i) acc[i] += w * v[u][i];
          }
        }
      }
    }
    if (wpr > 1) {
#pragma unroll
      for (int i = 0; i < PER; ++i) s_acc[warp][PER * lane + i] = acc[i];
      __syncthreads();
      if (part != 0 || !in_range) return;
      for (int w = 1; w < wpr; ++w) {
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] += s_acc[warp + w][PER * lane + i];
      }
    }
    if (!in_range) return;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += acc[i];
    if (__any_sync(0xffffffffu, sum != sum) && lse == lse) {
      const float4 f = attend_again<E, D>(p, row, heads_q.div(row), num_splits(p, len), len, lse);
      acc[0] = f.x, acc[1] = f.y;
      if constexpr (PER == 4) acc[2] = f.z, acc[3] = f.w;
    }
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<E*>(p.out) + (size_t)row * D + PER * lane);
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) dst[i] = Elem<E>::pack(acc[2 * i], acc[2 * i + 1]);
    if (lane == 0) p.lse[row] = lse * kLn2;
    return;
  }

  const int i = blockIdx.x - merge_blocks;
  const int pair = stretches.div(i);
  const int t0 = (i - pair * stretches.d) * kMassTokens;
  const int b = heads_kv.div(pair), h = pair - b * p.Hkv;
  const int len = seq_len(p, b);
  if (t0 >= len) return;
  const int n = num_splits(p, len);
  const float* sc = p.scores + (size_t)pair * p.Lmax * p.gs;
  const size_t mrow = (size_t)pair * p.mass_cap;
  const int t1 = min(t0 + kMassTokens, len);
  float mass[kMassUnroll], w[kMassUnroll];
#pragma unroll
  for (int u = 0; u < kMassUnroll; ++u) {
    const int t = t0 + u * kFinishThreads + (int)threadIdx.x;
    mass[u] = t < t1 ? p.mass_in[mrow + t] : 0.f;
    w[u] = 0.f;
  }
  wait_first();
  float4 first[kMassUnroll];  // scores of the first four heads, or of the only one or two
#pragma unroll
  for (int u = 0; u < kMassUnroll; ++u) {
    const int t = t0 + u * kFinishThreads + (int)threadIdx.x;
    first[u] = t < t1 ? load_scores(sc + (size_t)t * p.gs, 0, p.gs) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int hh = warp; hh < p.G; hh += kWarps) {
    const float z = merge_lse(p.lse_part + (size_t)b * p.Hq + (size_t)h * p.G + hh, plane, n, lane);
    // A head whose scores are all -inf gives no weight: +inf makes exp2(-inf - inf) = 0.
    if (lane == 0) s_lse[hh] = z == -INFINITY ? INFINITY : z;
  }
  __syncthreads();
  for (int h0 = 0; h0 < p.G; h0 += 4) {
    float z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = h0 + e < p.G ? s_lse[h0 + e] : INFINITY;
#pragma unroll
    for (int u = 0; u < kMassUnroll; ++u) {
      const int t = t0 + u * kFinishThreads + (int)threadIdx.x;
      float4 x = h0 == 0 ? first[u]
                 : t < t1 ? load_scores(sc + (size_t)t * p.gs, h0, p.gs) : make_float4(0.f, 0.f, 0.f, 0.f);
      // Heads past the group: 0, and z = +inf. An odd group's scores have one head of padding, at an odd place.
      // Its q is 0, but 0 times an infinite key is NaN.
      if (h0 + 1 >= p.G) x.y = 0.f;
      if (h0 + 3 >= p.G) x.w = 0.f;
      w[u] += (exp2f(x.x - z[0]) + exp2f(x.y - z[1])) + (exp2f(x.z - z[2]) + exp2f(x.w - z[3]));
    }
  }
#pragma unroll
  for (int u = 0; u < kMassUnroll; ++u) {
    const int t = t0 + u * kFinishThreads + (int)threadIdx.x;
    if (t < t1) p.mass_out[mrow + t] = mass[u] + w[u];
  }
}

// Tokens per split. One unit per warp of the grid where the padded batch is that small,
// but at least kMinChunk tokens, so that a unit's partial (G * D fp32) stays small next to
// its K and V; at most kMaxChunk, which gives a large batch units enough to even out.
constexpr int kMinChunk = 32;
constexpr int kMaxChunk = 256;
static int chunk_tokens(int B, int Hkv, int Lmax, int warps) {
  const long long total = (long long)B * Lmax * Hkv;
  long long c = (total + warps - 1) / warps;
  c = (c + T - 1) / T * T;
  if (c < kMinChunk) c = kMinChunk;
  return (int)(c > kMaxChunk ? kMaxChunk : c);
}

static int score_stride(int G) { return G == 1 ? 1 : (G + 1) & ~1; }

struct Layout {
  int chunk, splits;
  size_t o_bytes, lse_bytes, score_bytes;
  size_t total() const { return o_bytes + lse_bytes + score_bytes; }
};

static size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

static Layout layout(int B, int Lmax, int Hq, int Hkv, int D, bool mass) {
  Layout w;
  w.chunk = chunk_tokens(B, Hkv, Lmax, num_sms() * kCtas * NW);
  w.splits = (Lmax + w.chunk - 1) / w.chunk;
  const size_t rows = (size_t)w.splits * B * Hq;
  w.o_bytes = round256(rows * D * 4);
  w.lse_bytes = round256(rows * 4);
  w.score_bytes = mass ? round256((size_t)B * Hkv * Lmax * score_stride(Hq / Hkv) * 4) : 0;
  return w;
}

// CTAs per SM, asked once per kernel and device.
template <typename E, int D, int NT, bool MASS>
static int occupancy(int* out) {
  constexpr int kDevices = 64;
  static std::mutex mu;
  static int known[kDevices] = {};
  int dev = 0;
  FK_CHECK_CUDA(cudaGetDevice(&dev));
  FK_CHECK_ARG(dev >= 0 && dev < kDevices, "device index too large");
  std::lock_guard<std::mutex> lock(mu);
  if (known[dev] == 0) {
    auto kern = attend_kernel<E, D, NT, MASS>;
    FK_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, attend_smem<D>()));
    int occ = 0;
    FK_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, kThreads, attend_smem<D>()));
    known[dev] = occ < 1 ? 1 : occ;
  }
  *out = known[dev];
  return kOk;
}

template <typename E, int D, int NT, bool MASS>
static int launch_attend(const Params& p, cudaStream_t st) {
  int occ = 0;
  int rc = occupancy<E, D, NT, MASS>(&occ);
  if (rc) return rc;
  long long grid = (long long)num_sms() * occ;
  const int splits = (p.Lmax + p.chunk.d - 1) / p.chunk.d;
  const long long units = (long long)p.B * p.Hkv * splits;
  if (grid > (units + NW - 1) / NW) grid = (units + NW - 1) / NW;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = attend_smem<D>();
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attend_kernel<E, D, NT, MASS>, p));
  // One warp per (row, q head) takes 8 splits at a time; up to 8 warps share a longer row.
  int wpr_log = 0;
  while (wpr_log < 3 && (8 << wpr_log) < splits) ++wpr_log;
  const int rows = (kFinishThreads / 32) >> wpr_log;
  const int merge_blocks = (p.B * p.Hq + rows - 1) / rows;
  const int stretches = (p.Lmax + kMassTokens - 1) / kMassTokens;
  const long long blocks = merge_blocks + (MASS ? (long long)p.B * p.Hkv * stretches : 0);
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(kFinishThreads, 1, 1);
  cfg.dynamicSmemBytes = 0;
  FK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, finish_kernel<E, D>, p, merge_blocks, wpr_log, FastDiv::of(stretches),
                                   FastDiv::of(p.Hq), FastDiv::of(p.Hkv)));
  return kOk;
}

template <typename E, int D>
static int by_group(const Params& p, cudaStream_t st) {
  const bool mass = p.mass_out != nullptr;
  if (p.G <= 8) return mass ? launch_attend<E, D, 1, true>(p, st) : launch_attend<E, D, 1, false>(p, st);
  return mass ? launch_attend<E, D, 2, true>(p, st) : launch_attend<E, D, 2, false>(p, st);
}

static int check_sizes(int B, int Lmax, int Hq, int Hkv, int D) {
  FK_CHECK_ARG(B >= 1 && Lmax >= 1, "batch and max_seqlen must be >= 1");
  FK_CHECK_ARG(Lmax <= (1 << 30), "max_seqlen must be <= 2^30");
  FK_CHECK_ARG(D == 64 || D == 128, "head_dim must be 64 or 128");
  FK_CHECK_ARG(Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0, "num_heads_q must be a positive multiple of num_heads_kv");
  FK_CHECK_ARG(Hq / Hkv <= 16, "GQA group size (num_heads_q / num_heads_kv) must be <= 16");
  FK_CHECK_ARG((long long)B * Hq <= (1 << 24) && (long long)B * Lmax < (1LL << 31), "batch too large");
  const long long stretches = (Lmax + kMassTokens - 1) / kMassTokens;
  FK_CHECK_ARG((long long)B * Hkv * stretches < (1LL << 30), "batch * num_heads_kv * max_seqlen too large");
  return kOk;
}

}  // namespace cattn
}  // namespace fk

using namespace fk;

extern "C" int fk_cache_attn_workspace_bytes(int batch, int max_seqlen, int num_heads_q, int num_heads_kv,
                                             int head_dim, int with_mass, size_t* bytes_out) {
  FK_CHECK_ARG(bytes_out != nullptr, "bytes_out is null");
  int rc = cattn::check_sizes(batch, max_seqlen, num_heads_q, num_heads_kv, head_dim);
  if (rc) return rc;
  *bytes_out = cattn::layout(batch, max_seqlen, num_heads_q, num_heads_kv, head_dim, with_mass != 0).total();
  return kOk;
}

extern "C" int fk_cache_attn_fwd(const void* q, long long q_batch_stride, const void* k_cache, const void* v_cache,
                                 const int32_t* block_table, const int32_t* cache_seqlens, const float* mass_in,
                                 float* mass_out, long long mass_capacity, void* out, float* lse, int dtype,
                                 int batch, int max_seqlen, int block_size, int num_blocks, int num_heads_q,
                                 int num_heads_kv, int head_dim, float softmax_scale, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  FK_CHECK_ARG(q && k_cache && v_cache && cache_seqlens && out && lse && workspace, "null tensor pointer");
  FK_CHECK_ARG(dtype == FK_BF16 || dtype == FK_FP16, "dtype must be FK_BF16 or FK_FP16");
  int rc = cattn::check_sizes(batch, max_seqlen, num_heads_q, num_heads_kv, head_dim);
  if (rc) return rc;
  FK_CHECK_ARG(isfinite(softmax_scale), "softmax_scale must be finite");
  FK_CHECK_ARG(q_batch_stride >= (long long)num_heads_q * head_dim && q_batch_stride % 2 == 0,
               "q row stride must be even and >= num_heads_q * head_dim");
  FK_CHECK_ARG(((uintptr_t)q & 3) == 0 && ((uintptr_t)out & 3) == 0, "q and out must be 4-byte aligned");
  FK_CHECK_ARG(((uintptr_t)k_cache & 15) == 0 && ((uintptr_t)v_cache & 15) == 0 && ((uintptr_t)workspace & 15) == 0,
               "caches and workspace must be 16-byte aligned");
  FK_CHECK_ARG((mass_in == nullptr) == (mass_out == nullptr), "give both mass_in and mass_out, or neither");
  FK_CHECK_ARG(!mass_in || mass_capacity >= max_seqlen, "mass_capacity must be >= max_seqlen");
  FK_CHECK_ARG(!mass_in || mass_in == mass_out ||
                   !bytes_meet(mass_in, 4LL * batch * num_heads_kv * mass_capacity, mass_out,
                               4LL * batch * num_heads_kv * mass_capacity),
               "mass_out must be mass_in or other memory");
  if (block_table) {
    FK_CHECK_ARG(block_size >= 1 && num_blocks >= 1 && max_seqlen % block_size == 0,
                 "paged cache: max_seqlen must be max_blocks_per_seq * block_size, num_blocks >= 1");
    FK_CHECK_ARG((long long)num_blocks * block_size < (1LL << 31), "pool too large");
  }
  const cattn::Layout w = cattn::layout(batch, max_seqlen, num_heads_q, num_heads_kv, head_dim, mass_out != nullptr);
  FK_CHECK_ARG(workspace_bytes >= w.total(), "workspace too small");
  cattn::Params p = {};
  p.q = q;
  p.q_stride = q_batch_stride;
  p.k = k_cache;
  p.v = v_cache;
  p.block_table = block_table;
  p.block_size = block_table ? block_size : 1;
  p.page = FastDiv::of(p.block_size);
  p.max_blocks = block_table ? max_seqlen / block_size : 0;
  p.num_blocks = num_blocks;
  p.seqlens = cache_seqlens;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.o_part = reinterpret_cast<float*>(ws);
  p.lse_part = reinterpret_cast<float*>(ws + w.o_bytes);
  p.scores = mass_out ? reinterpret_cast<float*>(ws + w.o_bytes + w.lse_bytes) : nullptr;
  p.gs = cattn::score_stride(num_heads_q / num_heads_kv);
  p.mass_in = mass_in;
  p.mass_out = mass_out;
  p.mass_cap = mass_capacity;
  p.out = out;
  p.lse = lse;
  p.B = batch;
  p.Lmax = max_seqlen;
  p.Hq = num_heads_q;
  p.Hkv = num_heads_kv;
  p.G = num_heads_q / num_heads_kv;
  p.chunk = FastDiv::of(w.chunk);
  p.scale_log2 = softmax_scale * cattn::kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FK_BF16)
    return head_dim == 128 ? cattn::by_group<__nv_bfloat16, 128>(p, st) : cattn::by_group<__nv_bfloat16, 64>(p, st);
  return head_dim == 128 ? cattn::by_group<__half, 128>(p, st) : cattn::by_group<__half, 64>(p, st);
}
