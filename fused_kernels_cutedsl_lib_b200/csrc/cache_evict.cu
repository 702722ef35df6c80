// Eviction from a KV cache by accumulated attention weight.
//
// Per row b with len > budget and per kv head: of the tokens [0, len) the first
// `sinks`, the last `recent` and the budget - sinks - recent others of greatest
// mass stay (equal masses: the earlier token), in their order. Their K and V
// rows and masses are written to [0, budget) of the output cache, zeros to the
// masses behind, and the new length and old positions beside them. Rows of at
// most `budget` tokens are copied whole. The output cache is another one than
// the input cache, contiguous or paged, with pages of any size on either side.
//
// Bound: HBM. Every mass is read once (4 bytes), every kept token's K and V row
// is read and written once.
//
// `select_kernel`: a cluster of CL CTAs per (row, kv head) finds the threshold mass
// by radix selection. Floats map to order-preserving unsigned keys, kept in
// registers (each warp owns a contiguous stretch of the candidates). Starting from
// the interval [least key, greatest key], a pass counts the keys in 1024 equal
// parts of the interval and goes on with the part that holds the want-th greatest,
// until the part is one key or holds exactly the keys still wanted: at most four
// passes, two or three in practice. Starting from the keys' own range instead of
// their top bits spreads the counts: masses share few exponents, and equal bins
// serialise the shared-memory atomics. Each CTA counts its stretch, all CTAs
// read all counts through distributed shared memory and draw the same conclusion,
// so a pass is one cluster barrier. Then each warp counts what it keeps, one scan
// over the cluster's warps gives every warp its place, and kept positions and
// masses are written in order. No atomics decide an order: results do not depend
// on timing.
//
// `gather_kernel` (a programmatic dependent): copies the kept rows, 16 bytes per
// thread and cache, neighbouring threads along the heads of one output token.
//
// Measured, 8 kv heads of 128 dims: 32 ragged rows of up to 32768 tokens to 4096 213 us, 47 the
// selection and 166 the copy, at a plain copy's rate (the copy in the selection's
// kernel was slower: its CTAs are few). One row of 32768 to 2048 19.2 us, 18.7 without masses of 0 (one value
// for a tenth of the tokens): the passes' barriers.
#include <cooperative_groups.h>

#include "common.cuh"
#include "evict_key.cuh"
#include "fk_b200.h"

namespace fk {
namespace evict {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = kThreads;  // one per thread
constexpr int kBinBits = 10;
constexpr int kMaxCluster = 8;

struct Params {
  const uint8_t* k;          // [B, Lmax, Hkv, row_bytes] or [num_blocks, block_size, Hkv, row_bytes]
  const uint8_t* v;
  const int* table;          // [B, max_blocks] or null
  int max_blocks, block_size, num_blocks;
  const int* seqlens;
  const float* mass;         // [B, Hkv, mass_cap]
  long long mass_cap;
  uint8_t* k_out;
  uint8_t* v_out;
  const int* out_table;
  int out_max_blocks, out_block_size, out_num_blocks, out_max_seqlen;
  int* seqlens_out;
  float* mass_out;           // [B, Hkv, out_mass_cap]
  long long out_mass_cap;
  int* kept;                 // [B, Hkv, budget], -1 behind the new length
  int B, Lmax, Hkv, row_bytes, budget, sinks, recent;
  FastDiv heads;             // by Hkv
  int cl_log;                // log2 of the CTAs per cluster
};

// Both kernels are resident while kernels before them still write lengths, masses, tables, caches and `kept`. So
// nothing is read through the read-only path (__ldg): such loads may be moved ahead of the wait. These
// are ordinary loads that the compiler still moves past stores, which it does not know to go elsewhere (32
// ragged rows to 4096 tokens: 213 us, with plain reads 257).
__device__ __forceinline__ int load_now(const int* src) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(src));
  return v;
}
__device__ __forceinline__ float load_now(const float* src) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(src));
  return v;
}

__device__ __forceinline__ int seq_len(const Params& p, int b) {
  const int L = load_now(p.seqlens + b);
  return min(max(L, 0), p.Lmax);
}

__device__ __forceinline__ uint32_t mass_key(float f) { return key_of_bits(__float_as_uint(f + 0.f)); }  // -0 + 0 = +0

// KEYS: keys per lane kept in registers; 0: any number, read again from memory in every pass.
template <int KEYS>
__global__ void __launch_bounds__(kThreads, 1) select_kernel(const Params p) {
  __shared__ int s_hist[2][kBins];  // this CTA's counts, double-buffered over the passes
  __shared__ uint32_t s_below[kWarps], s_greatest[kWarps];
  __shared__ uint32_t s_range[2];   // this CTA's KeyRange
  __shared__ int s_warp[kWarps];    // sums of the scan
  __shared__ int s_bin, s_above, s_count;
  __shared__ int s_gt[kWarps], s_tie[kWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const int cl = cluster.num_blocks(), rank = cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pair = blockIdx.x >> p.cl_log;
  const int b = p.heads.div(pair), h = pair - b * p.Hkv;
  const int len = seq_len(p, b);
  const int kept = min(len, p.budget);
  const float* mass = p.mass + (size_t)pair * p.mass_cap;
  float* mass_out = p.mass_out + (size_t)pair * p.out_mass_cap;
  int* out = p.kept + (size_t)pair * p.budget;
  const int t0 = rank * kThreads + threadIdx.x, step = cl * kThreads;

  // Behind the new length: no positions, and masses that start at zero.
  for (int i = kept + t0; i < p.budget; i += step) out[i] = -1;
  for (long long i = kept + t0; i < p.out_mass_cap; i += step) mass_out[i] = 0.f;
  if (h == 0 && rank == 0 && threadIdx.x == 0) p.seqlens_out[b] = kept;
  if (len <= p.budget) {  // the same for the whole cluster
    for (int i = t0; i < len; i += step) {
      out[i] = i;
      mass_out[i] = mass[i];
    }
    return;
  }
  const int first = p.sinks, m = len - p.recent - p.sinks;  // the candidates [first, first + m)
  const int want = p.budget - p.sinks - p.recent;           // 0 <= want < m
  for (int i = t0; i < p.sinks; i += step) {
    out[i] = i;
    mass_out[i] = mass[i];
  }
  for (int i = t0; i < p.recent; i += step) {
    out[p.budget - p.recent + i] = len - p.recent + i;
    mass_out[p.budget - p.recent + i] = mass[len - p.recent + i];
  }
  if (want == 0) return;

  // Each warp of the cluster owns a contiguous stretch of the candidates, a whole number of
  // rounds of 32.
  const int gw = rank * kWarps + warp;
  const int seg = ((((m + 31) >> 5) + cl * kWarps - 1) >> (p.cl_log + 5)) << 5;
  const int w0 = min(gw * seg, m), w1 = min(w0 + seg, m);
  mass += first;
  uint32_t reg[KEYS > 0 ? KEYS : 1];
  if constexpr (KEYS > 0) {
    float f[KEYS];
#pragma unroll
    for (int u = 0; u < KEYS; ++u) f[u] = w0 + u * 32 + lane < w1 ? load_now(mass + w0 + u * 32 + lane) : 0.f;
#pragma unroll
    for (int u = 0; u < KEYS; ++u) reg[u] = w0 + u * 32 + lane < w1 ? mass_key(f[u]) : kNoKey;
  }
  // Calls f(key, index) for this lane's candidates, in order, whole warps at a time.
  auto each = [&](auto f) {
    if constexpr (KEYS > 0) {
#pragma unroll
      for (int u = 0; u < KEYS; ++u) f(reg[u], w0 + u * 32 + lane);
    } else {
      for (int i0 = w0; i0 < w1; i0 += 32) {
        const int i = i0 + lane;
        f(i < w1 ? mass_key(load_now(mass + i)) : kNoKey, i);
      }
    }
  };
  auto sync_all = [&]() {
    if (cl > 1) cluster.sync(); else __syncthreads();
  };

  // ---- the keys' range ----
  KeyRange range;
  each([&](uint32_t key, int) { range.add(key); });
  auto over_warp = [](KeyRange r) {
    r.below = __reduce_min_sync(0xffffffffu, r.below);
    r.greatest = __reduce_max_sync(0xffffffffu, r.greatest);
    return r;
  };
  range = over_warp(range);
  if (lane == 0) {
    s_below[warp] = range.below;
    s_greatest[warp] = range.greatest;
  }
  s_hist[0][threadIdx.x] = 0;
  __syncthreads();
  if (warp == 0) {
    range.below = s_below[lane];
    range.greatest = s_greatest[lane];
    range = over_warp(range);
    if (lane == 0) {
      s_range[0] = range.below;
      s_range[1] = range.greatest;
    }
  }
  sync_all();
  range.below = s_range[0];
  range.greatest = s_range[1];
  for (int q = 0; q < cl && cl > 1; ++q) {
    const uint32_t* r = cluster.map_shared_rank(s_range, q);
    range.join(r[0], r[1]);
  }
  uint32_t lo = range.least(), hi = range.greatest;

  // ---- narrow [lo, lo + 2^width) to the want-th greatest key ----
  int width = 32 - __clz(hi - lo);  // bits of the interval
  int above = 0;                    // candidates above the interval
  int inside = m;                   // candidates in it
  for (int pass = 0; width > 0 && inside > want - above; ++pass) {
    const int shift = max(0, width - kBinBits);
    int* hist = s_hist[pass & 1];
    each([&](uint32_t key, int) {
      const uint32_t d = key - lo;  // wraps to a great number below the interval, kNoKey's place
      if (d <= hi - lo) atomicAdd(&hist[d >> shift], 1);
    });
    sync_all();
    int n = hist[threadIdx.x];
    if (cl > 1) {
      n = 0;
      for (int q = 0; q < cl; ++q) n += cluster.map_shared_rank(hist, q)[threadIdx.x];
    }
    // The other buffer is free: whoever read it in the pass before has passed this barrier.
    s_hist[(pass & 1) ^ 1][threadIdx.x] = 0;
    // Candidates in greater bins: bin t of thread t, a suffix sum.
    int suffix = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_down_sync(0xffffffffu, suffix, off);
      if (lane + off < 32) suffix += o;
    }
    if (lane == 0) s_warp[warp] = suffix;
    __syncthreads();
    int later = lane > warp ? s_warp[lane] : 0;
    later = __reduce_add_sync(0xffffffffu, later);
    const int over = above + later + suffix - n;
    if (over < want && want <= over + n) {
      s_bin = threadIdx.x;
      s_above = over;
      s_count = n;
    }
    __syncthreads();
    lo += (uint32_t)s_bin << shift;
    hi = min(hi, lo + (shift == 0 ? 0u : (0xFFFFFFFFu >> (32 - shift))));
    width = shift;
    above = s_above;
    inside = s_count;
  }
  // All keys above the interval stay. Either all that are left in it are wanted, or it is one key,
  // of which the earliest want - above stay.
  const bool whole = inside == want - above;
  const int ties = whole ? 0 : want - above;
  const uint32_t under = whole ? lo - 1 : lo;  // greater keys stay

  int n_gt = 0, n_tie = 0;
  each([&](uint32_t key, int) {
    n_gt += key > under;
    n_tie += key == lo;  // all of them are above `under` if the interval stays whole
  });
  n_gt = __reduce_add_sync(0xffffffffu, n_gt);
  n_tie = __reduce_add_sync(0xffffffffu, n_tie);
  if (lane == 0) {
    s_gt[warp] = n_gt;
    s_tie[warp] = n_tie;
  }
  sync_all();
  // What the warps before this one hold.
  int b_gt = 0, b_tie = 0;
  for (int q = 0; q <= rank; ++q) {
    const int* gq = cl > 1 ? cluster.map_shared_rank(s_gt, q) : s_gt;
    const int* tq = cl > 1 ? cluster.map_shared_rank(s_tie, q) : s_tie;
    if (q < rank || lane < warp) {
      b_gt += gq[lane];
      b_tie += tq[lane];
    }
  }
  b_gt = __reduce_add_sync(0xffffffffu, b_gt);
  b_tie = __reduce_add_sync(0xffffffffu, b_tie);
  const uint32_t below = (1u << lane) - 1u;
  each([&](uint32_t key, int i) {
    const bool gt = key > under, tie = !whole && key == lo;
    const uint32_t bg = __ballot_sync(0xffffffffu, gt), bt = __ballot_sync(0xffffffffu, tie);
    const int tie_rank = b_tie + __popc(bt & below);
    if (gt || (tie && tie_rank < ties)) {
      const int pos = p.sinks + b_gt + __popc(bg & below) + min(tie_rank, ties);
      out[pos] = first + i;
      mass_out[pos] = load_now(mass + i);
    }
    b_gt += __popc(bg);
    b_tie += __popc(bt);
  });
  if (cl > 1) cluster.sync();  // no CTA leaves while another reads its counts
}

constexpr int kGatherThreads = 256;
constexpr int kUnroll = 4;  // 16-byte copies of K and of V in flight per thread

// How the pieces of 16 bytes of one row b's output tokens are dealt to threads: piece i of a
// block is piece in_tok of token tok, i = tok * per_tok + in_tok, heads and pieces fastest.
struct GatherPlan {
  FastDiv per_tok;    // pieces of a token: heads * row_bytes / 16
  FastDiv per_row;    // pieces of a head's row
  FastDiv page_in, page_out;
  int tokens;         // output tokens per block
  int slots;          // output tokens per row b at most
};

__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const Params p, const GatherPlan g) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.y, s0 = blockIdx.x * g.tokens;
  const int live = min(seq_len(p, b), p.budget);  // tokens of this row's output
  const int pieces = min(g.tokens, live - s0) * g.per_tok.d;
  const int* kept = p.kept + (size_t)b * p.Hkv * p.budget;
  const size_t row = (size_t)p.Hkv * p.row_bytes;
  for (int i0 = threadIdx.x; i0 < pieces; i0 += kGatherThreads * kUnroll) {
    uint4 kv[kUnroll], vv[kUnroll];
    long long from[kUnroll], to[kUnroll];
    int src[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = i0 + u * kGatherThreads;
      const int tok = g.per_tok.div(i), in_tok = i - tok * g.per_tok.d, s = s0 + tok;
      from[u] = in_tok * 16;  // offsets in bytes; the row is added below
      to[u] = -1;
      if (i < pieces) {
        src[u] = load_now(kept + (size_t)g.per_row.div(in_tok) * p.budget + s);
        long long r = (long long)b * p.out_max_seqlen + s;
        if (p.out_table) {
          const int page = load_now(p.out_table + (size_t)b * p.out_max_blocks + g.page_out.div(s));
          r = page < 0 || page >= p.out_num_blocks
                  ? -1
                  : (long long)page * p.out_block_size + (s - g.page_out.div(s) * p.out_block_size);
        }
        if (r >= 0) to[u] = r * (long long)row + in_tok * 16;
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (to[u] < 0) continue;
      long long r = (long long)b * p.Lmax + src[u];
      if (p.table) {
        const int pg = g.page_in.div(src[u]);
        const int page = load_now(p.table + (size_t)b * p.max_blocks + pg);
        r = page < 0 || page >= p.num_blocks ? -1 : (long long)page * p.block_size + (src[u] - pg * p.block_size);
      }
      from[u] = r < 0 ? -1 : from[u] + r * (long long)row;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      kv[u] = vv[u] = make_uint4(0u, 0u, 0u, 0u);
      if (to[u] >= 0 && from[u] >= 0) {
        kv[u] = *reinterpret_cast<const uint4*>(p.k + from[u]);
        vv[u] = *reinterpret_cast<const uint4*>(p.v + from[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (to[u] < 0) continue;
      *reinterpret_cast<uint4*>(p.k_out + to[u]) = kv[u];
      *reinterpret_cast<uint4*>(p.v_out + to[u]) = vv[u];
    }
  }
}

static int launch(Params p, cudaStream_t st) {
  // CTAs per (row, head): doubled while the pairs do not fill the SMs and the CTAs so far have fewer lanes than the
  // longest row has tokens, so that each warp has at least 16 candidates of it; and until a lane's keys
  // fit 32 registers (at 32 rows of up to 32768 tokens one CTA with 32 keys per lane measured 47 us, two with 16
  // each 55: a pass is latency, and a cluster's barrier costs more than a CTA's).
  p.cl_log = 0;
  while ((1 << p.cl_log) < kMaxCluster && p.Lmax > (kThreads << p.cl_log) &&
         (((long long)p.B * p.Hkv << p.cl_log) < num_sms() || p.Lmax > (32 * kThreads << p.cl_log)))
    ++p.cl_log;
  const int cl = 1 << p.cl_log;
  p.heads = FastDiv::of(p.Hkv);
  const int keys = (p.Lmax + cl * kThreads - 1) / (cl * kThreads);  // per lane, of a row as long as can be
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cl;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.B * p.Hkv * cl), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (keys <= 4)
    FK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, select_kernel<4>, p));
  else if (keys <= 16)
    FK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, select_kernel<16>, p));
  else if (keys <= 32)
    FK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, select_kernel<32>, p));
  else
    FK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, select_kernel<0>, p));
  GatherPlan g;
  g.slots = p.budget < p.Lmax ? p.budget : p.Lmax;
  const int per_row = p.row_bytes / 16, per_tok = p.Hkv * per_row;
  g.per_tok = FastDiv::of(per_tok);
  g.per_row = FastDiv::of(per_row);
  g.page_in = FastDiv::of(p.block_size);
  g.page_out = FastDiv::of(p.out_block_size);
  // Tokens per block: one round of the unrolled loop, or a token.
  g.tokens = (kGatherThreads * kUnroll + per_tok - 1) / per_tok;
  cfg.gridDim = dim3((unsigned)((g.slots + g.tokens - 1) / g.tokens), (unsigned)p.B, 1);
  cfg.blockDim = dim3(kGatherThreads, 1, 1);
  cfg.numAttrs = 1;
  FK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, gather_kernel, p, g));
  return kOk;
}

}  // namespace evict
}  // namespace fk

using namespace fk;

extern "C" int fk_cache_evict(const void* k_cache, const void* v_cache, const int32_t* block_table,
                              const int32_t* cache_seqlens, const float* mass, long long mass_capacity, void* k_out,
                              void* v_out, const int32_t* out_block_table, int32_t* seqlens_out, float* mass_out,
                              long long out_mass_capacity, int32_t* kept, int batch, int max_seqlen, int block_size,
                              int num_blocks, int out_max_seqlen, int out_block_size, int out_num_blocks,
                              int num_heads_kv, int row_bytes, int budget, int sinks, int recent, void* stream) {
  FK_CHECK_ARG(k_cache && v_cache && cache_seqlens && mass && k_out && v_out && seqlens_out && mass_out && kept,
               "null tensor pointer");
  FK_CHECK_ARG(batch >= 1 && max_seqlen >= 1 && num_heads_kv >= 1, "sizes must be positive");
  FK_CHECK_ARG(max_seqlen <= (1 << 30) && out_max_seqlen <= (1 << 30) && budget <= (1 << 30),
               "max_seqlen, out_max_seqlen and budget must be <= 2^30");
  FK_CHECK_ARG(row_bytes >= 16 && row_bytes % 16 == 0, "row_bytes must be a positive multiple of 16");
  FK_CHECK_ARG(budget >= 1 && sinks >= 0 && recent >= 0 && (long long)sinks + recent <= budget,
               "budget must be >= 1 and sinks + recent must lie in [0, budget]");
  FK_CHECK_ARG(out_max_seqlen >= (budget < max_seqlen ? budget : max_seqlen),
               "the output cache must hold min(budget, max_seqlen) tokens per row");
  FK_CHECK_ARG(mass_capacity >= max_seqlen && out_mass_capacity >= (budget < max_seqlen ? budget : max_seqlen),
               "mass arrays too short");
  FK_CHECK_ARG(batch <= 65535 && (long long)batch * num_heads_kv <= (1 << 24) &&
                   (long long)num_heads_kv * row_bytes <= (1 << 24),
               "batch or row too large");
  FK_CHECK_ARG((((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0,
               "caches must be 16-byte aligned");
  FK_CHECK_ARG(mass_out != mass && seqlens_out != cache_seqlens && k_out != v_out, "outputs must not alias");
  // One pool on both sides is fine with two tables over different pages.
  FK_CHECK_ARG((k_out != k_cache && v_out != v_cache && k_out != v_cache && v_out != k_cache) ||
                   (block_table && out_block_table && block_table != out_block_table && k_out == k_cache &&
                    v_out == v_cache),
               "the output cache must not alias the input cache");
  if (block_table)
    FK_CHECK_ARG(block_size >= 1 && num_blocks >= 1 && max_seqlen % block_size == 0,
                 "paged cache: max_seqlen must be max_blocks_per_seq * block_size, num_blocks >= 1");
  if (out_block_table)
    FK_CHECK_ARG(out_block_size >= 1 && out_num_blocks >= 1 && out_max_seqlen % out_block_size == 0,
                 "paged output: out_max_seqlen must be max_blocks_per_seq * out_block_size, out_num_blocks >= 1");
  evict::Params p = {};
  p.k = static_cast<const uint8_t*>(k_cache);
  p.v = static_cast<const uint8_t*>(v_cache);
  p.table = block_table;
  p.block_size = block_table ? block_size : 1;
  p.max_blocks = block_table ? max_seqlen / block_size : 0;
  p.num_blocks = num_blocks;
  p.seqlens = cache_seqlens;
  p.mass = mass;
  p.mass_cap = mass_capacity;
  p.k_out = static_cast<uint8_t*>(k_out);
  p.v_out = static_cast<uint8_t*>(v_out);
  p.out_table = out_block_table;
  p.out_block_size = out_block_table ? out_block_size : 1;
  p.out_max_blocks = out_block_table ? out_max_seqlen / out_block_size : 0;
  p.out_num_blocks = out_num_blocks;
  p.out_max_seqlen = out_max_seqlen;
  p.seqlens_out = seqlens_out;
  p.mass_out = mass_out;
  p.out_mass_cap = out_mass_capacity;
  p.kept = kept;
  p.B = batch;
  p.Lmax = max_seqlen;
  p.Hkv = num_heads_kv;
  p.row_bytes = row_bytes;
  p.budget = budget;
  p.sinks = sinks;
  p.recent = recent;
  return evict::launch(p, static_cast<cudaStream_t>(stream));
}
