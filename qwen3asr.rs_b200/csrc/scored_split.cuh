// scored_split.cuh — what the kernels of scored decode attention share: a CTA's
// split of a context, its stream of pages, and the end of its rows.
//
// A CTA takes one split of one (sequence, kv head)'s context and a tile of
// rows, row r = i * group + g for window row i and query head g of the kv
// head. Its pages stream through a ring of shared-memory stages by bulk
// copies; stage s belongs to warp s % 4, which consumes it and refills it with
// the pages one ring ahead. Each warp keeps its own running maximum, sum and
// O, joined at the end.
//
// The scored rows' raw scores x (log2 domain) stay in shared memory, or go to
// the workspace where they do not fit. The weights follow once the row's
// maximum and sum over the whole context are known: at once where one split is
// the whole context; else the split leaves x, O and (m, l) in the workspace
// and a second launch joins them. Measured slower at 512 sequences of 64 to
// 4096 tokens: the last CTA of a sequence joining it, found by a counter (its
// SM's place idles while its own loads are under way), and the splits as a
// thread-block cluster that join in distributed shared memory (a cluster
// waits for all its places at once: 360 against 324 us with the join as it was).
#pragma once

#include <type_traits>

#include "common.cuh"

namespace vasr {

constexpr int kScoredDim = 128;
constexpr int kScoredMaxRows = 128;       // rows of one (sequence, kv head)
constexpr int kScoredMaxPages = 64;       // pages of one split
constexpr int kScoredThreads = 128;

struct ScoredSplitParams {
  void *out;
  const void *q;
  const void *k_cache;
  const void *v_cache;
  float *score_cache;
  const uint32_t *block_tables;
  const uint32_t *context_lens;
  const float *k_scale;
  const float *v_scale;
  float *ws_o;         // [(b * Hkv + kvh) * max_splits + split][rows][D]
  float2 *ws_ml;       // [..same..][rows]  (m in log2 units, l)
  float *ws_x;         // [(b * Hkv + kvh) * scored_rows + r][x_stride]
  int64_t q_token_stride;
  int64_t num_blocks;
  int64_t x_stride;
  int num_heads;
  int num_kv_heads;
  int group;
  int query_len;
  int rows;            // query_len * group
  int scored_rows;     // score_rows * group
  int row_tiles;
  int cols;
  int max_context;
  int pages_per_split;
  int max_splits;
  int x_tokens;        // raw scores a row has in shared memory; 0: none, they go to the workspace
  float scale;
  float softcap;
  float decay;
};

// 2^x in one instruction (2 ulp, results below 2^-126 are 0): the arguments
// are a score less its row's maximum, whose own rounding is larger.
__device__ __forceinline__ float scored_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A page copy that leaves L2 first: pages are read once a step, and would
// push the raw scores out before the join reads them.
__device__ __forceinline__ uint64_t evict_first_policy() {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void bulk_g2s_hint(uint32_t dst_smem, const void *src, uint32_t bytes, uint32_t bar,
                                              uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          dst_smem),
      "l"(src), "r"(bytes), "r"(bar), "l"(policy)
      : "memory");
}

// The context length a kernel works with; too long a one is cut and recorded.
__device__ __forceinline__ int scored_context(const ScoredSplitParams &p, int b, int bs, bool report) {
  int64_t n = p.context_lens[b];
  const int64_t cap = min((int64_t)p.cols * bs, (int64_t)p.max_context);
  if (n > cap) {
    if (report) raise_device_error(VASR_PA_DERR_CTX_RANGE);
    n = cap;
  }
  return (int)n;
}

__device__ __forceinline__ int scored_splits(int n, int pages_per_split, int bs) {
  const int per = pages_per_split * bs;
  return (n + per - 1) / per;
}

// (m, 1 / l) of one row over the splits, by one warp. A row that saw nothing
// gets (0, 0): its raw scores are -inf and weigh 0.
__device__ __forceinline__ float2 scored_final_row(const ScoredSplitParams &p, int64_t pair, int n_splits, int r) {
  const int lane = threadIdx.x & 31;
  const float2 *ml = p.ws_ml + pair * p.max_splits * p.rows + r;
  float m = -INFINITY, l = 0.f;
  for (int s0 = 0; s0 < n_splits; s0 += 64) {
    float2 v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = s0 + 32 * i + lane;
      v[i] = s < n_splits ? ml[(int64_t)s * p.rows] : make_float2(-INFINITY, 0.f);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float m_new = fmaxf(m, v[i].x);
      if (v[i].y != 0.f) l = (l != 0.f ? l * scored_exp2(m - m_new) : 0.f) + v[i].y * scored_exp2(v[i].x - m_new);
      m = m_new;
    }
  }
  const float top = warp_max_xor(m, 32);
  l = warp_sum_xor(l != 0.f ? l * scored_exp2(m - top) : 0.f, 32);
  return l != 0.f ? make_float2(top, 1.f / l) : make_float2(0.f, 0.f);
}

// A row's state over some of the splits: 4 dims of O (lane: dims 4 lane ..),
// the maximum and the sum.
struct ScoredRow {
  float4 o;
  float m, l;
  __device__ __forceinline__ void add(const float4 &v, float vm, float vl) {
    if (vl == 0.f) return;  // saw nothing
    const float m_new = fmaxf(m, vm);
    const float a = l != 0.f ? scored_exp2(m - m_new) : 0.f, w = scored_exp2(vm - m_new);
    o.x = fmaf(v.x, w, o.x * a);
    o.y = fmaf(v.y, w, o.y * a);
    o.z = fmaf(v.z, w, o.z * a);
    o.w = fmaf(v.w, w, o.w * a);
    l = fmaf(vl, w, l * a);
    m = m_new;
  }
};
// Splits first, first + step, ... of a row, by one warp: (m, l) and O in one
// round of loads.
__device__ __forceinline__ ScoredRow scored_sum_splits(const ScoredSplitParams &p, int64_t pair, int n_splits, int r,
                                                       int first, int step) {
  const int lane = threadIdx.x & 31;
  ScoredRow row{make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f};
  constexpr int kBatch = 4;  // splits whose loads are under way together
  for (int s0 = first; s0 < n_splits; s0 += kBatch * step) {
    float2 ml[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int s = s0 + i * step;
      const int64_t at = (pair * p.max_splits + s) * p.rows + r;
      ml[i] = s < n_splits ? p.ws_ml[at] : make_float2(0.f, 0.f);
      v[i] = s < n_splits ? reinterpret_cast<const float4 *>(p.ws_o + at * kScoredDim)[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) row.add(v[i], ml[i].x, ml[i].y);
  }
  return row;
}

template <typename T>
__device__ __forceinline__ T *scored_out_row(const ScoredSplitParams &p, int b, int kvh, int r) {
  return static_cast<T *>(p.out) +
         (((int64_t)b * p.query_len + r / p.group) * p.num_heads + kvh * p.group + r % p.group) * kScoredDim;
}
template <typename T>
__device__ __forceinline__ void scored_store4(T *out, float4 o, float mul) {
  out[0] = Elem<T>::from_f32(o.x * mul);
  out[1] = Elem<T>::from_f32(o.y * mul);
  out[2] = Elem<T>::from_f32(o.z * mul);
  out[3] = Elem<T>::from_f32(o.w * mul);
}

// score <- decay score + sum of the scored rows' weights for up to
// kWeightTokens tokens from j0 (below j1), 4 tokens a thread and kWeightBatch
// such groups (page rows hold a multiple of 8 tokens). x: the rows' raw
// scores. load() starts the reads that do not need the rows' (m, 1 / l).
constexpr int kWeightBatch = 2;
constexpr int kWeightTokens = kScoredThreads * 4 * kWeightBatch;
constexpr int kWeightEarly = 2;  // rows whose raw scores load() reads too
struct ScoredWeights {
  float4 *at[kWeightBatch];
  float4 old[kWeightBatch], x[kWeightEarly][kWeightBatch];
  int j0, j1;
  __device__ __forceinline__ void load(const ScoredSplitParams &p, int b, int kvh, int bs, int first, int last,
                                       const float *xs, int64_t x_stride) {
    const uint32_t *table = p.block_tables + (int64_t)b * p.cols;
    const int shift = 31 - __clz(bs);
    j0 = first + threadIdx.x * 4;
    j1 = last;
#pragma unroll
    for (int u = 0; u < kWeightBatch; ++u) {
      const int j = j0 + u * kScoredThreads * 4;
      at[u] = nullptr;
      if (j < j1) {
        const uint32_t id = __ldg(table + (j >> shift));
        if ((int64_t)id < p.num_blocks)  // others are recorded where the page was read
          at[u] = reinterpret_cast<float4 *>(p.score_cache + (((int64_t)id * p.num_kv_heads + kvh) << shift) + (j & (bs - 1)));
#pragma unroll
        for (int r = 0; r < kWeightEarly; ++r)
          if (r < p.scored_rows)
            x[r][u] = *reinterpret_cast<const float4 *>(xs + r * x_stride + j);
      }
    }
#pragma unroll
    for (int u = 0; u < kWeightBatch; ++u) old[u] = at[u] ? *at[u] : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void finish(const ScoredSplitParams &p, const float2 *fin, const float *xs, int64_t x_stride) const {
    float4 w[kWeightBatch] = {};
    auto add = [&](int u, const float4 &v, const float2 &f) {
      w[u].x = fmaf(scored_exp2(v.x - f.x), f.y, w[u].x);
      w[u].y = fmaf(scored_exp2(v.y - f.x), f.y, w[u].y);
      w[u].z = fmaf(scored_exp2(v.z - f.x), f.y, w[u].z);
      w[u].w = fmaf(scored_exp2(v.w - f.x), f.y, w[u].w);
    };
#pragma unroll
    for (int u = 0; u < kWeightBatch; ++u) {
#pragma unroll
      for (int r = 0; r < kWeightEarly; ++r)
        if (at[u] && r < p.scored_rows) add(u, x[r][u], fin[r]);
    }
    for (int r = kWeightEarly; r < p.scored_rows; ++r)
#pragma unroll
      for (int u = 0; u < kWeightBatch; ++u)
        if (at[u]) add(u, *reinterpret_cast<const float4 *>(xs + r * x_stride + j0 + u * kScoredThreads * 4), fin[r]);
#pragma unroll
    for (int u = 0; u < kWeightBatch; ++u) {
      if (!at[u]) continue;
      const int left = j1 - (j0 + u * kScoredThreads * 4);  // places past the context keep their bits
      float4 s = old[u];
      s.x = fmaf(p.decay, s.x, w[u].x);
      if (left > 1) s.y = fmaf(p.decay, s.y, w[u].y);
      if (left > 2) s.z = fmaf(p.decay, s.z, w[u].z);
      if (left > 3) s.w = fmaf(p.decay, s.w, w[u].w);
      *at[u] = s;
    }
  }
};

template <typename TC, int BS, int NST>
struct ScoredCfg {
  static constexpr int D = kScoredDim;
  static constexpr int kWarps = kScoredThreads / 32;
  static constexpr int kSP = BS < 16 ? 16 / BS : 1;  // pages per stage
  static constexpr int kST = kSP * BS;               // tokens per stage
  static constexpr int kTiles = kST / 16;
  static constexpr int kPB = D * BS * (int)sizeof(TC);
  static constexpr int kNST = NST;
  static constexpr int kOffK = 0;
  static constexpr int kOffV = NST * kSP * kPB;
  static constexpr int kOffBlk = 2 * NST * kSP * kPB;
  static constexpr int kOffBar = kOffBlk + kScoredMaxPages * 8;
  static constexpr int kOffFin = kOffBar + NST * 8;                     // float2 [kScoredMaxRows]
  static constexpr int kOffML = kOffFin + kScoredMaxRows * 8;           // float2 [warps][16]
  static constexpr int kOffX = (kOffML + kWarps * 16 * 8 + 127) & ~127;  // raw scores [scored rows][x_tokens]
  static constexpr int kXBytes = 8192;
  static constexpr int kSmemBytes = kOffX + kXBytes;
  static_assert(NST % kWarps == 0, "stages split evenly over the warps");
  static_assert(kWarps * 16 * D * 4 <= kOffBlk, "the warps' O fits the drained ring");
};

// This CTA's split, tile of rows and pages.
template <typename TC, int BS, int NST>
struct ScoredSplit {
  using C = ScoredCfg<TC, BS, NST>;
  int split, kvh, tile, b;
  int n, n_splits;     // the context, and its splits
  int tok0, tok1;      // the split's tokens
  int n_pages, n_units;
  int64_t pair;
  const int64_t *page;  // element offset of each page
  uint32_t s_base;
  uint64_t policy;
  // raw scores: token tok0 + j of row r at x[r * x_stride + j]
  float *x_pair, *x;
  int64_t x_stride;

  // False where the CTA has nothing to do (an empty context's zeros are written).
  template <typename T>
  __device__ __forceinline__ bool begin(const ScoredSplitParams &p, unsigned char *smem, int rows_per_tile) {
    constexpr int D = C::D;
    const int tid = threadIdx.x;
    s_base = smem_addr(smem);
    split = blockIdx.x;
    kvh = blockIdx.y / p.row_tiles;
    tile = blockIdx.y % p.row_tiles;
    b = blockIdx.z;
    pair = (int64_t)b * p.num_kv_heads + kvh;
    if (tid < NST) mbar_init(s_base + C::kOffBar + tid * 8, 1);
    if (tid == 0) mbar_fence_init();
    // block ids of the split, loaded beside the context length (right unless
    // sharing the pages evenly moves the split's start)
    uint32_t spec_id = 0;
    const int spec_col = split * p.pages_per_split + tid;
    if (tid < p.pages_per_split && spec_col < p.cols) spec_id = __ldg(p.block_tables + (int64_t)b * p.cols + spec_col);
    n = scored_context(p, b, BS, split == 0 && tid == 0 && blockIdx.y == 0);
    n_splits = scored_splits(n, p.pages_per_split, BS);
    if (n == 0 && split == 0) {  // nothing cached: zeros
      for (int e = tid; e < rows_per_tile * D; e += kScoredThreads) {
        const int r = tile * rows_per_tile + e / D;
        if (r < p.rows) scored_out_row<T>(p, b, kvh, r)[e % D] = Elem<T>::from_f32(0.f);
      }
    }
    if (split >= n_splits) return false;
    const int seq_pages = (n + BS - 1) / BS;
    const int per = (seq_pages + n_splits - 1) / n_splits;  // pages shared evenly by the splits
    const int page0 = split * per;
    tok0 = page0 * BS;
    tok1 = min(n, tok0 + per * BS);
    n_pages = max(0, (tok1 - tok0 + BS - 1) / BS);
    n_units = (n_pages + C::kSP - 1) / C::kSP;
    int64_t *offsets = reinterpret_cast<int64_t *>(smem + C::kOffBlk);
    if (tid < n_pages) {
      uint32_t id = spec_id;
      if (page0 != split * p.pages_per_split) id = __ldg(p.block_tables + (int64_t)b * p.cols + page0 + tid);
      if ((int64_t)id >= p.num_blocks) {
        raise_device_error(VASR_PA_DERR_BLOCK_RANGE);
        id = 0;
      }
      offsets[tid] = ((int64_t)id * p.num_kv_heads + kvh) * (D * BS);
    }
    page = offsets;
    policy = evict_first_policy();
    x_pair = p.ws_x + pair * p.scored_rows * p.x_stride;
    x = p.x_tokens ? reinterpret_cast<float *>(smem + C::kOffX) : x_pair + tok0;
    x_stride = p.x_tokens ? p.x_tokens : p.x_stride;
    __syncthreads();
    const int warp = tid >> 5;
    if ((tid & 31) == 0)
      for (int u = warp; u < min(NST, n_units); u += C::kWarps) issue(p, u);
    return true;
  }
  // One thread: the pages of unit u into its stage.
  __device__ __forceinline__ void issue(const ScoredSplitParams &p, int u) const {
    const int s = u % NST, pg0 = u * C::kSP, np = min(C::kSP, n_pages - pg0);
    const uint32_t bar = s_base + C::kOffBar + s * 8;
    mbar_arrive_expect_tx(bar, (uint32_t)(2 * np * C::kPB));
    for (int i = 0; i < np; ++i) {
      const int64_t off = page[pg0 + i];
      // the page's scores are wanted at the end
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.score_cache + off / C::D));
      bulk_g2s_hint(s_base + C::kOffK + (s * C::kSP + i) * C::kPB, static_cast<const TC *>(p.k_cache) + off, C::kPB, bar, policy);
      bulk_g2s_hint(s_base + C::kOffV + (s * C::kSP + i) * C::kPB, static_cast<const TC *>(p.v_cache) + off, C::kPB, bar, policy);
    }
  }
  __device__ __forceinline__ bool wait(int u) const {
    return mbar_wait_bounded(s_base + C::kOffBar + (u % NST) * 8, (uint32_t)((u / NST) & 1));
  }
  // This warp is done with unit u: its stage takes the unit one ring ahead.
  __device__ __forceinline__ void refill(const ScoredSplitParams &p, int u) const {
    __syncwarp();
    if (u + NST < n_units && (threadIdx.x & 31) == 0) {
      fence_proxy_async_smem();
      issue(p, u + NST);
    }
  }
  // A warp whose wait for unit u gave up: the copies it has in flight land
  // before the ring is reused.
  __device__ __forceinline__ void drain(int u) const {
    for (int v = u; v < min(u + NST, n_units); v += C::kWarps) wait(v);
  }

  // The warps' O ([warp][kRows][D] over the drained ring) and (m, l) are in
  // shared memory: the tile's rows end here, or go to the join.
  template <typename T, int kRows>
  __device__ __forceinline__ void end(const ScoredSplitParams &p, unsigned char *smem, float v_mul) const {
    constexpr int D = C::D;
    const int tid = threadIdx.x, row0 = tile * kRows;
    const float *co = reinterpret_cast<const float *>(smem);
    const float2 *cml = reinterpret_cast<const float2 *>(smem + C::kOffML);  // [warp][16]
    float2 *fin = reinterpret_cast<float2 *>(smem + C::kOffFin);
    const int rows_here = min(kRows, p.rows - row0);
    // a row's (m, l) over the warps, and one dim of its O
    auto row_total = [&](int r) {
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) m = fmaxf(m, cml[w * 16 + r].x);
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) {
        const float2 ml = cml[w * 16 + r];
        if (ml.y != 0.f) l = fmaf(ml.y, scored_exp2(ml.x - m), l);
      }
      return make_float2(m, l);
    };
    auto row_dim = [&](int r, int d, float m) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) {
        const float2 ml = cml[w * 16 + r];
        if (ml.y != 0.f) v = fmaf(co[(w * kRows + r) * D + d], scored_exp2(ml.x - m), v);
      }
      return v;
    };
    if (n_splits == 1 && p.row_tiles == 1) {  // all there is of this (sequence, kv head)
      ScoredWeights weights;
      weights.load(p, b, kvh, BS, 0, n, x, x_stride);
      for (int e = tid; e < rows_here * D; e += kScoredThreads) {
        const int r = e / D, d = e % D;
        const float2 f = row_total(r);
        const float inv = f.y != 0.f ? 1.f / f.y : 0.f;
        if (d == 0) fin[r] = f.y != 0.f ? make_float2(f.x, inv) : make_float2(0.f, 0.f);
        scored_out_row<T>(p, b, kvh, r)[d] = Elem<T>::from_f32(row_dim(r, d, f.x) * inv * v_mul);
      }
      __syncthreads();
      weights.finish(p, fin, x, x_stride);  // all of the context: a split is at most kWeightTokens long
      return;
    }
    for (int e = tid; e < rows_here * D; e += kScoredThreads) {
      const int r = e / D, d = e % D;
      const float2 f = row_total(r);
      const int64_t at = (pair * p.max_splits + split) * p.rows + row0 + r;
      p.ws_o[at * D + d] = row_dim(r, d, f.x);
      if (d == 0) p.ws_ml[at] = f;
    }
    if (p.x_tokens) {
      const int count = max(0, tok1 - tok0);
      for (int r = row0; r < min(row0 + kRows, p.scored_rows); ++r)
        for (int j = tid * 4; j < count; j += kScoredThreads * 4)
          *reinterpret_cast<float4 *>(x_pair + r * p.x_stride + tok0 + j) =
              *reinterpret_cast<const float4 *>(x + r * x_stride + j);
    }
  }
};

// The end of every (sequence, kv head) of several splits (or row tiles):
// blocks [0, chunks) add the weights of `chunk` tokens each, the others join
// the rows: a warp has a row, or all warps share one where there are many
// splits (row_warps = 4). Eight CTAs a SM: with ten, registers spill and 512
// sequences take 324 us instead of 319, with six 321.
template <typename T>
__global__ void __launch_bounds__(kScoredThreads, 8) scored_join_kernel(const ScoredSplitParams p, int bs, int chunk,
                                                                         int chunks, int row_warps) {
  __shared__ float2 fin[kScoredMaxRows];
  __shared__ float4 part[kScoredThreads];
  constexpr int kWarps = kScoredThreads / 32;
  const int kvh = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = scored_context(p, b, bs, false);
  const int n_splits = scored_splits(n, p.pages_per_split, bs);
  const int64_t pair = (int64_t)b * p.num_kv_heads + kvh;
  const int j0 = blockIdx.x * chunk, j1 = min(n, j0 + chunk);
  if (n_splits == 0 || (n_splits == 1 && p.row_tiles == 1) || ((int)blockIdx.x < chunks && j0 >= n)) {
    // nothing to do; but a grid of which no CTA waited could end, and let the
    // stream go on, before the split kernel has
    if (blockIdx.x == 0 && kvh == 0 && b == 0) pdl_wait();
    return;
  }
  if ((int)blockIdx.x < chunks) {
    const float *x = p.ws_x + pair * p.scored_rows * p.x_stride;
    pdl_wait();
    ScoredWeights weights;
    weights.load(p, b, kvh, bs, j0, j1, x, p.x_stride);
    for (int r = warp; r < p.scored_rows; r += kWarps) {
      const float2 f = scored_final_row(p, pair, n_splits, r);
      if (lane == 0) fin[r] = f;
    }
    __syncthreads();
    weights.finish(p, fin, x, p.x_stride);
    for (int j = j0 + kWeightTokens; j < j1; j += kWeightTokens) {
      weights.load(p, b, kvh, bs, j, j1, x, p.x_stride);
      weights.finish(p, fin, x, p.x_stride);
    }
    return;
  }
  const int r = ((int)blockIdx.x - chunks) * (kWarps / row_warps) + warp / row_warps;
  pdl_wait();
  if (r < p.rows) {
    ScoredRow row = scored_sum_splits(p, pair, n_splits, r, warp % row_warps, row_warps);
    if (row_warps > 1) {
      part[threadIdx.x] = row.o;
      if (lane == 0) fin[warp] = make_float2(row.m, row.l);
      __syncthreads();  // r is the same for all warps
      if (warp != 0) return;
#pragma unroll
      for (int w = 1; w < kWarps; ++w) row.add(part[w * 32 + lane], fin[w].x, fin[w].y);
    }
    const float inv = row.l != 0.f ? 1.f / row.l : 0.f;
    scored_store4(scored_out_row<T>(p, b, kvh, r) + 4 * lane, row.o, inv * (p.v_scale ? __ldg(p.v_scale) : 1.f));
  }
}

}  // namespace vasr
