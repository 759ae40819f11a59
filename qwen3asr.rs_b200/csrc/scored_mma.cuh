// scored_mma.cuh — scored decode attention on the tensor cores (mma.sync
// m16n8k16, f32 accumulate) for 16-bit queries over 16-bit or fp8 pages,
// head_dim 128.
//
// A CTA takes one split of one (sequence, kv head)'s context and 8 or 16 rows,
// row r = i * group + g for window row i and query head g of the kv head. Its
// pages stream through a ring of shared-memory stages by bulk copies; stage s
// belongs to warp s % 4. Per 16 tokens a warp computes
//   S[16 rows x 16] = Q K^T     A = Q, B = K by ldmatrix from the page layout
//   O^T[128 x rows] += V^T P^T  A = V^T by ldmatrix, B = S's own fragments
// and keeps the scored rows' raw scores x (log2 domain) in shared memory (in
// the workspace where they do not fit). The weights follow once the row's
// maximum and sum over the whole context are known: at once where one split is
// the whole context; else the split leaves x, O and (m, l) in the workspace
// and a second launch joins them. Measured slower at 512 sequences of 64 to
// 4096 tokens: the last CTA of a sequence joining it, found by a counter (its
// SM's place idles while its own loads are under way), and the splits as a
// thread-block cluster that join in distributed shared memory (a cluster
// waits for all its places at once: 360 against 324 us).
//
// Up to 4 rows (kDup: one token, group <= 4) P^T has columns to spare: A holds
// every query row twice, so the score fragments of rows r and r + 4 are equal,
// and row r's P goes into the product rounded to the operand type while row
// r + 4 carries what that rounding left. O then has P's full f32 precision up
// to 2^-16, for no further MMA; with more rows P is rounded to the operand
// type (the output has that rounding anyway).
//
// Tokens that only some rows of a window see (the last query_len - 1) stay
// out of the P V product: a masked row would multiply their V by zero, and a
// NaN or infinite V would then reach a row that does not see it. They are
// added one by one in f32, row by row.
//
// fp8 pages: the products run in f16 (every E4M3 value is exact in f16), with
// each query row scaled by a power of two to the top of f16's range, so that
// bf16 rows of any magnitude keep their bits. The reduction index is permuted
// as in decode_mma.cuh, so that one ldmatrix row of 16 bytes feeds a k-step.
#pragma once

#include "decode_mma.cuh"

namespace vasr {

constexpr int kScoredDim = 128;
constexpr int kScoredMaxRows = 128;       // rows of one (sequence, kv head)
constexpr int kScoredMaxPages = 64;       // pages of one split
constexpr int kScoredThreads = 128;

struct ScoredMmaParams {
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
__device__ __forceinline__ int scored_context(const ScoredMmaParams &p, int b, int bs, bool report) {
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
__device__ __forceinline__ float2 scored_final_row(const ScoredMmaParams &p, int64_t pair, int n_splits, int r) {
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
__device__ __forceinline__ ScoredRow scored_sum_splits(const ScoredMmaParams &p, int64_t pair, int n_splits, int r,
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
__device__ __forceinline__ T *scored_out_row(const ScoredMmaParams &p, int b, int kvh, int r) {
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
  __device__ __forceinline__ void load(const ScoredMmaParams &p, int b, int kvh, int bs, int first, int last,
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
  __device__ __forceinline__ void finish(const ScoredMmaParams &p, const float2 *fin, const float *xs, int64_t x_stride) const {
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

template <typename T, typename TC, int BS, int NRT, bool kDup, int NST, int MINB>
__global__ void __launch_bounds__(kScoredThreads, MINB) scored_mma_kernel(const ScoredMmaParams p) {
  using C = ScoredCfg<TC, BS, NST>;
  constexpr bool kFp8 = std::is_same<TC, __nv_fp8_e4m3>::value;
  using TM = typename std::conditional<kFp8, __half, T>::type;  // MMA operand type
  constexpr int D = C::D, kKS = D / 16, kRows = kDup ? 4 : 8 * NRT;
  constexpr float kRescale = 8.f;  // the running maximum moves when a tile's exceeds it by 2^8
  static_assert(!kDup || NRT == 1, "doubled rows fill one tile of 8");
  extern __shared__ __align__(128) unsigned char smem[];
  pdl_launch_dependents();
  const uint32_t s_base = smem_addr(smem);
  const int split = blockIdx.x, kvh = blockIdx.y / p.row_tiles, tile = blockIdx.y % p.row_tiles, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = lane >> 2, tig = lane & 3;
  if (tid < NST) mbar_init(s_base + C::kOffBar + tid * 8, 1);
  if (tid == 0) mbar_fence_init();

  // block ids of the split, loaded beside the context length (right unless
  // sharing the pages evenly moves the split's start)
  uint32_t spec_id = 0;
  const int spec_col = split * p.pages_per_split + tid;
  if (tid < p.pages_per_split && spec_col < p.cols) spec_id = __ldg(p.block_tables + (int64_t)b * p.cols + spec_col);
  const int n = scored_context(p, b, BS, split == 0 && tid == 0 && blockIdx.y == 0);
  const int n_splits = scored_splits(n, p.pages_per_split, BS);
  const int row0 = tile * kRows;
  const float v_mul = p.v_scale ? __ldg(p.v_scale) : 1.f;
  if (n == 0 && split == 0) {  // nothing cached: zeros
    for (int e = tid; e < kRows * D; e += kScoredThreads) {
      const int r = row0 + e / D;
      if (r < p.rows)
        static_cast<T *>(p.out)[(((int64_t)b * p.query_len + r / p.group) * p.num_heads + kvh * p.group + r % p.group) * D +
                                e % D] = Elem<T>::from_f32(0.f);
    }
  }
  if (split >= n_splits) return;
  const int seq_pages = (n + BS - 1) / BS;
  const int per = (seq_pages + n_splits - 1) / n_splits;  // pages shared evenly by the splits
  const int page0 = split * per, tok0 = page0 * BS;
  const int tok1 = min(n, tok0 + per * BS);
  const int n_pages = max(0, (tok1 - tok0 + BS - 1) / BS);
  const int n_units = (n_pages + C::kSP - 1) / C::kSP;
  int64_t *page = reinterpret_cast<int64_t *>(smem + C::kOffBlk);  // element offset of each page of the split
  if (tid < n_pages) {
    uint32_t id = spec_id;
    if (page0 != split * p.pages_per_split) id = __ldg(p.block_tables + (int64_t)b * p.cols + page0 + tid);
    if ((int64_t)id >= p.num_blocks) {
      raise_device_error(VASR_PA_DERR_BLOCK_RANGE);
      id = 0;
    }
    page[tid] = ((int64_t)id * p.num_kv_heads + kvh) * (D * BS);
  }
  __syncthreads();

  const TC *kc = static_cast<const TC *>(p.k_cache);
  const TC *vc = static_cast<const TC *>(p.v_cache);
  const uint64_t policy = evict_first_policy();
  auto issue_unit = [&](int u) {
    const int s = u % NST, pg0 = u * C::kSP, np = min(C::kSP, n_pages - pg0);
    const uint32_t bar = s_base + C::kOffBar + s * 8;
    mbar_arrive_expect_tx(bar, (uint32_t)(2 * np * C::kPB));
    for (int i = 0; i < np; ++i) {
      const int64_t off = page[pg0 + i];
      // the page's scores are wanted at the end
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.score_cache + off / D));
      bulk_g2s_hint(s_base + C::kOffK + (s * C::kSP + i) * C::kPB, kc + off, C::kPB, bar, policy);
      bulk_g2s_hint(s_base + C::kOffV + (s * C::kSP + i) * C::kPB, vc + off, C::kPB, bar, policy);
    }
  };
  if (lane == 0)
    for (int u = warp; u < min(NST, n_units); u += C::kWarps) issue_unit(u);

  // ---- query fragments: rows grp (and grp + 8) of this tile; row[t] = its row or -1
  uint32_t qa[kKS][2 * NRT];
  float c_log2[NRT];
  int row[NRT];
  const float k_mul = p.k_scale ? p.scale * __ldg(p.k_scale) : p.scale;
#pragma unroll
  for (int t = 0; t < NRT; ++t) {
    const int r = row0 + (kDup ? (grp & 3) : grp + 8 * t);
    row[t] = r < p.rows ? r : -1;
    const int rr = r < p.rows ? r : 0;
    const T *qp = static_cast<const T *>(p.q) + ((int64_t)b * p.query_len + rr / p.group) * p.q_token_stride +
                  (int64_t)(kvh * p.group + rr % p.group) * D;
    c_log2[t] = k_mul;
    if constexpr (kFp8) {  // lane tig: dims 4 tig .. 4 tig + 3 of every k-step
      float big = 0.f;
      for (int ks = 0; ks < kKS; ++ks)
        for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(Elem<T>::to_f32(qp[ks * 16 + tig * 4 + e])));
      big = warp_max_xor(big, 4);
      // the row's largest value in [2^14, 2^15); exponents that would leave f32's range are cut
      const int ex = min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 127);
      const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
      c_log2[t] *= __uint_as_float((uint32_t)(127 - 14 + ex) << 23);
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        const T *q4 = qp + ks * 16 + tig * 4;
        qa[ks][2 * t] = dec_pack2<__half>(Elem<T>::to_f32(q4[0]) * up, Elem<T>::to_f32(q4[1]) * up);
        qa[ks][2 * t + 1] = dec_pack2<__half>(Elem<T>::to_f32(q4[2]) * up, Elem<T>::to_f32(q4[3]) * up);
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        qa[ks][2 * t] = __ldg(reinterpret_cast<const uint32_t *>(qp + ks * 16 + tig * 2));
        qa[ks][2 * t + 1] = __ldg(reinterpret_cast<const uint32_t *>(qp + ks * 16 + 8 + tig * 2));
      }
    }
    if (row[t] < 0) {
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) qa[ks][2 * t] = qa[ks][2 * t + 1] = 0u;
    }
  }
  const bool use_softcap = p.softcap != 1.f;
  // row i of the window sees tokens below n - query_len + 1 + i; all rows those below n_all
  const int n_all = n - p.query_len + 1;
  // this split's raw scores: token j of row r at x_split[r * x_stride + j - tok0]
  const int64_t pair = (int64_t)b * p.num_kv_heads + kvh;
  float *x_pair = p.ws_x + pair * p.scored_rows * p.x_stride;
  float *x_split = p.x_tokens ? reinterpret_cast<float *>(smem + C::kOffX) : x_pair + tok0;
  const int64_t x_stride = p.x_tokens ? p.x_tokens : p.x_stride;
  int seen[NRT];
  float *xrow[NRT];
#pragma unroll
  for (int t = 0; t < NRT; ++t) {
    seen[t] = row[t] < 0 ? 0 : n_all + row[t] / p.group - tok0;
    xrow[t] = nullptr;
    if (row[t] >= 0 && row[t] < p.scored_rows && !(kDup && grp >= 4))
      xrow[t] = x_split + row[t] * x_stride;
    if (!use_softcap) c_log2[t] *= kLog2e;
  }

  float o[NRT][D / 16][4];
  float m_used[NRT], l_part[NRT];
#pragma unroll
  for (int t = 0; t < NRT; ++t) {
    m_used[t] = -INFINITY;
    l_part[t] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[t][j][0] = o[t][j][1] = o[t][j][2] = o[t][j][3] = 0.f;
  }
  bool aborted = false;
  int u_abort = 0;
  for (int u = warp; u < n_units; u += C::kWarps) {
    const int s = u % NST;
    if (!mbar_wait_bounded(s_base + C::kOffBar + s * 8, (uint32_t)((u / NST) & 1))) {
      aborted = true;
      u_abort = u;
      break;
    }
    const uint32_t sk = s_base + C::kOffK + s * C::kSP * C::kPB;
    const uint32_t sv = s_base + C::kOffV + s * C::kSP * C::kPB;
    const int unit0 = u * C::kST;              // first token, relative to tok0
    const int valid = tok1 - tok0 - unit0;     // cached tokens of the stage
    const int whole = min(valid, n_all - tok0 - unit0);  // those that every row sees
#pragma unroll
    for (int ti = 0; ti < C::kTiles; ++ti) {
      const int t0 = ti * 16;
      if (t0 >= valid) break;
      // ---- S = Q K^T, two 8-token n-tiles
      float sacc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      if constexpr (kFp8) {
        const int r = lane & 7;
        const int ktok = t0 + 4 * (r >> 1) + 2 * ((lane >> 3) & 1) + (r & 1);
        const uint32_t krow = sk + (ktok / BS) * C::kPB + ((lane >> 4) * BS + ktok % BS) * 16;
#pragma unroll
        for (int kp = 0; kp < kKS / 2; ++kp) {
          uint32_t f[4];
          dec_ldmatrix_x4(krow + kp * 2 * (BS * 16), f[0], f[1], f[2], f[3]);
#pragma unroll
          for (int q2 = 0; q2 < 4; ++q2) {
            const int ks = 2 * kp + (q2 >> 1);
            dec_mma<TM>(sacc[q2 & 1], qa[ks][0], NRT > 1 ? qa[ks][2 * NRT - 2] : 0u, qa[ks][1],
                        NRT > 1 ? qa[ks][2 * NRT - 1] : 0u, fp8x2_to_h2(f[q2]), fp8x2_to_h2(f[q2] >> 16));
          }
        }
      } else {
        const int ktok = t0 + (lane & 7) + (lane >> 4) * 8;
        const uint32_t krow = sk + (ktok / BS) * C::kPB + (ktok % BS) * 16 + ((lane >> 3) & 1) * (BS * 16);
#pragma unroll
        for (int ks = 0; ks < kKS; ++ks) {
          uint32_t b0, b1, b2, b3;
          dec_ldmatrix_x4(krow + ks * 2 * (BS * 16), b0, b1, b2, b3);
          const uint32_t a1 = NRT > 1 ? qa[ks][2 * NRT - 2] : 0u, a3 = NRT > 1 ? qa[ks][2 * NRT - 1] : 0u;
          dec_mma<TM>(sacc[0], qa[ks][0], a1, qa[ks][1], a3, b0, b1);
          dec_mma<TM>(sacc[1], qa[ks][0], a1, qa[ks][1], a3, b2, b3);
        }
      }
      // ---- raw scores of the lane's rows, tokens tok(n, e) of the tile; only
      // a tile that not all rows see all of needs masks
      auto tok = [&](int nn, int e) { return kFp8 ? t0 + 4 * tig + 2 * nn + e : t0 + nn * 8 + tig * 2 + e; };
      const bool tail = t0 + 16 > whole;
      float pv[NRT][4];
      uint32_t pa[NRT][2];
#pragma unroll
      for (int t = 0; t < NRT; ++t) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = sacc[e >> 1][2 * t + (e & 1)] * c_log2[t];
          if (use_softcap) x[e] = p.softcap * tanhf(x[e] / p.softcap) * kLog2e;
        }
        if (tail) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = tok(e >> 1, e & 1);
            if (j >= valid || unit0 + j >= seen[t]) x[e] = -INFINITY;
          }
        }
        if (xrow[t]) {
          float *at = xrow[t] + unit0;
          if (tok(0, 0) < valid) *reinterpret_cast<float2 *>(at + tok(0, 0)) = make_float2(x[0], x[1]);
          if (tok(1, 0) < valid) *reinterpret_cast<float2 *>(at + tok(1, 0)) = make_float2(x[2], x[3]);
        }
        float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (__any_sync(0xffffffffu, mx > m_used[t] + kRescale)) {
          const float m_new = fmaxf(m_used[t], mx);
          const float alpha = m_used[t] == -INFINITY ? 0.f : scored_exp2(m_used[t] - m_new);
          m_used[t] = m_new;
          l_part[t] *= alpha;
          // O^T's columns 2 tig, 2 tig + 1 are rows whose alphas live in lanes 8 tig, 8 tig + 4
          const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * tig), a1 = __shfl_sync(0xffffffffu, alpha, 8 * tig + 4);
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            o[t][j][0] *= a0;
            o[t][j][1] *= a1;
            o[t][j][2] *= a0;
            o[t][j][3] *= a1;
          }
        }
        const float off = m_used[t] == -INFINITY ? 0.f : m_used[t];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pv[t][e] = scored_exp2(x[e] - off);
          l_part[t] += pv[t][e];
        }
#pragma unroll
        for (int nn = 0; nn < 2; ++nn) {
          pa[t][nn] = dec_pack2<TM>(pv[t][2 * nn], pv[t][2 * nn + 1]);
          if constexpr (kDup) {  // rows 4..7: what the rounding of rows 0..3 left
            const TM *h = reinterpret_cast<const TM *>(&pa[t][nn]);
            const uint32_t rest = dec_pack2<TM>(pv[t][2 * nn] - Elem<TM>::to_f32(h[0]),
                                                pv[t][2 * nn + 1] - Elem<TM>::to_f32(h[1]));
            if (grp >= 4) pa[t][nn] = rest;
          }
        }
      }
      // ---- O^T += V^T P^T over the tokens that every row sees
      if constexpr (kFp8) {
        const int vd = (lane >> 3) * 8 + (lane & 7);
        const uint32_t vrow = sv + (t0 / BS) * C::kPB + vd * BS + t0 % BS;
        const int tk = t0 + 4 * tig;
        const uint32_t mlo = (tk < whole ? 0xffffu : 0u) | (tk + 1 < whole ? 0xffff0000u : 0u);
        const uint32_t mhi = (tk + 2 < whole ? 0xffffu : 0u) | (tk + 3 < whole ? 0xffff0000u : 0u);
#pragma unroll
        for (int dq = 0; dq < D / 32; ++dq) {
          uint32_t r[4];
          dec_ldmatrix_x4(vrow + dq * 32 * BS, r[0], r[1], r[2], r[3]);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t a0 = fp8x2_to_h2(r[2 * hf]), a2 = fp8x2_to_h2(r[2 * hf] >> 16);
            uint32_t a1 = fp8x2_to_h2(r[2 * hf + 1]), a3 = fp8x2_to_h2(r[2 * hf + 1] >> 16);
            if (tail) {
              a0 &= mlo;
              a1 &= mlo;
              a2 &= mhi;
              a3 &= mhi;
            }
#pragma unroll
            for (int t = 0; t < NRT; ++t) dec_mma<TM>(o[t][dq * 2 + hf], a0, a1, a2, a3, pa[t][0], pa[t][1]);
          }
        }
      } else {
        const int vd = (lane & 7) + (lane >> 4) * 8;
        const int vtok = t0 + ((lane >> 3) & 1) * 8;
        const uint32_t vrow = sv + (vtok / BS) * C::kPB + (vd * BS + vtok % BS) * 2;
        const int tk = t0 + tig * 2;
        const uint32_t m0 = (tk < whole ? 0xffffu : 0u) | (tk + 1 < whole ? 0xffff0000u : 0u);
        const uint32_t m1 = (tk + 8 < whole ? 0xffffu : 0u) | (tk + 9 < whole ? 0xffff0000u : 0u);
#pragma unroll
        for (int dp = 0; dp < D / 16; ++dp) {
          uint32_t b0, b1, b2, b3;
          dec_ldmatrix_x4(vrow + dp * 16 * BS * 2, b0, b1, b2, b3);
          if (tail) {
            b0 &= m0;
            b2 &= m0;
            b1 &= m1;
            b3 &= m1;
          }
#pragma unroll
          for (int t = 0; t < NRT; ++t) dec_mma<TM>(o[t][dp], b0, b2, b1, b3, pa[t][0], pa[t][1]);
        }
      }
      // ---- tokens that only some rows see, one by one
      if (tail && whole < valid) {
        const unsigned char *vp = smem + C::kOffV + s * C::kSP * C::kPB;
        for (int j = max(t0, whole); j < min(t0 + 16, valid); ++j) {
          const int jt = j - t0;
          const int src = kFp8 ? jt >> 2 : (jt & 7) >> 1;                 // tig of the token's lane
          const int at = kFp8 ? jt & 3 : 2 * (jt >> 3) + (jt & 1);        // its place there
#pragma unroll
          for (int t = 0; t < NRT; ++t) {
            float w[2];
            bool sees[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {  // the lane's columns of O^T: rows 2 tig + e
              const int from = (2 * tig + e) * 4 + src;
              float v0 = __shfl_sync(0xffffffffu, pv[t][0], from), v1 = __shfl_sync(0xffffffffu, pv[t][1], from);
              float v2 = __shfl_sync(0xffffffffu, pv[t][2], from), v3 = __shfl_sync(0xffffffffu, pv[t][3], from);
              w[e] = at == 0 ? v0 : at == 1 ? v1 : at == 2 ? v2 : v3;
              sees[e] = unit0 + j < __shfl_sync(0xffffffffu, seen[t], (2 * tig + e) * 4);
              if (kDup && tig >= 2) sees[e] = false;  // the doubled rows' columns
            }
#pragma unroll
            for (int jd = 0; jd < D / 16; ++jd)
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                const int d = jd * 16 + hf * 8 + grp;
                const TC v = reinterpret_cast<const TC *>(vp + (j / BS) * C::kPB)[d * BS + j % BS];
                if (sees[0]) o[t][jd][2 * hf] = fmaf(w[0], Elem<TC>::to_f32(v), o[t][jd][2 * hf]);
                if (sees[1]) o[t][jd][2 * hf + 1] = fmaf(w[1], Elem<TC>::to_f32(v), o[t][jd][2 * hf + 1]);
              }
          }
        }
      }
    }
    __syncwarp();
    const int nu = u + NST;
    if (nu < n_units && lane == 0) {
      fence_proxy_async_smem();
      issue_unit(nu);
    }
  }
  if (aborted) {  // the copies this warp has in flight land before the ring is reused
    for (int v = u_abort; v < min(u_abort + NST, n_units); v += C::kWarps)
      mbar_wait_bounded(s_base + C::kOffBar + (v % NST) * 8, (uint32_t)((v / NST) & 1));
  }
  __syncthreads();  // every stage is read: the ring becomes the warps' O

  float *co = reinterpret_cast<float *>(smem);  // [warp][kRows][D]
  float2 *cml = reinterpret_cast<float2 *>(smem + C::kOffML);  // [warp][16]
#pragma unroll
  for (int t = 0; t < NRT; ++t) {
    float l = l_part[t];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (tig == 0 && !(kDup && grp >= 4))
      cml[warp * 16 + 8 * t + grp] = aborted ? make_float2(-INFINITY, 0.f) : make_float2(m_used[t], l);
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = o[t][j][e];
        if constexpr (kDup) v += __shfl_xor_sync(0xffffffffu, v, 2);  // rows r and r + 4
        const int r = 8 * t + 2 * tig + (e & 1), d = j * 16 + (e >> 1) * 8 + grp;
        if (r < kRows) co[(warp * kRows + r) * D + d] = v;
      }
  }
  __syncthreads();
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
    weights.load(p, b, kvh, BS, 0, n, x_split, x_stride);
    for (int e = tid; e < rows_here * D; e += kScoredThreads) {
      const int r = e / D, d = e % D;
      const float2 f = row_total(r);
      const float inv = f.y != 0.f ? 1.f / f.y : 0.f;
      if (d == 0) fin[r] = f.y != 0.f ? make_float2(f.x, inv) : make_float2(0.f, 0.f);
      scored_out_row<T>(p, b, kvh, r)[d] = Elem<T>::from_f32(row_dim(r, d, f.x) * inv * v_mul);
    }
    __syncthreads();
    weights.finish(p, fin, x_split, x_stride);
    for (int j = kWeightTokens; j < n; j += kWeightTokens) {  // splits of pages of 32 tokens may be longer
      weights.load(p, b, kvh, BS, j, n, x_split, x_stride);
      weights.finish(p, fin, x_split, x_stride);
    }
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
            *reinterpret_cast<const float4 *>(x_split + r * x_stride + j);
  }
}

// The end of every (sequence, kv head) of several splits (or row tiles):
// blocks [0, chunks) add the weights of `chunk` tokens each, the others join
// the rows: a warp has a row, or all warps share one where there are many
// splits (row_warps = 4).
template <typename T>
__global__ void __launch_bounds__(kScoredThreads, 10) scored_join_kernel(const ScoredMmaParams p, int bs, int chunk,
                                                                         int chunks, int row_warps) {
  __shared__ float2 fin[kScoredMaxRows];
  __shared__ float4 part[kScoredThreads];
  constexpr int kWarps = kScoredThreads / 32;
  const int kvh = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = scored_context(p, b, bs, false);
  const int n_splits = scored_splits(n, p.pages_per_split, bs);
  const int64_t pair = (int64_t)b * p.num_kv_heads + kvh;
  if (n_splits == 0 || (n_splits == 1 && p.row_tiles == 1)) return;
  if ((int)blockIdx.x < chunks) {
    const int j0 = blockIdx.x * chunk, j1 = min(n, j0 + chunk);
    if (j0 >= n) return;
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
