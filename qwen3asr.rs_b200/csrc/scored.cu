// scored.cu — paged attention of a few new tokens that also accumulates every
// cached token's attention weight.
//
// Row (i, head) of sequence b, i < query_len, sits at position
// len_b - query_len + i and sees the tokens up to there (a row before the
// first token sees none and gives zeros):
//   x_j = scale q . k_j   (softcapped when asked),  p_j = softmax(x)_j,
//   out = sum_j p_j v_j,
//   score_j <- decay score_j + sum over i < score_rows and the kv head's query
//              heads of p_j                       for every j < len_b.
// The weights need the whole row's maximum and sum, which a split of the
// context does not have: each split leaves its raw scores x (log2 domain) and
// its partial (o, m, l) in the workspace, a merge makes out and the final
// (m, l) of every row, and the last step turns the raw scores into weights.
// head_dim 128 runs scored_mma_kernel (16-bit queries, scored_mma.cuh) or
// scored_f32_kernel (f32 queries and pages, scored_f32.cuh); the kernels here
// serve the other shapes, one thread a token, three launches (121 us for one
// sequence of 16381 tokens, 2410 us for 512 of 64 to 4096, which the others
// take 17 and 317 us for). Comparisons below that name 324 us were made
// while the join's registers spilled, which cost 7 us on both sides.
#include "common.cuh"
#include "launch.h"
#include "scored_f32.cuh"
#include "scored_mma.cuh"

namespace vasr {
namespace {

constexpr int kSplitTokens = 256;
constexpr int kThreads = 128;
constexpr int kMergeThreads = 128;
constexpr int kWeightThreads = 256;

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// ---- the split kernels: which calls they take, their splits and workspace
bool takes_split(const ScoredArgs &a) {
  const int rows = a.query_len * (a.num_heads / a.num_kv_heads);
  const bool fp8 = a.cache_dtype == VASR_PA_FP8_E4M3;
  return a.head_dim == kScoredDim && rows <= kScoredMaxRows && !(fp8 && (a.block_size < 16 || a.dtype == VASR_PA_F32)) &&
         (int64_t)a.num_kv_heads * ((rows + 1) / 2) <= 65535;
}

constexpr int kSplitMostTokens = 1024, kSplitFewTokens = 640, kSplitFewPairs = 4 * 148;
static_assert(kSplitMostTokens <= kWeightTokens, "a context of one split has its scores added in one turn");

struct SplitLayout {
  int pages_per_split, max_splits;
  int64_t x_stride;
  size_t off_o, off_ml, off_x, total;
};
SplitLayout split_layout(int num_seqs, int query_len, int score_rows, int num_heads, int num_kv_heads, int block_size,
                     int max_context_len) {
  SplitLayout l;
  // Splits of 1024 tokens, or shorter ones that just fill the SMs once (three
  // CTAs each) where the longest contexts would leave some idle; at least 64.
  // 512 sequences of 64 to 4096 tokens, 8 kv heads: 324 us with 1024, 325 with
  // 768, 333 with 512, 393 with 256 (more partial results to join). One of
  // 16381: 17.9 us with three CTAs a SM, 21.1 with four, of which the last wait
  // for places. Few (sequence, kv head)s of up to two splits end at different
  // times: 640 tokens took 50.4 against 55.9 us for 64 windows of 5 rows over
  // 200 to 1500 tokens, 29.9 / 36.1 for 32, 42.4 / 45.2 for 64 of 4 rows, 38.3 /
  // 40.1 for 64 single tokens, 76 / 79 in f32, 30.9 / 30.8 from fp8 pages; but
  // (with P in one part) 82.6 / 78.7 for 128 windows, 192 / 186 for 64 windows
  // over 4000 tokens. Between 512 and 1024 pairs nothing was measured.
  const int64_t pairs = (int64_t)num_seqs * num_kv_heads;
  const int64_t pages = ((int64_t)max_context_len + block_size - 1) / block_size;
  int64_t per_pair = 3 * 148 / pairs;
  if (per_pair < 1) per_pair = 1;
  int64_t want = (pages + per_pair - 1) / per_pair;
  const int least = (64 + block_size - 1) / block_size;
  const bool few = pairs <= kSplitFewPairs && max_context_len <= 2 * kSplitMostTokens;
  const int most = (few ? kSplitFewTokens : kSplitMostTokens) / block_size;
  l.pages_per_split = (int)(want < least ? least : want > most ? most : want);
  if (l.pages_per_split > kScoredMaxPages) l.pages_per_split = kScoredMaxPages;
  const int per = l.pages_per_split * block_size;
  l.max_splits = (int)(((int64_t)max_context_len + per - 1) / per);
  l.x_stride = (int64_t)l.max_splits * per;
  const size_t rows = (size_t)num_seqs * num_kv_heads * l.max_splits * query_len * (num_heads / num_kv_heads);
  l.off_o = 0;
  l.off_ml = align256(l.off_o + rows * kScoredDim * sizeof(float));
  l.off_x = align256(l.off_ml + rows * sizeof(float2));
  l.total = l.off_x + align256((size_t)num_seqs * score_rows * num_heads * l.x_stride * sizeof(float));
  return l;
}

// ---- the other kernels
struct ScoredLayout {
  int splits;         // of max_context_len
  int64_t x_stride;   // raw scores of one row
  size_t off_o, off_ml, off_x, total;
};
ScoredLayout layout(int num_seqs, int query_len, int score_rows, int num_heads, int head_dim, int max_context_len) {
  ScoredLayout l;
  l.splits = (int)(((int64_t)max_context_len + kSplitTokens - 1) / kSplitTokens);
  l.x_stride = (int64_t)l.splits * kSplitTokens;
  const size_t rows = (size_t)num_seqs * query_len * num_heads;
  l.off_o = 0;
  l.off_ml = align256(l.off_o + rows * l.splits * head_dim * sizeof(float));
  l.off_x = align256(l.off_ml + rows * (l.splits + 1) * sizeof(float2));
  l.total = l.off_x + align256((size_t)num_seqs * score_rows * num_heads * l.x_stride * sizeof(float));
  return l;
}

struct ScoredParams {
  ScoredArgs a;
  float *o;       // [row][split][D]
  float2 *ml;     // [row][split], the merged one at [row][splits]
  float *x;       // [scored row][x_stride]
  int splits;
  int64_t x_stride;
  int group;      // query heads per kv head
};

__device__ __forceinline__ int context_of(const ScoredArgs &a, int b) {
  int64_t n = a.context_lens[b];
  const int64_t cap = min((int64_t)a.max_num_blocks_per_seq * a.block_size, (int64_t)a.max_context_len);
  if (n > cap) {
    raise_device_error(VASR_PA_DERR_CTX_RANGE);
    n = cap;
  }
  return (int)n;
}
// The page to read for token j: block 0 stands in for one that is none of the pool's.
__device__ __forceinline__ int64_t page_of(const ScoredArgs &a, int b, int j) {
  const uint32_t id = a.block_tables[(int64_t)b * a.max_num_blocks_per_seq + j / a.block_size];
  if ((int64_t)id < a.num_blocks) return id;
  raise_device_error(VASR_PA_DERR_BLOCK_RANGE);
  return 0;
}
// Row r = (i, head): i * num_heads + head.
__device__ __forceinline__ int64_t row_index(const ScoredArgs &a, int b, int i, int head) {
  return ((int64_t)b * a.query_len + i) * a.num_heads + head;
}

__device__ __forceinline__ float block_reduce(float v, bool is_max) {
  __shared__ float part[kThreads / 32];
  v = is_max ? warp_max_xor(v, 32) : warp_sum_xor(v, 32);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
  for (int w = 1; w < kThreads / 32; ++w) v = is_max ? fmaxf(v, part[w]) : v + part[w];
  __syncthreads();
  return v;
}

// One (split, query head, sequence): every row of the window over the split.
template <typename T, typename TC>
__global__ void __launch_bounds__(kThreads) scored_split_kernel(const ScoredParams p) {
  const ScoredArgs &a = p.a;
  const int split = blockIdx.x, head = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int D = a.head_dim, BS = a.block_size, kvh = head / p.group;
  constexpr int kX = Elem<TC>::kX;
  extern __shared__ float smem[];
  float *q = smem, *w = smem + D;
  const int n = context_of(a, b);
  const int t0 = split * kSplitTokens;
  if (t0 >= n) return;
  const int t1 = min(n, t0 + kSplitTokens);
  const TC *kc = static_cast<const TC *>(a.key_cache);
  const TC *vc = static_cast<const TC *>(a.value_cache);
  const float k_mul = a.k_scale ? a.scale * __ldg(a.k_scale) : a.scale;
  for (int i = 0; i < a.query_len; ++i) {
    const int64_t row = row_index(a, b, i, head);
    const int seen = min(t1, n - a.query_len + i + 1);  // tokens [t0, seen) are visible
    const T *qp = static_cast<const T *>(a.query) + ((int64_t)b * a.query_len + i) * a.q_token_stride + (int64_t)head * D;
    for (int d = tid; d < D; d += kThreads) q[d] = Elem<T>::to_f32(qp[d]);
    __syncthreads();
    float *x = nullptr;
    if (i < a.score_rows) x = p.x + (((int64_t)b * a.score_rows + i) * a.num_heads + head) * p.x_stride;
    float m = -INFINITY;
    for (int j = t0 + tid; j < t1; j += kThreads) {
      float s = -INFINITY;
      if (j < seen) {
        const TC *k = kc + (page_of(a, b, j) * a.num_kv_heads + kvh) * (int64_t)D * BS + (j % BS) * kX;
        float dot = 0.f;
        for (int c = 0; c < D / kX; ++c) {
          float f[kX];
          unpack_chunk<TC>(*reinterpret_cast<const uint4 *>(k + (int64_t)c * BS * kX), f);
#pragma unroll
          for (int e = 0; e < kX; ++e) dot = fmaf(q[c * kX + e], f[e], dot);
        }
        s = dot * k_mul;
        if (a.softcapping != 1.f) s = a.softcapping * tanhf(s / a.softcapping);
        s *= kLog2e;
      }
      if (x) x[j] = s;
      w[j - t0] = s;
      m = fmaxf(m, s);
    }
    m = block_reduce(m, true);
    float l = 0.f;
    for (int j = t0 + tid; j < t1; j += kThreads) {
      const float e = w[j - t0] == -INFINITY ? 0.f : exp2f(w[j - t0] - m);
      w[j - t0] = e;
      l += e;
    }
    l = block_reduce(l, false);
    for (int d = tid; d < D; d += kThreads) {
      float o = 0.f;
      for (int j = t0; j < seen; ++j) {
        const TC *v = vc + (page_of(a, b, j) * a.num_kv_heads + kvh) * (int64_t)D * BS;
        o = fmaf(w[j - t0], Elem<TC>::to_f32(v[(int64_t)d * BS + j % BS]), o);
      }
      p.o[(row * p.splits + split) * D + d] = o;
    }
    if (tid == 0) p.ml[row * (p.splits + 1) + split] = make_float2(m, l);
    __syncthreads();
  }
}

// One row: the splits' partials into out and the row's final (m, l).
template <typename T>
__global__ void __launch_bounds__(kMergeThreads) scored_merge_kernel(const ScoredParams p) {
  const ScoredArgs &a = p.a;
  const int64_t row = blockIdx.x;
  const int b = (int)(row / ((int64_t)a.query_len * a.num_heads));
  const int n = context_of(a, b);
  const int splits = (n + kSplitTokens - 1) / kSplitTokens;
  const float2 *ml = p.ml + row * (p.splits + 1);
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, ml[s].x);
  for (int s = 0; s < splits; ++s)
    if (ml[s].y != 0.f) l = fmaf(ml[s].y, exp2f(ml[s].x - m), l);
  const float v_mul = a.v_scale ? __ldg(a.v_scale) : 1.f;
  for (int d = threadIdx.x; d < a.head_dim; d += kMergeThreads) {
    float o = 0.f;
    for (int s = 0; s < splits; ++s)
      if (ml[s].y != 0.f) o = fmaf(p.o[(row * p.splits + s) * a.head_dim + d], exp2f(ml[s].x - m), o);
    static_cast<T *>(a.out)[row * a.head_dim + d] = Elem<T>::from_f32(l != 0.f ? o / l * v_mul : 0.f);
  }
  if (threadIdx.x == 0) p.ml[row * (p.splits + 1) + p.splits] = make_float2(m, l);
}

// The weights of the scored rows, added to the tokens' scores.
__global__ void __launch_bounds__(kWeightThreads) scored_weight_kernel(const ScoredParams p) {
  const ScoredArgs &a = p.a;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int n = context_of(a, b);
  const int j = blockIdx.x * kWeightThreads + threadIdx.x;
  if (j >= n) return;
  const uint32_t id = a.block_tables[(int64_t)b * a.max_num_blocks_per_seq + j / a.block_size];
  if ((int64_t)id >= a.num_blocks) return;  // no page of the pool's (recorded where it was read): no score
  float sum = 0.f;
  for (int i = 0; i < a.score_rows; ++i)
    for (int g = 0; g < p.group; ++g) {
      const int head = kvh * p.group + g;
      const float2 ml = p.ml[row_index(a, b, i, head) * (p.splits + 1) + p.splits];
      const float x = p.x[(((int64_t)b * a.score_rows + i) * a.num_heads + head) * p.x_stride + j];
      if (ml.y != 0.f) sum += exp2f(x - ml.x) / ml.y;
    }
  float *s = a.score_cache + ((int64_t)id * a.num_kv_heads + kvh) * a.block_size + j % a.block_size;
  *s = a.decay * *s + sum;
}

template <typename T, typename TC>
int launch_scored_t(const ScoredArgs &a, cudaStream_t s) {
  const ScoredLayout l =
      layout(a.num_seqs, a.query_len, a.score_rows, a.num_heads, a.head_dim, a.max_context_len);
  unsigned char *ws = static_cast<unsigned char *>(a.workspace);
  ScoredParams p{a, reinterpret_cast<float *>(ws + l.off_o), reinterpret_cast<float2 *>(ws + l.off_ml),
                 reinterpret_cast<float *>(ws + l.off_x), l.splits, l.x_stride, a.num_heads / a.num_kv_heads};
  const int64_t rows = (int64_t)a.num_seqs * a.query_len * a.num_heads;
  if (rows > 0x7fffffff) return VASR_PA_EINVAL_SHAPE;
  scored_split_kernel<T, TC><<<dim3((unsigned)l.splits, (unsigned)a.num_heads, (unsigned)a.num_seqs), kThreads,
                               (a.head_dim + kSplitTokens) * sizeof(float), s>>>(p);
  scored_merge_kernel<T><<<(unsigned)rows, kMergeThreads, 0, s>>>(p);
  const unsigned chunks = ((unsigned)a.max_context_len + kWeightThreads - 1) / kWeightThreads;
  scored_weight_kernel<<<dim3(chunks, (unsigned)a.num_kv_heads, (unsigned)a.num_seqs), kWeightThreads, 0, s>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? VASR_PA_OK : VASR_PA_ELAUNCH;
}

// Launches kern, a split kernel of tiles of tile_rows rows, and the join where one is needed.
template <typename T, typename C, int BS>
int launch_split(const ScoredArgs &a, void (*kern)(ScoredSplitParams), std::atomic<uint64_t> &attr_done, int tile_rows,
                 cudaStream_t s) {
  const SplitLayout l = split_layout(a.num_seqs, a.query_len, a.score_rows, a.num_heads, a.num_kv_heads, a.block_size,
                                 a.max_context_len);
  unsigned char *ws = static_cast<unsigned char *>(a.workspace);
  ScoredSplitParams p{};
  p.out = a.out;
  p.q = a.query;
  p.k_cache = a.key_cache;
  p.v_cache = a.value_cache;
  p.score_cache = a.score_cache;
  p.block_tables = a.block_tables;
  p.context_lens = a.context_lens;
  p.k_scale = a.k_scale;
  p.v_scale = a.v_scale;
  p.ws_o = reinterpret_cast<float *>(ws + l.off_o);
  p.ws_ml = reinterpret_cast<float2 *>(ws + l.off_ml);
  p.ws_x = reinterpret_cast<float *>(ws + l.off_x);
  p.q_token_stride = a.q_token_stride;
  p.num_blocks = a.num_blocks;
  p.x_stride = l.x_stride;
  p.num_heads = a.num_heads;
  p.num_kv_heads = a.num_kv_heads;
  p.group = a.num_heads / a.num_kv_heads;
  p.query_len = a.query_len;
  p.rows = a.query_len * p.group;
  p.scored_rows = a.score_rows * p.group;
  p.row_tiles = (p.rows + tile_rows - 1) / tile_rows;
  p.cols = a.max_num_blocks_per_seq;
  p.max_context = a.max_context_len;
  p.pages_per_split = l.pages_per_split;
  p.max_splits = l.max_splits;
  const int split_tokens = l.pages_per_split * BS;
  p.x_tokens = (size_t)p.scored_rows * split_tokens * sizeof(float) <= (size_t)C::kXBytes ? split_tokens : 0;
  p.scale = a.scale;
  p.softcap = a.softcapping;
  p.decay = a.decay;
  if (!ensure_smem_attr(kern, C::kSmemBytes, attr_done)) return VASR_PA_ELAUNCH;
  const dim3 grid((unsigned)l.max_splits, (unsigned)(a.num_kv_heads * p.row_tiles), (unsigned)a.num_seqs);
  kern<<<grid, kScoredThreads, C::kSmemBytes, s>>>(p);
  if (l.max_splits == 1 && p.row_tiles == 1) return cudaPeekAtLastError() == cudaSuccess ? VASR_PA_OK : VASR_PA_ELAUNCH;
  // the join: as many tokens a CTA as leave about 16 CTAs per SM, 512 at least
  // (512 for every call: 331 against 324 us for 512 sequences); rows of more
  // than 8 splits take a CTA each (18 us for one sequence, against 22 with a
  // warp each; at 4 splits the CTA is 326 against 324 us)
  const int64_t pairs = (int64_t)a.num_seqs * a.num_kv_heads;
  int chunk = 512;
  auto chunks_of = [&](int tokens) { return (int)(((int64_t)a.max_context_len + tokens - 1) / tokens); };
  while (chunk < a.max_context_len && chunk < 1 << 30 && pairs * chunks_of(chunk) > 16 * 148) chunk *= 2;
  const int chunks = chunks_of(chunk);
  const int row_warps = l.max_splits <= 8 ? 1 : kScoredThreads / 32;
  const int row_ctas = (p.rows * row_warps + kScoredThreads / 32 - 1) / (kScoredThreads / 32);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(chunks + row_ctas), (unsigned)a.num_kv_heads, (unsigned)a.num_seqs);
  cfg.blockDim = dim3(kScoredThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  return cudaLaunchKernelEx(&cfg, scored_join_kernel<T>, p, BS, chunk, chunks, row_warps) == cudaSuccess ? VASR_PA_OK : VASR_PA_ELAUNCH;
}

// Stages of the ring: 32 KB of pages or more in flight a CTA (with half of it
// and four CTAs a SM, 336 against 324 us for 512 sequences).
template <typename TC, int BS>
constexpr int ring_stages() {
  return 2 * (BS < 16 ? 16 : BS) * kScoredDim * (int)sizeof(TC) <= 8192 ? 8 : 4;
}

template <typename T, typename TC, int BS, int NRT, bool kDup>
int launch_mma_rows(const ScoredArgs &a, cudaStream_t s) {
  // one-byte pages leave room for four CTAs a SM: 31 against 34 us for 64
  // sequences of 200 to 1500 tokens; but windows, whose P comes in two
  // products, would spill there (windows of 4 rows 42.8 against 38.9 us)
  constexpr int kNST = ring_stages<TC, BS>(), kMinB = sizeof(TC) == 1 && kDup ? 4 : 3;
  static std::atomic<uint64_t> attr_done{0};
  return launch_split<T, ScoredCfg<TC, BS, kNST>, BS>(a, scored_mma_kernel<T, TC, BS, NRT, kDup, kNST, kMinB>, attr_done,
                                                      kDup ? 4 : 8 * NRT, s);
}

template <int BS, int kRows>
int launch_f32_rows(const ScoredArgs &a, cudaStream_t s) {
  constexpr int kNST = ring_stages<float, BS>();
  static std::atomic<uint64_t> attr_done{0};
  return launch_split<float, ScoredCfg<float, BS, kNST>, BS>(a, scored_f32_kernel<BS, kRows, kNST>, attr_done, kRows, s);
}

template <int BS>
int launch_f32_bs(const ScoredArgs &a, cudaStream_t s) {
  const int rows = a.query_len * (a.num_heads / a.num_kv_heads);
  if (rows <= 2) return launch_f32_rows<BS, 2>(a, s);
  if (rows <= 4) return launch_f32_rows<BS, 4>(a, s);
  return launch_f32_rows<BS, 8>(a, s);
}

template <typename T, typename TC, int BS>
int launch_mma_bs(const ScoredArgs &a, cudaStream_t s) {
  const int rows = a.query_len * (a.num_heads / a.num_kv_heads);
  // Doubled rows cost nothing in time (18.3 / 17.9 us without / with them for
  // one sequence) and are taken wherever they fit. Tiles of 16 rows for 8 rows
  // would: 50 against 44 us for 64 sequences' windows of 4 rows.
  if (rows <= 4) return launch_mma_rows<T, TC, BS, 1, true>(a, s);
  if (rows <= 8) return launch_mma_rows<T, TC, BS, 1, false>(a, s);
  return launch_mma_rows<T, TC, BS, 2, false>(a, s);
}

template <typename T>
int launch_scored_c(const ScoredArgs &a, cudaStream_t s) {
  if constexpr (std::is_same<T, float>::value) {
    if (takes_split(a)) {
      switch (a.block_size) {
        case 8: return launch_f32_bs<8>(a, s);
        case 16: return launch_f32_bs<16>(a, s);
        default: return launch_f32_bs<32>(a, s);
      }
    }
  } else {
    if (takes_split(a)) {
      if (a.cache_dtype == VASR_PA_FP8_E4M3)
        return a.block_size == 16 ? launch_mma_bs<T, __nv_fp8_e4m3, 16>(a, s) : launch_mma_bs<T, __nv_fp8_e4m3, 32>(a, s);
      switch (a.block_size) {
        case 8: return launch_mma_bs<T, T, 8>(a, s);
        case 16: return launch_mma_bs<T, T, 16>(a, s);
        default: return launch_mma_bs<T, T, 32>(a, s);
      }
    }
  }
  if (a.cache_dtype == VASR_PA_FP8_E4M3) return launch_scored_t<T, __nv_fp8_e4m3>(a, s);
  return launch_scored_t<T, T>(a, s);
}

}  // namespace

size_t scored_workspace_bytes(int num_seqs, int query_len, int score_rows, int num_heads, int num_kv_heads,
                              int head_dim, int block_size, int max_context_len) {
  const size_t mma =
      head_dim == kScoredDim
          ? split_layout(num_seqs, query_len, score_rows, num_heads, num_kv_heads, block_size, max_context_len).total
          : 0;
  const size_t other = layout(num_seqs, query_len, score_rows, num_heads, head_dim, max_context_len).total;
  return mma > other ? mma : other;
}

int launch_scored(const ScoredArgs &a, cudaStream_t s) {
  switch (a.dtype) {
    case VASR_PA_F32: return launch_scored_c<float>(a, s);
    case VASR_PA_BF16: return launch_scored_c<__nv_bfloat16>(a, s);
    case VASR_PA_F16: return launch_scored_c<__half>(a, s);
    default: return VASR_PA_EINVAL_DTYPE;
  }
}

uint32_t *error_word_scored() { return unit_error_word(); }

}  // namespace vasr
