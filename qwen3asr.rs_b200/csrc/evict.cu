// evict.cu — shrinking a sequence's cache to the tokens that were attended to.
//
// Per (sequence, kv head) the tokens that stay are the first num_sink, the
// last num_recent and, among the others, those of the largest accumulated
// attention weight (score_cache), budget of them in all; equal scores keep the
// lower index and NaN counts as the lowest score. They move, in their old
// order, to token places 0 .. budget - 1 of the sequence: every kv head keeps
// its own set, which the page layout allows because a block holds each head's
// tokens apart.
//
// Selection is a radix select over order-preserving keys of the scores, kept
// in shared memory: a histogram of one byte per pass, at most four passes, and
// a last one that lists the survivors by rank. A CTA has a (sequence, kv head);
// long contexts of few sequences take a cluster of CTAs, which add their
// histograms up over distributed shared memory. It is bound by latency: 8
// heads of 4099 tokens take about 8 us of launch, loads and barriers. Plain
// shared atomics count fastest, equal scores included: one count per distinct
// digit of a warp, found by a match, took 2 us more.
//
// The move copies bits, bound by memory: it reads every 32-byte sector that
// holds a kept token and writes the kept ones. A sector of V holds 16 tokens
// of one dim (16-bit pages), so that nearly all of V is read whatever stays:
// 640 of 700 to 1500 tokens of 64 sequences are 342 MB of kept K, V and scores,
// 428 MB of sectors, and take 92 us with the selection (the move alone 81% of
// the copy rate in sectors). In place, token r of the result comes from an
// index >= r, so places filled in ascending tiles never overwrite a token that
// is still needed, as long as a tile is read before it or a later one is
// written: a CTA moves its slices of the head dimension of one (sequence,
// head) that way. Measured slower: tables and indices fetched a tile or two
// ahead (114 us: the registers cost a fifth of the loads in flight), 6 CTAs an
// SM (127 us), 8 K chunks or 32 V rows a unit (97 and 99 us), and tiles of one
// (sequence, head) shared among CTAs when the pages do not overlap (no gain).
#include <cooperative_groups.h>

#include "common.cuh"
#include "launch.h"

namespace cg = cooperative_groups;

namespace vasr {
namespace {

constexpr int kSelectThreads = 512;
constexpr int kSelectMostThreads = 1024;  // at most 148 (sequence, head)s: 13.8 against 15.3 us for 8 of 4099 tokens
// Keys in a CTA's shared memory: 32 KB, or most of an SM's where every CTA has
// one to itself (one CTA a head of 20000 tokens: 43 against 57 us for 8 heads, 85
// / 101 for 32).
constexpr int kKeys = 8192, kMostKeys = 49152;
// Longer contexts of up to 74 (sequence, head)s take clusters of up to 8 CTAs:
// 20.5 against 22.5 us at 8 heads of 9000 tokens, 29 / 43 at 20000, 75 / 85 at 32
// heads of 20000; but 15.3 / 13.8 at 8 of 4099, 23 / 20 at 32 of 4099.
constexpr int kClusterTokens = 8192, kMostClusterCtas = 8;
constexpr int kMoveThreads = 256;
constexpr int kMoveMostThreads = 1024;
constexpr int kMoveCtas = 8 * 148;

// Unsigned keys in the order of the scores (-0 = 0, NaN lowest); tokens that
// always stay are above every score.
__device__ __forceinline__ uint32_t score_key(float s) {
  if (!(s == s)) s = -INFINITY;
  const uint32_t u = __float_as_uint(s + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Sequence {
  int len;     // tokens in the cache
  int budget;  // tokens that stay
};
__device__ __forceinline__ Sequence sequence_of(const EvictArgs &p, int b) {
  Sequence q;
  int64_t len = p.context_lens[b];
  const int64_t cap = min((int64_t)p.cols * p.block_size, (int64_t)p.max_context_len);
  if (len > cap) {
    raise_device_error(VASR_PA_DERR_CTX_RANGE);
    len = cap;
  }
  q.len = (int)len;
  q.budget = p.budget;
  if (p.budgets) q.budget = (int)min(p.budgets[b], (uint32_t)p.budget);
  q.budget = min(q.budget, q.len);
  return q;
}

// Block id of column `col`; -1 (and recorded) where it is none of the pool's.
__device__ __forceinline__ int64_t block_at(const uint32_t *table, int col, int64_t num_blocks) {
  const uint32_t id = __ldg(table + col);
  if ((int64_t)id < num_blocks) return id;
  raise_device_error(VASR_PA_DERR_BLOCK_RANGE);
  return -1;
}

// kept[b, h, :] = the indices that stay, ascending, then -1. The CTAs of a
// (sequence, head) form a cluster (kCluster; else there is one) and have a
// stretch of its tokens each; the keys of a stretch's first key_cap tokens fit
// the dynamic shared memory, those past them are made anew on every pass.
template <int kThreads, bool kCluster>
__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictArgs p, int key_cap) {
  extern __shared__ uint32_t s_key[];
  __shared__ int s_hist[4][256], s_total[256];  // a pass's own counts, and the cluster's
  __shared__ int s_above[kThreads / 32], s_ties[kThreads / 32];
  __shared__ int2 s_cta;
  __shared__ uint32_t s_prefix;
  __shared__ int s_rank, s_done;
  pdl_launch_dependents();
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = kCluster ? (int)cluster.num_blocks() : 1, cta = kCluster ? (int)cluster.block_rank() : 0;
  const int h = blockIdx.x / ctas, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int shift = 31 - __clz(p.block_size);
  const Sequence q = sequence_of(p, b);
  int32_t *kept = p.kept + ((int64_t)b * p.num_kv_heads + h) * p.budget;
  if (blockIdx.x == 0 && tid == 0) p.new_lens[b] = (uint32_t)q.budget;
  for (int i = q.budget + cta * kThreads + tid; i < p.budget; i += ctas * kThreads) kept[i] = -1;
  if (q.len == q.budget) {
    for (int i = cta * kThreads + tid; i < q.budget; i += ctas * kThreads) kept[i] = i;
    return;
  }
  if (q.budget == 0) return;
  const uint32_t *table = p.block_tables + (int64_t)b * p.cols;
  const int recent0 = q.len - p.num_recent;
  const int stretch = (q.len + ctas - 1) / ctas, t0 = min(cta * stretch, q.len), t1 = min(t0 + stretch, q.len);
  auto make_key = [&](int j) -> uint32_t {
    const int64_t blk = block_at(table, j >> shift, p.num_blocks);
    if (j < p.num_sink || j >= recent0) return 0xffffffffu;
    if (blk < 0) return 0u;
    return score_key(p.score_cache[((blk * p.num_kv_heads + h) << shift) + (j & (p.block_size - 1))]);
  };
#pragma unroll 4
  for (int j = tid; j < min(t1 - t0, key_cap); j += kThreads) s_key[j] = make_key(t0 + j);
  auto key_of = [&](int j) { return j - t0 < key_cap ? s_key[j - t0] : make_key(j); };
  for (int i = tid; i < 4 * 256; i += kThreads) s_hist[i / 256][i % 256] = 0;
  __syncthreads();
  // ---- the key of rank `budget` from above, one byte of it per pass
  uint32_t prefix = 0, mask = 0;
  int rank = q.budget;  // 1-based rank among the keys that match the prefix
  for (int shift8 = 24; shift8 >= 0; shift8 -= 8) {
    int *hist = s_hist[shift8 / 8];
    for (int j0 = t0; j0 < t1; j0 += kThreads) {
      const int j = j0 + tid;
      const uint32_t key = j < t1 ? key_of(j) : 0u;
      const bool in = j < t1 && (key & mask) == prefix;
      if (in) atomicAdd(&hist[(key >> shift8) & 255u], 1);
    }
    if constexpr (kCluster) {
      cluster.sync();
      if (tid < 256) {
        int sum = 0;
        for (int c = 0; c < ctas; ++c) sum += cluster.map_shared_rank(hist, c)[tid];
        s_total[tid] = sum;
      }
      hist = s_total;
    }
    __syncthreads();
    if (warp == 0) {  // lane l: digits 255 - 8 l downwards; which one holds the rank
      int c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += c[i] = hist[255 - 8 * lane - i];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      int before = upto - sum;
      if (before < rank && rank <= upto) {
        int i = 0;
        while (i < 7 && rank > before + c[i]) before += c[i++];
        s_prefix = prefix | (uint32_t)(255 - 8 * lane - i) << shift8;
        s_rank = rank - before;
        s_done = c[i] == rank - before;  // the whole digit stays: the lower bytes do not matter
      }
    }
    __syncthreads();
    prefix = s_prefix;
    rank = s_rank;
    mask |= 255u << shift8;
    if (s_done) break;
  }
  // ---- kept are the keys above the prefix and the first `rank` equal to it:
  // each warp counts its part of the stretch, then writes it
  const int per = (t1 - t0 + kThreads - 1) / kThreads * 32;  // tokens of a warp
  const int j0 = t0 + warp * per, j1 = min(t1, j0 + per);
  int above = 0, ties = 0;
  for (int j = j0 + lane; j < j1; j += 32) {
    const uint32_t key = key_of(j);
    above += key > prefix;
    ties += key == prefix;
  }
  above = __reduce_add_sync(0xffffffffu, above);
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0) {
    s_above[warp] = above;
    s_ties[warp] = ties;
  }
  __syncthreads();
  above = ties = 0;
  if constexpr (kCluster) {  // what the cluster's lower CTAs have
    if (warp == 0) {
      const int up = __reduce_add_sync(0xffffffffu, lane < kThreads / 32 ? s_above[lane] : 0);
      const int eq = __reduce_add_sync(0xffffffffu, lane < kThreads / 32 ? s_ties[lane] : 0);
      if (lane == 0) s_cta = make_int2(up, eq);
    }
    cluster.sync();
    const int2 lower_cta = lane < cta ? *cluster.map_shared_rank(&s_cta, lane) : make_int2(0, 0);
    above = __reduce_add_sync(0xffffffffu, lower_cta.x);
    ties = __reduce_add_sync(0xffffffffu, lower_cta.y);
    cluster.barrier_arrive();  // this CTA has read the others' shared memory
  }
  above += __reduce_add_sync(0xffffffffu, lane < warp ? s_above[lane] : 0);
  ties += __reduce_add_sync(0xffffffffu, lane < warp ? s_ties[lane] : 0);
  const uint32_t lower = (1u << lane) - 1u;
  for (int j = j0; j < j1; j += 32) {
    const int mine = j + lane;
    const uint32_t key = mine < j1 ? key_of(mine) : 0u;
    const bool up = mine < j1 && key > prefix, tie = mine < j1 && key == prefix;
    const uint32_t ups = __ballot_sync(0xffffffffu, up), eqs = __ballot_sync(0xffffffffu, tie);
    const int tie_at = ties + __popc(eqs & lower);
    if (up || (tie && tie_at < rank)) kept[above + __popc(ups & lower) + min(tie_at, rank)] = mine;
    above += __popc(ups);
    ties += __popc(eqs);
  }
  if constexpr (kCluster) cluster.barrier_wait();
}

// The move of one (sequence, head), in units that gridDim.x CTAs share: kBatch
// chunks of K, as many bytes of V rows, or the scores. A thread has a token of
// the tile, and works out where it comes from and goes to once for all its
// units. A unit is read before any of it is written; the K chunks and V rows
// of different units do not touch.
constexpr int kBatch = 4;
template <typename U>
constexpr int v_rows() { return 16 / (int)sizeof(U) * kBatch / 2; }

// count (at most N) elements, BS apart, of this thread's token: all threads'
// reads come before any write when the places overlap.
template <int N, int BS, typename E>
__device__ __forceinline__ void move_unit(const E *src, E *dst, int count, bool live, bool in_place) {
  E v[N];
  if (live) {
    if (count == N) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = src[i * BS];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < count) v[i] = src[i * BS];
    }
  }
  if (in_place) __syncthreads();
  if (live) {
    if (count == N) {
#pragma unroll
      for (int i = 0; i < N; ++i) dst[i * BS] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < count) dst[i * BS] = v[i];
    }
  }
}

template <typename U, int BS, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == kMoveThreads ? 4 : 1) evict_move_kernel(const EvictArgs p) {
  constexpr int kX = 16 / (int)sizeof(U), kRows = v_rows<U>();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const Sequence q = sequence_of(p, b);
  const bool in_place = !p.out_block_tables;
  if (in_place && q.len == q.budget) return;  // everything stays where it is
  const uint32_t *table = p.block_tables + (int64_t)b * p.cols;
  const uint32_t *out_table = in_place ? table : p.out_block_tables + (int64_t)b * p.out_cols;
  const int32_t *kept = p.kept + ((int64_t)b * p.num_kv_heads + h) * p.budget;
  const int D = p.head_dim, chunks = D / kX;
  const int k_units = (chunks + kBatch - 1) / kBatch, units = k_units + (D + kRows - 1) / kRows + 1;
  for (int r0 = 0; r0 < q.budget; r0 += kThreads) {
    const int r = r0 + tid;
    int64_t from = -1, to = -1;  // (block, head)
    int so = 0, dof = 0;
    if (r < q.budget) {
      const int j = kept[r];
      const int64_t sb = block_at(table, j / BS, p.num_blocks), db = block_at(out_table, r / BS, p.num_blocks);
      if (sb >= 0 && db >= 0) {
        from = sb * p.num_kv_heads + h;
        to = db * p.num_kv_heads + h;
        so = j % BS;
        dof = r % BS;
      }
    }
    const bool live = from >= 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      if (u < k_units) {  // K: 16 bytes a token and chunk
        const int c0 = u * kBatch;
        uint4 *cache = static_cast<uint4 *>(p.key_cache);
        move_unit<kBatch, BS>(cache + (from * chunks + c0) * BS + so, cache + (to * chunks + c0) * BS + dof,
                              min(kBatch, chunks - c0), live, in_place);
      } else if (u < units - 1) {  // V: an element a token and row, the tile's tokens along the rows
        const int d0 = (u - k_units) * kRows;
        U *cache = static_cast<U *>(p.value_cache);
        move_unit<kRows, BS>(cache + (from * D + d0) * BS + so, cache + (to * D + d0) * BS + dof, min(kRows, D - d0),
                             live, in_place);
      } else {
        move_unit<1, BS>(p.score_cache + from * BS + so, p.score_cache + to * BS + dof, 1, live, in_place);
      }
    }
  }
}

// CTAs per (sequence, head): enough to fill the SMs, at most one per unit.
// Where even that leaves most SMs' places empty, tiles of 1024 tokens take fewer
// turns: 13.8 against 15.2 us at one sequence of 4099 tokens, 29 / 42 at 20000.
template <typename U, int BS>
int launch_move_bs(const EvictArgs &a, cudaStream_t s) {
  const int chunks = a.head_dim * (int)sizeof(U) / 16;
  const int64_t pairs = (int64_t)a.num_seqs * a.num_kv_heads;
  const int units = (chunks + kBatch - 1) / kBatch + (a.head_dim + v_rows<U>() - 1) / v_rows<U>() + 1;
  int64_t parts = (kMoveCtas + pairs - 1) / pairs;
  parts = parts > units ? units : parts;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)parts, (unsigned)a.num_kv_heads, (unsigned)a.num_seqs);
  const bool wide = pairs * parts < kMoveCtas / 4 && a.budget > kMoveThreads;
  cfg.blockDim = dim3(wide ? kMoveMostThreads : kMoveThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, wide ? evict_move_kernel<U, BS, kMoveMostThreads> : evict_move_kernel<U, BS, kMoveThreads>, a) ==
                 cudaSuccess
             ? VASR_PA_OK
             : VASR_PA_ELAUNCH;
}

template <typename U>
int launch_move(const EvictArgs &a, cudaStream_t s) {
  switch (a.block_size) {
    case 8: return launch_move_bs<U, 8>(a, s);
    case 16: return launch_move_bs<U, 16>(a, s);
    default: return launch_move_bs<U, 32>(a, s);
  }
}

}  // namespace

int launch_evict(const EvictArgs &a, cudaStream_t s) {
  const int64_t pairs = (int64_t)a.num_seqs * a.num_kv_heads;
  int ctas = 1;
  while (a.max_context_len > kClusterTokens && ctas < kMostClusterCtas && 2 * ctas * pairs <= 148) ctas *= 2;
  const int64_t share = ((int64_t)a.max_context_len + ctas - 1) / ctas;
  const int most = pairs <= 148 ? kMostKeys : kKeys;
  const int key_cap = share > most ? most : (int)share;
  const int smem = key_cap * (int)sizeof(uint32_t);
  const dim3 grid((unsigned)(a.num_kv_heads * ctas), (unsigned)a.num_seqs);
  static std::atomic<uint64_t> one_done{0}, cluster_done{0};
  if (ctas > 1) {
    auto kern = evict_select_kernel<kSelectMostThreads, true>;
    if (!ensure_smem_attr(kern, kMostKeys * 4, cluster_done)) return VASR_PA_ELAUNCH;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kSelectMostThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)ctas, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, a, key_cap) != cudaSuccess) return VASR_PA_ELAUNCH;
  } else if (pairs <= 148) {
    auto kern = evict_select_kernel<kSelectMostThreads, false>;
    if (!ensure_smem_attr(kern, kMostKeys * 4, one_done)) return VASR_PA_ELAUNCH;
    kern<<<grid, kSelectMostThreads, smem, s>>>(a, key_cap);
  } else {  // at most kKeys keys: within the default limit
    evict_select_kernel<kSelectThreads, false><<<grid, kSelectThreads, smem, s>>>(a, key_cap);
  }
  switch (a.elem_size) {
    case 1: return launch_move<uint8_t>(a, s);
    case 2: return launch_move<uint16_t>(a, s);
    default: return launch_move<uint32_t>(a, s);
  }
}

uint32_t *error_word_evict() { return unit_error_word(); }

}  // namespace vasr
