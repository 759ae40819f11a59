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
// Selection is a radix select over order-preserving keys of the scores; the
// move copies bits. In place, token r of the result comes from an index >= r,
// so places filled in ascending tiles never overwrite a token that is still
// needed, as long as a tile is read before it or a later one is written: each
// CTA moves one slice of the head dimension of one (sequence, head) that way.
#include "common.cuh"
#include "launch.h"

namespace vasr {
namespace {

constexpr int kSelectThreads = 256;
constexpr int kMoveThreads = 256;

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

// Block id of column `col`, checked against the pool (block 0 otherwise).
__device__ __forceinline__ int64_t block_at(const uint32_t *table, int col, int64_t num_blocks) {
  const uint32_t id = table[col];
  if ((int64_t)id < num_blocks) return id;
  raise_device_error(VASR_PA_DERR_BLOCK_RANGE);
  return -1;
}

// Exclusive prefix sum of x over the block; *total the block's sum.
__device__ __forceinline__ int block_scan(int x, int *total) {
  __shared__ int part[kSelectThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  if (lane == 31) part[warp] = s;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    if (w < warp) before += part[w];
    all += part[w];
  }
  __syncthreads();
  *total = all;
  return before + s - x;
}

// kept[b, h, :] = the indices that stay, ascending, then -1.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictArgs p) {
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const Sequence q = sequence_of(p, b);
  int32_t *kept = p.kept + ((int64_t)b * p.num_kv_heads + h) * p.budget;
  if (h == 0 && tid == 0) p.new_lens[b] = (uint32_t)q.budget;
  for (int i = q.budget + tid; i < p.budget; i += kSelectThreads) kept[i] = -1;
  if (q.len == q.budget) {
    for (int i = tid; i < q.budget; i += kSelectThreads) kept[i] = i;
    return;
  }
  const uint32_t *table = p.block_tables + (int64_t)b * p.cols;
  auto key_of = [&](int j) -> uint32_t {
    if (j < p.num_sink || j >= q.len - p.num_recent) return 0xffffffffu;
    const int64_t blk = block_at(table, j / p.block_size, p.num_blocks);
    if (blk < 0) return 0u;
    return score_key(p.score_cache[(blk * p.num_kv_heads + h) * p.block_size + j % p.block_size]);
  };
  // the key of rank `budget` from above: one byte of it per pass
  __shared__ int hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_rank;
  uint32_t prefix = 0, mask = 0;
  int rank = q.budget;  // 1-based rank among the keys that match the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int j = tid; j < q.len; j += kSelectThreads) {
      const uint32_t key = key_of(j);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255;
      while (d > 0 && rank > hist[d]) rank -= hist[d--];
      s_prefix = prefix | ((uint32_t)d << shift);
      s_rank = rank;
    }
    __syncthreads();
    prefix = s_prefix;
    rank = s_rank;
    mask |= 255u << shift;
    __syncthreads();
  }
  // above the threshold, or equal to it and among the first `rank` equal ones
  int done = 0, ties = 0;
  for (int j0 = 0; j0 < q.len; j0 += kSelectThreads) {
    const int j = j0 + tid;
    const uint32_t key = j < q.len ? key_of(j) : 0u;
    const bool tie = j < q.len && key == prefix;
    int n;
    const int tie_at = ties + block_scan(tie, &n);
    ties += n;
    const bool keep = j < q.len && (key > prefix || (tie && tie_at < rank));
    const int at = done + block_scan(keep, &n);
    done += n;
    if (keep) kept[at] = j;
  }
}

// One slice of 16 bytes' worth of dims: K, V or the scores of one (sequence,
// head). Slices [0, nk) are K chunks, [nk, nk + nv) groups of kX V rows, the
// last one the scores.
template <typename U>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs p) {
  constexpr int kX = 16 / (int)sizeof(U);
  const int slice = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const Sequence q = sequence_of(p, b);
  const uint32_t *out_table = p.out_block_tables ? p.out_block_tables + (int64_t)b * p.out_cols
                                                 : p.block_tables + (int64_t)b * p.cols;
  const int out_cols = p.out_block_tables ? p.out_cols : p.cols;
  const uint32_t *table = p.block_tables + (int64_t)b * p.cols;
  const int32_t *kept = p.kept + ((int64_t)b * p.num_kv_heads + h) * p.budget;
  const int BS = p.block_size, D = p.head_dim, nk = D / kX;
  const int budget = min(q.budget, out_cols * BS);
  for (int r0 = 0; r0 < budget; r0 += kMoveThreads) {
    const int r = r0 + tid;
    int64_t from = -1, to = -1;
    int so = 0, dof = 0;
    if (r < budget) {
      const int j = kept[r];
      const int64_t sb = block_at(table, j / BS, p.num_blocks), db = block_at(out_table, r / BS, p.num_blocks);
      if (sb >= 0 && db >= 0) {
        from = sb * p.num_kv_heads + h;
        to = db * p.num_kv_heads + h;
        so = j % BS;
        dof = r % BS;
      }
    }
    if (slice < nk) {  // K chunk: 16 bytes a token
      uint4 v = make_uint4(0, 0, 0, 0);
      if (from >= 0) v = static_cast<const uint4 *>(p.key_cache)[(from * nk + slice) * BS + so];
      __syncthreads();
      if (from >= 0) static_cast<uint4 *>(p.key_cache)[(to * nk + slice) * BS + dof] = v;
    } else if (slice < 2 * nk) {  // kX rows of V
      U v[kX];
      const int d0 = (slice - nk) * kX;
      U *cache = static_cast<U *>(p.value_cache);
      if (from >= 0)
        for (int e = 0; e < kX; ++e) v[e] = cache[(from * D + d0 + e) * BS + so];
      __syncthreads();
      if (from >= 0)
        for (int e = 0; e < kX; ++e) cache[(to * D + d0 + e) * BS + dof] = v[e];
    } else {
      float s = 0.f;
      if (from >= 0) s = p.score_cache[from * BS + so];
      __syncthreads();
      if (from >= 0) p.score_cache[to * BS + dof] = s;
    }
  }
}

template <typename U>
int launch_move(const EvictArgs &a, cudaStream_t s) {
  const dim3 grid((unsigned)(2 * (a.head_dim * (int)sizeof(U) / 16) + 1), (unsigned)a.num_kv_heads,
                  (unsigned)a.num_seqs);
  evict_move_kernel<U><<<grid, kMoveThreads, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? VASR_PA_OK : VASR_PA_ELAUNCH;
}

}  // namespace

int launch_evict(const EvictArgs &a, cudaStream_t s) {
  evict_select_kernel<<<dim3((unsigned)a.num_kv_heads, (unsigned)a.num_seqs), kSelectThreads, 0, s>>>(a);
  switch (a.elem_size) {
    case 1: return launch_move<uint8_t>(a, s);
    case 2: return launch_move<uint16_t>(a, s);
    default: return launch_move<uint32_t>(a, s);
  }
}

int read_error_evict(uint32_t *bits, bool clear, cudaStream_t s) { return read_unit_error(bits, clear, s); }

}  // namespace vasr
