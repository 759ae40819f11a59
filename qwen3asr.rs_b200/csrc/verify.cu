// verify.cu — drafted tokens against the target's probabilities.
//
// Row i of a sequence's target logits gives p_i = softmax(logits_i / T); the
// drafter proposed x_i with probability q_i(x_i). Draft i is accepted while
//   u_i q_i(x_i) < p_i(x_i)
// for a given uniform u_i, and the token after the n accepted ones is drawn
// from r = max(p_n - q_n, 0) (a failed draft) or r = p_n (none failed) as
//   argmax_v r(v) / e_v,   e_v given Exp(1) noise,
// which takes v with probability r(v) / sum r: the times e_v / r(v) are
// exponential with rate r(v), and the first of them wins. Unlike a running
// sum over the vocabulary, the comparison does not depend on the order of a
// long f32 sum. T = 0: accept while x_i is the argmax of row i, then take row
// n's argmax. Lowest index on equal values; NaN logits count as -inf.
//
// Two launches. The first gives every chunk of every row its maximum and its
// sum of exp((x - max) / T) in one pass: a thread keeps its logits in
// registers between the maximum and the sum. The second, a programmatic
// dependent of the first, has a CTA per chunk of a sequence's vocabulary: it
// loads its noise and the drafts' logits early, joins the rows' chunks and
// decides on its own copy (a few hundred bytes), runs the race over its chunk
// of row n, and the last CTA of the sequence takes the winner. Only the row
// that is drawn from is read twice, the second time from L2.
#include <type_traits>

#include "common.cuh"
#include "launch.h"

namespace vasr {
namespace {

constexpr int kRowElems = 32;   // logits a thread of the first launch keeps in registers
constexpr int kEmitElems = 16;  // logits, drafter's values and noise each of the second's (80 registers)
constexpr int kMaxThreads = 256;

// One chunk of a row: its maximum (and, for greedy rows, the first place of
// it) and sum over the chunk of exp((x - max) / T).
struct ChunkStat {
  float max;
  float sum;
  uint32_t arg;
  uint32_t pad;
};

// (value, index): larger value first, then lower index.
struct Best {
  float v;
  uint32_t i;
};
constexpr uint32_t kNone = 0xffffffffu;
__device__ __forceinline__ Best better(Best x, Best y) {
  return (y.v > x.v || (y.v == x.v && y.i < x.i)) ? y : x;
}
__device__ __forceinline__ Best warp_best(Best x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
  return x;
}

__device__ __forceinline__ float temperature_of(const VerifyArgs &p, int b) {
  return p.temperatures ? p.temperatures[b] : p.temperature;
}
__device__ __forceinline__ int drafts_of(const VerifyArgs &p, int b) {
  return p.draft_lens ? min(max(p.draft_lens[b], 0), p.num_drafts) : p.num_drafts;
}
// exp((x - max) / T) with c = log2(e) / T. exp2 in its one-instruction form
// (2 ulp): the product's own rounding is no smaller, and the precise form's
// range checks took a third of the kernels' instructions. weight_of also
// holds where max is +inf (the entries there share the mass) or 1 / T is.
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float plain_weight(float x, float max, float c) { return exp2_approx((x - max) * c); }
__device__ __forceinline__ float weight_of(float x, float max, float c) {
  return x == max ? 1.f : x == x ? plain_weight(x, max, c) : 0.f;
}

// A thread's elements of a chunk of a row: groups of 8, group tid + k threads
// being its k-th whatever the type, so that rows of different types line up.
// Vector loads where the group is 16-byte aligned and whole, else one by one
// (what lies past the chunk reads as 0).
constexpr int kGroup = 8;
template <typename T, int kGroups>
struct Held {
  static constexpr int kVec = 16 / (int)sizeof(T);
  static constexpr int kVecs = kGroup / kVec;
  uint4 raw[kGroups][kVecs];
  __device__ __forceinline__ void load(const T *row, int len, int tid, int threads) {
    const bool aligned = reinterpret_cast<uintptr_t>(row) % 16 == 0;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int j = (tid + k * threads) * kGroup;
      if (aligned && j + kGroup <= len) {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) raw[k][v] = __ldg(reinterpret_cast<const uint4 *>(row + j) + v);
      } else {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          T e[kVec];
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            const int at = j + v * kVec + i;
            e[i] = at < len ? row[at] : Elem<T>::from_f32(0.f);
          }
          raw[k][v] = *reinterpret_cast<const uint4 *>(e);
        }
      }
    }
  }
  __device__ __forceinline__ void group(int k, float (&out)[kGroup]) const {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      float f[kVec];
      unpack_chunk<T>(raw[k][v], f);
#pragma unroll
      for (int i = 0; i < kVec; ++i) out[v * kVec + i] = f[i];
    }
  }
  // the largest element of group k; NaN is passed over
  __device__ __forceinline__ float group_max(int k) const {
    if constexpr (sizeof(T) == 2) {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2 *h = reinterpret_cast<const T2 *>(&raw[k][0]);
      const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(Elem<T>::to_f32(m.x), Elem<T>::to_f32(m.y));
    } else {
      float v[kGroup];
      group(k, v);
      float m = v[0];
#pragma unroll
      for (int i = 1; i < kGroup; ++i) m = fmaxf(m, v[i]);
      return m;
    }
  }
};

// The guarded forms for a chunk's rest (fewer than 8 elements of a group) and
// for logits that are not finite.
template <typename T, int kGroups, typename F>
__device__ __forceinline__ void each_guarded(const Held<T, kGroups> &x, int len, int tid, int threads, F f) {
  for (int k = 0; k < kGroups; ++k) {
    float v[kGroup];
    x.group(k, v);
    const int j = (tid + k * threads) * kGroup;
#pragma unroll
    for (int i = 0; i < kGroup; ++i)
      if (j + i < len && v[i] == v[i]) f(v[i], j + i);
  }
}

template <typename T>
__global__ void __launch_bounds__(kMaxThreads) verify_rows_kernel(const VerifyArgs p) {
  pdl_launch_dependents();
  constexpr int kGroups = kRowElems / kGroup;
  const int chunk = blockIdx.x, i = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, threads = blockDim.x;
  if (i > drafts_of(p, b)) return;
  const int size = threads * kRowElems;
  const int64_t lo = (int64_t)chunk * size;
  const int len = (int)min((int64_t)size, p.vocab - lo);
  const T *row = static_cast<const T *>(p.logits) + b * p.logits_seq_stride + i * p.logits_row_stride + lo;
  Held<T, kGroups> x;
  x.load(row, len, tid, threads);
  const float t = temperature_of(p, b);
  float m = -INFINITY;
  if (len == size) {
#pragma unroll
    for (int k = 0; k < kGroups; ++k) m = fmaxf(m, x.group_max(k));
  } else {
    each_guarded(x, len, tid, threads, [&](float v, int) { m = fmaxf(m, v); });
  }
  __shared__ float part[kMaxThreads / 32];
  __shared__ uint32_t s_arg;
  const int warps = threads >> 5;
  m = warp_max_xor(m, 32);
  if ((tid & 31) == 0) part[tid >> 5] = m;
  if (tid == 0) s_arg = kNone;
  __syncthreads();
  for (int w = 0; w < warps; ++w) m = fmaxf(m, part[w]);
  __syncthreads();
  float sum = 0.f;
  if (t > 0.f) {
    const float c = kLog2e / t;
    if (m > -INFINITY) {
      if (len == size) {
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          float v[kGroup];
          x.group(k, v);
#pragma unroll
          for (int e = 0; e < kGroup; ++e) sum += plain_weight(v[e], m, c);
        }
      }
      if (len != size || !(sum == sum)) {
        sum = 0.f;
        each_guarded(x, len, tid, threads, [&](float v, int) { sum += weight_of(v, m, c); });
      }
    }
    sum = warp_sum_xor(sum, 32);
    if ((tid & 31) == 0) part[tid >> 5] = sum;
    __syncthreads();
    sum = 0.f;
    for (int w = 0; w < warps; ++w) sum += part[w];
  } else {
    uint32_t first = kNone;
    each_guarded(x, len, tid, threads, [&](float v, int j) {
      if (v == m) first = min(first, (uint32_t)j);
    });
    if (first != kNone) atomicMin(&s_arg, first);
    __syncthreads();
  }
  if (tid == 0) {
    ChunkStat *out = static_cast<ChunkStat *>(p.stats);
    out[((int64_t)b * (p.num_drafts + 1) + i) * p.row_chunks + chunk] =
        ChunkStat{m, sum, s_arg != kNone ? (uint32_t)lo + s_arg : 0u, 0u};
  }
}

// A whole row from its chunks, by one warp.
__device__ __forceinline__ ChunkStat join_chunks(const VerifyArgs &p, int64_t row, float t) {
  const int lane = threadIdx.x & 31;
  const ChunkStat *s = static_cast<const ChunkStat *>(p.stats) + row * p.row_chunks;
  Best top{-INFINITY, kNone};
  for (int c = lane; c < p.row_chunks; c += 32)
    if (s[c].max > -INFINITY) top = better(top, Best{s[c].max, s[c].arg});
  top = warp_best(top);
  float sum = 0.f;
  if (t > 0.f && top.v > -INFINITY) {
    const float k = kLog2e / t;
    for (int c = lane; c < p.row_chunks; c += 32)
      if (s[c].sum != 0.f) sum = fmaf(s[c].sum, weight_of(s[c].max, top.v, k), sum);
    sum = warp_sum_xor(sum, 32);
  }
  return ChunkStat{top.v, sum, top.i != kNone ? top.i : 0u, 0u};
}

template <typename T, typename TQ>
__global__ void __launch_bounds__(kMaxThreads, 4) verify_emit_kernel(const VerifyArgs p) {
  extern __shared__ ChunkStat s_row[];  // [num_drafts + 1]
  __shared__ int s_fail;
  __shared__ Best part[kMaxThreads / 32];
  __shared__ uint32_t s_last;
  const int chunk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, threads = blockDim.x;
  const int warp = tid >> 5, lane = tid & 31, warps = threads >> 5;
  const int k = drafts_of(p, b);
  const float t = temperature_of(p, b);
  const T *rows = static_cast<const T *>(p.logits) + b * p.logits_seq_stride;
  const TQ *probs = p.draft_probs ? static_cast<const TQ *>(p.draft_probs) + b * p.probs_seq_stride : nullptr;
  const int32_t *drafts = p.draft_tokens + (int64_t)b * p.num_drafts;
  constexpr int kGroups = kEmitElems / kGroup;
  const int size = threads * kEmitElems;
  const int64_t lo = (int64_t)chunk * size;
  const int len = (int)min((int64_t)size, p.vocab - lo);
  if (tid == 0) s_fail = k;
  // inputs that the first launch does not write
  Held<float, kGroups> race;
  if (t > 0.f) race.load(p.race + b * p.race_seq_stride + lo, len, tid, threads);
  int32_t x0 = -1;
  float logit0 = -INFINITY, q0 = 1.f, u0 = 0.f;
  if (tid < k) {
    x0 = drafts[tid];
    if (x0 >= 0 && x0 < p.vocab) {
      logit0 = fmaxf(Elem<T>::to_f32(rows[tid * p.logits_row_stride + x0]), -INFINITY);
      if (probs) q0 = Elem<TQ>::to_f32(probs[tid * p.probs_row_stride + x0]);
    }
    if (t > 0.f) u0 = p.uniform[(int64_t)b * p.num_drafts + tid];
  }
  pdl_wait();
  for (int i = warp; i <= k; i += warps) {
    const ChunkStat s = join_chunks(p, (int64_t)b * (p.num_drafts + 1) + i, t);
    if (lane == 0) s_row[i] = s;
  }
  __syncthreads();
  const float c = t > 0.f ? kLog2e / t : 0.f;
  for (int i = tid; i < k; i += threads) {
    int32_t x = x0;
    float logit = logit0, q = q0, u = u0;
    if (i != tid) {
      x = drafts[i];
      logit = -INFINITY;
      q = 1.f;
      u = t > 0.f ? p.uniform[(int64_t)b * p.num_drafts + i] : 0.f;
      if (x >= 0 && x < p.vocab) {
        logit = fmaxf(Elem<T>::to_f32(rows[i * p.logits_row_stride + x]), -INFINITY);
        if (probs) q = Elem<TQ>::to_f32(probs[i * p.probs_row_stride + x]);
      }
    }
    const ChunkStat s = s_row[i];
    bool ok = x >= 0 && x < p.vocab && s.max > -INFINITY;
    if (ok) ok = t > 0.f ? u * q < weight_of(logit, s.max, c) / s.sum : (uint32_t)x == s.arg;
    if (!ok) atomicMin(&s_fail, i);
  }
  __syncthreads();
  const int n = s_fail;
  const ChunkStat s = s_row[n];
  const T *row = rows + n * p.logits_row_stride;
  const int64_t failed = n < k ? (int64_t)drafts[n] : -1;
  const TQ *qrow = probs && n < k ? probs + n * p.probs_row_stride : nullptr;
  const bool drawn = t > 0.f && s.max > -INFINITY;
  uint32_t next = s.arg;
  if (drawn) {
    // ---- the race over this chunk. The quotient takes one reciprocal
    // instruction (1 ulp); only r / e > 0 can win, so NaN and r <= 0 drop out.
    Held<T, kGroups> x;
    x.load(row + lo, len, tid, threads);
    Held<TQ, kGroups> q;
    if (qrow) q.load(qrow + lo, len, tid, threads);
    const float inv = 1.f / s.sum;
    const bool finite = s.max < INFINITY && c < INFINITY;
    const int skip = failed >= lo && failed < lo + len && !qrow ? (int)(failed - lo) : -1;
    Best best{0.f, kNone};
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int j = (tid + g * threads) * kGroup;
      float w[kGroup], e[kGroup], qv[kGroup];
      x.group(g, w);
      race.group(g, e);
      if (qrow) {
        q.group(g, qv);
      } else {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) qv[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const float pw = finite ? plain_weight(w[i], s.max, c) : weight_of(w[i], s.max, c);
        float a = fmaf(pw, inv, -qv[i]) * rcp_approx(e[i]);
        if (j + i >= len || j + i == skip) a = 0.f;
        if (a > best.v) best = Best{a, (uint32_t)(j + i)};
      }
    }
    if (best.i != kNone) best.i += (uint32_t)lo;
    best = warp_best(best);
    if (lane == 0) part[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < warps; ++w) best = better(best, part[w]);
      Best *slots = static_cast<Best *>(p.bests) + (int64_t)b * gridDim.x;
      slots[chunk] = best;
      __threadfence();
      s_last = atomicAdd(p.counters + b, 1u) == gridDim.x - 1;
      __threadfence();
    }
    __syncthreads();
    if (!s_last) return;
    // ---- the sequence's last CTA: the winner over all chunks
    best = Best{0.f, kNone};
    const Best *slots = static_cast<const Best *>(p.bests) + (int64_t)b * gridDim.x;
    for (int i = tid; i < (int)gridDim.x; i += threads) best = better(best, Best{__ldcg(&slots[i].v), __ldcg(&slots[i].i)});
    best = warp_best(best);
    if (lane == 0) part[warp] = best;
    __syncthreads();
    best = part[0];
    for (int w = 1; w < warps; ++w) best = better(best, part[w]);
    if (best.i == kNone) {  // r is 0 everywhere (the drafter covers the target): draw from p
      __syncthreads();
      const float *noise = p.race + b * p.race_seq_stride;
      for (int64_t v = tid; v < p.vocab; v += threads) {
        const float a = weight_of(Elem<T>::to_f32(row[v]), s.max, c) * inv * rcp_approx(noise[v]);
        if (a > best.v) best = Best{a, (uint32_t)v};
      }
      best = warp_best(best);
      if (lane == 0) part[warp] = best;
      __syncthreads();
      best = part[0];
      for (int w = 1; w < warps; ++w) best = better(best, part[w]);
    }
    next = best.i != kNone ? best.i : 0u;  // all noise NaN
    if (tid == 0) p.counters[b] = 0u;
  } else if (chunk != 0) {
    return;
  }
  int32_t *out = p.out_tokens + (int64_t)b * (p.num_drafts + 1);
  for (int i = tid; i <= p.num_drafts; i += threads) out[i] = i < n ? drafts[i] : i == n ? (int32_t)next : -1;
  if (tid == 0) p.num_accepted[b] = n;
}

// 8192 logits a chunk (256 threads); calls whose chunks would not fill the SMs
// take chunks of 2048 (64 threads), which cost more CTAs per byte.
int chunk_threads(int num_seqs, int num_drafts, int64_t vocab) {
  const int64_t ctas = (int64_t)num_seqs * (num_drafts + 1) * ((vocab + 8191) / 8192);
  return ctas >= 2 * 148 ? 256 : 64;
}

struct VerifyLayout {
  int threads, row_chunks, emit_chunks;
  size_t off_stats, off_bests, total;
};
constexpr size_t kCounterBytes = 65536 * sizeof(uint32_t);  // one per sequence, left at zero
VerifyLayout verify_layout(int num_seqs, int num_drafts, int64_t vocab) {
  VerifyLayout l;
  l.threads = chunk_threads(num_seqs, num_drafts, vocab);
  auto chunks = [&](int elems) { return (int)((vocab + l.threads * elems - 1) / (l.threads * elems)); };
  l.row_chunks = chunks(kRowElems);
  l.emit_chunks = chunks(kEmitElems);
  l.off_stats = kCounterBytes;
  l.off_bests = l.off_stats + (size_t)num_seqs * (num_drafts + 1) * l.row_chunks * sizeof(ChunkStat);
  l.total = l.off_bests + (size_t)num_seqs * l.emit_chunks * sizeof(Best);
  return l;
}

template <typename T, typename TQ>
int launch_verify_tq(VerifyArgs a, cudaStream_t s) {
  const VerifyLayout l = verify_layout(a.num_seqs, a.num_drafts, a.vocab);
  unsigned char *ws = static_cast<unsigned char *>(a.workspace);
  a.counters = reinterpret_cast<uint32_t *>(ws);
  a.stats = ws + l.off_stats;
  a.bests = ws + l.off_bests;
  a.row_chunks = l.row_chunks;
  verify_rows_kernel<T><<<dim3((unsigned)l.row_chunks, (unsigned)a.num_drafts + 1, (unsigned)a.num_seqs),
                          (unsigned)l.threads, 0, s>>>(a);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)l.emit_chunks, (unsigned)a.num_seqs);
  cfg.blockDim = dim3((unsigned)l.threads);
  cfg.dynamicSmemBytes = (size_t)(a.num_drafts + 1) * sizeof(ChunkStat);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, verify_emit_kernel<T, TQ>, a) == cudaSuccess ? VASR_PA_OK : VASR_PA_ELAUNCH;
}

template <typename T>
int launch_verify_t(const VerifyArgs &a, cudaStream_t s) {
  if (!a.draft_probs) return launch_verify_tq<T, float>(a, s);
  switch (a.probs_dtype) {
    case VASR_PA_BF16: return launch_verify_tq<T, __nv_bfloat16>(a, s);
    case VASR_PA_F16: return launch_verify_tq<T, __half>(a, s);
    default: return launch_verify_tq<T, float>(a, s);
  }
}

}  // namespace

size_t verify_workspace_bytes(int num_seqs, int num_drafts, int64_t vocab) {
  return verify_layout(num_seqs, num_drafts, vocab).total;
}

int launch_verify(const VerifyArgs &a, cudaStream_t s) {
  switch (a.dtype) {
    case VASR_PA_F32: return launch_verify_t<float>(a, s);
    case VASR_PA_BF16: return launch_verify_t<__nv_bfloat16>(a, s);
    case VASR_PA_F16: return launch_verify_t<__half>(a, s);
    default: return VASR_PA_EINVAL_DTYPE;
  }
}

}  // namespace vasr
