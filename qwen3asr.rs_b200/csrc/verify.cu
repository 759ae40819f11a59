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
// Three launches, each a programmatic dependent of the one before. The first
// gives every chunk of every row its maximum and its sum of exp((x - max) / T)
// in one pass over the logits, which a thread keeps in registers between its
// maximum and its sum. The second, a CTA per sequence, joins the chunks and
// writes the verdict (n, row n's maximum and sum); a counter that elects the
// sequence's last CTA of the first launch instead made every CTA of that
// launch wait for its own atomic (40 against 30 us at 64 x 5 rows of 151936).
// The third runs the race over row n, a CTA per chunk of the vocabulary: it
// has its noise in registers by the time the verdict is there, and the last
// CTA of a sequence takes the winner, found by a counter that the second launch
// has zeroed (so the workspace needs no clearing). Only the row that is drawn from is read
// twice, the second time from L2.
//
// A large call is bound by memory and, nearly as much, by the exponentials: 64
// sequences of 5 bf16 rows of 151936 logits with an f32 drafter take 43 us for
// the 175 MB that must be read (4.1 TB/s), 32 x 8 f32 rows without a drafter
// 40 us (4.4 TB/s). One sequence takes 9.1 us, the latency of three launches
// that each wait for one round of loads; CTAs of 64 threads, four times as
// many, took 11.7 us there (more chunks to join) and 5 us more for the large call.
// CTAs that stay and load the next chunk ahead of the current one's work need
// registers for two, and were slower by 3 us.
#include <type_traits>

#include "common.cuh"
#include "launch.h"

namespace vasr {
namespace {

constexpr int kThreads = 256;
constexpr int kRowElems = 32;   // logits a thread of the first launch keeps (16: 49 us for the large call)
constexpr int kEmitElems = 16;  // of logits, drafter's values and noise each, in the third (8: 59 us, 32: 48 us)
// CTAs a SM whose registers suffice: at 64 x 5 bf16 rows 42.7 us with 8 and 5,
// 46.0 with 6 and 4, 47.6 with 8 and 6; at 32 x 8 f32 rows, which hold twice the
// registers, 39.8 with 5, 41.6 with 4, 47.4 with 6.
template <typename T>
constexpr int kRowCtas = sizeof(T) == 2 ? 8 : 5;
template <typename T>
constexpr int kEmitCtas = sizeof(T) == 2 ? 5 : 4;

// One chunk of a row: its maximum (and, for greedy rows, the first place of
// it) and sum over the chunk of exp((x - max) / T).
struct ChunkStat {
  float max;
  float sum;
  uint32_t arg;
  uint32_t pad;
};

// What the second launch found out about a sequence.
struct Verdict {
  int n;        // accepted drafts
  float max;    // of row n
  float inv;    // 1 / its sum
  int32_t drawn;  // the race is to be run (else the tokens are written already)
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
  __device__ __forceinline__ void load(const T *row, int len, int tid) {
    const bool aligned = reinterpret_cast<uintptr_t>(row) % 16 == 0;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int j = (tid + k * kThreads) * kGroup;
      if (aligned && (k + 1) * kThreads * kGroup <= len) {  // the whole CTA's groups
#pragma unroll
        for (int v = 0; v < kVecs; ++v) raw[k][v] = __ldg(reinterpret_cast<const uint4 *>(row + j) + v);
      } else {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          raw[k][v] = make_uint4(0, 0, 0, 0);
          if (aligned && j + kGroup <= len) {
            raw[k][v] = __ldg(reinterpret_cast<const uint4 *>(row + j) + v);
          } else if (j < len) {
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

// f(value, index) for the thread's elements of group k that lie in the chunk
// and are not NaN; groups past a chunk's end have none.
template <typename T, int kGroups, typename F>
__device__ __forceinline__ void each_of_group(const Held<T, kGroups> &x, int k, int len, int tid, F f) {
  const int j = (tid + k * kThreads) * kGroup;
  if (j >= len) return;
  float v[kGroup];
  x.group(k, v);
#pragma unroll
  for (int i = 0; i < kGroup; ++i)
    if (j + i < len && v[i] == v[i]) f(v[i], j + i);
}

// grid = (chunk, row, sequence)
template <typename T>
__global__ void __launch_bounds__(kThreads, kRowCtas<T>) verify_rows_kernel(const VerifyArgs p) {
  pdl_launch_dependents();
  constexpr int kGroups = kRowElems / kGroup;
  __shared__ float2 part[kThreads / 32];
  __shared__ uint32_t s_arg;
  const int chunk = blockIdx.x, i = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int warp = tid >> 5, lane = tid & 31, warps = kThreads >> 5;
  if (i > drafts_of(p, b)) return;
  const float t = temperature_of(p, b);
  const int size = kThreads * kRowElems;
  const int64_t lo = (int64_t)chunk * size;
  const int len = (int)min((int64_t)size, p.vocab - lo);
  Held<T, kGroups> x;
  x.load(static_cast<const T *>(p.logits) + b * p.logits_seq_stride + i * p.logits_row_stride + lo, len, tid);
  // the thread's own maximum and sum, then the warp's, then the chunk's
  const int whole = len / (kThreads * kGroup);  // groups that all threads have
  float m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    if (g < whole) m = fmaxf(m, x.group_max(g));
    else each_of_group(x, g, len, tid, [&](float v, int) { m = fmaxf(m, v); });
  }
  const float c = kLog2e / t;
  if (t > 0.f && m > -INFINITY) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (g < whole) {
        float v[kGroup];
        x.group(g, v);
#pragma unroll
        for (int e = 0; e < kGroup; ++e) sum += plain_weight(v[e], m, c);
      } else {
        each_of_group(x, g, len, tid, [&](float v, int) { sum += weight_of(v, m, c); });
      }
    }
    if (!(sum == sum)) {  // an infinite maximum or a NaN among the logits
      sum = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        each_of_group(x, g, len, tid, [&](float v, int) { sum += weight_of(v, m, c); });
    }
  }
  const float wm = warp_max_xor(m, 32);
  if (t > 0.f) sum = warp_sum_xor(m > -INFINITY ? sum * weight_of(m, wm, c) : 0.f, 32);
  if (lane == 0) part[warp] = make_float2(wm, sum);
  if (tid == 0) s_arg = kNone;
  __syncthreads();
  const bool greedy = !(t > 0.f);
  if (!greedy && warp != 0) return;
  const float2 mine = part[lane < warps ? lane : 0];
  const float cm = warp_max_xor(mine.x, 32);
  if (greedy) {  // the first place of the maximum
    uint32_t first = kNone;
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      each_of_group(x, g, len, tid, [&](float v, int j) {
        if (v == cm) first = min(first, (uint32_t)j);
      });
    if (first != kNone) atomicMin(&s_arg, first);
    __syncthreads();
  } else {
    sum = warp_sum_xor(lane < warps && mine.y != 0.f ? mine.y * weight_of(mine.x, cm, c) : 0.f, 32);
  }
  if (tid == 0)
    static_cast<ChunkStat *>(p.stats)[((int64_t)b * (p.num_drafts + 1) + i) * gridDim.x + chunk] =
        ChunkStat{cm, sum, s_arg != kNone ? (uint32_t)lo + s_arg : 0u, 0u};
}

// A whole row from its chunks, by one warp.
__device__ __forceinline__ ChunkStat join_chunks(const VerifyArgs &p, int64_t row, float t) {
  const int lane = threadIdx.x & 31, chunks = p.row_chunks;
  const float4 *s = static_cast<const float4 *>(p.stats) + row * chunks;
  Best top{-INFINITY, kNone};
  for (int c = lane; c < chunks; c += 32) {
    const float4 v = s[c];
    if (v.x > -INFINITY) top = better(top, Best{v.x, __float_as_uint(v.z)});
  }
  top = warp_best(top);
  float sum = 0.f;
  if (t > 0.f && top.v > -INFINITY) {
    const float k = kLog2e / t;
    for (int c = lane; c < chunks; c += 32) {
      const float4 v = s[c];
      if (v.y != 0.f) sum = fmaf(v.y, weight_of(v.x, top.v, k), sum);
    }
    sum = warp_sum_xor(sum, 32);
  }
  return ChunkStat{top.v, sum, top.i != kNone ? top.i : 0u, 0u};
}

// One CTA per sequence: every row's sum, then the verdict.
template <typename T, typename TQ>
__global__ void __launch_bounds__(kThreads) verify_verdict_kernel(const VerifyArgs p) {
  pdl_launch_dependents();
  extern __shared__ ChunkStat s_row[];  // [num_drafts + 1]
  __shared__ int s_fail;
  const int b = blockIdx.x, tid = threadIdx.x, threads = blockDim.x, warp = tid >> 5, lane = tid & 31;
  const int k = drafts_of(p, b);
  const float t = temperature_of(p, b);
  const T *rows = static_cast<const T *>(p.logits) + b * p.logits_seq_stride;
  const int32_t *drafts = p.draft_tokens + (int64_t)b * p.num_drafts;
  const TQ *probs = p.draft_probs ? static_cast<const TQ *>(p.draft_probs) + b * p.probs_seq_stride : nullptr;
  // a draft's target logit, drafter's probability and uniform (inputs: read ahead of the first launch's end)
  auto draft = [&](int r, int32_t &x, float &logit, float &q, float &u) {
    x = drafts[r];
    if (x < 0 || x >= p.vocab) x = -1;
    logit = x >= 0 ? Elem<T>::to_f32(rows[r * p.logits_row_stride + x]) : -INFINITY;
    q = probs && x >= 0 ? Elem<TQ>::to_f32(probs[r * p.probs_row_stride + x]) : 1.f;
    u = t > 0.f ? p.uniform[(int64_t)b * p.num_drafts + r] : 0.f;
  };
  int32_t x0 = -1;
  float logit0 = 0.f, q0 = 0.f, u0 = 0.f;
  if (tid < k) draft(tid, x0, logit0, q0, u0);
  if (tid == 0) s_fail = k;
  pdl_wait();
  for (int r = warp; r <= k; r += threads >> 5) {
    const ChunkStat s = join_chunks(p, (int64_t)b * (p.num_drafts + 1) + r, t);
    if (lane == 0) s_row[r] = s;
  }
  __syncthreads();
  for (int r = tid; r < k; r += threads) {
    int32_t x = x0;
    float logit = logit0, q = q0, u = u0;
    if (r != tid) draft(r, x, logit, q, u);
    const ChunkStat s = s_row[r];
    bool ok = x >= 0 && s.max > -INFINITY;
    if (ok) ok = t > 0.f ? u * q < weight_of(logit, s.max, kLog2e / t) / s.sum : (uint32_t)x == s.arg;
    if (!ok) atomicMin(&s_fail, r);
  }
  __syncthreads();
  const int n = s_fail;
  const ChunkStat s = s_row[n];
  const bool drawn = t > 0.f && s.max > -INFINITY;
  if (tid == 0) {
    static_cast<Verdict *>(p.verdicts)[b] = Verdict{n, s.max, 1.f / s.sum, drawn};
    p.counters[b] = 0u;  // of the race's CTAs
    p.num_accepted[b] = n;
  }
  int32_t *out = p.out_tokens + (int64_t)b * (p.num_drafts + 1);  // all but the drawn token
  for (int r = tid; r <= p.num_drafts; r += threads)
    if (r != n || !drawn) out[r] = r < n ? drafts[r] : r == n ? (int32_t)s.arg : -1;
}

// grid = (chunk, sequence)
template <typename T, typename TQ>
__global__ void __launch_bounds__(kThreads, kEmitCtas<T>) verify_emit_kernel(const VerifyArgs p) {
  constexpr int kGroups = kEmitElems / kGroup;
  __shared__ Best part[kThreads / 32];
  const int chunk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int warp = tid >> 5, lane = tid & 31, warps = kThreads >> 5;
  const float t = temperature_of(p, b);
  const int size = kThreads * kEmitElems;
  const int64_t lo = (int64_t)chunk * size;
  const int len = (int)min((int64_t)size, p.vocab - lo);
  // inputs come early, while the launches before still run
  Held<float, kGroups> race;
  if (t > 0.f) race.load(p.race + b * p.race_seq_stride + lo, len, tid);
  const int k = drafts_of(p, b);
  pdl_wait();
  const float4 raw = __ldcg(static_cast<const float4 *>(p.verdicts) + b);
  const Verdict s{__float_as_int(raw.x), raw.y, raw.z, __float_as_int(raw.w)};
  if (!s.drawn) return;
  const float c = kLog2e / t;
  const T *row = static_cast<const T *>(p.logits) + b * p.logits_seq_stride + s.n * p.logits_row_stride;
  // ---- the race over this chunk. The quotient takes one reciprocal
  // instruction (1 ulp); only r / e > 0 can win, so NaN and r <= 0 drop out.
  Held<T, kGroups> x;
  x.load(row + lo, len, tid);
  const bool with_q = p.draft_probs && s.n < k;
  Held<TQ, kGroups> q;
  if (with_q)
    q.load(static_cast<const TQ *>(p.draft_probs) + b * p.probs_seq_stride + s.n * p.probs_row_stride + lo, len, tid);
  int skip = -1;  // a failed draft that the drafter was certain of
  if (s.n < k && !with_q) {
    const int64_t failed = (int64_t)p.draft_tokens[(int64_t)b * p.num_drafts + s.n] - lo;
    if (failed >= 0 && failed < len) skip = (int)failed;
  }
  const bool finite = s.max < INFINITY && c < INFINITY;
  float top = 0.f;
  int place = -1;  // g * 8 + i of the winner
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int j = (tid + g * kThreads) * kGroup;
    float w[kGroup], e[kGroup], qv[kGroup];
    x.group(g, w);
    race.group(g, e);
    if (with_q) {
      q.group(g, qv);
    } else {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) qv[i] = 0.f;
    }
    if (finite && j + kGroup <= len && (skip < j || skip >= j + kGroup)) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const float a = fmaf(plain_weight(w[i], s.max, c), s.inv, -qv[i]) * rcp_approx(e[i]);
        if (a > top) {
          top = a;
          place = g * kGroup + i;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const float a = fmaf(weight_of(w[i], s.max, c), s.inv, -qv[i]) * rcp_approx(e[i]);
        if (a > top && j + i < len && j + i != skip) {
          top = a;
          place = g * kGroup + i;
        }
      }
    }
  }
  Best best{top, kNone};
  if (place >= 0) best.i = (uint32_t)(lo + (tid + place / kGroup * kThreads) * kGroup + place % kGroup);
  best = warp_best(best);
  if (lane == 0) part[warp] = best;
  __syncthreads();
  if (warp != 0) return;
  best = lane < warps ? part[lane] : Best{0.f, kNone};
  best = warp_best(best);
  uint64_t *slots = static_cast<uint64_t *>(p.bests) + (int64_t)b * gridDim.x;
  uint32_t last = 0;
  if (lane == 0) {
    slots[chunk] = (uint64_t)__float_as_uint(best.v) << 32 | best.i;
    __threadfence();
    last = atomicAdd(p.counters + b, 1u) == gridDim.x - 1;
    __threadfence();
  }
  if (!__shfl_sync(0xffffffffu, last, 0)) return;
  // ---- the sequence's last CTA: the winner over all chunks
  best = Best{0.f, kNone};
  for (int i = lane; i < (int)gridDim.x; i += 32) {
    const uint64_t v = __ldcg(reinterpret_cast<const unsigned long long *>(slots) + i);
    best = better(best, Best{__uint_as_float((uint32_t)(v >> 32)), (uint32_t)v});
  }
  best = warp_best(best);
  if (best.i == kNone) {  // r is 0 everywhere (the drafter covers the target): draw from p
    const float *noise = p.race + b * p.race_seq_stride;
    for (int64_t v = lane; v < p.vocab; v += 32) {
      const float a = weight_of(Elem<T>::to_f32(row[v]), s.max, c) * s.inv * rcp_approx(noise[v]);
      if (a > best.v) best = Best{a, (uint32_t)v};
    }
    best = warp_best(best);
  }
  if (lane == 0)
    p.out_tokens[(int64_t)b * (p.num_drafts + 1) + s.n] = best.i != kNone ? (int32_t)best.i : 0;  // 0: all noise NaN
}

struct VerifyLayout {
  int row_chunks, emit_chunks;
  size_t off_stats, off_verdicts, off_bests, total;
};
constexpr size_t kCounterBytes = 65536 * sizeof(uint32_t);  // one per sequence, zeroed by the second launch
VerifyLayout verify_layout(int num_seqs, int num_drafts, int64_t vocab) {
  VerifyLayout l;
  auto chunks = [&](int elems) { return (int)((vocab + kThreads * elems - 1) / (kThreads * elems)); };
  l.row_chunks = chunks(kRowElems);
  l.emit_chunks = chunks(kEmitElems);
  l.off_stats = kCounterBytes;
  l.off_verdicts = l.off_stats + (size_t)num_seqs * (num_drafts + 1) * l.row_chunks * sizeof(ChunkStat);
  l.off_bests = l.off_verdicts + (size_t)num_seqs * sizeof(Verdict);
  l.total = l.off_bests + (size_t)num_seqs * l.emit_chunks * sizeof(uint64_t);
  return l;
}

template <typename T, typename TQ>
int launch_verify_tq(VerifyArgs a, cudaStream_t s) {
  const VerifyLayout l = verify_layout(a.num_seqs, a.num_drafts, a.vocab);
  unsigned char *ws = static_cast<unsigned char *>(a.workspace);
  a.counters = reinterpret_cast<uint32_t *>(ws);
  a.stats = ws + l.off_stats;
  a.verdicts = ws + l.off_verdicts;
  a.bests = ws + l.off_bests;
  a.row_chunks = l.row_chunks;
  verify_rows_kernel<T><<<dim3((unsigned)l.row_chunks, (unsigned)a.num_drafts + 1, (unsigned)a.num_seqs),
                          kThreads, 0, s>>>(a);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = s;
  const int row_warps = a.num_drafts + 1 < kThreads / 32 ? a.num_drafts + 1 : kThreads / 32;
  cfg.gridDim = dim3((unsigned)a.num_seqs);
  cfg.blockDim = dim3((unsigned)row_warps * 32);
  cfg.dynamicSmemBytes = (size_t)(a.num_drafts + 1) * sizeof(ChunkStat);
  if (cudaLaunchKernelEx(&cfg, verify_verdict_kernel<T, TQ>, a) != cudaSuccess) return VASR_PA_ELAUNCH;
  cfg.gridDim = dim3((unsigned)l.emit_chunks, (unsigned)a.num_seqs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 0;
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
