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
#include "common.cuh"
#include "launch.h"

namespace vasr {
namespace {

constexpr int kThreads = 512;

// What row i says: its maximum (and where), the sum of exp((x - max) / T).
struct RowStat {
  float max;
  float sum;
  uint32_t arg;
  uint32_t pad;
};

template <typename T>
__device__ __forceinline__ float load_logit(const T *row, int64_t v) {
  const float x = Elem<T>::to_f32(row[v]);
  return x == x ? x : -INFINITY;
}

__device__ __forceinline__ float load_prob(const void *row, int64_t v, int dtype) {
  switch (dtype) {
    case VASR_PA_BF16: return __bfloat162float(static_cast<const __nv_bfloat16 *>(row)[v]);
    case VASR_PA_F16: return __half2float(static_cast<const __half *>(row)[v]);
    default: return static_cast<const float *>(row)[v];
  }
}

// (value, index): larger value first, then lower index.
struct Best {
  float v;
  uint32_t i;
};
__device__ __forceinline__ Best better(Best x, Best y) {
  return (y.v > x.v || (y.v == x.v && y.i < x.i)) ? y : x;
}
__device__ __forceinline__ Best block_best(Best x) {
  __shared__ Best part[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
  __syncthreads();
  x = part[0];
  for (int w = 1; w < kThreads / 32; ++w) x = better(x, part[w]);
  __syncthreads();
  return x;
}
__device__ __forceinline__ float block_sum(float x) {
  __shared__ float part[kThreads / 32];
  x = warp_sum_xor(x, 32);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0.f;
  for (int w = 0; w < kThreads / 32; ++w) x += part[w];
  __syncthreads();
  return x;
}

__device__ __forceinline__ float temperature_of(const VerifyArgs &p, int b) {
  return p.temperatures ? p.temperatures[b] : p.temperature;
}
__device__ __forceinline__ int drafts_of(const VerifyArgs &p, int b) {
  return p.draft_lens ? min(max(p.draft_lens[b], 0), p.num_drafts) : p.num_drafts;
}
// exp((x - max) / T); the entries at an infinite maximum share the mass.
__device__ __forceinline__ float weight_of(float x, float max, float inv_t) {
  return x == max ? 1.f : expf((x - max) * inv_t);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(const VerifyArgs p) {
  const int i = blockIdx.x, b = blockIdx.y;
  if (i > drafts_of(p, b)) return;
  const T *row = static_cast<const T *>(p.logits) + b * p.logits_seq_stride + i * p.logits_row_stride;
  Best best{-INFINITY, 0xffffffffu};
  for (int64_t v = threadIdx.x; v < p.vocab; v += kThreads) {
    const float x = load_logit(row, v);
    if (x > best.v) best = Best{x, (uint32_t)v};
  }
  best = block_best(best);
  const float t = temperature_of(p, b);
  float sum = 0.f;
  if (t > 0.f && best.v > -INFINITY) {
    const float inv_t = 1.f / t;
    for (int64_t v = threadIdx.x; v < p.vocab; v += kThreads) sum += weight_of(load_logit(row, v), best.v, inv_t);
    sum = block_sum(sum);
  }
  if (threadIdx.x == 0)
    static_cast<RowStat *>(p.workspace)[(int64_t)b * (p.num_drafts + 1) + i] =
        RowStat{best.v, sum, best.v > -INFINITY ? best.i : 0u, 0u};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_emit_kernel(const VerifyArgs p) {
  const int b = blockIdx.x;
  const int k = drafts_of(p, b);
  const float t = temperature_of(p, b);
  const float inv_t = t > 0.f ? 1.f / t : 0.f;
  const RowStat *stats = static_cast<const RowStat *>(p.workspace) + (int64_t)b * (p.num_drafts + 1);
  const T *rows = static_cast<const T *>(p.logits) + b * p.logits_seq_stride;
  const int32_t *drafts = p.draft_tokens + (int64_t)b * p.num_drafts;
  const unsigned char *probs = nullptr;
  const int prob_size = p.probs_dtype == VASR_PA_F32 ? 4 : 2;
  if (p.draft_probs) probs = static_cast<const unsigned char *>(p.draft_probs) + b * p.probs_seq_stride * prob_size;
  int n = 0;
  for (; n < k; ++n) {
    const int32_t x = drafts[n];
    const RowStat s = stats[n];
    if (x < 0 || x >= p.vocab || !(s.max > -INFINITY)) break;
    if (t > 0.f) {
      const float px = weight_of(load_logit(rows + n * p.logits_row_stride, x), s.max, inv_t) / s.sum;
      const float qx = probs ? load_prob(probs + n * p.probs_row_stride * prob_size, x, p.probs_dtype) : 1.f;
      if (!(p.uniform[(int64_t)b * p.num_drafts + n] * qx < px)) break;
    } else if ((uint32_t)x != s.arg) {
      break;
    }
  }
  const RowStat s = stats[n];
  uint32_t next = s.arg;
  if (t > 0.f && s.max > -INFINITY) {
    const T *row = rows + n * p.logits_row_stride;
    const float *race = p.race + b * p.race_seq_stride;
    const int64_t failed = n < k ? (int64_t)drafts[n] : -1;
    const unsigned char *q = probs && n < k ? probs + n * p.probs_row_stride * prob_size : nullptr;
    Best rest{0.f, 0xffffffffu}, all{0.f, 0xffffffffu};  // only positive values win
    for (int64_t v = threadIdx.x; v < p.vocab; v += kThreads) {
      const float pv = weight_of(load_logit(row, v), s.max, inv_t) / s.sum;
      float r = pv;
      if (q) r = pv - load_prob(q, v, p.probs_dtype);
      else if (v == failed) r = 0.f;
      const float e = race[v];
      const float a = r / e, c = pv / e;
      if (r > 0.f && a > rest.v) rest = Best{a, (uint32_t)v};
      if (pv > 0.f && c > all.v) all = Best{c, (uint32_t)v};
    }
    rest = block_best(rest);
    all = block_best(all);
    if (all.i == 0xffffffffu) all.i = s.arg;  // no weight over its noise is positive
    next = rest.i != 0xffffffffu ? rest.i : all.i;
  }
  if (threadIdx.x == 0) {
    int32_t *out = p.out_tokens + (int64_t)b * (p.num_drafts + 1);
    for (int i = 0; i <= p.num_drafts; ++i) out[i] = i < n ? drafts[i] : i == n ? (int32_t)next : -1;
    p.num_accepted[b] = n;
  }
}

template <typename T>
int launch_verify_t(const VerifyArgs &a, cudaStream_t s) {
  verify_rows_kernel<T><<<dim3((unsigned)a.num_drafts + 1, (unsigned)a.num_seqs), kThreads, 0, s>>>(a);
  verify_emit_kernel<T><<<(unsigned)a.num_seqs, kThreads, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? VASR_PA_OK : VASR_PA_ELAUNCH;
}

}  // namespace

size_t verify_workspace_bytes(int num_seqs, int num_drafts, int64_t) {
  return (size_t)num_seqs * (num_drafts + 1) * sizeof(RowStat);
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
