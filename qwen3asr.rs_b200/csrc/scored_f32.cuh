// scored_f32.cuh — scored decode attention in f32 (queries and pages),
// head_dim 128, on the CUDA cores.
//
// The split, its page ring and its end are those of scored_split.cuh; a tile
// has 2, 4 or 8 rows. Per 16 tokens of a stage, lane (token t, half hf) sums
// q . k over its half of the dims of every row (K chunks of 4 dims are
// adjacent for adjacent tokens, the rows' q are broadcast from shared memory),
// the halves meet in one shuffle, and the weights p go through shared memory
// to the P V sums, where a lane owns dims lane, lane + 32, lane + 64, lane +
// 96. Each lane starts its V row at another quad of tokens, so that the rows'
// 16-byte reads fall into different banks. Both sums run as packed f32x2 FMAs
// over neighbouring dims or tokens.
//
// Bound by the pages' bytes up to about 4 rows and by shared-memory reads
// above (a row more costs 32 q reads and 4 p reads per 16 tokens). 8 sequences
// of 4000 tokens, 16 heads over 8 (263 MB), take 62 us (4.2 TB/s); one thread a
// token took 201 us. 64 windows of 4 rows over 200 to 1500 tokens: 168 us.
#pragma once

#include "scored_split.cuh"

namespace vasr {

__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

template <int BS, int kRows, int NST>
__global__ void __launch_bounds__(kScoredThreads, BS <= 16 ? 3 : 1) scored_f32_kernel(const ScoredSplitParams p) {
  using C = ScoredCfg<float, BS, NST>;
  constexpr int D = C::D, kDims = D / 32;
  constexpr float kRescale = 8.f;  // the running maximum moves when a tile's exceeds it by 2^8
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(16) float s_q[kRows][D];
  __shared__ __align__(16) float s_p[C::kWarps][kRows][16];
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = lane & 15, hf = lane >> 4;
  ScoredSplit<float, BS, NST> sp;
  if (!sp.template begin<float>(p, smem, kRows)) return;
  const int row0 = sp.tile * kRows;
  for (int e = tid; e < kRows * D; e += kScoredThreads) {
    const int r = row0 + e / D, rr = r < p.rows ? r : 0;
    const float q = static_cast<const float *>(p.q)[((int64_t)sp.b * p.query_len + rr / p.group) * p.q_token_stride +
                                                    (int64_t)(sp.kvh * p.group + rr % p.group) * D + e % D];
    s_q[e / D][e % D] = r < p.rows ? q : 0.f;
  }
  __syncthreads();
  const bool use_softcap = p.softcap != 1.f;
  const float c_log2 = use_softcap ? p.scale : p.scale * kLog2e;
  // row i of the window sees tokens below n - query_len + 1 + i; all rows those below n_all
  const int n_all = sp.n - p.query_len + 1;
  const uint32_t a_q = smem_addr(&s_q[0][0]) + hf * (D / 2) * 4, a_p = smem_addr(&s_p[warp][0][0]);
  float o[kRows][kDims][2], m_used[kRows], l_part[kRows];  // O's even and odd tokens
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    m_used[r] = -INFINITY;
    l_part[r] = 0.f;
#pragma unroll
    for (int i = 0; i < kDims; ++i) o[r][i][0] = o[r][i][1] = 0.f;
  }
  bool aborted = false;
  int u_abort = 0;
  for (int u = warp; u < sp.n_units; u += C::kWarps) {
    const int s = u % NST;
    if (!sp.wait(u)) {
      aborted = true;
      u_abort = u;
      break;
    }
    const uint32_t sk = sp.s_base + C::kOffK + s * C::kSP * C::kPB;
    const uint32_t sv = sp.s_base + C::kOffV + s * C::kSP * C::kPB;
    const int unit0 = u * C::kST;                    // first token, relative to tok0
    const int valid = sp.tok1 - sp.tok0 - unit0;     // cached tokens of the stage
    const int whole = min(valid, n_all - sp.tok0 - unit0);  // those that every row sees
#pragma unroll
    for (int ti = 0; ti < C::kTiles; ++ti) {
      const int t0 = ti * 16, j = t0 + t;
      if (t0 >= valid) break;
      const bool tail = t0 + 16 > whole;
      // ---- q . k of the lane's token and half
      float dot[kRows][2];
#pragma unroll
      for (int r = 0; r < kRows; ++r) dot[r][0] = dot[r][1] = 0.f;
      const uint32_t krow = sk + (j / BS) * C::kPB + (hf * (D / 8) * BS + j % BS) * 16;
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const float4 k = lds_f4(krow + c * BS * 16);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float4 q = lds_f4(a_q + (r * D + c * 4) * 4);
          fma2(dot[r][0], dot[r][1], q.x, q.y, k.x, k.y);
          fma2(dot[r][0], dot[r][1], q.z, q.w, k.z, k.w);
        }
      }
      // ---- softmax over the tile
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        float x = dot[r][0] + dot[r][1];
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        x *= c_log2;
        if (use_softcap) x = p.softcap * tanhf(x / p.softcap) * kLog2e;
        const int row = row0 + r;
        if (tail && (j >= valid || unit0 + j >= n_all + row / p.group - sp.tok0)) x = -INFINITY;
        if (hf == 0 && row < p.scored_rows && j < valid) sp.x[row * sp.x_stride + unit0 + j] = x;
        if (__any_sync(0xffffffffu, x > m_used[r] + kRescale)) {
          const float m_new = fmaxf(m_used[r], warp_max_xor(x, 16));
          const float alpha = m_used[r] == -INFINITY ? 0.f : scored_exp2(m_used[r] - m_new);
          m_used[r] = m_new;
          l_part[r] *= alpha;
#pragma unroll
          for (int i = 0; i < kDims; ++i) {
            o[r][i][0] *= alpha;
            o[r][i][1] *= alpha;
          }
        }
        const float w = scored_exp2(x - (m_used[r] == -INFINITY ? 0.f : m_used[r]));
        l_part[r] += w;
        if (hf == 0) s_p[warp][r][t] = w;
      }
      __syncwarp();
      // ---- O += P V
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int quad = (q4 + (lane >> (BS == 8 ? 2 : BS == 16 ? 1 : 0))) & 3, jv = t0 + quad * 4;
        float4 v[kDims];
#pragma unroll
        for (int i = 0; i < kDims; ++i) v[i] = lds_f4(sv + (jv / BS) * C::kPB + ((lane + 32 * i) * BS + jv % BS) * 4);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float4 w = lds_f4(a_p + (r * 16 + quad * 4) * 4);
#pragma unroll
          for (int i = 0; i < kDims; ++i) {
            if (!tail) {
              fma2(o[r][i][0], o[r][i][1], w.x, w.y, v[i].x, v[i].y);
              fma2(o[r][i][0], o[r][i][1], w.z, w.w, v[i].z, v[i].w);
            } else {  // a token that the row does not see (weight 0) may hold anything
              if (w.x != 0.f) o[r][i][0] = fmaf(w.x, v[i].x, o[r][i][0]);
              if (w.y != 0.f) o[r][i][1] = fmaf(w.y, v[i].y, o[r][i][1]);
              if (w.z != 0.f) o[r][i][0] = fmaf(w.z, v[i].z, o[r][i][0]);
              if (w.w != 0.f) o[r][i][1] = fmaf(w.w, v[i].w, o[r][i][1]);
            }
          }
        }
      }
      __syncwarp();
    }
    sp.refill(p, u);
  }
  if (aborted) sp.drain(u_abort);
  __syncthreads();  // every stage is read: the ring becomes the warps' O
  float *co = reinterpret_cast<float *>(smem);                 // [warp][kRows][D]
  float2 *cml = reinterpret_cast<float2 *>(smem + C::kOffML);  // [warp][16]
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const float l = warp_sum_xor(l_part[r], 16);
    if (lane == 0) cml[warp * 16 + r] = aborted ? make_float2(-INFINITY, 0.f) : make_float2(m_used[r], l);
#pragma unroll
    for (int i = 0; i < kDims; ++i) co[(warp * kRows + r) * D + lane + 32 * i] = o[r][i][0] + o[r][i][1];
  }
  __syncthreads();
  sp.template end<float, kRows>(p, smem, 1.f);
}

}  // namespace vasr
