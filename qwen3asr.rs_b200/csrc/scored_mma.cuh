// scored_mma.cuh — scored decode attention on the tensor cores (mma.sync
// m16n8k16, f32 accumulate) for 16-bit queries over 16-bit or fp8 pages,
// head_dim 128.
//
// The split, its page ring and its end are those of scored_split.cuh. Per 16
// tokens a warp computes
//   S[16 rows x 16] = Q K^T     A = Q, B = K by ldmatrix from the page layout
//   O^T[128 x rows] += V^T P^T  A = V^T by ldmatrix, B = S's own fragments
//
// P enters its product in two parts of the operand type, what it rounds to and
// what that rounding left, so that O has P to 2^-16 (bf16) or 2^-22 (f16) and a
// window's rows answer as single tokens do. Up to 4 rows (kDup: one token,
// group <= 4) P^T has columns to spare: A holds every query row twice, so the
// score fragments of rows r and r + 4 are equal, and row r + 4 carries row r's
// rest for no further MMA. With more rows the rest takes MMAs of its own. P
// rounded alone was 2.8 instead of 2.1 parts in 10^4 off 64 bits for windows of
// 5 f16 rows (2.1 is the output's own rounding) and took, in us through the
// public call, 50.7 against 52.9 there, 43.9 / 45.1 for windows of 4 bf16 rows,
// 326 / 348 for 256 windows of 5 over 500 to 4000 tokens, 121 / 129 for 16 rows
// all scored, 37.6 / 38.9 for windows of 4 over fp8 pages.
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
//
// With bf16 pages and one token a sequence this is bound by memory: 512
// sequences of 64 to 4096 tokens, 16 heads over 8, are 2.00 GB and take 317 us
// with the join (6.3 TB/s; 291 us without any scores). mma.sync suffices: at 2
// to 10 rows a 128-row tcgen05 tile would be empty. One sequence of 16381
// tokens (68 MB) takes 17 us (3.9 TB/s; the split alone 13.4). fp8 pages and
// windows are bound by how evenly the contexts fall on the SMs and by the chain
// from MMA to softmax to MMA: 64 sequences of 200 to 1500 tokens take 31 us from
// fp8 pages (99 MB; SMs busy 72% of the time, issuing in 45% of those cycles) and
// 51 us for windows of 5 f16 rows (197 MB; 79% and 39%).
#pragma once

#include "decode_mma.cuh"
#include "scored_split.cuh"

namespace vasr {

template <typename T, typename TC, int BS, int NRT, bool kDup, int NST, int MINB>
__global__ void __launch_bounds__(kScoredThreads, MINB) scored_mma_kernel(const ScoredSplitParams p) {
  using C = ScoredCfg<TC, BS, NST>;
  constexpr bool kFp8 = std::is_same<TC, __nv_fp8_e4m3>::value;
  using TM = typename std::conditional<kFp8, __half, T>::type;  // MMA operand type
  constexpr int D = C::D, kKS = D / 16, kRows = kDup ? 4 : 8 * NRT;
  constexpr float kRescale = 8.f;  // the running maximum moves when a tile's exceeds it by 2^8
  // P is 2^(x - m + kLift): in f16 it then fills the range up to 2^15, and
  // weights down to 2^-31 of the largest are not lost
  constexpr float kLift = std::is_same<TM, __half>::value ? 7.f : 0.f;
  static_assert(!kDup || NRT == 1, "doubled rows fill one tile of 8");
  extern __shared__ __align__(128) unsigned char smem[];
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = lane >> 2, tig = lane & 3;
  ScoredSplit<TC, BS, NST> sp;
  if (!sp.template begin<T>(p, smem, kRows)) return;
  const uint32_t s_base = sp.s_base;
  const int kvh = sp.kvh, b = sp.b, n = sp.n, tok0 = sp.tok0, tok1 = sp.tok1, n_units = sp.n_units;
  const int row0 = sp.tile * kRows;
  const float v_mul = p.v_scale ? __ldg(p.v_scale) : 1.f;

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
  int seen[NRT];
  float *xrow[NRT];
#pragma unroll
  for (int t = 0; t < NRT; ++t) {
    seen[t] = row[t] < 0 ? 0 : n_all + row[t] / p.group - tok0;
    xrow[t] = nullptr;
    if (row[t] >= 0 && row[t] < p.scored_rows && !(kDup && grp >= 4))
      xrow[t] = sp.x + row[t] * sp.x_stride;
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
    if (!sp.wait(u)) {
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
      uint32_t pa[NRT][2], rest[NRT][2];  // P in the operand type, and what that rounding left
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
        const float off = m_used[t] == -INFINITY ? 0.f : m_used[t] - kLift;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pv[t][e] = scored_exp2(x[e] - off);
          l_part[t] += pv[t][e];
        }
#pragma unroll
        for (int nn = 0; nn < 2; ++nn) {
          pa[t][nn] = dec_pack2<TM>(pv[t][2 * nn], pv[t][2 * nn + 1]);
          const TM *h = reinterpret_cast<const TM *>(&pa[t][nn]);
          rest[t][nn] = dec_pack2<TM>(pv[t][2 * nn] - Elem<TM>::to_f32(h[0]), pv[t][2 * nn + 1] - Elem<TM>::to_f32(h[1]));
          if (kDup && grp >= 4) pa[t][nn] = rest[t][nn];  // rows 4..7: the rest of rows 0..3
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
            for (int t = 0; t < NRT; ++t) {
              dec_mma<TM>(o[t][dq * 2 + hf], a0, a1, a2, a3, pa[t][0], pa[t][1]);
              if constexpr (!kDup) dec_mma<TM>(o[t][dq * 2 + hf], a0, a1, a2, a3, rest[t][0], rest[t][1]);
            }
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
          for (int t = 0; t < NRT; ++t) {
            dec_mma<TM>(o[t][dp], b0, b2, b1, b3, pa[t][0], pa[t][1]);
            if constexpr (!kDup) dec_mma<TM>(o[t][dp], b0, b2, b1, b3, rest[t][0], rest[t][1]);
          }
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
    sp.refill(p, u);
  }
  if (aborted) sp.drain(u_abort);
  __syncthreads();  // every stage is read: the ring becomes the warps' O

  float *co = reinterpret_cast<float *>(smem);  // [warp][kRows][D]
  float2 *cml = reinterpret_cast<float2 *>(smem + C::kOffML);  // [warp][16]
#pragma unroll
  for (int t = 0; t < NRT; ++t) {
    float l = l_part[t];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (tig == 0 && !(kDup && grp >= 4))
      cml[warp * 16 + 8 * t + grp] = aborted ? make_float2(-INFINITY, 0.f) : make_float2(m_used[t] - kLift, l);
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
  sp.template end<T, kRows>(p, smem, v_mul);
}

}  // namespace vasr
