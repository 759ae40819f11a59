// mrope.cu — rotary embedding with several position axes: fused with the
// per-head q/k RMSNorm and the KV append, and alone (forwards or inverted).
//
// A token has one position per axis (time, height, width); frequency i of the
// R / 2 rotated pairs takes the angle of one axis, by sections laid out one
// after another or interleaved:
//   n = x rsqrt(mean(x^2) + eps) w                    (fused form; w may be absent)
//   y_i       = n_i cos - n_(i + R/2) sin             cos, sin = table[pos[axis(i)], i]
//   y_(i+R/2) = n_(i+R/2) cos + n_i sin
// The inverse turns by the negative angle; as the rotation is orthogonal it is
// also the gradient of the forward form. All arithmetic is f32 and each output
// is rounded once, when it is stored.
#include "common.cuh"
#include "launch.h"

namespace vasr {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxDim = 512;

__device__ __forceinline__ int axis_of(const MropeAngles &r, int i) {
  if (r.interleaved) {
    const int a = i % r.num_axes;
    return i / r.num_axes < r.sections[a] ? a : 0;
  }
  int a = 0, end = r.sections[0];
  while (a + 1 < r.num_axes && i >= end) end += r.sections[++a];
  return a;
}

// cos and sin of frequency i for token t; a position outside the table is
// clamped to it and recorded.
__device__ __forceinline__ float2 angle_of(const MropeAngles &r, int64_t t, int i) {
  int64_t pos = r.positions[axis_of(r, i) * r.axis_stride + t];
  if (pos < 0 || pos >= r.max_position) {
    raise_device_error(VASR_PA_DERR_POSITION_RANGE);
    pos = pos < 0 ? 0 : r.max_position - 1;
  }
  const int64_t at = pos * r.half + i;
  return make_float2(__ldg(r.cos_table + at), __ldg(r.sin_table + at));
}

template <typename T>
__device__ __forceinline__ void store_elem(T *p, float v, float) { *p = Elem<T>::from_f32(v); }
template <>
__device__ __forceinline__ void store_elem(__nv_fp8_e4m3 *p, float v, float scale) {
  *p = __nv_fp8_e4m3(v / scale);
}

// One warp per (token, head row), the row in shared memory as f32; any even
// rotary size and any head_dim up to 512.
template <typename T, typename TC>
__global__ void __launch_bounds__(32 * kWarps) mrope_append_rows_kernel(const MropeAppendArgs p) {
  __shared__ float rows[kWarps][kMaxDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tasks = p.num_heads + 2 * p.num_kv_heads;
  const int64_t gw = (int64_t)blockIdx.x * kWarps + warp;
  if (gw >= p.num_tokens * tasks) return;
  const int64_t t = gw / tasks;
  const int task = (int)(gw - t * tasks);
  const int D = p.head_dim, BS = p.block_size;
  const T *src = static_cast<const T *>(p.qkv) + t * p.qkv_token_stride + (int64_t)task * D;
  const bool is_q = task < p.num_heads;
  const bool is_v = task >= p.num_heads + p.num_kv_heads;
  const int h = is_q ? task : (task - p.num_heads) % p.num_kv_heads;
  int64_t slot = -1;
  if (!is_q) {
    slot = p.slot_mapping[t];
    if (slot >= p.num_blocks * BS) {
      if (lane == 0) raise_device_error(VASR_PA_DERR_SLOT_RANGE);
      slot = -1;
    }
    if (slot < 0) return;
  }
  float *row = rows[warp];
  float ss = 0.f;
  for (int d = lane; d < D; d += 32) {
    const float v = Elem<T>::to_f32(src[d]);
    row[d] = v;
    ss = fmaf(v, v, ss);
  }
  const int64_t blk = slot < 0 ? 0 : slot / BS;
  const int off = slot < 0 ? 0 : (int)(slot % BS);
  const int64_t page = (blk * p.num_kv_heads + h) * (int64_t)D * BS;
  if (is_v) {
    TC *v = static_cast<TC *>(p.value_cache) + page + off;
    const float scale = p.v_scale ? __ldg(p.v_scale) : 1.f;
    for (int d = lane; d < D; d += 32) store_elem<TC>(v + (int64_t)d * BS, row[d], scale);
    return;
  }
  if (p.q_norm_weight) {
    const float inv = rsqrtf(warp_sum_xor(ss, 32) / (float)D + p.eps);
    const T *w = static_cast<const T *>(is_q ? p.q_norm_weight : p.k_norm_weight);
    for (int d = lane; d < D; d += 32) row[d] *= inv * Elem<T>::to_f32(w[d]);
  }
  __syncwarp();
  for (int i = lane; i < p.rope.half; i += 32) {
    const float2 cs = angle_of(p.rope, t, i);
    const float a = row[i], b = row[i + p.rope.half];
    row[i] = a * cs.x - b * cs.y;
    row[i + p.rope.half] = b * cs.x + a * cs.y;
  }
  __syncwarp();
  if (is_q) {
    T *q = static_cast<T *>(p.q_out) + (t * p.num_heads + h) * (int64_t)D;
    for (int d = lane; d < D; d += 32) q[d] = Elem<T>::from_f32(row[d]);
    return;
  }
  constexpr int kX = Elem<TC>::kX;
  TC *k = static_cast<TC *>(p.key_cache) + page;
  const float scale = p.k_scale ? __ldg(p.k_scale) : 1.f;
  for (int d = lane; d < D; d += 32) store_elem<TC>(k + ((int64_t)(d / kX) * BS + off) * kX + d % kX, row[d], scale);
  if (p.score_cache && lane == 0) p.score_cache[(blk * p.num_kv_heads + h) * BS + off] = 0.f;
}

// One warp per (token, head) of x [T, H, D]; a lane owns whole pairs, so
// out may be x itself.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) mrope_rows_kernel(const MropeArgs p) {
  const int lane = threadIdx.x & 31;
  const int64_t gw = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (gw >= p.num_tokens * p.num_heads) return;
  const int64_t t = gw / p.num_heads;
  const int h = (int)(gw - t * p.num_heads);
  const T *x = static_cast<const T *>(p.x) + t * p.x_token_stride + h * p.x_head_stride;
  T *y = static_cast<T *>(p.out) + t * p.out_token_stride + h * p.out_head_stride;
  const int half = p.rope.half;
  for (int i = lane; i < half; i += 32) {
    float2 cs = angle_of(p.rope, t, i);
    if (p.inverse) cs.y = -cs.y;
    const float a = Elem<T>::to_f32(x[i]), b = Elem<T>::to_f32(x[i + half]);
    y[i] = Elem<T>::from_f32(a * cs.x - b * cs.y);
    y[i + half] = Elem<T>::from_f32(b * cs.x + a * cs.y);
  }
  for (int d = 2 * half + lane; d < p.head_dim; d += 32) y[d] = x[d];
}

template <typename T, typename TC>
int launch_append_tc(const MropeAppendArgs &a, cudaStream_t s) {
  const int64_t warps = a.num_tokens * (a.num_heads + 2 * a.num_kv_heads);
  const int64_t ctas = (warps + kWarps - 1) / kWarps;
  if (ctas > 0x7fffffff) return VASR_PA_EINVAL_SHAPE;
  mrope_append_rows_kernel<T, TC><<<(unsigned)ctas, 32 * kWarps, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? VASR_PA_OK : VASR_PA_ELAUNCH;
}

template <typename T>
int launch_append_t(const MropeAppendArgs &a, cudaStream_t s) {
  if (a.cache_dtype == VASR_PA_FP8_E4M3) return launch_append_tc<T, __nv_fp8_e4m3>(a, s);
  return launch_append_tc<T, T>(a, s);
}

template <typename T>
int launch_rows_t(const MropeArgs &a, cudaStream_t s) {
  const int64_t ctas = (a.num_tokens * a.num_heads + kWarps - 1) / kWarps;
  if (ctas > 0x7fffffff) return VASR_PA_EINVAL_SHAPE;
  mrope_rows_kernel<T><<<(unsigned)ctas, 32 * kWarps, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? VASR_PA_OK : VASR_PA_ELAUNCH;
}

}  // namespace

int launch_mrope_append(const MropeAppendArgs &a, cudaStream_t s) {
  switch (a.dtype) {
    case VASR_PA_F32: return launch_append_t<float>(a, s);
    case VASR_PA_BF16: return launch_append_t<__nv_bfloat16>(a, s);
    case VASR_PA_F16: return launch_append_t<__half>(a, s);
    default: return VASR_PA_EINVAL_DTYPE;
  }
}

int launch_mrope(const MropeArgs &a, cudaStream_t s) {
  switch (a.dtype) {
    case VASR_PA_F32: return launch_rows_t<float>(a, s);
    case VASR_PA_BF16: return launch_rows_t<__nv_bfloat16>(a, s);
    case VASR_PA_F16: return launch_rows_t<__half>(a, s);
    default: return VASR_PA_EINVAL_DTYPE;
  }
}

int read_error_mrope(uint32_t *bits, bool clear, cudaStream_t s) {
  return read_unit_error(bits, clear, s);
}

}  // namespace vasr
