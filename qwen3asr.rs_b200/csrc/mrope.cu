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
//
// Calls of a few tokens are bound by the latency of a launch and three
// dependent loads (position, angle, store): 64 tokens of 16 + 8 + 8 heads of
// 128 take 4.1 us. Long ones are bound by memory: 8192 such tokens (139 MB in
// bf16, prompts into pages) take 29 us, 4.7 TB/s; 4099 tokens of 24 heads
// turned back (52 MB) 12 us, 4.3 TB/s: a thread asks for its rows only once its
// angles are there, and the grid starts and ends. A torch elementwise kernel
// over the same bytes takes 36.9 and 15.3 us. The general kernels below, a warp a row, took 157 and 35 us there.
#include <type_traits>

#include "common.cuh"
#include "launch.h"

namespace vasr {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxDim = 512;

__device__ __forceinline__ int axis_of(const MropeAngles &r, int i) {
  return (int)(r.axis_bits[i / 16] >> (2 * (i % 16))) & 3;
}

// Position of token t on axis a; one outside the table is clamped to it and
// recorded.
__device__ __forceinline__ int64_t position_of(const MropeAngles &r, int64_t t, int a) {
  const int64_t pos = r.positions[a * r.axis_stride + t];
  if (pos >= 0 && pos < r.max_position) return pos;
  raise_device_error(VASR_PA_DERR_POSITION_RANGE);
  return pos < 0 ? 0 : r.max_position - 1;
}

// cos and sin of frequency i for token t.
__device__ __forceinline__ float2 angle_of(const MropeAngles &r, int64_t t, int i) {
  const int64_t at = position_of(r, t, axis_of(r, i)) * r.half + i;
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

// ------------------------------------------------------------ vector kernels
// Rows whose D / 2 rotated pairs fall into whole 16-byte chunks: a thread owns
// chunk c and its partner c + C / 2 of a token's row (C chunks a row), so both
// halves of its pairs are its own and the norm is a sum over the C / 2 lanes
// of the row. It loads its cos and sin once and runs over the heads with them
// (a warp a row loads them again for every head). Every other R, head_dim,
// stride or alignment takes the general kernels.
template <int kX>
struct Angles {
  float c[kX], s[kX];
  // frequencies [i0, i0 + kX), i0 a multiple of kX (4 or 8): one word of axis
  // bits; every axis' row in vectors (16-byte aligned), then a choice per frequency
  __device__ __forceinline__ void load(const MropeAngles &r, int64_t t, int i0) {
    const uint32_t bits = r.axis_bits[i0 / 16] >> (2 * (i0 % 16));
#pragma unroll
    for (int a = 0; a < kMropeMaxAxes; ++a) {
      if (a >= r.num_axes) break;
      const int64_t at = position_of(r, t, a) * r.half + i0;
#pragma unroll
      for (int v = 0; v < kX / 4; ++v) {
        const float4 cv = __ldg(reinterpret_cast<const float4 *>(r.cos_table + at) + v);
        const float4 sv = __ldg(reinterpret_cast<const float4 *>(r.sin_table + at) + v);
        const float cf[4] = {cv.x, cv.y, cv.z, cv.w}, sf[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool mine = a == 0 || (bits >> (2 * (4 * v + e)) & 3u) == (uint32_t)a;
          c[4 * v + e] = mine ? cf[e] : c[4 * v + e];
          s[4 * v + e] = mine ? sf[e] : s[4 * v + e];
        }
      }
    }
  }
  // (a, b) turned, all pairs; sums and products of two frequencies at a time
  __device__ __forceinline__ void turn(float (&a)[kX], float (&b)[kX]) const {
#pragma unroll
    for (int e = 0; e < kX; e += 2) {
      float x0 = a[e], x1 = a[e + 1], y0 = b[e], y1 = b[e + 1];
      mul2(a[e], a[e + 1], x0, x1, c[e], c[e + 1]);
      mul2(b[e], b[e + 1], y0, y1, c[e], c[e + 1]);
      fma2(a[e], a[e + 1], y0, y1, -s[e], -s[e + 1]);
      fma2(b[e], b[e + 1], x0, x1, s[e], s[e + 1]);
    }
  }
};

template <typename T>
__device__ __forceinline__ uint4 pack_chunk(const float (&f)[Elem<T>::kX]) {
  uint4 u;
  if constexpr (sizeof(T) == 4) {
    u = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 *e = reinterpret_cast<T2 *>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) e[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      else e[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    }
  }
  return u;
}

// kX consecutive dims of one token into a K page (dims d0 .. of a chunk).
template <typename TC, int kX>
__device__ __forceinline__ void store_key(TC *at, const float (&f)[kX], float scale) {
  if constexpr (sizeof(TC) == 1) {
    uint32_t w[kX / 4];
#pragma unroll
    for (int i = 0; i < kX; ++i)
      reinterpret_cast<__nv_fp8_e4m3 *>(w)[i] = __nv_fp8_e4m3(f[i] / scale);
    if constexpr (kX == 8) *reinterpret_cast<uint2 *>(at) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t *>(at) = w[0];
  } else {
    (void)scale;
    *reinterpret_cast<uint4 *>(at) = pack_chunk<TC>(f);
  }
}

// A prompt's CTA has a tile of 16 tokens and a warp for each warp's worth of
// them (at most 8), which runs over all heads of its part with one set of
// angles; a decode step's CTA one warp's worth of tokens and 8 warps that
// split the heads.
constexpr int tile_tokens(int tokens_per_warp, bool prompt) {
  return !prompt ? tokens_per_warp : 8 * tokens_per_warp < 16 ? 8 * tokens_per_warp : 16;
}
template <typename T, int D>
constexpr int tile_warps(bool prompt) {
  return prompt ? tile_tokens(64 / (D / Elem<T>::kX), true) / (64 / (D / Elem<T>::kX)) : 8;
}

// Prompts: the part's heads of the tile's rows arrive by one bulk copy a token
// (a token's heads are adjacent), so that the bytes in flight cost shared
// memory and not registers; rows are 16 bytes apart modulo 128 to spread banks.
// Smaller parts mean more CTAs per SM and less imbalance at the end, until the
// angles are loaded too often: 29 us at 8192 tokens, against 32 with parts of
// 2048 bytes, 30 with 1536 and 31 with 1024.
constexpr int kPartBytes = 1280;  // of one token's row at most
template <typename T, int D>
constexpr int part_heads() { return kPartBytes / (D * (int)sizeof(T)) > 0 ? kPartBytes / (D * (int)sizeof(T)) : 1; }
template <typename T, int D>
constexpr int part_pitch() { return part_heads<T, D>() * D * (int)sizeof(T) + 16; }

// grid = (token tile, part): the first qk_parts parts share the tile's q and k
// heads, the others its V. Warps split a tile's tokens and its heads. V goes
// out element by element with the tile's tokens across the lanes: consecutive
// slots fill a page row's 32-byte sectors whole in one store, and any other
// slots need no case of their own.
template <typename T, typename TC, int D, bool kPrompt>
__global__ void __launch_bounds__(32 * tile_warps<T, D>(kPrompt)) mrope_append_tile_kernel(const MropeAppendArgs p,
                                                                                          int qk_parts) {
  pdl_launch_dependents();  // a decode behind this kernel reads nothing it writes before it has ended
  constexpr int kX = Elem<T>::kX, C = D / kX, L = C / 2, kPerWarp = 32 / L;
  constexpr int kTile = tile_tokens(kPerWarp, kPrompt), kGroups = kTile / kPerWarp;
  constexpr int kCtaWarps = tile_warps<T, D>(kPrompt), kHeadLanes = kCtaWarps / kGroups;
  constexpr int kXc = Elem<TC>::kX;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int shift = 31 - __clz(p.block_size);
  const int64_t tile0 = (int64_t)blockIdx.x * kTile;
  auto slot_of = [&](int64_t t) -> int64_t {
    if (t >= p.num_tokens) return -1;
    const int64_t slot = p.slot_mapping[t];
    if (slot < p.num_blocks << shift) return slot;
    raise_device_error(VASR_PA_DERR_SLOT_RANGE);
    return -1;
  };
  const bool is_v = (int)blockIdx.y >= qk_parts;
  const int part = is_v ? blockIdx.y - qk_parts : blockIdx.y, parts = is_v ? gridDim.y - qk_parts : qk_parts;
  const int heads = is_v ? p.num_kv_heads : p.num_heads + p.num_kv_heads;
  // prompts: a part has its heads [h0, h1) in shared memory; else they are dealt out
  constexpr int kPitch = part_pitch<T, D>();
  const int per = (heads + parts - 1) / parts;
  const int h0 = kPrompt ? part * per : 0, h1 = kPrompt ? min(heads, h0 + per) : heads;
  extern __shared__ __align__(128) unsigned char rows[];
  __shared__ __align__(8) uint64_t s_bar;
  if constexpr (kPrompt) {
    const uint32_t bar = smem_addr(&s_bar);
    const int ntok = (int)min((int64_t)kTile, p.num_tokens - tile0);
    const uint32_t bytes = (uint32_t)(max(h1 - h0, 0) * D * (int)sizeof(T));
    if (threadIdx.x == 0) {
      mbar_init(bar, 1);
      mbar_fence_init();
      mbar_arrive_expect_tx(bar, ntok * bytes);
    }
    __syncthreads();
    if ((int)threadIdx.x < ntok && bytes > 0)
      bulk_g2s(smem_addr(rows) + threadIdx.x * kPitch,
               static_cast<const T *>(p.qkv) + (tile0 + threadIdx.x) * p.qkv_token_stride +
                   (int64_t)((is_v ? p.num_heads + p.num_kv_heads : 0) + h0) * D,
               bytes, bar);
  }
  // false: the copies did not come (recorded); waited for once more, so that they do not outlive the CTA
  auto rows_here = [&]() {
    if constexpr (kPrompt) {
      if (mbar_wait_bounded(smem_addr(&s_bar), 0)) return true;
      mbar_wait_bounded(smem_addr(&s_bar), 0);
      return false;
    }
    return true;
  };
  if (!is_v) {
    const int c = lane % L;
    const int64_t t = tile0 + (warp % kGroups) * kPerWarp + lane / L;
    const bool live = t < p.num_tokens;
    const int64_t tt = live ? t : p.num_tokens - 1;  // lanes past the end follow, for the shuffles
    const T *src = static_cast<const T *>(p.qkv) + tt * p.qkv_token_stride + c * kX;
    const int step = kPrompt ? kHeadLanes : kHeadLanes * parts;
    int h = h0 + warp / kGroups + (kPrompt ? 0 : kHeadLanes * part);
    const int64_t slot = slot_of(t);
    auto load = [&](int head, uint4 (&r)[2]) {
      if constexpr (kPrompt) {
        const unsigned char *at = rows + (tt - tile0) * kPitch + ((head - h0) * D + c * kX) * (int)sizeof(T);
        r[0] = *reinterpret_cast<const uint4 *>(at);
        r[1] = *reinterpret_cast<const uint4 *>(at + D / 2 * (int)sizeof(T));
      } else {
        r[0] = __ldg(reinterpret_cast<const uint4 *>(src + (int64_t)head * D));
        r[1] = __ldg(reinterpret_cast<const uint4 *>(src + (int64_t)head * D + D / 2));
      }
    };
    uint4 raw[2], w[2];
    if (!kPrompt && h < h1) load(h, raw);
    Angles<kX> ang;
    ang.load(p.rope, tt, c * kX);
    if (!rows_here()) return;
    const float k_scale = p.k_scale ? __ldg(p.k_scale) : 1.f;
    const int64_t page0 = (slot >> shift) * p.num_kv_heads;
    const int off = (int)(slot & (p.block_size - 1));
    const T *weight = nullptr;
    for (; h < h1; h += step) {
      if constexpr (kPrompt) load(h, raw);
      const bool is_q = h < p.num_heads;
      const T *mine = static_cast<const T *>(is_q ? p.q_norm_weight : p.k_norm_weight);
      if (mine != weight) {
        weight = mine;
        w[0] = __ldg(reinterpret_cast<const uint4 *>(weight + c * kX));
        w[1] = __ldg(reinterpret_cast<const uint4 *>(weight + c * kX + D / 2));
      }
      float a[kX], b[kX];
      unpack_chunk<T>(raw[0], a);
      unpack_chunk<T>(raw[1], b);
      if (!kPrompt && h + step < h1) load(h + step, raw);  // while this row is worked on
      if (weight) {
        float s0 = 0.f, s1 = 0.f, wa[kX], wb[kX];
#pragma unroll
        for (int e = 0; e < kX; e += 2) {
          fma2(s0, s1, a[e], a[e + 1], a[e], a[e + 1]);
          fma2(s0, s1, b[e], b[e + 1], b[e], b[e + 1]);
        }
        const float inv = rsqrtf(warp_sum_xor(s0 + s1, L) / (float)D + p.eps);
        unpack_chunk<T>(w[0], wa);
        unpack_chunk<T>(w[1], wb);
#pragma unroll
        for (int e = 0; e < kX; e += 2) {
          mul2(wa[e], wa[e + 1], wa[e], wa[e + 1], inv, inv);
          mul2(wb[e], wb[e + 1], wb[e], wb[e + 1], inv, inv);
          mul2(a[e], a[e + 1], a[e], a[e + 1], wa[e], wa[e + 1]);
          mul2(b[e], b[e + 1], b[e], b[e + 1], wb[e], wb[e + 1]);
        }
      }
      ang.turn(a, b);
      if (is_q) {
        if (live) {
          T *q = static_cast<T *>(p.q_out) + (t * p.num_heads + h) * D + c * kX;
          *reinterpret_cast<uint4 *>(q) = pack_chunk<T>(a);
          *reinterpret_cast<uint4 *>(q + D / 2) = pack_chunk<T>(b);
        }
      } else if (slot >= 0) {
        const int64_t page = page0 + h - p.num_heads;
        auto place = [&](int d) {
          return static_cast<TC *>(p.key_cache) + (((page * (D / kXc) + d / kXc) << shift) + off) * kXc + d % kXc;
        };
        store_key<TC, kX>(place(c * kX), a, k_scale);
        store_key<TC, kX>(place(c * kX + D / 2), b, k_scale);
        if (p.score_cache && c == 0) p.score_cache[(page << shift) + off] = 0.f;
      }
    }
    return;
  }
  // ---- v: item = (head, group of chunks), the tile's tokens across the lanes
  constexpr int kChunks = 32 / kTile, kItems = C / kChunks;
  const int64_t t = tile0 + lane % kTile;
  const int cc = lane / kTile;
  const int64_t slot = slot_of(t);
  if (!rows_here() || slot < 0) return;
  const T *src = static_cast<const T *>(p.qkv) + t * p.qkv_token_stride + (int64_t)(p.num_heads + p.num_kv_heads) * D;
  TC *dst = static_cast<TC *>(p.value_cache) + (((slot >> shift) * p.num_kv_heads * D) << shift) +
            (slot & (p.block_size - 1));
  const float v_scale = p.v_scale ? __ldg(p.v_scale) : 1.f;
  const int step = kPrompt ? kCtaWarps : kCtaWarps * parts;
#pragma unroll 4
  for (int i = h0 * kItems + warp + (kPrompt ? 0 : kCtaWarps * part); i < h1 * kItems; i += step) {
    const int d = (i * kChunks + cc) * kX;  // dim of the token's V row, over the heads
    uint4 raw;
    if constexpr (kPrompt)
      raw = *reinterpret_cast<const uint4 *>(rows + lane % kTile * kPitch + (d - h0 * D) * (int)sizeof(T));
    else
      raw = __ldg(reinterpret_cast<const uint4 *>(src + d));
    TC *at = dst + ((int64_t)d << shift);
    if constexpr (std::is_same<T, TC>::value) {
      const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
      for (int k = 0; k < kX; ++k) at[(int64_t)k << shift] = e[k];
    } else {
      float f[kX];
      unpack_chunk<T>(raw, f);
#pragma unroll
      for (int k = 0; k < kX; ++k) at[(int64_t)k << shift] = __nv_fp8_e4m3(f[k] / v_scale);
    }
  }
}

// x [T, H, D] turned: a warp per C / 2-lane token group and part of the heads.
template <typename T, int D>
__global__ void __launch_bounds__(32 * kWarps) mrope_tile_kernel(const MropeArgs p) {
  constexpr int kX = Elem<T>::kX, L = D / kX / 2, kTile = 32 * kWarps / L;  // tokens of a CTA
  const int c = threadIdx.x % L;
  const int64_t t = (int64_t)blockIdx.x * kTile + threadIdx.x / L;
  if (t >= p.num_tokens) return;
  Angles<kX> ang;
  ang.load(p.rope, t, c * kX);
#pragma unroll
  for (int e = 0; e < kX; ++e)
    if (p.inverse) ang.s[e] = -ang.s[e];
  const T *x = static_cast<const T *>(p.x) + t * p.x_token_stride + c * kX;
  T *y = static_cast<T *>(p.out) + t * p.out_token_stride + c * kX;
#pragma unroll 4
  for (int h = blockIdx.y; h < p.num_heads; h += gridDim.y) {
    float a[kX], b[kX];
    // plain loads: y may be x
    unpack_chunk<T>(*reinterpret_cast<const uint4 *>(x + h * p.x_head_stride), a);
    unpack_chunk<T>(*reinterpret_cast<const uint4 *>(x + h * p.x_head_stride + D / 2), b);
    ang.turn(a, b);
    *reinterpret_cast<uint4 *>(y + h * p.out_head_stride) = pack_chunk<T>(a);
    *reinterpret_cast<uint4 *>(y + h * p.out_head_stride + D / 2) = pack_chunk<T>(b);
  }
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
// Calls of kPromptTokens or more take the prompt form: 5.1 against 5.4 us at
// 512 tokens (16 + 8 heads of 128), 5.6 / 7.0 at 1000, 4.5 / 4.0 at 256.
constexpr int kPromptTokens = 512;
// Short calls split the heads over more CTAs until there are this many: 12.1 us
// at 4099 tokens of 24 heads, against 15.3 with half and 13.3 with twice as many.
constexpr int kTargetCtas = 4 * 148;

template <typename T, typename TC, int D, bool kPrompt>
int launch_append_tile(const MropeAppendArgs &a, cudaStream_t s) {
  constexpr int kPerWarp = 32 / (D / Elem<T>::kX / 2);
  constexpr int kTile = tile_tokens(kPerWarp, kPrompt), kCtaWarps = tile_warps<T, D>(kPrompt);
  constexpr int kHeadLanes = kCtaWarps / (kTile / kPerWarp);
  const int64_t tiles = (a.num_tokens + kTile - 1) / kTile;
  int64_t qk, v;
  int smem = 0;
  if (kPrompt) {
    qk = (a.num_heads + a.num_kv_heads + part_heads<T, D>() - 1) / part_heads<T, D>();
    v = (a.num_kv_heads + part_heads<T, D>() - 1) / part_heads<T, D>();
    smem = kTile * part_pitch<T, D>();
  } else {  // as many parts as give kTargetCtas, a part per row at most; V's share of them as its rows are of all
    const int qk_most = (a.num_heads + a.num_kv_heads + kHeadLanes - 1) / kHeadLanes;
    const int v_most = (a.num_kv_heads * (D / Elem<T>::kX) * kTile / 32 + kCtaWarps - 1) / kCtaWarps;
    const int64_t parts = kTargetCtas / tiles > 2 ? kTargetCtas / tiles : 2;
    v = parts * a.num_kv_heads / (a.num_heads + 2 * a.num_kv_heads);
    v = v < 1 ? 1 : v > v_most ? v_most : v;
    qk = parts - v;
    qk = qk > qk_most ? qk_most : qk;
  }
  if (tiles > 0x7fffffff || qk + v > 65535) return VASR_PA_EINVAL_SHAPE;
  mrope_append_tile_kernel<T, TC, D, kPrompt><<<dim3((unsigned)tiles, (unsigned)(qk + v)), 32 * kCtaWarps, smem, s>>>(a, (int)qk);
  return cudaPeekAtLastError() == cudaSuccess ? VASR_PA_OK : VASR_PA_ELAUNCH;
}

template <typename T, typename TC, int D>
int launch_append_d(const MropeAppendArgs &a, cudaStream_t s) {
  if (a.num_tokens >= kPromptTokens) return launch_append_tile<T, TC, D, true>(a, s);
  return launch_append_tile<T, TC, D, false>(a, s);
}

template <typename T, int D>
int launch_tile(const MropeArgs &a, cudaStream_t s) {
  constexpr int kTile = 32 * kWarps / (D / Elem<T>::kX / 2);
  const int64_t tiles = (a.num_tokens + kTile - 1) / kTile;
  int64_t parts = kTargetCtas / tiles;
  parts = parts < 1 ? 1 : parts > a.num_heads ? a.num_heads : parts;
  if (tiles > 0x7fffffff || parts > 65535) return VASR_PA_EINVAL_SHAPE;
  mrope_tile_kernel<T, D><<<dim3((unsigned)tiles, (unsigned)parts), 32 * kWarps, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? VASR_PA_OK : VASR_PA_ELAUNCH;
}

template <typename T, typename TC>
int launch_append_tc(const MropeAppendArgs &a, cudaStream_t s) {
  if (2 * a.rope.half == a.head_dim && aligned16(a.rope.cos_table) && aligned16(a.rope.sin_table) && aligned16(a.qkv) && (a.qkv_token_stride * (int64_t)sizeof(T)) % 16 == 0 &&
      aligned16(a.q_out) && aligned16(a.q_norm_weight) && aligned16(a.k_norm_weight)) {
    switch (a.head_dim) {
      case 64: return launch_append_d<T, TC, 64>(a, s);
      case 128: return launch_append_d<T, TC, 128>(a, s);
      case 256: return launch_append_d<T, TC, 256>(a, s);
      default: break;
    }
  }
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
  auto whole = [](int64_t stride) { return stride * (int64_t)sizeof(T) % 16 == 0; };
  if (2 * a.rope.half == a.head_dim && aligned16(a.rope.cos_table) && aligned16(a.rope.sin_table) && aligned16(a.x) && aligned16(a.out) && whole(a.x_token_stride) &&
      whole(a.x_head_stride) && whole(a.out_token_stride) && whole(a.out_head_stride)) {
    switch (a.head_dim) {
      case 64: return launch_tile<T, 64>(a, s);
      case 128: return launch_tile<T, 128>(a, s);
      case 256: return launch_tile<T, 256>(a, s);
      default: break;
    }
  }
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

uint32_t *error_word_mrope() { return unit_error_word(); }

}  // namespace vasr
