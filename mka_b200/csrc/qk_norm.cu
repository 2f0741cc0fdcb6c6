// Norms of the query and key heads with the position rotation, in one pass.
//
// For every token t and head h, with x = q[t, h, :] or k[t, h, :] (128 channels):
//   n = x * rsqrt(mean(x^2) + eps) * w            (w of the q or the k norm)
//   y[d]      = n[d]      * cos[d]      - n[d + 64] * sin[d]         d < 64
//   y[d + 64] = n[d + 64] * cos[d + 64] + n[d]      * sin[d + 64]
// all in fp32, rounded to bf16 once (a chain of modules rounds after the norm,
// after the weight and after each product; one rounding is closer to the
// formula). Either half may be left out: no weight is no norm, no table is no
// rotation.
//
// Bound by HBM: each row of 256 bytes is read once and written once, and each
// token's cos and sin rows (1 KB) are read once per warp that serves it. Eight
// lanes own a row: lane l holds channels [8l, 8l+8) and their partners
// [64 + 8l, 64 + 8l + 8) in two 16-byte loads, so the rotation needs no
// exchange and the sum of squares three shuffles; a warp takes four rows at a
// time, and several heads of one token in turn, so that the cos and sin
// registers are loaded once for all of them.
#include "fmka_internal.h"
#include "ptx.cuh"

namespace fmka {

namespace {

constexpr int kHeadDim = 128;
constexpr int kWarps = 4;
constexpr int kRowsPerWarp = 4;

__device__ __forceinline__ void unpack8(const uint4& a, float* f) {
  const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf16lo_to_f32(u[i]);
    f[2 * i + 1] = bf16hi_to_f32(u[i]);
  }
}

__device__ __forceinline__ void load_f32x8(const float* p, float* f) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

__device__ __forceinline__ void load_weight(const void* w, int f32, int l, float* f) {
  if (f32) {
    load_f32x8(static_cast<const float*>(w) + 8 * l, f);
    load_f32x8(static_cast<const float*>(w) + 64 + 8 * l, f + 8);
  } else {
    const uint4* p = static_cast<const uint4*>(w);
    unpack8(__ldg(p + l), f);
    unpack8(__ldg(p + 8 + l), f + 8);
  }
}

__global__ void __launch_bounds__(kWarps * 32) qk_norm_rope_kernel(const __grid_constant__ QkNormParams p) {
  const int lane = lane_id();
  const int l = lane & 7;
  const int sub = lane >> 3;
  const int heads = p.Hq + p.Hk;
  const int per_warp = kRowsPerWarp * p.iters;
  const int chunks = (heads + per_warp - 1) / per_warp;
  const int64_t unit = (int64_t)blockIdx.x * kWarps + warp_id();
  const int64_t token = unit / chunks;
  if (token >= (int64_t)p.B * p.T) return;
  const int h0 = (int)(unit - token * chunks) * per_warp;
  const int b = (int)(token / p.T);
  const int t = (int)(token - (int64_t)b * p.T);

  float c[16], s[16];
  const bool rotate = p.cos != nullptr;
  if (rotate) {
    int64_t off = (int64_t)b * p.rope_sb + (int64_t)t * p.rope_st;
    if (p.positions != nullptr) {
      const int64_t pos = p.pos_i64 ? __ldg(static_cast<const long long*>(p.positions) + token)
                                    : (int64_t)__ldg(static_cast<const int*>(p.positions) + token);
      if (pos < 0 || pos >= p.n_pos) {
        // -1 marks a padding token: its rows stay as they are; any other
        // position outside the table is an error that the host can read
        if (pos != -1 && lane == 0) atomicOr(p.status, kStatusBadLaunch);
        return;
      }
      off = pos * p.rope_st;
    }
    load_f32x8(p.cos + off + 8 * l, c);
    load_f32x8(p.cos + off + 64 + 8 * l, c + 8);
    load_f32x8(p.sin + off + 8 * l, s);
    load_f32x8(p.sin + off + 64 + 8 * l, s + 8);
  }
  for (int it = 0; it < p.iters; ++it) {
    const int h = h0 + it * kRowsPerWarp + sub;
    if (h0 + it * kRowsPerWarp >= heads) break;
    const bool live = h < heads;
    const int which = h >= p.Hq;
    const int hh = which ? h - p.Hq : h;
    float v[16];
    if (live) {
      const __nv_bfloat16* src = p.x[which] + b * p.x_sb[which] + t * p.x_st[which] + hh * p.x_sh[which];
      unpack8(*reinterpret_cast<const uint4*>(src + 8 * l), v);  // may be written over: a plain load
      unpack8(*reinterpret_cast<const uint4*>(src + 64 + 8 * l), v + 8);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(v[i], v[i], ss);
    ss += __shfl_xor_sync(0xffffffffu, ss, 1);
    ss += __shfl_xor_sync(0xffffffffu, ss, 2);
    ss += __shfl_xor_sync(0xffffffffu, ss, 4);
    if (!live) continue;
    if (p.w[which] != nullptr) {
      float w[16];
      load_weight(p.w[which], p.w_f32[which], l, w);
      const float r = rsqrtf(ss * (1.0f / kHeadDim) + p.eps);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = v[i] * r * w[i];
    }
    uint32_t o[8];
    if (rotate) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a0 = v[2 * i], a1 = v[2 * i + 1], b0 = v[8 + 2 * i], b1 = v[9 + 2 * i];
        o[i] = pack_bf16x2(a0 * c[2 * i] - b0 * s[2 * i], a1 * c[2 * i + 1] - b1 * s[2 * i + 1]);
        o[4 + i] = pack_bf16x2(b0 * c[8 + 2 * i] + a0 * s[8 + 2 * i], b1 * c[9 + 2 * i] + a1 * s[9 + 2 * i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    }
    __nv_bfloat16* dst = p.y[which] + b * p.y_sb[which] + t * p.y_st[which] + hh * p.y_sh[which];
    *reinterpret_cast<uint4*>(dst + 8 * l) = make_uint4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<uint4*>(dst + 64 + 8 * l) = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

}  // namespace

int launch_qk_norm_rope(QkNormParams p, cudaStream_t stream) {
  const int64_t tokens = (int64_t)p.B * p.T;
  const int heads = p.Hq + p.Hk;
  p.iters = 1;
  p.status = device_status_word();
  if (p.status == nullptr) return set_error(kErrDevice, "qk_norm_rope: device status word unavailable");
  const int chunks = (heads + kRowsPerWarp * p.iters - 1) / (kRowsPerWarp * p.iters);
  const int64_t grid = (tokens * chunks + kWarps - 1) / kWarps;
  if (grid > 0x7FFFFFFF) return set_error(kErrUnsupported, "qk_norm_rope: problem too large");
  qk_norm_rope_kernel<<<(unsigned)grid, kWarps * 32, 0, stream>>>(p);
  return check_cuda(cudaGetLastError(), "qk_norm_rope launch");
}

}  // namespace fmka
