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
// time, and the heads of one token in turn, so that weights and angles are
// multiplied once per token (y = r * (x * w cos + partner * w' sin)) and a row
// costs three packed operations per pair of channels. 32768 tokens of 28 + 4
// heads: 104 us, 5.24 TB/s of 6.56 measured for a copy (192 us with one group of
// rows per warp; when it took 108: 115 with weights and angles apart, 114 with the
// next rows prefetched, which costs registers and so warps, 137 at 80 registers).
#include "fmka_internal.h"
#include "ptx.cuh"

namespace fmka {

namespace {

constexpr int kHeadDim = 128;
constexpr int kWarps = 4;
constexpr int kRowsPerWarp = 4;
constexpr int kGroupsAhead = 2;   // four-row groups loaded before the first is used (32768 tokens of 28 + 4 heads: 104 us, with one 121)
// A token's heads share one warp once that still leaves this many warps per SM (20 are resident). 32 + 8 heads, in us with
// 1 / 13 / 32 of them: 256 tokens 5.9 / 3.5 / 3.5;  512: 7.3 / 4.7 / 5.6;  1024: 8.3 / 7.0 / 7.0;  2048: 9.8 / 9.9 / 12.0.
constexpr int kWarpsPerSm = 13;

__device__ __forceinline__ void load_f32x8(const float* p, float2* f) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = make_float2(a.x, a.y);
  f[1] = make_float2(a.z, a.w);
  f[2] = make_float2(b.x, b.y);
  f[3] = make_float2(b.z, b.w);
}

// f[0..3]: channels 8l .. 8l+7, f[4..7]: 64 + 8l .. 64 + 8l + 7.
__device__ __forceinline__ void load_weight(const void* w, int f32, int l, float2* f) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (f32) {
      load_f32x8(static_cast<const float*>(w) + half * 64 + 8 * l, f + 4 * half);
    } else {
      const uint4 a = __ldg(static_cast<const uint4*>(w) + half * 8 + l);
      const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) f[4 * half + i] = make_float2(bf16lo_to_f32(u[i]), bf16hi_to_f32(u[i]));
    }
  }
}

// own[i] = w[d] cos[d]; other[i] = -w[d + 64] sin[d] for d < 64 and w[d - 64] sin[d] above: the factor of the partner.
__device__ __forceinline__ void factors(const QkNormParams& p, int which, int64_t rope_off, bool rotate, int l,
                                        float2 (&own)[8], float2 (&other)[8]) {
  float2 w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = make_float2(1.f, 1.f);
  if (p.w[which] != nullptr) load_weight(p.w[which], p.w_f32[which], l, w);
  if (rotate) {
    load_f32x8(p.cos + rope_off + 8 * l, own);
    load_f32x8(p.cos + rope_off + 64 + 8 * l, own + 4);
    load_f32x8(p.sin + rope_off + 8 * l, other);
    load_f32x8(p.sin + rope_off + 64 + 8 * l, other + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      own[i] = fmul2(own[i], w[i]);
      other[i] = fmul2(other[i], w[i ^ 4]);
      if (i < 4) other[i] = make_float2(-other[i].x, -other[i].y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) own[i] = w[i];
  }
}

// U groups of four heads are loaded before the first of them is used.
template <int U>
__global__ void __launch_bounds__(kWarps * 32, 5) qk_norm_rope_kernel(const __grid_constant__ QkNormParams p) {
  const int lane = lane_id();
  const int l = lane & 7;
  const int sub = lane >> 3;
  const int heads = p.Hq + p.Hk;
  const int groups = (heads + kRowsPerWarp - 1) / kRowsPerWarp;
  const int chunks = (groups + p.iters - 1) / p.iters;
  const int64_t unit = (int64_t)blockIdx.x * kWarps + warp_id();
  const int64_t token = unit / chunks;
  if (token >= (int64_t)p.B * p.T) return;
  const int first = (int)(unit - token * chunks) * p.iters;
  const int last = min(groups, first + p.iters);
  const int b = (int)(token / p.T);
  const int t = (int)(token - (int64_t)b * p.T);

  int64_t rope_off = (int64_t)b * p.rope_sb + (int64_t)t * p.rope_st;
  if (p.positions != nullptr) {
    const int64_t pos = p.pos_i64 ? __ldg(static_cast<const long long*>(p.positions) + token)
                                  : (int64_t)__ldg(static_cast<const int*>(p.positions) + token);
    if (pos < 0 || pos >= p.n_pos) {
      // -1 marks a padding token: its rows stay as they are; any other
      // position outside the table is an error that the host can read
      if (pos != -1 && lane == 0) atomicOr(p.status, kStatusBadLaunch);
      return;
    }
    rope_off = pos * p.rope_st;
  }
  const __nv_bfloat16* xq = p.x[0] + b * p.x_sb[0] + t * p.x_st[0] + 8 * l;
  const __nv_bfloat16* xk = p.x[1] + b * p.x_sb[1] + t * p.x_st[1] + 8 * l;
  __nv_bfloat16* yq = p.y[0] + b * p.y_sb[0] + t * p.y_st[0] + 8 * l;
  __nv_bfloat16* yk = p.y[1] + b * p.y_sb[1] + t * p.y_st[1] + 8 * l;
  // Weight and angle in one factor: y = r * (x * own + partner * other), r = rsqrt(mean + eps); made once for the
  // query heads and once for the key heads of the token.
  float2 own[8], other[8];
  int made_for = -1;
  const bool rotate = p.cos != nullptr;
  for (int g0 = first; g0 < last; g0 += U) {
    uint4 raw[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = (g0 + u) * kRowsPerWarp + sub;
      raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
      if (g0 + u < last && h < heads) {
        const __nv_bfloat16* src = h < p.Hq ? xq + h * p.x_sh[0] : xk + (h - p.Hq) * p.x_sh[1];
        raw[u][0] = __ldcs(reinterpret_cast<const uint4*>(src));
        raw[u][1] = __ldcs(reinterpret_cast<const uint4*>(src + 64));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (g0 + u >= last) break;
      const int h = (g0 + u) * kRowsPerWarp + sub;
      const int which = h >= p.Hq;
      if (made_for != which) {
        factors(p, which, rope_off, rotate, l, own, other);
        made_for = which;
      }
      const uint32_t x[8] = {raw[u][0].x, raw[u][0].y, raw[u][0].z, raw[u][0].w,
                             raw[u][1].x, raw[u][1].y, raw[u][1].z, raw[u][1].w};
      float2 v[8];
      float2 sq = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = make_float2(bf16lo_to_f32(x[i]), bf16hi_to_f32(x[i]));
        sq = ffma2(v[i], v[i], sq);
      }
      float ss = sq.x + sq.y;
      ss += __shfl_xor_sync(0xffffffffu, ss, 1);
      ss += __shfl_xor_sync(0xffffffffu, ss, 2);
      ss += __shfl_xor_sync(0xffffffffu, ss, 4);
      if (h >= heads) continue;
      const float r = p.w[which] != nullptr ? rsqrtf(ss * (1.0f / kHeadDim) + p.eps) : 1.f;
      const float2 r2 = make_float2(r, r);
      uint32_t o[8];
      if (rotate) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 y = fmul2(r2, ffma2(v[i], own[i], fmul2(v[i ^ 4], other[i])));
          o[i] = pack_bf16x2(y.x, y.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 y = fmul2(r2, fmul2(v[i], own[i]));
          o[i] = pack_bf16x2(y.x, y.y);
        }
      }
      __nv_bfloat16* dst = which ? yk + (h - p.Hq) * p.y_sh[1] : yq + h * p.y_sh[0];
      *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
      *reinterpret_cast<uint4*>(dst + 64) = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

}  // namespace

int launch_qk_norm_rope(QkNormParams p, cudaStream_t stream) {
  const int64_t tokens = (int64_t)p.B * p.T;
  const int groups = (p.Hq + p.Hk + kRowsPerWarp - 1) / kRowsPerWarp;
  p.status = device_status_word();
  if (p.status == nullptr) return set_error(kErrDevice, "qk_norm_rope: device status word unavailable");
  // All heads of a token in one warp, so that its angles are read once, unless that leaves the GPU short of warps; a
  // warp with one group of four rows has none to load ahead.
  const int64_t want = (int64_t)num_sms_current_device() * kWarpsPerSm;
  p.iters = groups;
  while (p.iters > 1 && tokens * ((groups + p.iters - 1) / p.iters) < want) p.iters = (p.iters + 1) / 2;
  const int chunks = (groups + p.iters - 1) / p.iters;
  const int64_t grid = (tokens * chunks + kWarps - 1) / kWarps;
  if (grid > 0x7FFFFFFF) return set_error(kErrUnsupported, "qk_norm_rope: problem too large");
  if (p.iters >= kGroupsAhead)
    qk_norm_rope_kernel<kGroupsAhead><<<(unsigned)grid, kWarps * 32, 0, stream>>>(p);
  else
    qk_norm_rope_kernel<1><<<(unsigned)grid, kWarps * 32, 0, stream>>>(p);
  return check_cuda(cudaGetLastError(), "qk_norm_rope launch");
}

}  // namespace fmka
