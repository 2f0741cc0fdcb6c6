// Attention for few or short rows, on mma.sync: packed sequences of different
// lengths, and single tokens against a small prefix shared by the batch plus
// the request's own keys (those also beside a long prefix).
//
//   o_r = sum_{j <= lim(r)} softmax_j(scale * q_r k_j) v_j,  lse_r = log sum_j exp(scale * q_r k_j)
//
// A row r is a (token, query head) pair: the G query heads of a kv head are
// rows of one tile, so grouped heads read each K/V row once. One CTA of four
// warps holds 16 * WM rows; WK = 4 / WM warps share the same rows and take
// different keys of each 64-key tile (merged at the end through shared memory).
// K and V tiles arrive by 16-byte cp.async copies into a ring of three stages;
// rows past the last visible key are filled with zeros instead of being read,
// so what lies there (another sequence, an unused slot) has no influence, not
// even as an infinity times a zero weight.
//
// Online softmax in fp32 (running max m and sum l per row, base 2); P is
// rounded to bf16 for the second product because the tensor cores take bf16:
// up to 2^-8 of each weight (half a step of 8 bits), the same size as the
// rounding of the output.
#include <algorithm>
#include <cfloat>

#include "fmka_internal.h"
#include "ptx.cuh"

namespace fmka {

namespace {

constexpr int kHeadDim = 128;
constexpr int kTileKeys = 64;
constexpr int kStages = 3;
constexpr int kTileBytes = kTileKeys * kHeadDim * 2;  // 16 KB
constexpr int kThreads = 128;
constexpr int kRingBytes = kStages * 2 * kTileBytes;
constexpr int kSmemBytes = kRingBytes + 16;

enum RowsMode : int {
  kModeVarlen = 0,  // packed sequences, every tile found from the offsets
  kModeList = 1,    // packed sequences, items of a plan (attn_plan.cu)
  kModeShared = 2,  // shared prefix (the first prefix_blocks blocks) and own keys
  kModeOnce = 3,    // the same without parts: a cluster of kOnceCtas takes all keys of a request and joins them itself
  kModeOnceVarlen = 4  // tiles found from the offsets as in kModeVarlen, each taken by a cluster as in kModeOnce
};
constexpr int kOnceCtas = 8;

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16-byte copy global -> shared; live == false writes zeros and reads nothing.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Byte offset of 16-byte chunk `chunk` (0..15) of row `row` in a tile of 256-byte rows; the XOR spreads the eight
// rows of an ldmatrix over all banks.
__device__ __forceinline__ uint32_t tile_off(int row, int chunk) {
  return row * 256 + ((chunk ^ (row & 7)) << 4);
}

struct RowsItem {
  int row0, n_tok;   // first packed token (request), tokens of this tile
  int64_t kv_off;    // element offset of key 0 of the kv head
  int kb, ke;        // keys [kb, ke)
  int lim0;          // last key token 0 sees (token i sees lim0 + i)
};

// The tile `idx` of the packed sequences: sequence, tokens and keys. Every warp computes it alike. False when idx is
// past the last tile, or when the offsets are not non-decreasing within the tensors (the status word then says so).
__device__ __forceinline__ bool find_tile(const PackedAttnParams& p, int tok_per_tile, int idx, RowsItem& it) {
  const int lane = lane_id();
  int base = 0;
  bool found = false;
  for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
    const int s = s0 + lane;
    int q0 = 0, q1 = 0, k0 = 0, k1 = 0;
    if (s < p.n_seqs) {
      q0 = __ldg(p.cu_q + s);
      q1 = __ldg(p.cu_q + s + 1);
      k0 = __ldg(p.cu_k + s);
      k1 = __ldg(p.cu_k + s + 1);
    }
    const bool bad = q0 < 0 || q1 < q0 || q1 > p.total_q || k0 < 0 || k1 < k0 || k1 > p.total_k;
    if (__any_sync(0xffffffffu, bad)) {
      if (lane == 0) atomicOr(p.status, kStatusBadLaunch);
      return false;
    }
    const int nt = (q1 - q0 + tok_per_tile - 1) / tok_per_tile;
    int incl = nt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += x;
    }
    const int excl = base + incl - nt;
    const unsigned hit = __ballot_sync(0xffffffffu, idx >= excl && idx < excl + nt);
    if (hit) {
      const int src = __ffs(hit) - 1;
      // the late tiles of a causal sequence have the most keys: they come first
      const int tile = __shfl_sync(0xffffffffu, nt - 1 - (idx - excl), src);
      q0 = __shfl_sync(0xffffffffu, q0, src);
      q1 = __shfl_sync(0xffffffffu, q1, src);
      k0 = __shfl_sync(0xffffffffu, k0, src);
      k1 = __shfl_sync(0xffffffffu, k1, src);
      const int t0 = tile * tok_per_tile;
      it.row0 = q0 + t0;
      it.n_tok = min(tok_per_tile, q1 - q0 - t0);
      it.kv_off = (int64_t)k0 * p.kv_st;
      it.kb = 0;
      it.ke = k1 - k0;
      if (p.causal) {
        it.lim0 = t0 + (k1 - k0) - (q1 - q0);
        it.ke = max(0, min(it.ke, it.lim0 + it.n_tok));
      } else {
        it.lim0 = k1 - k0;
      }
      found = true;  // the rest of the list is still checked
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  return found;
}

template <int WM, int MODE>
__global__ void __launch_bounds__(kThreads, 2) attn_rows_kernel(const __grid_constant__ PackedAttnParams p) {
  constexpr int WK = 4 / WM;
  constexpr int kRows = 16 * WM;
  constexpr int kWarpKeys = kTileKeys / WK;  // keys of a tile per warp
  constexpr int NT = kWarpKeys / 8;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = warp_id();
  const int lane = lane_id();
  const int wm = warp % WM;
  const int wk = warp / WM;
  const int hkv = blockIdx.y / p.n_gs;
  const int g0 = (blockIdx.y % p.n_gs) * p.Gs;
  const int gn = min(p.Gs, p.G - g0);
  const int tpt = kRows / p.Gs;  // tokens per tile

  grid_launch_dependents();
  RowsItem it;
  const __nv_bfloat16 *kp = p.k, *vp = p.v;
  int64_t kv_st = p.kv_st;
  int64_t part = -1;  // part row of token 0, head 0 of the slice, or -1: the output itself
  int part_ts = p.Hq;
  if constexpr (MODE == kModeVarlen) {
    if (!find_tile(p, tpt, blockIdx.x, it)) return;
    it.kv_off += hkv * p.kv_sh;
  } else if constexpr (MODE == kModeList) {
    grid_dependency_wait();
    if ((int)blockIdx.x >= __ldcg(p.header)) return;
    const int4 a = __ldcg(p.list + 2 * blockIdx.x), c = __ldcg(p.list + 2 * blockIdx.x + 1);
    it.row0 = a.x;
    it.n_tok = a.y;
    it.kv_off = (int64_t)a.z * p.kv_st + hkv * p.kv_sh;
    it.kb = a.w;
    it.ke = c.x;
    it.lim0 = c.y;
    part_ts = p.Gs;
    if (c.z >= 0) part = (int64_t)c.z + (int64_t)blockIdx.y * a.y * p.Gs;
  } else if constexpr (MODE == kModeOnceVarlen) {
    if (!find_tile(p, tpt, blockIdx.x / kOnceCtas, it)) return;  // all of a cluster or none
    it.kv_off += hkv * p.kv_sh;
    const int per = ((it.ke + kTileKeys - 1) / kTileKeys + kOnceCtas - 1) / kOnceCtas * kTileKeys;
    it.kb = (blockIdx.x % kOnceCtas) * per;
    it.ke = min(it.ke, it.kb + per);
  } else if constexpr (MODE == kModeOnce) {
    it.row0 = blockIdx.x / kOnceCtas;
    it.n_tok = 1;
    it.kv_off = it.row0 * p.kv_sb + hkv * p.kv_sh;
    const int len = p.lens != nullptr ? max(0, min(p.cap, __ldg(p.lens + it.row0))) : p.cap;
    const int tiles = (p.P + len + kTileKeys - 1) / kTileKeys;
    const int per = (tiles + kOnceCtas - 1) / kOnceCtas * kTileKeys;
    it.kb = (blockIdx.x % kOnceCtas) * per;
    it.ke = min(p.P + len, it.kb + per);
    it.lim0 = 0x3FFFFFFF;
    if (p.cap == 0) {  // rows that are filled with zeros still name an address: one that exists
      kp = p.kp;
      vp = p.vp;
      it.kv_off = 0;
    }
  } else {
    int split;
    if ((int)blockIdx.x < p.prefix_blocks) {
      const int tile = blockIdx.x / p.prefix_splits;
      split = blockIdx.x - tile * p.prefix_splits;
      it.row0 = tile * tpt;
      it.n_tok = min(tpt, p.B - it.row0);
      it.kv_off = hkv * p.kp_sh;
      it.kb = split * p.prefix_keys;
      it.ke = min(p.P, it.kb + p.prefix_keys);
      kp = p.kp;
      vp = p.vp;
      kv_st = p.kp_st;
    } else {
      const int x = blockIdx.x - p.prefix_blocks;
      it.row0 = x / p.own_splits;
      split = x - it.row0 * p.own_splits;
      it.n_tok = 1;
      it.kv_off = it.row0 * p.kv_sb + hkv * p.kv_sh;
      it.kb = split * p.own_keys;
      const int len = p.lens != nullptr ? max(0, min(p.cap, __ldg(p.lens + it.row0))) : p.cap;
      it.ke = min(len, it.kb + p.own_keys);
      split += p.prefix_splits;
    }
    it.lim0 = 0x3FFFFFFF;
    part = ((int64_t)split * p.B + it.row0) * p.Hq + hkv * p.G + g0;
  }
  // tiles from this one on hold keys that some rows see and others do not
  constexpr bool kCausal = MODE == kModeVarlen || MODE == kModeList || MODE == kModeOnceVarlen;
  constexpr bool kCluster = MODE == kModeOnce || MODE == kModeOnceVarlen;
  const int diag_tile = kCausal && it.n_tok > 1 ? max(0, it.lim0 + 1 - it.kb) / kTileKeys : 0x3FFFFFF;
  volatile int* bad_v = reinterpret_cast<volatile int*>(smem + kRingBytes);
  if (threadIdx.x == 0) *bad_v = 0;
  const int n_tiles = it.ke > it.kb ? (it.ke - it.kb + kTileKeys - 1) / kTileKeys : 0;

  kp += it.kv_off;
  vp += it.kv_off;
  const uint32_t s_base = smem_u32(smem);
  const int own0 = MODE == kModeOnce ? p.P : 0;  // key of kp's first row
  auto load_tile = [&](int i) {
    if (i < n_tiles) {
      const uint32_t ks = s_base + (i % kStages) * 2 * kTileBytes;
      const int key0 = it.kb + i * kTileKeys;
#pragma unroll
      for (int c = 0; c < kTileKeys * 16 / kThreads; ++c) {
        const int id = c * kThreads + threadIdx.x;
        const int row = id >> 4, ch = id & 15;
        const bool live = key0 + row < it.ke;
        if (MODE == kModeOnce && key0 + row < p.P) {  // the prefix's rows first
          const int64_t off = (int64_t)(key0 + row) * p.kp_st + hkv * p.kp_sh + ch * 8;
          cp_async16(ks + tile_off(row, ch), p.kp + (live ? off : 0), live);
          cp_async16(ks + kTileBytes + tile_off(row, ch), p.vp + (live ? off : 0), live);
        } else {
          const int64_t off = live ? (int64_t)(key0 + row - own0) * kv_st + ch * 8 : 0;
          cp_async16(ks + tile_off(row, ch), kp + off, live);
          cp_async16(ks + kTileBytes + tile_off(row, ch), vp + off, live);
        }
      }
    }
    cp_async_commit();
  };
  for (int i = 0; i < kStages - 1; ++i) load_tile(i);

  // rows of this thread: r_lo and r_lo + 8 of the warp's 16
  const int kq = (lane & 3) * 2;
  int lim[2], tok[2], head[2];
  bool row_ok[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = wm * 16 + (lane >> 2) + 8 * e;
    const int i = r / p.Gs, g = r % p.Gs;
    row_ok[e] = i < it.n_tok && g < gn;
    tok[e] = it.row0 + i;
    head[e] = hkv * p.G + g0 + g;
    lim[e] = min(it.ke - 1, it.lim0 + i);
  }
  uint32_t qa[8][4];
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const __nv_bfloat16* src = p.q + tok[e] * p.q_st + head[e] * p.q_sh + ks * 16 + kq;
      qa[ks][e] = row_ok[e] ? *reinterpret_cast<const uint32_t*>(src) : 0u;
      qa[ks][2 + e] = row_ok[e] ? *reinterpret_cast<const uint32_t*>(src + 8) : 0u;
    }
  }

  if constexpr (kCausal) __syncthreads();  // bad_v is zero before any warp may set it (a first tile can be masked)

  float o[16][4];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY};
  float l[2] = {0.f, 0.f};
  const int mrow = lane & 7;
  const int msel = lane >> 3;

  for (int i = 0; i < n_tiles; ++i) {
    cp_async_wait<kStages - 2>();
    if (kCausal && i >= diag_tile) {
      // this thread's own copies are visible to it before the barrier
#pragma unroll
      for (int c = 0; c < kTileKeys * 16 / kThreads; ++c) {
        const int id = c * kThreads + threadIdx.x;
        uint4* at = reinterpret_cast<uint4*>(smem + ((i % kStages) * 2 + 1) * kTileBytes + tile_off(id >> 4, id & 15));
        uint4 x = *at;
        if (zero_nonfinite(x)) {
          *at = x;
          *bad_v = 1;
        }
      }
    }
    __syncthreads();
    load_tile(i + kStages - 1);
    const uint32_t kt = s_base + (i % kStages) * 2 * kTileBytes;
    const uint32_t vt = kt + kTileBytes;
    const int key0 = it.kb + i * kTileKeys + wk * kWarpKeys;
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
      const int row = wk * kWarpKeys + nt * 8 + mrow;
#pragma unroll
      for (int s4 = 0; s4 < 4; ++s4) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4(kt + tile_off(row, s4 * 4 + msel), b0, b1, b2, b3);
        mma16816(sc[nt], qa[2 * s4], b0, b1);
        mma16816(sc[nt], qa[2 * s4 + 1], b2, b3);
      }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int key = key0 + nt * 8 + kq + (c & 1);
        sc[nt][c] = key > lim[c >> 1] ? -INFINITY : sc[nt][c] * p.scale_log2;
        mx[c >> 1] = fmaxf(mx[c >> 1], sc[nt][c]);
      }
    }
    float al[2], sub[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
      const float mn = fmaxf(m[e], mx[e]);
      sub[e] = mn == -INFINITY ? 0.f : mn;
      al[e] = fast_exp2(m[e] - sub[e]);
      m[e] = mn;
      l[e] *= al[e];
    }
    uint32_t pa[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        sc[nt][c] = fast_exp2(sc[nt][c] - sub[c >> 1]);
        l[c >> 1] += sc[nt][c];
      }
      pa[nt][0] = pack_bf16x2(sc[nt][0], sc[nt][1]);
      pa[nt][1] = pack_bf16x2(sc[nt][2], sc[nt][3]);
    }
#pragma unroll
    for (int dt = 0; dt < 16; ++dt) {
      o[dt][0] *= al[0];
      o[dt][1] *= al[0];
      o[dt][2] *= al[1];
      o[dt][3] *= al[1];
    }
#pragma unroll
    for (int kt2 = 0; kt2 < NT / 2; ++kt2) {
      const uint32_t a[4] = {pa[2 * kt2][0], pa[2 * kt2][1], pa[2 * kt2 + 1][0], pa[2 * kt2 + 1][1]};
      const int row = wk * kWarpKeys + kt2 * 16 + (msel & 1) * 8 + mrow;
#pragma unroll
      for (int dp = 0; dp < 8; ++dp) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4_trans(vt + tile_off(row, dp * 2 + (msel >> 1)), b0, b1, b2, b3);
        mma16816(o[2 * dp], a, b0, b1);
        mma16816(o[2 * dp + 1], a, b2, b3);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
  }
  cp_async_wait<0>();
  // Started beside the prefix's kernel, this one must not end before it: whatever comes next waits for this one only.
  if (MODE == kModeShared && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1) grid_dependency_wait();

  if constexpr (WK > 1) {
    // The four warps hold other keys of the same rows: through shared memory, then eight threads per row
    static_assert(WM == 1, "16 rows");
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);     // [4][16][128]
    float* sm = so + 4 * 16 * kHeadDim;              // [4][16][2]
    const int r0 = lane >> 2;
#pragma unroll
    for (int dt = 0; dt < 16; ++dt) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float2*>(so + (warp * 16 + r0 + 8 * e) * kHeadDim + ((dt ^ r0) * 8 + kq)) =
            make_float2(o[dt][2 * e], o[dt][2 * e + 1]);
    }
    if ((lane & 3) == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sm[(warp * 16 + r0 + 8 * e) * 2] = m[e];
        sm[(warp * 16 + r0 + 8 * e) * 2 + 1] = l[e];
      }
    }
    __syncthreads();
    const int row = threadIdx.x >> 3, seg = threadIdx.x & 7;  // channels [16 seg, 16 seg + 16)
    const int i = row / p.Gs, g = row - i * p.Gs;
    const bool live_row = i < it.n_tok && g < gn;
    const int64_t tok0 = it.row0 + i;
    const int head0 = hkv * p.G + g0 + g;
    const int lim_row = min(it.ke - 1, it.lim0 + i);
    float L = 0.f, M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm[(w * 16 + row) * 2]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float wt[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      wt[w] = fast_exp2(sm[(w * 16 + row) * 2] - Ms);
      L += wt[w] * sm[(w * 16 + row) * 2 + 1];
    }
    if (!kCluster && !live_row) return;
    float acc[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) acc[c] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int dt = seg * 2 + (q4 >> 1);
        const float4 x = *reinterpret_cast<const float4*>(so + (w * 16 + row) * kHeadDim + (dt ^ (row & 7)) * 8 + (q4 & 1) * 4);
        acc[q4 * 4 + 0] = fmaf(wt[w], x.x, acc[q4 * 4 + 0]);
        acc[q4 * 4 + 1] = fmaf(wt[w], x.y, acc[q4 * 4 + 1]);
        acc[q4 * 4 + 2] = fmaf(wt[w], x.z, acc[q4 * 4 + 2]);
        acc[q4 * 4 + 3] = fmaf(wt[w], x.w, acc[q4 * 4 + 3]);
      }
    }
    if constexpr (kCausal) {
      // rare: the infinities and NaNs taken out above go to the rows that see them
      if (n_tiles > diag_tile && *bad_v) {
        for (int j = it.kb + diag_tile * kTileKeys; j <= lim_row; ++j) {
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float x = __bfloat162float(vp[j * kv_st + seg * 16 + c]);
            if (!(fabsf(x) <= 3.4e38f)) acc[c] += x;
          }
        }
      }
    }
    if constexpr (kCluster) {
      // This CTA's keys are done: sums (not yet divided), maximum and weight of each row to where the others read them;
      // then every CTA joins 16 channels of all rows.
      float* xo = so + 4 * 16 * kHeadDim + 128;  // [16][128], behind so and sm
      float* xm = xo + 16 * kHeadDim;            // [16][2]
#pragma unroll
      for (int c = 0; c < 4; ++c)
        reinterpret_cast<float4*>(xo + row * kHeadDim + seg * 16)[c] =
            make_float4(acc[c * 4], acc[c * 4 + 1], acc[c * 4 + 2], acc[c * 4 + 3]);
      if (seg == 0) {
        xm[row * 2] = M;
        xm[row * 2 + 1] = L;
      }
      cluster_sync();
      const uint32_t rank = cluster_ctarank();
      float2 ml[kOnceCtas], v[kOnceCtas];
#pragma unroll
      for (int r = 0; r < kOnceCtas; ++r) {
        ml[r] = ld_cluster_f2(cluster_addr(xm + row * 2, r));
        v[r] = ld_cluster_f2(cluster_addr(xo + row * kHeadDim + rank * 16 + seg * 2, r));
      }
      float Mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < kOnceCtas; ++r) Mx = fmaxf(Mx, ml[r].x);
      const float Mxs = Mx == -INFINITY ? 0.f : Mx;
      float Lx = 0.f;
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int r = 0; r < kOnceCtas; ++r) {
        const float w = fast_exp2(ml[r].x - Mxs);
        Lx = fmaf(w, ml[r].y, Lx);
        sum.x = fmaf(w, v[r].x, sum.x);
        sum.y = fmaf(w, v[r].y, sum.y);
      }
      if (live_row) {
        const float inv = Lx == 0.f ? 0.f : 1.f / Lx;
        *reinterpret_cast<uint32_t*>(p.o + tok0 * p.o_st + head0 * p.o_sh + rank * 16 + seg * 2) =
            pack_bf16x2(sum.x * inv, sum.y * inv);
        if (rank == 0 && seg == 0 && p.lse != nullptr)
          p.lse[tok0 * p.lse_st + head0 * p.lse_sh] = Lx == 0.f ? -INFINITY : (Mx + __log2f(Lx)) * 0.69314718055994531f;
      }
      cluster_sync();  // no CTA leaves while its rows are read
      return;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;  // a row that sees no key gives zeros
    const float lse2 = L == 0.f ? -INFINITY : M + __log2f(L);
    if (part < 0) {
      uint4* dst = reinterpret_cast<uint4*>(p.o + tok0 * p.o_st + head0 * p.o_sh + seg * 16);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        dst[h] = make_uint4(pack_bf16x2(acc[h * 8 + 0] * inv, acc[h * 8 + 1] * inv),
                            pack_bf16x2(acc[h * 8 + 2] * inv, acc[h * 8 + 3] * inv),
                            pack_bf16x2(acc[h * 8 + 4] * inv, acc[h * 8 + 5] * inv),
                            pack_bf16x2(acc[h * 8 + 6] * inv, acc[h * 8 + 7] * inv));
      if (seg == 0 && p.lse != nullptr) p.lse[tok0 * p.lse_st + head0 * p.lse_sh] = lse2 * 0.69314718055994531f;
    } else {
      const int64_t rec = part + (int64_t)i * part_ts + g;
      if (L != 0.f) {
        float4* dst = reinterpret_cast<float4*>(p.part_o + rec * kHeadDim + seg * 16);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          dst[c] = make_float4(acc[c * 4] * inv, acc[c * 4 + 1] * inv, acc[c * 4 + 2] * inv, acc[c * 4 + 3] * inv);
      }
      if (seg == 0) p.part_lse[rec] = lse2;
    }
  } else {
    static_assert(MODE == kModeVarlen, "whole rows");
    if (n_tiles > diag_tile && *bad_v) {
      // rare, as above
      for (int e = 0; e < 2; ++e) {
        for (int j = diag_tile * kTileKeys; row_ok[e] && j <= lim[e]; ++j) {
          const __nv_bfloat16* src = vp + j * kv_st + kq;
#pragma unroll
          for (int dt = 0; dt < 16; ++dt) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(src + dt * 8);
            if ((x & 0x7F80u) == 0x7F80u) o[dt][2 * e] += bf16lo_to_f32(x);
            if ((x & 0x7F800000u) == 0x7F800000u) o[dt][2 * e + 1] += bf16hi_to_f32(x);
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (!row_ok[e]) continue;
      const float inv = l[e] == 0.f ? 0.f : 1.f / l[e];
      __nv_bfloat16* dst = p.o + tok[e] * p.o_st + head[e] * p.o_sh + kq;
#pragma unroll
      for (int dt = 0; dt < 16; ++dt)
        *reinterpret_cast<uint32_t*>(dst + dt * 8) = pack_bf16x2(o[dt][2 * e] * inv, o[dt][2 * e + 1] * inv);
      if ((lane & 3) == 0 && p.lse != nullptr)
        p.lse[tok[e] * p.lse_st + head[e] * p.lse_sh] =
            l[e] == 0.f ? -INFINITY : (m[e] + __log2f(l[e])) * 0.69314718055994531f;
    }
  }
}

// Joins prefix and own parts of every request: one warp per (request, query head).
__global__ void __launch_bounds__(128) join_parts_kernel(const __grid_constant__ PackedAttnParams p, int n_parts) {
  grid_dependency_wait();
  const int row = blockIdx.x * 4 + warp_id();
  const int rows = p.B * p.Hq;
  if (row >= rows) return;
  const int b = row / p.Hq, h = row - b * p.Hq;
  join_row(p.part_o + (int64_t)row * kHeadDim, p.part_lse + row, rows, n_parts, p.o + b * p.o_st + h * p.o_sh,
           p.lse == nullptr ? nullptr : p.lse + b * p.lse_st + h * p.lse_sh);
}

// One launch, clusters of kOnceCtas: tile x kv head (x slice of its group).
template <int MODE>
int launch_once(const PackedAttnParams& p, int64_t tiles, cudaStream_t stream, const char* what) {
  auto kern = attn_rows_kernel<1, MODE>;
  static std::atomic<uint64_t> devices{0};
  int rc = check_cuda(allow_smem(kern, kSmemBytes, devices), what);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * kOnceCtas), (unsigned)(p.Hkv * p.n_gs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kOnceCtas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, p), what);
}

template <int WM, int MODE>
int launch_rows(const PackedAttnParams& p, int64_t gx, bool dependent, cudaStream_t stream, const char* what) {
  auto kern = attn_rows_kernel<WM, MODE>;
  static std::atomic<uint64_t> devices{0};
  int rc = check_cuda(allow_smem(kern, kSmemBytes, devices), what);
  if (rc) return rc;
  if (gx > 0x7FFFFFFF) return set_error(kErrUnsupported, std::string(what) + ": problem too large");
  return check_cuda(launch_after(kern, dim3((unsigned)gx, (unsigned)(p.Hkv * p.n_gs)), kThreads, kSmemBytes, dependent,
                                 stream, p),
                    what);
}

void slice_group(PackedAttnParams& p, int rows) {
  p.n_gs = (p.G + rows - 1) / rows;
  p.Gs = (p.G + p.n_gs - 1) / p.n_gs;
}

// Whether a tensor map can hold rows and heads with these strides: an expanded view's zero cannot be one.
bool mappable(int64_t st, int rows, int64_t sh, int heads) {
  return (rows == 1 || st > 0) && (heads == 1 || sh > 0);
}

// Whether the pair kernel may scale by this: it masks scores with -inf first and multiplies then, and a factor of zero
// (or one that the kernels flush to zero) would make NaNs of them. This file's kernel masks behind the multiplication.
bool pair_scale(float scale_log2) { return scale_log2 >= FLT_MIN; }

// Tiles of `tokens` tokens of a packed batch, at most (every sequence may end in a tile that it does not fill).
int64_t tile_bound(int n_seqs, int total_q, int tokens) {
  return ((int64_t)total_q + (int64_t)n_seqs * (tokens - 1)) / tokens;
}

// How a packed batch runs:
//   kShort: one launch, every CTA of 64 rows finds its tile in the offsets itself. A CTA takes about 19 ns a key, so it
//     is for keys (times the waves of CTAs) that are done before a plan would be.
//   kOnce: one launch, every tile of 16 rows is found in the same way and taken by a cluster that cuts its keys in
//     eight: few tiles with more keys.
//   kThin: tiles of 16 rows from a plan, long sequences split: batches of few rows per sequence, where the time goes to
//     reading K and V.
//   kPair: 256 rows per cluster on tcgen05, from a plan: the rest.
// Measured in us on the device (short / thin / pair), 32 heads over 8, on both sides of each limit:
//   waves x keys: 40 prompts' keys 5.3 / 8.2 / 12.5;  200: 8.6 / 15.8 / 16.9;  250: 9.3 / 17.7 / 17.1;
//     400: 18.6 / 26.7 / 15.8;  500 (32 single tokens): 19.8 / 14.4 / 27.9;
//     the offsets cost a key for eight sequences in every CTA, and a wave 5 us: short / better plan for 300 x 8 tokens, 2
//     kv heads, 3 waves, 24 / 43;  256 x 1, 7 waves, 41 / 26;  1000 x 1, 1 kv head, 4 waves, 55 / 21;
//   rows per sequence (64 sequences of 100 to 16000 keys in even steps, 515 k keys): 4: 648 / 362 / 438;
//     16: 670 / 380 / 460;  32: 740 / 510 / 460;  32 as one kv head: 308 / 96 / 89;  prompts of 64 to 2048 tokens:
//     340 / 775 / 104.
//   a prompt among single tokens of 100 keys and more in even steps (thin / pair): 512 tokens among 60 of up to 4000:
//     118 / 117, of up to 16000: 369 / 412;  1024 among 400 of up to 4000: 530 / 786;  2048 among 800 of up to 2000:
//     654 / 888. (The rule goes by sizes that the host knows, and takes the pair for the first two.)
// and once / the better of thin and pair (which take a launch or two and a workspace more on the host, 5 us):
//   1 wave: 1 token on 500 keys 5.1 / 11.2, on 4000 9.5 / 17.5, on 8000 14.7 / 19.0, on 16000 24.6 / 22.0; 100 on 1000,
//     1 kv head, 9.0 / 21.6;
//   2 waves: 8 tokens on 1000 each 14.4 / 17.8, on 2000 17.6 / 18.6, on 100 to 4000 22.3 / 19.3; 3 x 40 tokens of 8
//     heads over 1 on 500 15.2 / 12.9;  4 waves: 16 tokens on 600 26.0 / 17.2.
enum class VarlenPath { kShort, kOnce, kThin, kPair };
constexpr int kShortKeys = 320;
constexpr int kOnceVarlenKeys = 12000;

VarlenPath varlen_path(int n_seqs, int total_q, int max_k, int Hkv, int G) {
  PackedAttnParams p = {};
  p.G = G;
  const int64_t slots = 2 * num_sms_current_device();
  auto waves = [&](int rows, int ctas) {  // of CTAs on all SMs, with `rows` rows and `ctas` CTAs a tile
    slice_group(p, rows);
    return (tile_bound(n_seqs, total_q, rows / p.Gs) * Hkv * p.n_gs * ctas + slots - 1) / slots;
  };
  const int64_t shorts = waves(64, 1);
  if (shorts <= 5 && shorts * ((int64_t)max_k + n_seqs / 8) < kShortKeys) return VarlenPath::kShort;
  const bool thin = (int64_t)total_q * G <= (int64_t)n_seqs * 16;
  const int64_t w = waves(16, kOnceCtas);
  if (w <= (thin ? 2 : 1) && w * w * max_k <= kOnceVarlenKeys) return VarlenPath::kOnce;
  return thin ? VarlenPath::kThin : VarlenPath::kPair;
}

PackedPlan thin_plan(int n_seqs, int total_q, int max_k, int Hkv, PackedAttnParams& p) {
  slice_group(p, 16);
  return packed_plan(n_seqs, total_q, max_k, Hkv, p.G, p.Gs, 16 / p.Gs, 2 * num_sms_current_device());
}

struct SharedPlan {
  int prefix_splits, prefix_keys;  // parts over the prefix, keys per part
  int own_splits, own_keys;
  bool pair;                       // the prefix goes to the pair kernel
  bool once;                       // no parts: one launch of clusters
};
constexpr int kOnceKeys = 2048;

// Few requests with few keys are one launch of clusters, if these all run at once: no parts in memory, no join, no
// workspace, which also saves the caller 5 of 22 us. In us on the device, clusters / parts:
//   batch 1, 8 kv heads, 64 own slots: prefix 1024: 6.4 / 7.5;  2048: 8.4 / 8.0;  4096: 11.9 / 10.2;
//   batch 4, 4 kv heads of 7, prefix 1000 and 64: 8.1 / 8.4;  batch 30, 1 kv head, prefix 1000 and 100: 8.4 / 8.5.
// Else the prefix belongs on the pair kernel (128 rows of the batch read a key once, on tcgen05) unless it is small: then
// this kernel's 16-row tiles, in the same launch as the own keys, spare a launch and the clusters' start. What they
// read is (tiles) x (keys); measured in us, rows here / pair kernel, 8 kv heads of 4 query heads:
//   batch 4, prefix 1024 (8 k keys read): 8.4 / 12.7;   batch 16, prefix 1024 (33 k): 11.3 / 13.1;
//   batch 16, prefix 2048 (66 k): 16.2 / 14.7;          batch 1, prefix 16384 (131 k): 25.8 / 25.3;
//   batch 33, prefix 5003 (440 k): 60.5 / 25.6;         batch 64, prefix 32768: 488 / 67.
// Parts of 256 keys: the 33 k case takes 18.5 with 64, 14.6 with 128, 11.3 with 256.
// Own keys in parts of 512 (256 and 1024 were slower on batches of 33 to 256 with 400 to 1024 own slots), but a cache
// with much room in parts as large as 8 waves of CTAs, or 8 parts, make them: parts that turn out empty are not free.
// 16 requests, 8 kv heads, room for 131072 keys, 8 / 32 / 256 parts, in us: 100 keys each 22 / 41 / 213; all full 816 /
// 815 / 1050; one full 224 / 128 / 323. 64 requests, room for 32768, 8 / 32 / 64 parts: 39 / 115 / 209; 800 / 878 / 991.
// A stride of zero over several heads or tokens (an expanded view) is not for tensor maps, and a scale of zero not for
// the pair kernel; they stay here, and with the parts that the sizes ask for, as the workspace's size is asked for
// without strides and scale.
SharedPlan plan_shared(int B, int Hq, int Hkv, int P, int cap) {
  SharedPlan s{0, kTileKeys, 0, kTileKeys, false, false};
  PackedAttnParams r = {};
  r.G = Hq / Hkv;
  slice_group(r, 16);
  s.once = (int64_t)B * Hkv * r.n_gs * kOnceCtas <= 2 * num_sms_current_device() && (int64_t)P + cap <= kOnceKeys;
  if (s.once) return s;
  if (P > 0) {
    const int tpt = 16 / r.Gs;
    s.pair = (int64_t)((B + tpt - 1) / tpt) * Hkv * r.n_gs * P >= (1 << 16);
    if (s.pair) {
      s.prefix_splits = attn_pair_prefix_splits(B, Hq, Hkv, P, cap, &s.prefix_keys);
    } else {
      s.prefix_keys = 256;
      s.prefix_splits = (P + s.prefix_keys - 1) / s.prefix_keys;
    }
  }
  if (cap > 0) {
    const int64_t units = (int64_t)B * Hkv * r.n_gs;
    const int most = (int)std::max<int64_t>(8, 16 * num_sms_current_device() / units);
    s.own_keys = std::max(512, (cap + most * kTileKeys - 1) / (most * kTileKeys) * kTileKeys);
    s.own_splits = (cap + s.own_keys - 1) / s.own_keys;
  }
  return s;
}

}  // namespace

size_t attn_varlen_workspace_bytes(int n_seqs, int total_q, int max_k, int Hq, int Hkv) {
  PackedAttnParams p = {};
  p.G = Hq / Hkv;
  switch (varlen_path(n_seqs, total_q, max_k, Hkv, p.G)) {
    case VarlenPath::kShort:
    case VarlenPath::kOnce: return 0;
    case VarlenPath::kThin: return thin_plan(n_seqs, total_q, max_k, Hkv, p).total;
    default: return attn_pair_plan(n_seqs, total_q, max_k, Hq, Hkv).total;
  }
}

int launch_attn_varlen(PackedAttnParams p, int max_k, void* workspace, cudaStream_t stream) {
  p.status = device_status_word();
  if (p.status == nullptr) return set_error(kErrDevice, "attn_varlen: device status word unavailable");
  const VarlenPath path = varlen_path(p.n_seqs, p.total_q, max_k, p.Hkv, p.G);
  // expanded views and a scale of zero are right on the first path whatever the size, and it needs no workspace
  if (path == VarlenPath::kShort || p.total_k == 0 ||
      (path == VarlenPath::kPair && (!pair_scale(p.scale_log2) || !mappable(p.q_st, p.total_q, p.q_sh, p.Hq) ||
                                     !mappable(p.kv_st, p.total_k, p.kv_sh, p.Hkv)))) {
    slice_group(p, 64);
    return launch_rows<4, kModeVarlen>(p, tile_bound(p.n_seqs, p.total_q, 64 / p.Gs), false, stream, "attn_varlen launch");
  }
  if (path == VarlenPath::kOnce) {
    slice_group(p, 16);
    return launch_once<kModeOnceVarlen>(p, tile_bound(p.n_seqs, p.total_q, 16 / p.Gs), stream, "attn_varlen launch");
  }
  PackedPlan w = path == VarlenPath::kThin ? thin_plan(p.n_seqs, p.total_q, max_k, p.Hkv, p)
                                           : attn_pair_plan(p.n_seqs, p.total_q, max_k, p.Hq, p.Hkv);
  int rc = launch_plan(p, w, workspace, stream);
  if (rc) return rc;
  if (path == VarlenPath::kThin) {
    p.header = w.header;
    p.list = w.list;
    p.part_o = w.part_o;
    p.part_lse = w.part_lse;
    rc = launch_rows<1, kModeList>(p, w.max_list, true, stream, "attn_varlen launch");
  } else {
    rc = launch_attn_pair_varlen(p, w, stream);
  }
  return rc ? rc : launch_join(p, w, stream);
}

size_t attn_decode_shared_workspace_bytes(int B, int Hq, int Hkv, int P, int cap) {
  const SharedPlan s = plan_shared(B, Hq, Hkv, P, cap);
  return (size_t)(s.prefix_splits + s.own_splits) * B * Hq * (kHeadDim + 1) * sizeof(float);
}

int launch_attn_decode_shared(PackedAttnParams p, void* workspace, cudaStream_t stream) {
  p.status = device_status_word();
  if (p.status == nullptr) return set_error(kErrDevice, "attn_decode_shared: device status word unavailable");
  SharedPlan s = plan_shared(p.B, p.Hq, p.Hkv, p.P, p.cap);
  if (!pair_scale(p.scale_log2) || !mappable(p.q_st, p.B, p.q_sh, p.Hq) || !mappable(p.kp_st, p.P, p.kp_sh, p.Hkv))
    s.pair = false;
  if (s.once) {
    slice_group(p, 16);
    return launch_once<kModeOnce>(p, p.B, stream, "attn_decode_shared launch");
  }
  const int parts = s.prefix_splits + s.own_splits;
  p.part_o = static_cast<float*>(workspace);
  p.part_lse = p.part_o + (int64_t)parts * p.B * p.Hq * kHeadDim;
  p.prefix_splits = s.prefix_splits;
  p.prefix_keys = s.prefix_keys;
  p.own_splits = s.own_splits;
  p.own_keys = s.own_keys;
  if (s.pair) {
    const int rc = launch_attn_pair_prefix(p, stream);
    if (rc) return rc;
  }
  slice_group(p, 16);
  const int tpt = 16 / p.Gs;
  p.prefix_blocks = s.pair ? 0 : (p.B + tpt - 1) / tpt * s.prefix_splits;
  const int64_t blocks = p.prefix_blocks + (int64_t)p.B * s.own_splits;
  if (blocks > 0) {
    // Behind the pair kernel it depends on nothing of it and does not wait: its blocks fill what SMs the other
    // leaves free.
    const int rc = launch_rows<1, kModeShared>(p, blocks, s.pair, stream, "attn_decode_shared launch");
    if (rc) return rc;
  }
  const int64_t rows = (int64_t)p.B * p.Hq;
  return check_cuda(launch_after(join_parts_kernel, dim3((unsigned)((rows + 3) / 4)), 128, 0, true, stream,
                                 p, parts),
                    "attn_decode_shared join launch");
}

}  // namespace fmka
