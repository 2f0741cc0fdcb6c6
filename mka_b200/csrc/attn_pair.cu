// Attention for many rows on tcgen05, by pairs of CTAs: packed sequences of
// different lengths, and the shared prefix of a decode batch.
//
//   o_r = sum_{j <= lim(r)} softmax_j(scale * q_r k_j) v_j,  lse_r = log sum_j exp(scale * q_r k_j)
//
// Work is cut into items: a tile of rows ((token, query head of one kv head's
// group) pairs, 128 per CTA, 256 per pair) against a range of keys. A persistent
// grid of CTA pairs takes the items in a fixed order, heavy ones first. Items
// that cover only a part of a row's keys leave a normalised fp32 partial output
// and a log2-sum-exp, joined by a second kernel.
//
// Each pair multiplies with the 2-SM MMA (M = 256, cta_group::2): every CTA
// holds its own 128 rows of Q, S, P and O and only half of each K tile (64
// keys) and V tile (64 channels), which halves the operand traffic per SM.
// TMEM of each CTA (512 columns): O | S0 | S1 | P0 | P1. With one row tile per CTA,
// two softmax warpgroups take the key tiles of the same rows in turn, each with
// its own S and P (bf16) buffer: an S buffer is free again once its scores are in
// registers, so S of the next tiles is made during the exponentials and nothing
// waits for the chain S -> softmax -> P V -> next S of a tile. (With P written
// over S, three S buffers and that chain, a tile took 1700 cycles; it takes 1412
// now, the rate of the MMAs under the power limit, and an item about 3000 more
// for its start and end.) 4 causal sequences of 4096 to 12288 tokens, 28 heads
// over 4: 1.48 ms, 1286 TFLOP/s; what bounds long items is the tensor pipe, what
// bounds short ones their start (Q and the first K, TMEM hand-over of O).
//
// Warp roles (16 warps per CTA):
//   warp 0      producer: Q, K, V tiles by TMA (128-byte swizzle)
//   warp 1      issues S = Q K^T (the even CTA's, for both), ahead of P V and
//               across item borders
//   warp 2      TMEM allocation; issues O += P V (the even CTA's). Two issuers,
//               because one warp's waits, commits and bookkeeping for both
//               products took longer (2050 cycles a tile) than the MMAs (1024)
//   warp 3      V gate: hands each V tile to the MMA. On tiles with keys that some
//               rows do not see it first looks for infinities and NaNs, because a
//               zero weight times such a value would not be zero. Only if there are
//               any, zeros go over the rows past the last key and over those values
//               (when every such tile was rewritten, the products waited for it:
//               32 x 512 tokens took 166 us instead of 140)
//   warps 4-7   output: O of a finished item from TMEM, divided by the joined sums,
//               while the softmax warps are already in the next item (when the
//               warpgroup with the last tile did this, an item cost 10000 cycles
//               more)
//   warps 8-11, 12-15  softmax of the even / odd key tiles, thread = row. The
//               running maximum passes from one warpgroup to the other through
//               shared memory; it moves only when a row outgrows it by 2^8, and
//               then O is rescaled in TMEM (exact: the sums use the same
//               maximum). Each warpgroup keeps its own sum.
#include <algorithm>

#include "fmka_internal.h"
#include "ptx.cuh"

namespace fmka {

namespace {

constexpr int kBN = 128;        // keys per tile
constexpr int kHeadDim = 128;
constexpr int kThreads = 512;
constexpr int kAhead = 3;       // key tiles that K is loaded ahead of V
constexpr int kKStages = 4;
constexpr int kVStages = 4;
constexpr int kQBytes = 32768;   // 128 rows x 128 channels
constexpr int kQHalf = 16384;    // 64 channels
constexpr int kKBytes = 16384;   // 64 keys x 128 channels
constexpr int kVBytes = 16384;   // 128 keys x 64 channels
constexpr int kStageBytes = 4 * 4096;  // 4 KB per output warp
constexpr int kTileSmem = 2 * kQBytes + kKStages * kKBytes + kVStages * kVBytes + kStageBytes;
constexpr int kMaxItems = 128;         // items of a pair in one launch
constexpr int kCtrlBytes = 5 * 1024 + 512;
constexpr int kSmemBytes = kTileSmem + kCtrlBytes + kMaxItems * 48;
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr uint32_t kTmemO = 0, kTmemS = 128, kTmemP = 384;  // S: 2 x 128 columns, P: 2 x 64
// Register split between the control warps and the softmax warps (setmaxnreg);
// the sum has to fit in what the block is launched with.
constexpr int kRegsControl = 56;
constexpr int kRegsOutput = 88;
constexpr int kRegsSoftmax = 184;
constexpr int kMinLaunchRegs = (128 * (kRegsControl + kRegsOutput) + 256 * kRegsSoftmax + kThreads - 1) / kThreads;

// One item as the roles read it, in shared memory. Keys are counted from the item's first.
struct PairItem {
  int q0, nq;      // first row token, tokens (over both CTAs)
  int k0, n;       // packed row of the first key, key tiles
  int klen;        // keys
  int lim0;        // last key token 0 sees (token i sees lim0 + i)
  int hkv, head0;  // kv head, first query head
  int gn;          // query heads
  int part_ts;     // partial rows per token
  int64_t part;    // first partial row, or -1
};
static_assert(sizeof(PairItem) == 48, "three 16-byte words");

// Division by a number known on the host, by Granlund and Montgomery's multiplication for invariant integers:
// q = (umulhi(n, m) + n) >> s for 0 <= n < 2^31.
struct FastDiv {
  uint32_t m, s;
  int d;
  static FastDiv of(int d) {
    FastDiv f;
    f.d = d;
    f.s = 0;
    while ((1ll << f.s) < d) ++f.s;
    f.m = (uint32_t)(((1ull << 32) * ((1ull << f.s) - (uint64_t)d)) / (uint64_t)d + 1);
    return f;
  }
  __device__ __forceinline__ int div(int n) const { return (int)((__umulhi((uint32_t)n, m) + (uint32_t)n) >> s); }
};

struct PairParams {
  __nv_bfloat16* o;
  int64_t o_st, o_sh;
  float* lse;
  int64_t lse_st, lse_sh;
  const __nv_bfloat16* v;
  int64_t kv_st, kv_sh;
  int Hq, G, Gs, n_gs, nh;   // nh = kv heads x group slices
  int tpt;                   // tokens per CTA
  FastDiv by_nh, by_ngs, by_nrt;
  float scale_log2;          // not zero and no denormal: masked scores are -inf before they are multiplied by it
  const int* header;         // [0] list entries; null: uniform items
  const int4* list;          // {q0, nq, k0, kb}, {ke, lim0, part, 0}
  int B, P, n_rt, n_splits, keys_per_split;  // uniform items
  int round0;                // first round of this launch
  float* part_o;
  float* part_lse;
  uint32_t* status;
};

__device__ __forceinline__ int pair_item_count(const PairParams& p) {
  const int n = p.header != nullptr ? __ldcg(p.header) : p.n_rt * p.n_splits;
  return __shfl_sync(0xffffffffu, n, 0) * p.nh;
}

// The items of one pair: a snake over the list, which is sorted by falling work.
__device__ __forceinline__ int pair_item_index(int r, int pair, int pairs) {
  return r * pairs + ((r & 1) ? pairs - 1 - pair : pair);
}

__device__ __forceinline__ PairItem make_item(const PairParams& p, int idx) {
  PairItem it;
  const int li = p.by_nh.div(idx), h = idx - li * p.nh;
  it.hkv = p.by_ngs.div(h);
  const int g0 = (h - it.hkv * p.n_gs) * p.Gs;
  it.head0 = it.hkv * p.G + g0;
  it.gn = min(p.Gs, p.G - g0);
  int kb, ke;
  if (p.header != nullptr) {
    const int4 a = __ldcg(p.list + 2 * li), b = __ldcg(p.list + 2 * li + 1);
    it.q0 = a.x;
    it.nq = a.y;
    it.k0 = a.z + a.w;
    kb = a.w;
    ke = b.x;
    it.lim0 = b.y - kb;
    it.part = b.z < 0 ? -1 : (int64_t)b.z + (int64_t)h * a.y * p.Gs;
    it.part_ts = p.Gs;
  } else {
    const int split = p.by_nrt.div(li), rt = li - split * p.n_rt;
    it.q0 = rt * 2 * p.tpt;
    it.nq = min(2 * p.tpt, p.B - it.q0);
    kb = split * p.keys_per_split;
    ke = min(p.P, kb + p.keys_per_split);
    it.k0 = kb;
    it.lim0 = p.P;
    it.part = ((int64_t)split * p.B + it.q0) * p.Hq + it.head0;
    it.part_ts = p.Hq;
  }
  it.klen = max(0, ke - kb);
  it.n = (it.klen + kBN - 1) / kBN;
  return it;
}

// The same value in all lanes, and known to be so by the compiler.
__device__ __forceinline__ int uni(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Keys (from the item's first) that every row sees: beyond them tiles have masked or missing keys.
__device__ __forceinline__ int keys_all_see(const PairItem& it) {
  return it.nq > 1 ? min(it.klen, max(0, it.lim0 + 1)) : it.klen;
}

// Position in a ring of N stages and the parity of its current round.
template <int N>
struct Ring {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void step() {
    if (++s == N) {
      s = 0;
      ph ^= 1u;
    }
  }
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    attn_pair_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PairParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * kQBytes;
  uint8_t* sV = sK + kKStages * kKBytes;
  uint8_t* sStage = sV + kVStages * kVBytes;
  float* s_m = reinterpret_cast<float*>(sStage + kStageBytes);  // [128] running maximum
  float* s_lm = s_m + 128;  // [warpgroup][2 slots][sum, maximum][128] handed on at an item's end
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_lm + 1024);
  uint64_t* q_full = bars;                 // [2] even CTA
  uint64_t* q_empty = q_full + 2;          // [2] both
  uint64_t* k_full = q_empty + 2;          // [kKStages] even CTA
  uint64_t* k_empty = k_full + kKStages;   // [kKStages] both
  uint64_t* v_land = k_empty + kKStages;   // [kVStages] own loads have landed
  uint64_t* v_ready = v_land + kVStages;   // [kVStages] even CTA: both gates passed
  uint64_t* v_empty = v_ready + kVStages;  // [kVStages] both
  uint64_t* s_full = v_empty + kVStages;   // [2] both
  uint64_t* s_free = s_full + 2;           // [2] even CTA, 8 warps
  uint64_t* p_full = s_free + 2;           // [2] even CTA, 8 warps
  uint64_t* pv_done = p_full + 2;          // [4] both, by tile number
  uint64_t* o_free = pv_done + 4;          // even CTA, 8 warps
  uint64_t* m_bar = o_free + 1;            // [2][4] maximum handed on, per quarter
  uint64_t* l_bar = m_bar + 8;             // [2][2][4] sum handed on: warpgroup, its count's parity, quarter
  uint64_t* mma_done = l_bar + 16;         // [2] S, P V
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* bad_v = abort_flag + 1;    // [8] by item number: 1 + the last item with taken-out values
  PairItem* items = reinterpret_cast<PairItem*>(smem + kTileSmem + kCtrlBytes);
  static_assert(512 * 9 + 8 * (2 * 2 + 2 * kKStages + 3 * kVStages + 6 + 4 + 1 + 24 + 2) + 48 <= kCtrlBytes,
                "control block fits behind the tiles");

  const int warp = __shfl_sync(0xffffffffu, warp_id(), 0);
  const int lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1;
  const int pairs = gridDim.x >> 1;
  if (smem_u32(smem) & 1023u) {  // the swizzled tiles need it; the same in every CTA
    if (threadIdx.x == 0) atomicOr(p.status, kStatusBadLaunch);
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < kKStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < kVStages; ++i) {
      mbar_init(&v_land[i], 1);
      mbar_init(&v_ready[i], 2);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 8);
      mbar_init(&p_full[i], 8);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&pv_done[i], 1);
    mbar_init(o_free, 8);  // output warps of both CTAs
    for (int i = 0; i < 8; ++i) mbar_init(&m_bar[i], 1);
    for (int i = 0; i < 16; ++i) mbar_init(&l_bar[i], 1);
    mbar_init(&mma_done[0], 1);
    mbar_init(&mma_done[1], 1);
    *abort_flag = 0;
    for (int i = 0; i < 8; ++i) bad_v[i] = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 2) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  // rows that no Q box reaches
  for (int i = threadIdx.x; i < 4 * (128 - p.Gs * p.tpt) * 8; i += kThreads) {
    const int per = (128 - p.Gs * p.tpt) * 8, half = i / per;
    reinterpret_cast<uint4*>(sQ + half * kQHalf + p.Gs * p.tpt * 128)[i - half * per] = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();  // the item list (or the previous kernel's outputs) is complete
  grid_launch_dependents();
  // this pair's items, decoded once for all roles
  const int n_items = pair_item_count(p);
  const int cnt = min(kMaxItems, max(0, (n_items + pairs - 1) / pairs - p.round0));
  if (threadIdx.x < kMaxItems && (int)threadIdx.x < cnt) {
    const int idx = pair_item_index(p.round0 + threadIdx.x, pair, pairs);
    PairItem it = {};  // the last round may have none for this pair
    it.part = -1;
    if (idx < n_items) it = make_item(p, idx);
    items[threadIdx.x] = it;
  }
  __syncthreads();

  if (warp == 0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    // ------------------------------------------------------------ producer --
    // K runs kAhead tiles ahead of V, as S runs ahead of P V.
    const uint32_t q_full_even = cluster_addr(&q_full[0], 0);
    const uint32_t k_full_even = cluster_addr(&k_full[0], 0);
    const int q_box = p.Gs * p.tpt * 128;  // bytes of one 64-channel box
    int ki = -1, vi = -1;  // items of the K and the V walk
    int kn = 0, vn = 0, k_row = 0, v_row = 0, k_head = 0, v_head = 0;
    int kj = 0, vj = 0, ahead = 0, gk = 0, gv = 0, q_use = -1;
    bool k_more = true;
    Ring<kKStages> kr;
    Ring<kVStages> vr;
    bool ok = true;
    while (ok) {
      while (k_more && ahead < kAhead) {
        if (kj == kn) {
          kj = kn = 0;
          while (++ki < cnt && (kn = uni(items[ki].n)) == 0) {}
          if (!(k_more = ki < cnt)) break;
          k_row = uni(items[ki].k0) + (int)rank * 64;
          k_head = uni(items[ki].hkv);
          ++q_use;
          const int qs = q_use & 1;
          if (!(ok = !__any_sync(0xffffffffu, *abort_flag) &&
                     warp_wait(&q_empty[qs], ((q_use >> 1) & 1) ^ 1u, p.status))) break;
          if (elect_one()) {
            if (rank == 0) mbar_arrive_expect_tx(&q_full[qs], 4 * q_box);
            const int tok = items[ki].q0 + (int)rank * p.tpt, head = items[ki].head0;
            tma_load_3d_pair(sQ + qs * kQBytes, &tmQ, q_full_even + qs * 8, 0, head, tok);
            tma_load_3d_pair(sQ + qs * kQBytes + kQHalf, &tmQ, q_full_even + qs * 8, 64, head, tok);
          }
          __syncwarp();
        }
        if (!(ok = warp_wait(&k_empty[kr.s], kr.ph ^ 1u, p.status))) break;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&k_full[kr.s], 2 * kKBytes);
          tma_load_3d_pair(sK + kr.s * kKBytes, &tmK, k_full_even + kr.s * 8, 0, k_row, k_head);
          tma_load_3d_pair(sK + kr.s * kKBytes + kKBytes / 2, &tmK, k_full_even + kr.s * 8, 64, k_row, k_head);
        }
        __syncwarp();
        k_row += kBN;
        ++gk;
        ++ahead;
        ++kj;
        kr.step();
      }
      if (!ok) break;
      if (vj == vn) {
        vj = vn = 0;
        while (++vi < cnt && (vn = uni(items[vi].n)) == 0) {}
        if (vi >= cnt) break;
        v_row = uni(items[vi].k0);
        v_head = uni(items[vi].hkv);
      }
      if (!(ok = warp_wait(&v_empty[vr.s], vr.ph ^ 1u, p.status))) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(&v_land[vr.s], kVBytes);
        tma_load_3d(sV + vr.s * kVBytes, &tmV, &v_land[vr.s], 64 * (int)rank, v_row, v_head);
      }
      __syncwarp();
      v_row += kBN;
      ++gv;
      --ahead;
      ++vj;
      vr.step();
    }
    if (!ok) *abort_flag = 1;
    // Drain: every load has landed, and its tile has been consumed, before the CTA goes.
#pragma unroll 1
    for (int g = gv - 1; g >= 0 && g >= gv - kVStages; --g)
      mbar_sleep(&v_land[g % kVStages], (g / kVStages) & 1, p.status);
#pragma unroll 1
    for (int g = gk - 1; g >= 0 && g >= gk - kKStages; --g)
      mbar_sleep(&k_empty[g % kKStages], (g / kKStages) & 1, p.status);
  } else if (warp == 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    // ----------------------------------- S = Q K^T (the even CTA issues) --
    if (rank == 0) {
      constexpr uint32_t id_s = make_idesc_bf16(256, kBN, false, false);
      const uint64_t q_desc = desc_kmajor_sw128(smem_u32(sQ));
      const uint64_t k_desc = desc_kmajor_sw128(smem_u32(sK));
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      Ring<kKStages> kr;
      Ring<2> sr, qr;
      bool ok = true;
      for (int i = 0; ok && i < cnt; ++i) {
        const int n = uni(items[i].n);
        if (n == 0) continue;
        if (!(ok = warp_wait(&q_full[qr.s], qr.ph, p.status))) break;
        const uint64_t qd = q_desc + (uint64_t)(qr.s * (kQBytes >> 4));
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
          // the K tile, and the S buffer (its last scores are in registers)
          if (!(ok = warp_wait(&k_full[kr.s], kr.ph, p.status) && warp_wait(&s_free[sr.s], sr.ph ^ 1u, p.status))) break;
          tc_fence_after();
          const uint64_t kd = k_desc + (uint64_t)(kr.s * (kKBytes >> 4));
          const uint32_t d = tm + kTmemS + sr.s * 128;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kHeadDim / 16; ++k)
              umma_ss_pair(d, qd + (k >> 2) * (kQHalf >> 4) + (k & 3) * 2, kd + (k >> 2) * (kKBytes >> 5) + (k & 3) * 2,
                           id_s, k > 0 ? 1u : 0u);
            tc_commit_pair(&s_full[sr.s], 0x3);
            tc_commit_pair(&k_empty[kr.s], 0x3);
          }
          __syncwarp();
          kr.step();
          sr.step();
        }
        if (ok && elect_one()) tc_commit_pair(&q_empty[qr.s], 0x3);
        __syncwarp();
        qr.step();
        if (__any_sync(0xffffffffu, *abort_flag)) ok = false;
      }
      if (!ok) *abort_flag = 1;
      if (elect_one()) tc_commit_pair(&mma_done[0], 0x1);
      __syncwarp();
      mbar_sleep(&mma_done[0], 0, p.status);
    }
  } else if (warp == 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    // ------------------------------------ O += P V (the even CTA issues) --
    if (rank == 0) {
      constexpr uint32_t id_pv = make_idesc_bf16(256, kHeadDim, false, true);
      const uint64_t v_desc = desc_mnmajor_sw128(smem_u32(sV), kVBytes);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      Ring<kVStages> vr;
      Ring<2> pr;
      Ring<4> dr;
      uint32_t o_phase = 1;  // nothing to wait for before the first item
      bool ok = true;
      for (int i = 0; ok && i < cnt; ++i) {
        const int n = uni(items[i].n), gated = uni(keys_all_see(items[i])) / kBN;
        if (n == 0) continue;
        if (!(ok = warp_wait(o_free, o_phase, p.status))) break;
        o_phase ^= 1u;
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
          // a tile that the gates may have written to is acquired from the other CTA as well
          ok = j >= gated ? __all_sync(0xffffffffu, mbar_wait_cluster(&v_ready[vr.s], vr.ph, p.status))
                          : warp_wait(&v_ready[vr.s], vr.ph, p.status);
          if (!ok || !(ok = warp_wait(&p_full[pr.s], pr.ph, p.status))) break;
          tc_fence_after();
          const uint64_t vd = v_desc + (uint64_t)(vr.s * (kVBytes >> 4));
          const uint32_t a = tm + kTmemP + pr.s * 64;
          const uint32_t add = j > 0 ? 1u : 0u;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kBN / 16; ++k)
              umma_ts_pair(tm + kTmemO, a + k * 8, vd + k * (2048 >> 4), id_pv, k > 0 ? 1u : add);
            tc_commit_pair(&pv_done[dr.s], 0x3);
            tc_commit_pair(&v_empty[vr.s], 0x3);
          }
          __syncwarp();
          vr.step();
          pr.step();
          dr.step();
        }
        if (__any_sync(0xffffffffu, *abort_flag)) ok = false;
      }
      if (!ok) *abort_flag = 1;
      if (elect_one()) tc_commit_pair(&mma_done[1], 0x1);
      __syncwarp();
      mbar_sleep(&mma_done[1], 0, p.status);
    }
  } else if (warp == 3) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    // -------------------------------------------------------------- V gate --
    const uint32_t ready_even = cluster_addr(&v_ready[0], 0);
    const uint32_t bad_peer = cluster_addr(const_cast<int*>(bad_v), rank ^ 1u);
    Ring<kVStages> vr;
    int item = 0;  // items with key tiles so far
    bool ok = true;
    for (int i = 0; ok && i < cnt; ++i) {
      const int n = uni(items[i].n), klen = uni(items[i].klen), see = uni(keys_all_see(items[i]));
      item += n > 0;
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        if (!(ok = warp_wait(&v_land[vr.s], vr.ph, p.status))) break;
        const int some = max(0, see - j * kBN);  // rows that every query sees
        // 16-byte chunk (row, ch) sits at ch ^ (row & 7) of its 128-byte row; a warp takes 32 rows at a time
        uint8_t* tile = sV + vr.s * kVBytes + (lane >> 3) * 128 + (lane & 7) * 16;
        uint32_t odd = 0;
#pragma unroll 1
        for (int row0 = some & ~31; row0 < kBN; row0 += 32) {
          uint4 x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = *reinterpret_cast<const uint4*>(tile + (row0 + k * 4) * 128);
#pragma unroll
          for (int k = 0; k < 8; ++k) odd |= nonfinite_bits(x[k]);
        }
        if (__any_sync(0xffffffffu, odd != 0)) {
          const int live = klen - j * kBN;  // rows that hold keys
          bool bad = false;
#pragma unroll 1
          for (int row0 = some & ~15; row0 < kBN; row0 += 16) {
            uint4 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<uint4*>(tile + (row0 + k * 4) * 128);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int row = row0 + k * 4 + (lane >> 3);
              const bool gone = row >= live;
              const bool taken = zero_nonfinite(x[k]) && !gone;
              if (gone) x[k] = make_uint4(0, 0, 0, 0);
              if (row >= some && (taken || gone)) *reinterpret_cast<uint4*>(tile + (row0 + k * 4) * 128) = x[k];
              bad |= taken && row >= some;
            }
          }
          if (__any_sync(0xffffffffu, bad) && lane == 0) {
            // the gate is at most four tiles ahead of the products, so eight slots never meet
            bad_v[item & 7] = item;
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(bad_peer + 4 * (item & 7)), "r"(item) : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(ready_even + vr.s * 8);
        } else if (lane == 0) {
          mbar_arrive_cluster_cta(ready_even + vr.s * 8);
        }
        vr.step();
      }
    }
    if (!ok) *abort_flag = 1;
  } else if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOutput));
    // -------------------------------------------------------------- output --
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t o_free_even = cluster_addr(o_free, 0);
    const int ri = r / p.Gs, rg = r - ri * p.Gs;
    const int ti = (int)rank * p.tpt + ri;
    uint8_t* stage = sStage + quarter * 4096;  // 128 bytes of each row; chunk c of row i at c ^ (i & 7)
    uint4* mine = reinterpret_cast<uint4*>(stage + lane * 128);
    int g0 = 0, item = 0;
    int took0 = 0, took1 = 0;
    bool ok = true;
    for (int i = 0; ok && i < cnt; ++i) {
      const PairItem it = items[i];
      const bool row_ok = ri < p.tpt && ti < it.nq && rg < it.gn;
      const int n = uni(it.n);
      const int tok = it.q0 + ti, head = it.head0 + rg;
      const bool direct = it.part < 0;
      float L = 0.f, m_end = -INFINITY;
      bool bad = false;
      if (n > 0) {
        // the sums of the two warpgroups, at the maximum of the one with the last tile
        const int last = (g0 + n - 1) & 1;
        float l_other = 0.f, m_other = -INFINITY;
#pragma unroll 1
        for (int k = n >= 2 ? 0 : 1; k < 2; ++k) {  // the other one's, the last one's
          const int e = last ^ k ^ 1;
          const int took = e ? took1++ : took0++;
          const int slot = e * 2 + (took & 1);
          if (!(ok = warp_wait(&l_bar[slot * 4 + quarter], (took >> 1) & 1, p.status))) break;
          if (k == 0) {
            l_other = s_lm[(slot * 2 + 0) * 128 + r];
            m_other = s_lm[(slot * 2 + 1) * 128 + r];
          } else {
            L = s_lm[(slot * 2 + 0) * 128 + r];
            m_end = s_lm[(slot * 2 + 1) * 128 + r];
          }
        }
        const int gl = g0 + n - 1;
        if (!ok || !(ok = warp_wait(&pv_done[gl & 3], (gl >> 2) & 1, p.status))) break;
        tc_fence_after();
        L += l_other * (m_other == m_end ? 1.f : fast_exp2(m_other - m_end));
        g0 += n;
        ++item;
        bad = bad_v[item & 7] == item;
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const float lse2 = L == 0.f ? -INFINITY : m_end + __log2f(L);
      const bool live = row_ok && (direct || L != 0.f);  // a part without a visible key leaves only its -inf
      const int64_t rec = it.part + (int64_t)ti * it.part_ts + rg;
      const int64_t row_off = direct ? tok * p.o_st + head * p.o_sh : rec * kHeadDim;  // elements
      uint8_t* row_out = (direct ? reinterpret_cast<uint8_t*>(p.o) : reinterpret_cast<uint8_t*>(p.part_o)) +
                         row_off * (direct ? 2 : 4);
      if (!live) row_out = nullptr;
#pragma unroll 1
      for (int pass = 0; pass < 4; ++pass) {  // 32 channels
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(lane_addr + kTmemO + pass * 32, o);
          tmem_wait_ld();
          if (pass == 3) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_cta(o_free_even);
          }
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * inv);
        } else {  // no row of the tile sees a key
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = 0u;
        }
        if (direct) {
          const int c0 = (pass & 1) * 4;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w4[e] = pack_bf16x2(__uint_as_float(o[c * 8 + 2 * e]), __uint_as_float(o[c * 8 + 2 * e + 1]));
            mine[(c0 + c) ^ (lane & 7)] = make_uint4(w4[0], w4[1], w4[2], w4[3]);
          }
          if (c0 == 0) continue;
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) mine[c ^ (lane & 7)] = make_uint4(o[c * 4], o[c * 4 + 1], o[c * 4 + 2], o[c * 4 + 3]);
        }
        // 128 bytes of every row are staged. Four rows per store instruction, whole lines (a thread storing its own
        // row would touch 32 lines with 16 bytes each); the loads of four come before their stores.
        const int line = (direct ? pass >> 1 : pass) * 128 + (lane & 7) * 16;
        __syncwarp();
#pragma unroll 1
        for (int k0 = lane >> 3; k0 < 32; k0 += 16) {
          uint4 x[4];
          unsigned long long dst[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int rr = k0 + k * 4;
            dst[k] = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row_out), rr);
            x[k] = *reinterpret_cast<const uint4*>(stage + rr * 128 + (((lane ^ rr) & 7) << 4));
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (dst[k] != 0ull) *reinterpret_cast<uint4*>(dst[k] + line) = x[k];
        }
        __syncwarp();
      }
      if (direct) {
        if (row_ok && p.lse != nullptr) p.lse[tok * p.lse_st + head * p.lse_sh] = lse2 * 0.69314718055994531f;
      } else if (row_ok) {
        p.part_lse[rec] = lse2;
      }
      if (bad && live) {
        // rare: values that the V gate took out go to the rows that see them (the row's stores by other lanes come
        // first: they are ordered by the barrier after them)
        const int lim = min(it.klen - 1, it.lim0 + ti);
        const __nv_bfloat16* vrow = p.v + (int64_t)it.k0 * p.kv_st + it.hkv * p.kv_sh;
#pragma unroll 1
        for (int key = max(0, it.lim0 + 1); key <= lim; ++key) {
#pragma unroll 1
          for (int d = 0; d < kHeadDim; ++d) {
            const float x = __bfloat162float(vrow[key * p.kv_st + d]);
            if (fabsf(x) <= 3.4e38f) continue;
            if (direct) {
              __nv_bfloat16* y = p.o + row_off + d;
              *y = __float2bfloat16(__bfloat162float(*y) + x);
            } else {
              p.part_o[row_off + d] += x;
            }
          }
        }
      }
    }
    if (!ok) *abort_flag = 1;
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ------------------------------------------------------------- softmax --
    const int wg = (warp - 8) >> 2;
    const int quarter = warp & 3;  // the TMEM lanes this warp may touch
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t p_full_even = cluster_addr(&p_full[wg], 0);
    const uint32_t s_free_even = cluster_addr(&s_free[wg], 0);
    const int ri = r / p.Gs, rg = r - ri * p.Gs;  // token of the CTA's tile, head of the slice
    const int ti = (int)rank * p.tpt + ri;         // token of the pair's tile
    const uint32_t s_col = kTmemS + wg * 128, p_col = kTmemP + wg * 64;
    int g0 = 0;                                    // tiles before this item
    int gave = 0;                                  // sums handed to the output warps so far
    bool ok = true;
    for (int i = 0; ok && i < cnt; ++i) {
      const int n = uni(items[i].n);
      if (n == 0) continue;
      const int klen = items[i].klen, lim0 = items[i].lim0;
      const bool row_ok = ri < p.tpt && ti < items[i].nq && rg < items[i].gn;
      // Last visible key. Rows that are not there (behind the last token, or the last rows where the group does not
      // divide 128) multiply whatever their Q holds; nothing of theirs is stored or has a say in the rescaling.
      const int lim = row_ok ? min(klen - 1, lim0 + ti) : 0x3FFFFFFF;
      float m_own = -INFINITY, l = 0.f;
      // from this tile on, some row of this CTA does not see every key
      const int first_masked = uni(min(klen, max(0, lim0 + 1 + (int)rank * p.tpt))) / kBN;
#pragma unroll 1
      for (int j = (g0 & 1) == wg ? 0 : 1; j < n; j += 2) {
        const int g = g0 + j;  // g & 1 == wg
        if (!(ok = warp_wait(&s_full[wg], (g >> 1) & 1, p.status))) break;
        tc_fence_after();
        uint32_t s[128];
        tmem_ld32(lane_addr + s_col + 0, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
        tmem_ld32(lane_addr + s_col + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
        tmem_ld32(lane_addr + s_col + 64, *reinterpret_cast<uint32_t(*)[32]>(&s[64]));
        tmem_ld32(lane_addr + s_col + 96, *reinterpret_cast<uint32_t(*)[32]>(&s[96]));
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_cta(s_free_even);
        if (j >= first_masked) {
          const int seen = lim - j * kBN;  // last visible column of the tile
          const int all_see = __reduce_min_sync(0xffffffffu, seen);
#pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 16) {
            if (all_see < c0 + 15) {
#pragma unroll
              for (int c = c0; c < c0 + 16; ++c)
                if (c > seen) s[c] = 0xFF800000u;  // -inf
            }
          }
        }
        float mxa[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) mxa[a] = -INFINITY;
#pragma unroll
        for (int c = 0; c < 128; c += 16) {
#pragma unroll
          for (int a = 0; a < 8; ++a) mxa[a] = fmax3(mxa[a], __uint_as_float(s[c + a]), __uint_as_float(s[c + 8 + a]));
        }
        const float mx = p.scale_log2 * fmax3(fmax3(mxa[0], mxa[1], mxa[2]), fmax3(mxa[3], mxa[4], mxa[5]),
                                              fmaxf(mxa[6], mxa[7]));
        // The maximum after the tile before (the other warpgroup's, same rows), and this warpgroup's P buffer (its
        // last P has been multiplied): one poll for both, which are there in the long run.
        if (g > 0) {
          uint64_t* mb = &m_bar[(wg ^ 1) * 4 + quarter];
          uint64_t* pb = &pv_done[(g - 2) & 3];
          const uint32_t m_ph = ((g - 1) >> 1) & 1, p_ph = ((g - 2) >> 2) & 1;
          if (!__all_sync(0xffffffffu, mbar_try_wait(mb, m_ph) && (g == 1 || mbar_try_wait(pb, p_ph)))) {
            if (!(ok = warp_wait(mb, m_ph, p.status) && (g == 1 || warp_wait(pb, p_ph, p.status)))) break;
          }
        }
        float m_ref = j > 0 ? s_m[r] : -INFINITY;
        float alpha = 1.f;
        const bool grow = __any_sync(0xffffffffu, row_ok && mx > m_ref + kRescaleThreshold);
        if (grow) {
          const float m_new = fmaxf(m_ref, mx);
          alpha = m_new == m_ref ? 1.f : fast_exp2(m_ref - m_new);
          m_ref = m_new;
        }
        if (grow || j == 0) s_m[r] = m_ref;
        __syncwarp();
        if (lane == 0) mbar_arrive(&m_bar[wg * 4 + quarter]);
        if (grow && j > 0) {
          // O holds the tiles before this one: wait for the last product, then move O to the new maximum. (No phase
          // of the barrier is skipped: the other warpgroup has waited for tile g - 5 before it wrote P of tile g - 3,
          // whose product comes before that of tile g - 2.)
          if (!(ok = warp_wait(&pv_done[(g - 1) & 3], ((g - 1) >> 2) & 1, p.status))) break;
          tc_fence_after();
#pragma unroll 1
          for (int c4 = 0; c4 < 8; ++c4) {
            uint32_t o[16];
            tmem_ld16(lane_addr + kTmemO + c4 * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
            tmem_st16(lane_addr + kTmemO + c4 * 16, o);
          }
        }
        l *= m_own == m_ref ? 1.f : fast_exp2(m_own - m_ref);
        m_own = m_ref;
        const float msub = m_ref == -INFINITY ? 0.f : m_ref;
        const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
        const float2 nm2 = make_float2(-msub, -msub);
        float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          const uint32_t* sc = s + 32 * ch;
          uint32_t pk[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float2 xx =
                ffma2(make_float2(__uint_as_float(sc[2 * c]), __uint_as_float(sc[2 * c + 1])), sl2, nm2);
            const float2 pp = make_float2(fast_exp2(xx.x), fast_exp2(xx.y));
            acc[c & 3] = fadd2(acc[c & 3], pp);
            pk[c] = pack_bf16x2(pp.x, pp.y);
          }
          tmem_st16(lane_addr + p_col + 16 * ch, pk);
        }
        const float2 asum = fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3]));
        l += asum.x + asum.y;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_cta(p_full_even);
      }
      if (!ok) break;
      if (n >= 2 || (g0 & 1) == wg) {
        // This warpgroup's sum and maximum go to the output warps. Two slots: before the one after next is written,
        // a product has been waited for that comes after the output warps have read this one.
        s_lm[((wg * 2 + (gave & 1)) * 2 + 0) * 128 + r] = l;
        s_lm[((wg * 2 + (gave & 1)) * 2 + 1) * 128 + r] = m_own;
        __syncwarp();
        if (lane == 0) mbar_arrive(&l_bar[(wg * 2 + (gave & 1)) * 4 + quarter]);
        ++gave;
      }
      g0 += n;
    }
    if (!ok) *abort_flag = 1;
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync();  // nothing aimed at either CTA is still under way
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Tensor map over [rows][heads][128] with a box of box_h heads x box_r rows x 64 channels. The stride of a dimension
// of one element says nothing.
int rows_map(CUtensorMap* out, const __nv_bfloat16* base, int64_t rows, int64_t st, int heads, int64_t sh, int box_h,
             int box_r, bool head_inner) {
  // the callers send expanded views (a stride of zero over several) elsewhere
  if (rows == 1) st = 128;
  if (heads == 1) sh = 128;
  if (head_inner) {
    const uint64_t dims[3] = {128, (uint64_t)heads, (uint64_t)rows};
    const uint64_t strides[2] = {(uint64_t)sh * 2, (uint64_t)st * 2};
    const uint32_t box[3] = {64, (uint32_t)box_h, (uint32_t)box_r};
    return make_tmap_bf16(out, base, 3, dims, strides, box, true);
  }
  const uint64_t dims[3] = {128, (uint64_t)rows, (uint64_t)heads};
  const uint64_t strides[2] = {(uint64_t)st * 2, (uint64_t)sh * 2};
  const uint32_t box[3] = {64, (uint32_t)box_r, 1};
  return make_tmap_bf16(out, base, 3, dims, strides, box, true);
}

void pair_tile(PairParams& p) {
  p.n_gs = (p.G + 127) / 128;
  p.Gs = (p.G + p.n_gs - 1) / p.n_gs;
  p.tpt = 128 / p.Gs;
  p.nh = (p.Hq / p.G) * p.n_gs;
}

int launch_pair(const PairParams& given, const __nv_bfloat16* q, int64_t q_rows, int64_t q_st, int64_t q_sh,
                const __nv_bfloat16* k, const __nv_bfloat16* v, int64_t kv_rows, int64_t kv_st, int64_t kv_sh,
                int pairs, int64_t max_items, bool dependent, cudaStream_t stream, const char* what) {
  PairParams p = given;
  p.by_nh = FastDiv::of(p.nh);
  p.by_ngs = FastDiv::of(p.n_gs);
  p.by_nrt = FastDiv::of(std::max(p.n_rt, 1));
  CUtensorMap tmQ, tmK, tmV;
  int rc = rows_map(&tmQ, q, q_rows, q_st, p.Hq, q_sh, p.Gs, p.tpt, true);
  if (rc) return rc;
  rc = rows_map(&tmK, k, kv_rows, kv_st, p.Hq / p.G, kv_sh, 1, 64, false);
  if (rc) return rc;
  rc = rows_map(&tmV, v, kv_rows, kv_st, p.Hq / p.G, kv_sh, 1, 128, false);
  if (rc) return rc;
  static std::atomic<int> launch_regs{0};
  if (launch_regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes fa;
    rc = check_cuda(cudaFuncGetAttributes(&fa, attn_pair_kernel), what);
    if (rc) return rc;
    launch_regs.store(fa.numRegs, std::memory_order_relaxed);
  }
  if (launch_regs.load(std::memory_order_relaxed) < kMinLaunchRegs)
    return set_error(kErrUnsupported, std::string(what) + ": compiled register count too small for the warpgroup split");
  static std::atomic<uint64_t> devices{0};
  rc = check_cuda(allow_smem(attn_pair_kernel, kSmemBytes, devices), what);
  if (rc) return rc;
  // kMaxItems of each pair per launch; the bound on the items is loose, a launch without any ends at once
  const int64_t rounds = (max_items + pairs - 1) / pairs;
  for (int64_t r0 = 0; r0 < rounds; r0 += kMaxItems) {
    p.round0 = (int)r0;
    rc = check_cuda(launch_after(attn_pair_kernel, dim3(2 * pairs), kThreads, kSmemBytes, dependent || r0 > 0, stream,
                                 tmQ, tmK, tmV, p),
                    what);
    if (rc) return rc;
  }
  return kOk;
}

}  // namespace

PackedPlan attn_pair_plan(int n_seqs, int total_q, int max_k, int Hq, int Hkv) {
  PairParams p = {};
  p.Hq = Hq;
  p.G = Hq / Hkv;
  pair_tile(p);
  return packed_plan(n_seqs, total_q, max_k, Hkv, p.G, p.Gs, 2 * p.tpt, num_sms_current_device() / 2);
}

int launch_attn_pair_varlen(const PackedAttnParams& a, const PackedPlan& w, cudaStream_t stream) {
  PairParams p = {};
  p.o = a.o;
  p.o_st = a.o_st;
  p.o_sh = a.o_sh;
  p.lse = a.lse;
  p.lse_st = a.lse_st;
  p.lse_sh = a.lse_sh;
  p.v = a.v;
  p.kv_st = a.kv_st;
  p.kv_sh = a.kv_sh;
  p.Hq = a.Hq;
  p.G = a.G;
  pair_tile(p);
  p.scale_log2 = a.scale_log2;
  p.status = a.status;
  p.header = w.header;
  p.list = w.list;
  p.part_o = w.part_o;
  p.part_lse = w.part_lse;
  return launch_pair(p, a.q, a.total_q, a.q_st, a.q_sh, a.k, a.v, a.total_k, a.kv_st, a.kv_sh, w.workers,
                     (int64_t)w.max_list * p.nh, true, stream, "attn_varlen launch");
}

// Parts of the shared prefix. The own keys' kernel cannot share an SM with this one (registers and shared memory are
// taken whole), so a cut that fills every pair leaves it waiting: the cut is the one with the least time for both, own
// keys filling the SMs beside a single round of pairs. Against cuts that fill all pairs, in us with own keys and join:
// 33 requests, 5003 + 400 keys, 25.6 -> 23.1; 64, 32768 + 1024, 67 -> 60; 256, 4096 + 512, 76.6 -> 71.9.
int attn_pair_prefix_splits(int B, int Hq, int Hkv, int P, int cap, int* keys_per_split) {
  PairParams p = {};
  p.Hq = Hq;
  p.G = Hq / Hkv;
  pair_tile(p);
  const int sms = num_sms_current_device(), pairs = sms / 2;
  const int64_t units = (int64_t)((B + 2 * p.tpt - 1) / (2 * p.tpt)) * p.nh;
  const int tiles = (P + kBN - 1) / kBN;
  // SM x us that the own keys take at the memory's rate (half of the slots in use, 512 bytes a key, 6.5 KB a ns)
  const double own = (double)B * Hkv * cap * 0.5 * 512 / 6.5e6 * sms;
  const int most = (int)std::min<int64_t>({64, tiles, 2 * pairs / units + 1});  // two rounds or less
  int per = tiles;
  double prefix = 0, beside = 0;
  auto cut = [&](int parts) {
    per = (tiles + parts - 1) / parts;
    const int64_t items = units * ((tiles + per - 1) / per);
    const int64_t rounds = (items + pairs - 1) / pairs;
    prefix = 0.75 * (double)rounds * (per + 4) + 0.1 * parts;  // four tiles' time per item for its start and end
    beside = rounds == 1 ? (double)(sms - 2 * items) * prefix : 0.0;
  };
  double alone = 1e30;  // the least time of the prefix by itself; it may take twice that, as slots may hold few keys
  for (int s = 1; s <= most; ++s) {
    cut(s);
    alone = std::min(alone, prefix);
  }
  int best = 1;
  double best_us = 1e30;
  for (int s = 1; s <= most; ++s) {
    cut(s);
    const double us = prefix + std::max(0.0, own - beside) / sms;
    if (prefix <= 2 * alone && us < best_us) {
      best_us = us;
      best = s;
    }
  }
  cut(best);
  *keys_per_split = per * kBN;
  return (tiles + per - 1) / per;
}

int launch_attn_pair_prefix(const PackedAttnParams& a, cudaStream_t stream) {
  PairParams p = {};
  p.v = a.vp;
  p.kv_st = a.kp_st;
  p.kv_sh = a.kp_sh;
  p.Hq = a.Hq;
  p.G = a.G;
  pair_tile(p);
  p.scale_log2 = a.scale_log2;
  p.status = a.status;
  p.B = a.B;
  p.P = a.P;
  p.n_rt = (a.B + 2 * p.tpt - 1) / (2 * p.tpt);
  p.n_splits = a.prefix_splits;
  p.keys_per_split = a.prefix_keys;
  p.part_o = a.part_o;
  p.part_lse = a.part_lse;
  const int64_t items = (int64_t)p.n_rt * p.n_splits * p.nh;
  if (items > 0x3FFFFFFF) return set_error(kErrUnsupported, "attn_decode_shared: problem too large");
  const int pairs = (int)std::min<int64_t>(num_sms_current_device() / 2, items);
  return launch_pair(p, a.q, a.B, a.q_st, a.q_sh, a.kp, a.vp, a.P, a.kp_st, a.kp_sh, pairs, items, false, stream,
                     "attn_decode_shared prefix launch");
}

}  // namespace fmka
