// The plan of a packed batch: what is computed where, made on the device from the sequences' offsets, and the kernel
// that joins the parts of rows whose keys were cut.
#include <algorithm>

#include "fmka_internal.h"
#include "ptx.cuh"

namespace fmka {

namespace {

constexpr int kHeadDim = 128;
constexpr int kBN = 128;  // keys per unit of work

// One CTA turns the sequences' offsets into the item list: row tiles of tok_tile
// tokens, each against the keys its rows see, sorted by falling work (a counting
// sort over kBins classes of tile counts), so that the workers, who take items in
// turn or as CTAs are scheduled, get about the same. A tile with more work than a
// worker's fair share is cut along its keys into parts that are joined afterwards.
// Offsets that fall or leave the tensors give an empty list and a status bit.
// It takes 4 to 6 us in a stream of calls for lists that fit shared memory (6.7 with
// cold caches), nearly all of it latency (smaller code in loops and calls measured no
// faster).
// (List, header and parts are read past L1: the reading kernels start before their writers end.)
constexpr int kPlanThreads = 512;
constexpr int kBins = 512;
constexpr int kPlanSeqs = 1024;
constexpr int kMinPartTiles = 4;  // a part is worth its partial output from 512 keys on (256 and 128: no faster)

struct PlanParams {
  const int* cu_q;
  const int* cu_k;
  int n_seqs, total_q, total_k, causal;
  PackedPlan w;
  uint32_t* status;
};

struct TileOf {
  int q0, nq, k0, ke, lim0, tiles;
};

// Row tile f: `first` holds the tiles before each sequence.
__device__ __forceinline__ TileOf tile_of(const PlanParams& p, const int* cu_q, const int* cu_k, const int* first,
                                          int f) {
  int lo = 0, hi = p.n_seqs - 1;  // the last sequence whose first tile is at or before f
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= f) lo = mid;
    else hi = mid - 1;
  }
  const int q0 = cu_q[lo], lq = cu_q[lo + 1] - q0;
  const int k0 = cu_k[lo], lk = cu_k[lo + 1] - k0;
  const int t0 = (f - first[lo]) * p.w.tok_tile;
  TileOf t;
  t.q0 = q0 + t0;
  t.nq = min(p.w.tok_tile, lq - t0);
  t.k0 = k0;
  t.lim0 = p.causal ? t0 + lk - lq : lk;
  t.ke = p.causal ? max(0, min(lk, t.lim0 + t.nq)) : lk;
  t.tiles = (t.ke + kBN - 1) / kBN;
  return t;
}

// Inclusive sum over the block (kPlanThreads threads); `all` gets the total. s_warp: one int per warp.
__device__ __forceinline__ int block_sum(int x, int* s_warp, int& all) {
  const int lane = lane_id(), warp = warp_id();
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int w = lane < kPlanThreads / 32 ? s_warp[lane] : 0;
#pragma unroll
  for (int d = 1; d < kPlanThreads / 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, d);
    if (lane >= d) w += y;
  }
  all = __shfl_sync(0xffffffffu, w, kPlanThreads / 32 - 1);
  const int before = __shfl_sync(0xffffffffu, w, max(0, warp - 1));
  __syncthreads();
  return x + (warp > 0 ? before : 0);
}

__global__ void __launch_bounds__(kPlanThreads) attn_plan_kernel(const __grid_constant__ PlanParams p) {
  __shared__ int s_warp[kPlanThreads / 32];
  __shared__ int s_hist[kBins];
  __shared__ unsigned long long s_total;
  __shared__ int s_groups, s_rows, s_max;
  __shared__ int s_seq[3][kPlanSeqs + 1];  // offsets and tiles of up to kPlanSeqs sequences; more stay in memory
  const int tid = threadIdx.x, lane = lane_id();
  grid_launch_dependents();
  s_hist[tid] = 0;
  static_assert(kBins == kPlanThreads, "one bin per thread");
  if (tid == 0) {
    s_total = 0;
    s_groups = s_rows = s_max = 0;
  }
  const bool small = p.n_seqs <= kPlanSeqs;
  const int* cu_q = small ? s_seq[0] : p.cu_q;
  const int* cu_k = small ? s_seq[1] : p.cu_k;
  int* first = small ? s_seq[2] : p.w.seq_tiles;
  // tiles before each sequence
  int n_tiles = 0;
  bool bad = false;
  for (int s0 = 0; s0 < p.n_seqs; s0 += kPlanThreads) {
    const int s = s0 + tid;
    int nt = 0;
    if (s < p.n_seqs) {
      const int q0 = __ldg(p.cu_q + s), q1 = __ldg(p.cu_q + s + 1);
      const int k0 = __ldg(p.cu_k + s), k1 = __ldg(p.cu_k + s + 1);
      bad |= q0 < 0 || q1 < q0 || q1 > p.total_q || k0 < 0 || k1 < k0 || k1 > p.total_k;
      nt = bad ? 0 : (q1 - q0 + p.w.tok_tile - 1) / p.w.tok_tile;
      if (small) {
        s_seq[0][s] = q0;
        s_seq[1][s] = k0;
        if (s == p.n_seqs - 1) {
          s_seq[0][s + 1] = q1;
          s_seq[1][s + 1] = k1;
        }
      }
    }
    int all;
    const int incl = block_sum(nt, s_warp, all);
    if (s < p.n_seqs) first[s] = n_tiles + incl - nt;
    n_tiles += all;
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) {
      atomicOr(p.status, kStatusBadLaunch);
      p.w.header[0] = p.w.header[1] = 0;
    }
    return;
  }
  // all work, and the largest tile
  unsigned sum = 0;
  int most = 1;
  for (int f = tid; f < n_tiles; f += kPlanThreads) {
    const int c = tile_of(p, cu_q, cu_k, first, f).tiles;
    sum += c;  // below 2^32: total_q / tok_tile tiles per thread of at most 2^24 key tiles would be needed
    most = max(most, c);
  }
  const unsigned warp_sum = __reduce_add_sync(0xffffffffu, sum & 0xFFFFFu);
  const unsigned warp_high = __reduce_add_sync(0xffffffffu, sum >> 20);
  const int warp_most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) {
    atomicAdd(&s_total, (unsigned long long)warp_sum + ((unsigned long long)warp_high << 20));
    atomicMax(&s_max, warp_most);
  }
  __syncthreads();
  const unsigned long long work = s_total * p.w.nh;
  const int share = (int)max((unsigned long long)kMinPartTiles, (work + p.w.workers - 1) / p.w.workers);
  const int top = min(s_max, p.w.split ? share : s_max);
  const float scale = (float)kBins / (float)(top + 1);
  auto parts_of = [&](int tiles) { return p.w.split && tiles > share ? (tiles + share - 1) / share : 1; };
  auto bin_of = [&](int tiles) { return kBins - 1 - min(kBins - 1, (int)((float)tiles * scale)); };
  for (int f = tid; f < n_tiles; f += kPlanThreads) {
    const int c = tile_of(p, cu_q, cu_k, first, f).tiles, np = parts_of(c);
    atomicAdd(&s_hist[bin_of((c + np - 1) / np)], np);
  }
  __syncthreads();
  // exclusive sums over the bins, heavy bins first
  {
    const int n = s_hist[tid];
    int all;
    const int incl = block_sum(n, s_warp, all);
    s_hist[tid] = incl - n;
    if (tid == 0) p.w.header[0] = all;
  }
  __syncthreads();
  for (int f = tid; f < n_tiles; f += kPlanThreads) {
    const TileOf t = tile_of(p, cu_q, cu_k, first, f);
    const int np = parts_of(t.tiles);
    const int per = (t.tiles + np - 1) / np;
    const int at = atomicAdd(&s_hist[bin_of(per)], np);
    if (np > 1) {
      const int rows = t.nq * p.w.Gs * p.w.nh;
      const int row0 = atomicAdd(&s_rows, np * rows);
      p.w.groups[atomicAdd(&s_groups, 1)] = make_int4(t.q0, t.nq, np, row0);
      for (int i = 0; i < np; ++i) {
        p.w.list[2 * (at + i)] = make_int4(t.q0, t.nq, t.k0, i * per * kBN);
        p.w.list[2 * (at + i) + 1] = make_int4(min(t.ke, (i + 1) * per * kBN), t.lim0, row0 + i * rows, 0);
      }
    } else {
      p.w.list[2 * at] = make_int4(t.q0, t.nq, t.k0, 0);
      p.w.list[2 * at + 1] = make_int4(t.ke, t.lim0, -1, 0);
    }
  }
  __syncthreads();
  if (tid == 0) p.w.header[1] = s_groups;
}

// Joins the parts of the rows whose keys were cut: a block per group of parts (x) and slice of its rows (y), a warp
// per row. A lane holds the weight of one part; the outputs are summed four parts at a time.
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ PackedAttnParams a,
                                                        const __grid_constant__ PackedPlan w) {
  grid_dependency_wait();
  if ((int)blockIdx.x >= __ldcg(w.header + 1)) return;
  const int4 gr = __ldcg(w.groups + blockIdx.x);
  const int item_rows = gr.y * w.Gs, rows = item_rows * w.nh;
  for (int row = blockIdx.y * 8 + warp_id(); row < rows; row += gridDim.y * 8) {
    const int h = row / item_rows, ti = (row - h * item_rows) / w.Gs, g = row % w.Gs;
    const int hkv = h / w.n_gs, hg = (h - hkv * w.n_gs) * w.Gs + g;
    if (hg >= a.G) continue;
    join_row(w.part_o + ((int64_t)gr.w + row) * kHeadDim, w.part_lse + (int64_t)gr.w + row, rows, gr.z,
             a.o + (int64_t)(gr.x + ti) * a.o_st + (hkv * a.G + hg) * a.o_sh,
             a.lse == nullptr ? nullptr : a.lse + (int64_t)(gr.x + ti) * a.lse_st + (hkv * a.G + hg) * a.lse_sh);
  }
}

size_t up16(size_t x) { return (x + 15) & ~size_t(15); }

}  // namespace

PackedPlan packed_plan(int n_seqs, int total_q, int max_k, int Hkv, int G, int Gs, int tok_tile, int workers) {
  PackedPlan w = {};
  w.Gs = Gs;
  w.n_gs = (G + Gs - 1) / Gs;
  w.nh = Hkv * w.n_gs;
  w.tok_tile = tok_tile;
  w.workers = workers;
  // An item with more than a worker's share of the work is cut into less than twice work / share parts, so the parts
  // of all nh slices number at most twice the workers.
  w.split = max_k > kMinPartTiles * kBN;
  w.max_parts = w.split ? 2 * workers / w.nh : 0;
  w.split = w.max_parts > 0;
  w.max_list = (int)(((int64_t)total_q + (int64_t)n_seqs * (tok_tile - 1)) / tok_tile) + w.max_parts;
  w.part_rows = (int64_t)w.max_parts * tok_tile * Gs * w.nh;
  size_t at = 16;
  w.at_seq = at;
  at = up16(at + sizeof(int) * (size_t)(n_seqs + 1));
  w.at_list = at;
  at += sizeof(int4) * 2 * (size_t)w.max_list;
  w.at_groups = at;
  at += sizeof(int4) * (size_t)w.max_parts;
  w.at_part_o = at;
  at += sizeof(float) * kHeadDim * (size_t)w.part_rows;
  w.at_part_lse = at;
  at += sizeof(float) * (size_t)w.part_rows;
  w.total = up16(at);
  return w;
}

int launch_plan(const PackedAttnParams& a, PackedPlan& w, void* workspace, cudaStream_t stream) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  w.header = reinterpret_cast<int*>(ws);
  w.seq_tiles = reinterpret_cast<int*>(ws + w.at_seq);
  w.list = reinterpret_cast<int4*>(ws + w.at_list);
  w.groups = reinterpret_cast<int4*>(ws + w.at_groups);
  w.part_o = reinterpret_cast<float*>(ws + w.at_part_o);
  w.part_lse = reinterpret_cast<float*>(ws + w.at_part_lse);
  PlanParams p = {};
  p.cu_q = a.cu_q;
  p.cu_k = a.cu_k;
  p.n_seqs = a.n_seqs;
  p.total_q = a.total_q;
  p.total_k = a.total_k;
  p.causal = a.causal;
  p.w = w;
  p.status = a.status;
  attn_plan_kernel<<<1, kPlanThreads, 0, stream>>>(p);
  return check_cuda(cudaGetLastError(), "attn_varlen plan launch");
}

int launch_join(const PackedAttnParams& a, const PackedPlan& w, cudaStream_t stream) {
  if (!w.split) return kOk;
  // a group has two parts or more; about four blocks per SM over all groups, at most one per eight rows of a group
  const int groups = std::max(1, w.max_parts / 2);
  const int slices = std::min((w.tok_tile * w.Gs * w.nh + 7) / 8, (4 * num_sms_current_device() + groups - 1) / groups);
  return check_cuda(launch_after(attn_join_kernel, dim3(groups, slices), 256, 0, true, stream, a, w),
                    "attn_varlen join launch");
}

}  // namespace fmka
