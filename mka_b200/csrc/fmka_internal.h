// Internal declarations shared by the FastMKA CUDA translation units: launch
// parameter structs, kernel launchers and the per-thread error channel that the
// C-ABI entry points report through.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <string>
#include <utility>

namespace fmka {

// ----------------------------------------------------------------- errors --
// Status codes returned by every C-ABI entry point (0 = success).
enum Status : int {
  kOk = 0,
  kErrInvalidArgument = 1,
  kErrUnsupported = 2,
  kErrCuda = 3,
  kErrWorkspace = 4,
  kErrDevice = 5,
};

// Records `msg` as this thread's last error and returns `code`.
int set_error(int code, const std::string& msg);
// Checks a CUDA runtime result; on failure records it and returns kErrCuda.
int check_cuda(cudaError_t e, const char* what);

// ------------------------------------------------------------- tensor maps --
// Encodes a bf16 tiled tensor map (rank 2 to 5), with or without 128-byte swizzle.
// dims/strides are innermost first; strides are in bytes for dims 1..rank-1.
int make_tmap_bf16(CUtensorMap* out, const void* base, int rank, const uint64_t* dims,
                   const uint64_t* strides_bytes, const uint32_t* box, bool swizzle128);
// The same for fp32 elements, without swizzle.
int make_tmap_f32(CUtensorMap* out, const void* base, int rank, const uint64_t* dims,
                  const uint64_t* strides_bytes, const uint32_t* box);

// ------------------------------------------------------------ peer memory --
// Most ranks (GPUs of one box) that exchange data through peer mappings.
constexpr int kMaxPeers = 8;

// Pointers into the same buffer as mapped in each rank (index = rank in group).
struct PeerPtrs {
  __nv_bfloat16* p[kMaxPeers];
};

// ------------------------------------------------------------------- GEMM --
enum SegKind : int { kSegRowMajor = 0, kSegHeads = 1, kSegRouter = 2, kSegSwiGLU = 3, kSegRowMajorF32 = 4 };

struct GemmSeg {
  int kind;
  int n_begin;           // first global column of this segment
  int n_end;             // one past the last column of this segment
  __nv_bfloat16* out;    // row-major: [M, ld]; heads: [B, H, Tcap, Dh] through strides
  int64_t ld;            // row-major row stride (elements)
  const float* bias;     // indexed by (n - n_begin); may be null
  int T;                 // tokens per batch row (rows m = b*T + t)
  int head_dim;          // 128
  int64_t s_b, s_h, s_t; // element strides of the head-split output
  int t_offset;          // first token slot written in the head-split output
  const float* rope_cos; // [*, T, head_dim] fp32 or null (no RoPE)
  const float* rope_sin;
  int64_t rope_sb, rope_st;
  const float* w2;       // router second layer [L, R] fp32
  int L;
  int act;               // 0 = SiLU, 1 = GELU (erf)
  float* logits;         // [M, L] fp32, accumulated
  float* out_f32;        // kSegRowMajorF32: [M, ld] fp32 output (row stride ld)
  // SwiGLU: columns come in blocks of 256, gate rows then up rows of the same
  // 128 output channels; out [M, ld] receives silu(gate) * up per channel.
};

struct GemmParams {
  int M, N, K;
  int a_kblk;            // > 0: A is stored as K / a_kblk blocks of [M, a_kblk]
  int64_t a_blk_stride;  // element distance between those blocks
  int n_split;  // columns < n_split use seg[0], the rest seg[1]
  GemmSeg seg[2];
  uint32_t* status;
  // Scatter epilogue (n_dst > 0, replaces the segments): bias seg[0].bias,
  // output row m written to row dst_row0 + m of every dst.p[0 .. n_dst-1]
  // (row stride dst_ld), each a local or a peer-mapped [*, N] bf16 buffer.
  int n_dst;
  int64_t dst_row0;
  int64_t dst_ld;
  PeerPtrs dst;
  // Tile order (set by launch_gemm): bands of raster_group row blocks with the
  // row block running fastest inside a band; 1 is plain row-major order.
  int raster_group;
};

// Row block mb and column block nb of persistent-GEMM tile `tile` (see
// GemmParams::raster_group); a bijection of [0, num_m * num_n) onto the grid.
__host__ __device__ __forceinline__ void gemm_tile_coords(int tile, int num_m, int num_n, int group, int& mb,
                                                          int& nb) {
  const int band_tiles = group * num_n;
  const int band = tile / band_tiles;
  const int first = band * group;
  const int rows = group < num_m - first ? group : num_m - first;
  const int r = tile - band * band_tiles;
  mb = first + r % rows;
  nb = r / rows;
}

// C = A[M,K] * B[N,K]^T with the segment epilogues. A and B are row-major bf16
// with row strides lda / ldb (elements).
int launch_gemm(const __nv_bfloat16* A, int64_t lda, const __nv_bfloat16* B, int64_t ldb, const GemmParams& p,
                int num_sms, cudaStream_t stream);

// ------------------------------------------------- packed serving operators --
struct QkNormParams {
  const __nv_bfloat16* x[2];   // q, k: x[b, t, h, :]
  __nv_bfloat16* y[2];
  int64_t x_sb[2], x_st[2], x_sh[2];
  int64_t y_sb[2], y_st[2], y_sh[2];
  const void* w[2];            // [128] or null (no norm)
  int w_f32[2];                // weights are fp32 instead of bf16
  float eps;
  const float* cos;            // rows of 128 or null (no rotation)
  const float* sin;
  int64_t rope_sb, rope_st;    // row of token (b, t) without positions
  const void* positions;       // [B * T] rows of the table, or null
  int pos_i64;
  int n_pos;                   // rows of the table
  int B, T, Hq, Hk;
  int iters;                   // groups of four heads per warp (set by the launcher)
  uint32_t* status;
};

// Attention over packed sequences, and over a shared prefix plus own keys.
// Rows are (token, query head of a kv head's group) pairs.
struct PackedAttnParams {
  const __nv_bfloat16* q;      // q[row, head, :], row = packed token or request
  int64_t q_st, q_sh;
  const __nv_bfloat16* k;      // packed: k[token, head, :]; own keys: k[request, head, slot, :]
  const __nv_bfloat16* v;
  int64_t kv_sb, kv_st, kv_sh;
  __nv_bfloat16* o;            // o[row, head, :]
  int64_t o_st, o_sh;
  float* lse;                  // lse[row * lse_st + head * lse_sh], may be null
  int64_t lse_st, lse_sh;
  int Hq, Hkv;
  int G;                       // query heads per kv head
  int Gs, n_gs;                // heads per slice of the group, slices
  float scale_log2;            // softmax scale * log2(e)
  // packed sequences
  const int* cu_q;
  const int* cu_k;
  int n_seqs, total_q, total_k, causal;
  // packed sequences with a plan (attn_plan.cu)
  const int* header;
  const int4* list;
  // shared prefix / own keys
  const __nv_bfloat16* kp;     // prefix[head, key, :]
  const __nv_bfloat16* vp;
  int64_t kp_sh, kp_st;
  int B, P, cap;
  const int* lens;             // own keys of each request, may be null (all cap)
  int prefix_splits, prefix_keys, prefix_blocks;  // parts of the prefix, keys of a part
  int own_splits, own_keys;
  float* part_o;               // [parts][B * Hq][128]
  float* part_lse;             // [parts][B * Hq] log2-sum-exp
  uint32_t* status;
};

// How a packed batch is cut into items, and where the item list, the parts of rows whose keys are cut and what joins
// them lie in the scratch memory (attn_plan.cu).
struct PackedPlan {
  int n_gs, Gs, nh;      // slices of a kv head's group, heads of a slice, kv heads x slices
  int tok_tile;          // tokens per item
  int workers;           // CTAs (or pairs) that share the work
  int split;             // items may be cut along their keys
  int max_list, max_parts;
  int64_t part_rows;
  size_t at_seq, at_list, at_groups, at_part_o, at_part_lse, total;
  int* header;           // [0] list entries, [1] groups of parts
  int* seq_tiles;        // [n_seqs + 1] tiles before each sequence
  int4* list;            // {q0, nq, k0, kb}, {ke, lim0, first part row or -1, 0}, heavy ones first
  int4* groups;          // {q0, nq, parts, first part row}
  float* part_o;         // [part_rows][128] normalised
  float* part_lse;       // [part_rows] log2-sum-exp
};
PackedPlan packed_plan(int n_seqs, int total_q, int max_k, int Hkv, int G, int Gs, int tok_tile, int workers);
int launch_plan(const PackedAttnParams& a, PackedPlan& w, void* workspace, cudaStream_t stream);
int launch_join(const PackedAttnParams& a, const PackedPlan& w, cudaStream_t stream);

// attn_pair.cu: the tcgen05 form for many rows.
PackedPlan attn_pair_plan(int n_seqs, int total_q, int max_k, int Hq, int Hkv);
int launch_attn_pair_varlen(const PackedAttnParams& a, const PackedPlan& w, cudaStream_t stream);
// Parts of a shared prefix: `cap` own slots per request follow, whose kernel runs beside this one on the SMs left free.
int attn_pair_prefix_splits(int B, int Hq, int Hkv, int P, int cap, int* keys_per_split);
int launch_attn_pair_prefix(const PackedAttnParams& a, cudaStream_t stream);

// Lets `kern` use `bytes` of dynamic shared memory, asked of the runtime once per device.
template <class... Params>
cudaError_t allow_smem(void (*kern)(Params...), int bytes, std::atomic<uint64_t>& devices) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (devices.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) devices.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Launch that may start while the kernel before it in the stream still runs (that kernel lets it, and it waits itself
// before it reads what the other writes).
template <class... Params, class... Args>
cudaError_t launch_after(void (*kern)(Params...), dim3 grid, int threads, size_t smem, bool dependent,
                         cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// Device status word used by kernels to report bounded-wait timeouts; one per
// device, allocated lazily.
uint32_t* device_status_word();
int num_sms_current_device();

}  // namespace fmka
