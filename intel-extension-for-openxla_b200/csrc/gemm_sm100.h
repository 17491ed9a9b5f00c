// Interface between the GEMM entry points (validation, normalisation) and the
// tcgen05 kernel launcher.
#pragma once

#include "host_common.h"

namespace ixk {
namespace gemm {

enum : int { kActNone = 0, kActRelu = 1, kActGelu = 2 };
// tcgen05.mma kinds (the values of ptx::kKind*, restated for host-only code)
enum : int { kKindF16 = 0, kKindF8 = 1, kKindTf32 = 2, kKindI8 = 3 };
constexpr int kMaxScatter = 8;  // destinations of a scattered output (= the most ranks a communicator has)

// A GEMM after normalisation: D is row-major [M,N]; A is [M,K], B is [K,N], each with
// either dimension contiguous.
struct Problem {
  int64_t M = 0, N = 0, K = 0, batch = 1;
  bool fp8 = false;          // any operand type other than the 16-bit floats
  int kind = 0;              // tcgen05.mma kind: kKindF16 / kKindF8 / kKindTf32 / kKindI8
  int ab_dtype = IXK_BF16;   // 16-bit operand type when kind == kKindF16
  uint32_t a_fmt = 0, b_fmt = 0;  // tcgen05 operand format codes
  bool a_mn_major = false;  // A stored with M contiguous (column-major A)
  bool b_mn_major = false;  // B stored with N contiguous (row-major B)
  const void* a = nullptr;
  const void* b = nullptr;
  int64_t lda = 0, ldb = 0, a_batch_stride = 0, b_batch_stride = 0;
  bool a_broadcast = false;        // every batch reads the same A (three projections of one input)
  int64_t bias_batch_stride = 0;   // elements between the bias vectors of consecutive batches
  const void* c = nullptr;
  const void* bias = nullptr;
  void* d = nullptr;
  void* aux = nullptr;             // pre-activation values (the *_AUX epilogues); D's type and shape
  int64_t ld_aux = 0, aux_batch_stride = 0;
  int64_t ldc = 0, ldd = 0, c_batch_stride = 0, d_batch_stride = 0;
  int out_dtype = IXK_BF16;
  int bias_dtype = IXK_BF16;
  int act = kActNone;
  float acc_scale = 1.0f;
  float beta = 0.0f;
  // What only the GPU knows, nullptr: nothing.  launch_two only, the other launches refuse it: acc_scale is multiplied by
  // *acc_scale_dev; D's rows from *m_limit on are not computed; K ends at *k_limit (at most K; the operands hold zeros from there
  // to a multiple of 64).
  const int* m_limit = nullptr;
  const int* k_limit = nullptr;
  const float* acc_scale_dev = nullptr;
  bool needs_two() const { return m_limit != nullptr || k_limit != nullptr || acc_scale_dev != nullptr; }
  int force_block_n = 0;  // tuning override; 0 = heuristic
  int k_chunk = 0;        // > 0: the batches are chunks of K, this many slabs each (the last one what is left), of one A and B
  // Scattered output (row-parallel projection feeding an all-reduce): row block o of D, rows
  // [o * M / scatter_world, (o + 1) * M / scatter_world), is stored dense ([M / world, N], pitch N)
  // at scatter_dest[o], which may be another GPU's memory.  0 = D goes to `d` as usual.
  int scatter_world = 0;
  void* scatter_dest[kMaxScatter] = {};
};

// Kernel parameter block (passed by value).
struct KernelArgs {
  int M, N, K, batch;
  int tiles_m, tiles_n;
  int a_mn_major, b_mn_major;
  int k_chunk;                 // slabs of K per batch, 0: all of them (single-CTA kernel)
  uint32_t idesc;
  uint32_t idesc_tail;         // CTA-pair kernel: the narrower tiles of the last round
  int tail_from, tail_parts;   // tiles from here on are cut into this many (1: none is)
  const void* bias;
  const void* c;
  void* d;
  int64_t ldd, ldc, d_batch_stride, c_batch_stride;
  int out_dtype, bias_dtype, act;
  float acc_scale, beta;
  const int *m_limit, *k_limit;   // see Problem
  const float* acc_scale_dev;
  int d_vec_ok, c_vec_ok, bias_vec_ok;
  int d_tma;  // 16-bit D with 16-byte-aligned rows: stored through shared memory + TMA
  int a_broadcast;
  int64_t bias_batch_stride;
  void* aux;
  int64_t ld_aux, aux_batch_stride;
  int aux_vec_ok;
  int scatter_rows;  // rows per destination of a scattered output; 0 = one destination
  int* status_word;
};

// D by whichever kernel suits the problem, K cut as far as the scratch goes.
int run_problem(const Problem& p, void* workspace, size_t workspace_bytes, const DeviceInfo& dev, cudaStream_t stream);
// Scratch that run_problem can use for a 16-bit problem of one batch.
size_t problem_workspace_bytes(int64_t M, int64_t N, int64_t K);

// Two products in one launch, for the gradients of a layer whose weight is much longer one way than the other:
//   p[0]  D0 (+)= A0.B0, fp32, unscaled, few tiles and a long K: cut along K into planes (at most `batch`), d_batch_stride
//         elements apart, which the caller adds up; beta 0 or 1 with c = d; rows of whole 16-byte pieces
//   p[1]  D1 = A1.B1, many tiles and a short K
// Either may be absent (M = 0).  The pairs of CTAs that have one unit less of the long product begin with the other's tiles,
// so that all end together.  `plan` (device): the slabs of K per plane, from two_plan.  16-bit operands; p[0].m_limit and
// p[1].k_limit hold the same number.
int launch_two(const Problem (&p)[2], const int* plan, const DeviceInfo& dev, cudaStream_t stream);
constexpr int kTwoTile = 256;    // of either product

// Slabs of 64 of the long product's K per plane: as few planes as let the longest pair's share of it end with the whole, of 8
// slabs or more (at least 16: 3 of 14 to 50 us more where it matters; 4: no further gain).
// tiles and slabs: of the long product (0), of the other (1).  Called by a whole warp: a lane looks at as many planes as its
// number says, one after the other these divisions took 2 us.
__device__ inline int two_plan(int64_t tiles0, int slabs0, int64_t tiles1, int slabs1, int pairs, int max_planes) {
  const int64_t share = (tiles0 * slabs0 + tiles1 * slabs1 + pairs - 1) / pairs;
  const int s = (threadIdx.x & 31) + 1, chunk = (slabs0 + s - 1) / s, planes = (slabs0 + chunk - 1) / chunk;
  const int64_t longest = (tiles0 * planes + pairs - 1) / pairs * chunk, time = longest > share ? longest : share;
  const unsigned allowed = __ballot_sync(0xffffffffu, s <= max_planes && (s == 1 || slabs0 / s >= 8));
  int best = 0;
  int64_t best_time = __shfl_sync(0xffffffffu, time, 0);
  for (int i = 1; i < 32 && (allowed >> i & 1u) != 0 && best_time * 100 > share * 102; ++i) {
    const int64_t t = __shfl_sync(0xffffffffu, time, i);
    if (t * 100 < best_time * 97) {    // (a further plane is written, read and added up)
      best = i;
      best_time = t;
    }
  }
  return __shfl_sync(0xffffffffu, chunk, best);
}

int pick_block_n(int64_t M, int64_t N, int64_t batch, int sm_count);
int launch(const Problem& p, const DeviceInfo& dev, cudaStream_t stream);

// Split-K for skinny problems (gemm_splitk.cu): number of K chunks for a problem (1 = do not
// split; depends on the shape only, so the workspace query needs no device), the fp32 scratch it
// takes, and the two-kernel launch (partial GEMMs as a batch, then reduce + epilogue).
int split_k_factor(int64_t M, int64_t N, int64_t K, int64_t batch, bool fp8);
// The same for problems of more rows whose tiles leave most SMs idle, as far as the scratch goes.
int tiled_splits(int64_t M, int64_t N, int64_t K, int64_t batch, int elem_bytes, size_t workspace_bytes);
size_t split_k_workspace_bytes(int64_t M, int64_t N, int splits);
// (geglu: the N columns are [gate | up]; the reduce writes gelu(gate) * up, N / 2 columns, to p.d / p.ldd;
// splits may be 1 then: one GEMM into the scratch + the GeGLU pass)
int launch_split_k(const Problem& p, int splits, void* workspace, const DeviceInfo& dev, cudaStream_t stream,
                   bool geglu = false);

// Few rows: the problem as a stream of the weights (gemm_stream.cu).
bool stream_takes(int64_t M);
bool stream_applies(const Problem& p);
bool stream_alone(const Problem& p);   // also without scratch for chunks of K
int stream_splits(int64_t M, int64_t N, int64_t K, int elem_bytes, size_t workspace_bytes, bool summed = false);
int launch_stream(const Problem& p, int splits, float* partial, const DeviceInfo& dev, cudaStream_t stream);

}  // namespace gemm
}  // namespace ixk
