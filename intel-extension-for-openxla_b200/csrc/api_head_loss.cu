// Losses at the vocabulary head: softmax cross entropy against labels, and distillation from a teacher's top logits, with
// their gradients.  The tensor-core kernel that makes the logits is in head_loss_sm100.cu; here are the entry points and
// the short kernels around it.
//
//   forward    [lists: a row's teacher entries sorted, their softmax]   (distillation)
//              [gather: rows with a target side by side]                 (more than one row block)
//              statistics of every row's logits -> loss: partials to lse and loss
//   backward   [lists], gather, then per piece of the vocabulary: G = dloss/dlogits in 16 bits, dw = G^T x and dx += G w (the
//              framework's GEMM kernels, both in one launch; fp32 accumulator across the pieces), [dbias = sums of G]; scatter: dx to its rows
//
// Rows without a target cost nothing beyond the gather's copy: their number is known on the GPU only, and the kernels take
// their row count from there.  Their hidden states are never multiplied, so nothing that they hold reaches a result.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "gemm_sm100.h"
#include "head_loss.h"
#include "head_pieces.h"
#include "ptx.cuh"

namespace ixk {
namespace head {

namespace {

constexpr int kMaxEntries = 256;
constexpr size_t kSplitBytes = size_t(64) << 20;   // of the GEMMs' K chunks, for few rows
constexpr size_t kPlaneBytes = size_t(128) << 20;  // of dx's planes, for more
constexpr int kMaxPlanes = 16;
constexpr int64_t kPitchUnit = 64;               // rows of whole 128-byte lines: a box that straddles lines reads one more of each
constexpr int kSlabRows = 64;                    // rows that the product along the rows reads at a time
constexpr float kLn2 = 0.6931471805599453f, kLog2E = 1.4426950408889634f;

template <bool kBf16>
__device__ __forceinline__ float from16(uint32_t bits) {
  if constexpr (kBf16) return __uint_as_float(bits << 16);
  else return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t to16(float f) {
  if constexpr (kBf16) return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  else return __half_as_ushort(__float2half_rn(f));
}

// ------------------------------------------------------------------------------------------------ lists

struct Lists {
  const void *index, *teacher;
  int64_t index_stride, teacher_stride;
  int wide, teacher_dtype, rows, entries, vocab;
  float inv_temperature;
  int* column;       // [rows][entries] ascending
  float* weight;
  uint16_t* start;   // [rows][starts]: the first entry at or behind column i * kStartUnit
  int starts;
  int* has;          // [rows]: any entry
};

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dtype) {
  if (dtype == IXK_F32) return static_cast<const float*>(p)[i];
  if (dtype == IXK_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

constexpr int kListWarps = 4;

// 4096 rows of 64 entries: 11 us, the latency of a row's chain (reads, softmax, ranks) four rows a CTA.
// One warp per row: softmax over the entries that are there (index inside the vocabulary, logit above -inf), and their
// ranks by index, ties by position, as their places in the list.  kListPer entries a lane.
template <int kListPer>
__global__ void __launch_bounds__(32 * kListWarps) lists_kernel(const Lists a) {
  __shared__ int columns[kListWarps][32 * kListPer], sorted[kListWarps][32 * kListPer];
  ptx::grid_dependency_sync();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kListWarps + warp; row < a.rows; row += static_cast<int64_t>(gridDim.x) * kListWarps) {
    int col[kListPer];
    float t[kListPer];
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < kListPer; ++e) {
      const int k = lane + 32 * e;
      col[e] = kNoColumn;
      t[e] = -INFINITY;
      if (k < a.entries) {
        const int64_t at = row * a.index_stride + k;
        const int64_t c = a.wide ? static_cast<const int64_t*>(a.index)[at] : static_cast<const int*>(a.index)[at];
        const float logit = load_as_float(a.teacher, row * a.teacher_stride + k, a.teacher_dtype);
        if (c >= 0 && c < a.vocab && logit != -INFINITY) {
          col[e] = static_cast<int>(c);
          t[e] = logit;
          top = fmaxf(top, logit);
        }
        columns[warp][k] = col[e];
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kListPer; ++e) {
      t[e] = col[e] != kNoColumn ? expf((t[e] - top) * a.inv_temperature) : 0.0f;   // (a logit over T may be infinite)
      sum += t[e];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const bool any = __any_sync(0xffffffffu, [&] {
      bool here = false;
#pragma unroll
      for (int e = 0; e < kListPer; ++e) here |= col[e] != kNoColumn;
      return here;
    }());
    __syncwarp();
    int rank[kListPer];
#pragma unroll
    for (int e = 0; e < kListPer; ++e) rank[e] = 0;
    for (int k = 0; k < a.entries; ++k) {
      const int c = columns[warp][k];
#pragma unroll
      for (int e = 0; e < kListPer; ++e) rank[e] += c < col[e] || (c == col[e] && k < lane + 32 * e);
    }
#pragma unroll
    for (int e = 0; e < kListPer; ++e) {
      if (lane + 32 * e < a.entries) {
        a.column[row * a.entries + rank[e]] = col[e];
        sorted[warp][rank[e]] = col[e];
        a.weight[row * a.entries + rank[e]] = col[e] != kNoColumn ? t[e] / sum : 0.0f;
      }
    }
    if (lane == 0) a.has[row] = any ? 1 : 0;
    __syncwarp();
    // entry k is the first of the units behind the one before it, up to its own; behind the last entry there is none
    for (int k = lane; k <= a.entries; k += 32) {
      const int from = k == 0 ? 0 : min(sorted[warp][k - 1] / kStartUnit + 1, a.starts);
      const int to = k == a.entries ? a.starts : min(sorted[warp][k] / kStartUnit + 1, a.starts);
      for (int i = from; i < to; ++i) a.start[row * a.starts + i] = static_cast<uint16_t>(k);
    }
    __syncwarp();
  }
}

// ------------------------------------------------------------------------------------------------ gather

struct HasTarget {
  const void* labels;
  const int* has;
  int wide, vocab;
  int64_t ignore_index;
  __device__ __forceinline__ bool counts(int64_t l) const { return l != ignore_index && l >= 0 && l < vocab; }
  __device__ __forceinline__ bool operator()(int64_t row) const {
    if (labels == nullptr) return has[row] != 0;
    return counts(wide ? static_cast<const int64_t*>(labels)[row] : static_cast<const int*>(labels)[row]);
  }
  __device__ __forceinline__ int label(int64_t row) const {      // of a row that has one
    return wide ? static_cast<int>(static_cast<const int64_t*>(labels)[row]) : static_cast<const int*>(labels)[row];
  }
};

// Numbers that the GPU finds out and later kernels read.
struct Control {
  int active;          // rows with a target
  int plane_slabs;     // slabs of the vocabulary's piece per plane of dx (gemm::two_plan), and the planes
  int planes;
  int pad;
  float range[2];      // what G is multiplied by, and the inverse
};

struct Gather {
  HasTarget has;
  const uint16_t* x;
  uint16_t* packed;            // the rows with a target, pitch ldp
  int64_t ldx, ldp;
  int rows, hidden, rows_per_cta;
  Control* control;
  RowInfo* info;
  int* inverse;                // may be nullptr
  float *loss, *lse;           // zeroed where there is no target; may be nullptr
  // backward: G is made of grad_loss over its largest size in the batch.  With equal grad_loss, a mean, a label's entry is then
  // p - 1, which 16 bits hold well where p is small, and not (p - 1) / tokens, whose rounding error every row shares (3.9e-3 of
  // the gradient in the worst case); times `top` (fp16: 2^13), as G = g (p - q) with g = 1 / tokens and p = 1 / vocabulary
  // would be lost below fp16's smallest numbers.
  const float *lse_in, *grad_loss;
  int64_t grad_stride;
  float factor;
  float top;                   // 0: forward
  // labels apart: the label's p - 1, from its fp32 logit and lse.  What the products over all of K lose of a logit of 15 is 6e-5, as
  // much as 1 - p of a token that the model is sure of.
  float* gap;
  const uint16_t *w, *bias;
  int64_t ldw;
  int w_column_major;
  float scale;
  // and the products' plan: tiles of a row block of dx, of dw; slabs of a piece
  int dx_tiles_n, piece_slabs, dw_tiles, pairs, max_planes;
};

// The label's logit of a row, scale (x . w[label] + bias[label]) in fp32, is made by a CTA of the loss kernel that has kShares warps
// for it, and again by one warp of the gather in front of the gradient.  Both add up in the same order, so that what the sum's
// rounding does to the logit is in lse as well and p - 1 does not see it: share i takes every kShares-th group of 32 vectors (w
// row-major) or elements, the lanes' sums meet in a butterfly, the shares' in ascending order.
template <bool kBf16>
__device__ __forceinline__ float dot_vec(const uint4& p, const uint4& q, float t) {
  const uint32_t pw[4] = {p.x, p.y, p.z, p.w}, qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    t = fmaf(from16<kBf16>(pw[j] & 0xffffu), from16<kBf16>(qw[j] & 0xffffu), t);
    t = fmaf(from16<kBf16>(pw[j] >> 16), from16<kBf16>(qw[j] >> 16), t);
  }
  return t;
}
// call(rows, threads of a CTA of the loss kernel): rows side by side are one read of up to 256 bytes; few rows want a CTA each.
// Hidden 2048, vocabulary 32000, 1, 8 and 32 rows a CTA, us with what is left of the kernel before it: 300 rows 59, 61, 63; 700 rows
// 27, 28, 34; 3000 rows 44, 36, 39; 4096 rows 54, 42, 43; 8192 rows 90, 69, 53.
template <typename Call>
int loss_shape(int64_t rows, const Call& call) {
  using std::integral_constant;
  if (rows >= 4096) return call(integral_constant<int, 32>{}, integral_constant<int, 1024>{});
  if (rows >= 512) return call(integral_constant<int, 8>{}, integral_constant<int, 1024>{});
  return call(integral_constant<int, 1>{}, integral_constant<int, 256>{});
}

// 2048 x 4096: 8 us, 34 MB moved, and 51 where the labels' logits are wanted; every CTA first counts the rows with a target in
// front of its own, which saves a launch.
constexpr int kGatherThreads = 256;
constexpr int kCopyVecs = 8, kCountAtOnce = 8;

// kShares: of the label's logit, 0: it is not wanted.
template <bool kBf16, int kShares>
__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const Gather a) {
  __shared__ int warp_count[kGatherThreads / 32];
  __shared__ int source[kGatherThreads];
  __shared__ float warp_top[kGatherThreads / 32];
  ptx::grid_dependency_sync();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x * a.rows_per_cta, end = min(first + a.rows_per_cta, a.rows);
  auto block_sum = [&](int v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) warp_count[warp] = v;
    __syncthreads();
    int t = 0;
    for (int w = 0; w < kGatherThreads / 32; ++w) t += warp_count[w];
    return t;
  };
  // every CTA counts the rows in front of its own
  int before = 0;
  float largest = 0.0f;        // (the last CTA: of grad_loss)
  const bool ranges = a.top > 0.0f && end == a.rows;
  auto count = [&](const auto* targets, auto none, auto test) {
    for (int i0 = threadIdx.x; i0 < first; i0 += kCountAtOnce * kGatherThreads) {
      decltype(none) t[kCountAtOnce];      // (all loads out before the first test)
      float g[kCountAtOnce];
#pragma unroll
      for (int j = 0; j < kCountAtOnce; ++j) {
        const int i = i0 + j * kGatherThreads;
        t[j] = i < first ? targets[i] : none;
        g[j] = ranges && i < first ? a.grad_loss[i * a.grad_stride] : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < kCountAtOnce; ++j) {
        if (test(t[j])) {
          ++before;
          largest = fmaxf(largest, fabsf(g[j] * a.factor));
        }
      }
    }
  };
  const auto is_label = [&](int64_t l) { return a.has.counts(l); };
  if (a.has.labels == nullptr) count(a.has.has, 0, [](int h) { return h != 0; });
  else if (a.has.wide) count(static_cast<const int64_t*>(a.has.labels), int64_t(-1), is_label);
  else count(static_cast<const int*>(a.has.labels), -1, is_label);
  before = block_sum(before);
  const int whole = a.hidden / 8;
  for (int from = first; from < end; from += kGatherThreads) {      // (a row a thread; block_sum's barriers part the rounds)
    const int row = from + threadIdx.x;
    const bool mine = row < end;
    const bool keep = mine && a.has(row);
    const unsigned ballot = __ballot_sync(0xffffffffu, keep);
    const int here = block_sum(lane == 0 ? __popc(ballot) : 0);
    if (mine) {
      int at = __popc(ballot & ((1u << lane) - 1u));
      for (int w = 0; w < warp; ++w) at += warp_count[w];
      if (keep) {
        source[at] = row;
        RowInfo info{row, kNoColumn, 0.0f, 0.0f};
        if (a.has.labels != nullptr) info.label = a.has.label(row);
        if (a.grad_loss != nullptr) {
          info.lse2 = a.lse_in[row] * kLog2E;
          info.coef = a.grad_loss[row * a.grad_stride] * a.factor;
          largest = fmaxf(largest, fabsf(info.coef));
        }
        a.info[before + at] = info;
      } else if (a.loss != nullptr) {
        a.loss[row] = 0.0f;
        a.lse[row] = 0.0f;
      }
      if (a.inverse != nullptr) a.inverse[row] = keep ? before + at : -1;
    }
    __syncthreads();
    for (int i = warp; i < here; i += kGatherThreads / 32) {
      const uint16_t* src = a.x + source[i] * a.ldx;
      uint16_t* dst = a.packed + (before + i) * a.ldp;
      constexpr bool kLogit = kShares > 0;
      const int label = kLogit ? a.has.label(source[i]) : 0;
      // (with more than kDirectRows rows, a column-major weight's labels are not apart)
      constexpr bool kByColumn = kShares == 8;
      const bool by_row = kLogit && !(kByColumn && a.w_column_major);
      const uint16_t* of_label = !kLogit ? nullptr : by_row ? a.w + label * a.ldw : a.w + label;
      float share[kLogit ? kShares : 1] = {};
      float lse = 0.0f, bias = 0.0f;
      if constexpr (kLogit) {
        lse = a.lse_in[source[i]];
        if (a.bias != nullptr) bias = from16<kBf16>(a.bias[label]);
        static_assert(kCopyVecs % kShares == 0, "a lane's vectors belong to the shares in turn");
        if (kByColumn && !by_row) {
          constexpr int kAtOnce = 16;
          for (int c0 = lane; c0 < a.hidden; c0 += 32 * kAtOnce) {
            uint16_t p[kAtOnce], q[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
              const int c = c0 + 32 * j;
              p[j] = c < a.hidden ? src[c] : 0;
              q[j] = c < a.hidden ? of_label[c * a.ldw] : 0;
            }
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
              if (c0 + 32 * j < a.hidden) share[j % kShares] = fmaf(from16<kBf16>(p[j]), from16<kBf16>(q[j]), share[j % kShares]);
          }
        }
      }
      for (int v0 = lane; v0 < whole; v0 += 32 * kCopyVecs) {
        uint4 w[kCopyVecs], q[kLogit ? kCopyVecs : 1];      // (all loads out before the first store)
#pragma unroll
        for (int j = 0; j < kCopyVecs; ++j) {
          if (v0 + 32 * j < whole) {
            w[j] = reinterpret_cast<const uint4*>(src)[v0 + 32 * j];
            if constexpr (kLogit)
              if (by_row) q[j] = reinterpret_cast<const uint4*>(of_label)[v0 + 32 * j];
          }
        }
#pragma unroll
        for (int j = 0; j < kCopyVecs; ++j) {
          if (v0 + 32 * j < whole) {
            reinterpret_cast<uint4*>(dst)[v0 + 32 * j] = w[j];
            if constexpr (kLogit)
              if (by_row) share[j % kShares] = dot_vec<kBf16>(w[j], q[j], share[j % kShares]);
          }
        }
      }
      for (int c = whole * 8 + lane; c < a.hidden; c += 32) {
        dst[c] = src[c];
        if constexpr (kLogit)
          if (by_row) share[0] = fmaf(from16<kBf16>(src[c]), from16<kBf16>(of_label[c]), share[0]);
      }
      if constexpr (kLogit) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
          for (int j = 0; j < kShares; ++j) share[j] += __shfl_xor_sync(0xffffffffu, share[j], o);
        }
        share[0] += bias;
        float own = 0.0f;
#pragma unroll
        for (int j = 0; j < kShares; ++j) own += share[j];
        own *= a.scale;
        // (no probability is above 1, however lse was rounded; NaN stays)
        const float gap = expm1f(own - lse);
        if (lane == 0) a.gap[before + i] = gap > 0.0f ? 0.0f : gap;
      }
    }
    before += here;
  }
  if (end != a.rows) return;
  // the last CTA: how many there are, zeros behind them as far as the products read, and the gradient's range
  const int total = before;
  if (threadIdx.x == 0) a.control->active = total;
  if (warp == 0 && a.dx_tiles_n > 0) {
    const int64_t tiles = (static_cast<int64_t>(total) + gemm::kTwoTile - 1) / gemm::kTwoTile * a.dx_tiles_n;
    const int slabs = gemm::two_plan(tiles, a.piece_slabs, a.dw_tiles, max((total + kSlabRows - 1) / kSlabRows, 1), a.pairs, a.max_planes);
    if (lane == 0) {
      a.control->plane_slabs = slabs;
      a.control->planes = (a.piece_slabs + slabs - 1) / slabs;
    }
  }
  const int zero_end = a.rows <= kDirectRows ? a.rows : min((total + kSlabRows - 1) / kSlabRows * kSlabRows, a.rows);
  for (int i = total + warp; i < zero_end; i += kGatherThreads / 32)
    for (int c = lane; c < a.hidden; c += 32) a.packed[i * a.ldp + c] = 0;
  if (ranges) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    if (lane == 0) warp_top[warp] = largest;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 0; w < kGatherThreads / 32; ++w) largest = fmaxf(largest, warp_top[w]);
      const bool fit = largest >= 0x1p-100f && largest <= 0x1p100f;      // (both quotients are finite)
      a.control->range[0] = fit ? a.top / largest : 1.0f;
      a.control->range[1] = fit ? largest / a.top : 1.0f;
    }
  }
}

// ------------------------------------------------------------------------------------------------ loss

struct Loss {
  HasTarget has;               // (without a gather)
  const float2* partial;       // [slots][rows]
  const float* at_target;      // [batch rows][entries]
  const float* weight;         // [batch rows][entries]; nullptr: one label of weight 1
  const int* active;           // nullptr: all rows, in place
  const RowInfo* info;
  int rows, slots, entries;
  float factor;
  float *loss, *lse;
  // labels apart: the label's logit, scale (x . w[label] + bias[label]), is made here (and left out of the partials)
  int apart;
  const uint16_t *x, *w, *bias;
  int64_t ldx, ldw;
  int hidden, w_column_major;
  float scale;
};


// A lane's share of x . w[label]: every step-th vector from `first` on (w row-major), or element.
template <bool kBf16>
__device__ __forceinline__ float dot_share(const Loss& a, int64_t row, int label, int first, int step) {
  const uint16_t* x = a.x + row * a.ldx;
  float t = 0.0f;
  if (a.w_column_major) {
    const uint16_t* w = a.w + label;
#pragma unroll 8
    for (int c = first; c < a.hidden; c += step) t = fmaf(from16<kBf16>(x[c]), from16<kBf16>(w[c * a.ldw]), t);
    return t;
  }
  const uint16_t* w = a.w + label * a.ldw;
  const int whole = a.hidden / 8;
#pragma unroll 4
  for (int v = first; v < whole; v += step) t = dot_vec<kBf16>(reinterpret_cast<const uint4*>(x)[v], reinterpret_cast<const uint4*>(w)[v], t);
  for (int c = whole * 8 + first; c < a.hidden; c += step) t = fmaf(from16<kBf16>(x[c]), from16<kBf16>(w[c]), t);
  return t;
}

// kRows rows per CTA, side by side in memory; their partials dealt out over the remaining threads, their labels' logits over
// the warps.  2048 rows of 4096: 13 us, of which the labels' rows of w (17 MB here and there) are half.  The loss of a label apart
// and largest is ln(1 + the others' share): lse - logit would have nothing left of a loss below 1e-6.
template <int kRows, int kThreads, bool kBf16>
__global__ void __launch_bounds__(kThreads) loss_kernel(const Loss a) {
  constexpr int kParts = kThreads / kRows;
  __shared__ float2 stat[kParts][kRows];
  __shared__ float row_lse[kRows], share[kParts][kRows], logit[kThreads / 32 / kRows][kRows];
  ptx::grid_dependency_sync();
  const int active_rows = a.active != nullptr ? *a.active : a.rows;
  if (a.apart) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wr = warp % kRows, wrow = blockIdx.x * kRows + wr;
    constexpr int kShares = kThreads / 32 / kRows;
    int label = kNoColumn;
    if (wrow < active_rows) {
      if (a.info != nullptr) label = a.info[wrow].label;
      else if (a.has(wrow)) label = a.has.label(wrow);
    }
    float t = label != kNoColumn ? dot_share<kBf16>(a, wrow, label, warp / kRows * 32 + lane, kShares * 32) : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) logit[warp / kRows][wr] = warp < kRows && a.bias != nullptr && label != kNoColumn ? t + from16<kBf16>(a.bias[label]) : t;
  }
  const int r = threadIdx.x % kRows, part = threadIdx.x / kRows;
  const int row = blockIdx.x * kRows + r;
  const bool there = row < active_rows;
  const int64_t orig = !there ? 0 : a.info != nullptr ? a.info[row].row : row;
  auto join = [](float2 p, float2 q) {
    const float top = fmaxf(p.x, q.x);
    return make_float2(top, p.y * exp2f(p.x - top) + q.y * exp2f(q.x - top));
  };
  float2 s = make_float2(-FLT_MAX, 0.0f);
  if (there) {
#pragma unroll 8
    for (int i = part; i < a.slots; i += kParts) s = join(s, a.partial[static_cast<int64_t>(i) * a.rows + row]);
  }
  stat[part][r] = s;
  __syncthreads();
  for (int n = kParts / 2; n > 0; n /= 2) {
    if (part < n) stat[part][r] = join(stat[part][r], stat[part + n][r]);
    __syncthreads();
  }
  float of_label = 0.0f;      // labels apart: the loss
  if (part == 0) {
    float2 all = stat[0][r];
    if (a.apart) {
      float own = 0.0f;       // the label's logit
#pragma unroll
      for (int i = 0; i < kThreads / 32 / kRows; ++i) own += logit[i][r];
      own *= a.scale;
      const float t2 = own * kLog2E;
      if (t2 < INFINITY && all.x <= t2) {
        // at least as large as all others: ln(1 + their sum over its exponential), as small as it may be
        of_label = log1pf(all.y * exp2f(all.x - t2));
        row_lse[r] = own + of_label;
      } else {
        // (an infinite logit has to make the sum infinite, not undefined)
        all = t2 == INFINITY ? make_float2(FLT_MAX, INFINITY) : t2 == -INFINITY ? all : join(all, make_float2(t2, 1.0f));
        const float lse = fmaf(all.x, kLn2, logf(all.y));
        of_label = lse - own;
        row_lse[r] = lse;
      }
    } else {
      row_lse[r] = fmaf(all.x, kLn2, logf(all.y));
    }
  }
  __syncthreads();
  const float lse = row_lse[r];
  float t = 0.0f;
  if (a.apart) {
    t = of_label;
  } else if (there) {
    for (int k = part; k < a.entries; k += kParts) {
      const float q = a.weight != nullptr ? a.weight[orig * a.entries + k] : 1.0f;
      if (q != 0.0f) t += q * (logf(q) + (lse - a.at_target[orig * a.entries + k]));   // (0 ln 0 = 0; NaN goes on)
    }
  }
  share[part][r] = t;
  __syncthreads();
  for (int n = kParts / 2; n > 0; n /= 2) {
    if (part < n) share[part][r] += share[part + n][r];
    __syncthreads();
  }
  if (part == 0 && there) {
    const bool counts = a.active != nullptr || a.has(orig);
    // (lse - logit of a label that is all there is may come out below 0 by a rounding; a divergence from entries that appear
    // twice is below 0 by its definition)
    const float sum = a.weight == nullptr && share[0][r] < 0.0f ? 0.0f : share[0][r];
    a.loss[orig] = counts ? sum * a.factor : 0.0f;
    a.lse[orig] = counts ? lse : 0.0f;
  }
}

// ------------------------------------------------------------------------------------------------ behind the products

// dbias of a piece: the sums of G's columns, as they were rounded for the products, another read of G (2048 x 51200: 45 us, 4.7 TB/s; the products before it leave
// little of a large G in L2, and the kernel that makes G has a row a thread).  256 columns per CTA, kGroups warps that take rows in turn; where the columns alone
// leave SMs idle the rows are dealt out to gridDim.y CTAs, which leave partial sums for bias_sum_kernel.
constexpr int kFewGroups = 4;
constexpr int64_t kFewBiasRows = 32;      // 5 x 176783: 6.9 us with 32 warps, 4.3 with four; 76 x 99763: 7.7 and 13
template <bool kBf16, int kGroups>
__global__ void __launch_bounds__(32 * kGroups) bias_kernel(const uint16_t* g, int64_t ldg, const Control* control, int count, float* partial,
                                                              uint16_t* out) {
  __shared__ float sums[kGroups][kBiasCols];
  ptx::grid_dependency_sync();
  const int group = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = control->active;
  const int c0 = blockIdx.x * kBiasCols + lane * 8;
  float t[8] = {};
  if (c0 < count) {      // (G's pitch is whole vectors)
    const uint16_t* p = g + c0;
#pragma unroll 8
    for (int row = blockIdx.y * kGroups + group; row < rows; row += gridDim.y * kGroups) {
      const uint4 w = *reinterpret_cast<const uint4*>(p + row * ldg);
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t[2 * j] += from16<kBf16>(words[j] & 0xffffu);
        t[2 * j + 1] += from16<kBf16>(words[j] >> 16);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[group][lane * 8 + j] = t[j];
  __syncthreads();
  for (int col = threadIdx.x; col < kBiasCols; col += 32 * kGroups) {
    const int c = blockIdx.x * kBiasCols + col;
    if (c >= count) return;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) s += sums[i][col];
    if (gridDim.y > 1) partial[static_cast<int64_t>(blockIdx.y) * count + c] = s;
    else out[c] = static_cast<uint16_t>(to16<kBf16>(s * control->range[1]));
  }
}
template <bool kBf16>
__global__ void __launch_bounds__(128) bias_sum_kernel(const float* partial, int parts, const Control* control, int count, uint16_t* out) {
  ptx::grid_dependency_sync();
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= count) return;
  float s = 0.0f;
#pragma unroll 8
  for (int i = 0; i < parts; ++i) s += partial[static_cast<int64_t>(i) * count + c];
  out[c] = static_cast<uint16_t>(to16<kBf16>(s * control->range[1]));
}

// dx: the accumulator's rows, their planes added up, back to where they came from, rounded once; zeros where there was no
// target.  `width` threads a row.  2048 x 4096: 11 us.
template <bool kBf16>
__global__ void __launch_bounds__(256) scatter_kernel(const float* acc, int64_t ld_acc, int64_t plane, const int* inverse, const Control* control,
                                                      int rows, int hidden, int vec, int width, uint16_t* dx, int64_t ld) {
  ptx::grid_dependency_sync();
  const int in = threadIdx.x / width, thread = threadIdx.x % width, per_cta = blockDim.x / width;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * per_cta + in;
  if (in >= per_cta || row >= rows) return;
  const int from = inverse[row], planes = control->planes;
  const float scale = control->range[1];
  const float* src = acc + from * ld_acc;
  uint16_t* dst = dx + row * ld;
  const int vecs = vec ? hidden / 8 : 0;
  for (int v = thread; v < vecs; v += width) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (from >= 0) {
      float4 a = reinterpret_cast<const float4*>(src)[2 * v], b = reinterpret_cast<const float4*>(src)[2 * v + 1];
#pragma unroll 8
      for (int i = 1; i < planes; ++i) {
        const float4 c = reinterpret_cast<const float4*>(src + i * plane)[2 * v], d = reinterpret_cast<const float4*>(src + i * plane)[2 * v + 1];
        a = make_float4(a.x + c.x, a.y + c.y, a.z + c.z, a.w + c.w);
        b = make_float4(b.x + d.x, b.y + d.y, b.z + d.z, b.w + d.w);
      }
      w.x = to16<kBf16>(a.x * scale) | to16<kBf16>(a.y * scale) << 16;
      w.y = to16<kBf16>(a.z * scale) | to16<kBf16>(a.w * scale) << 16;
      w.z = to16<kBf16>(b.x * scale) | to16<kBf16>(b.y * scale) << 16;
      w.w = to16<kBf16>(b.z * scale) | to16<kBf16>(b.w * scale) << 16;
    }
    reinterpret_cast<uint4*>(dst)[v] = w;
  }
  for (int c = vecs * 8 + thread; c < hidden; c += width) {
    float t = 0.0f;
    if (from >= 0) {
#pragma unroll 8
      for (int i = 0; i < planes; ++i) t += src[i * plane + c];
    }
    dst[c] = static_cast<uint16_t>(to16<kBf16>(t * scale));
  }
}

// The same for few rows in many planes: 256 columns per CTA, eight groups of threads that take planes in turn.
constexpr int kFewCols = 256, kFewPlaneGroups = 8;
template <bool kBf16>
__global__ void __launch_bounds__(32 * kFewPlaneGroups) scatter_few_kernel(const float* acc, int64_t ld_acc, int64_t plane, int planes, const int* inverse,
                                                                         const Control* control, int hidden, uint16_t* dx, int64_t ld) {
  __shared__ float sums[kFewPlaneGroups][kFewCols];
  ptx::grid_dependency_sync();
  const int64_t row = blockIdx.x;
  const int from = inverse[row], lane = threadIdx.x & 31, group = threadIdx.x >> 5, c0 = blockIdx.y * kFewCols;
  if (from >= 0) {
    const float* src = acc + from * ld_acc + c0;
    float t[8] = {};
#pragma unroll 4
    for (int i = group; i < planes; i += kFewPlaneGroups) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + lane + 32 * j < hidden) t[j] += src[i * plane + lane + 32 * j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[group][lane + 32 * j] = t[j];
  }
  __syncthreads();
  const int c = c0 + threadIdx.x;
  if (c >= hidden) return;
  float s = 0.0f;
  if (from >= 0) {
#pragma unroll
    for (int i = 0; i < kFewPlaneGroups; ++i) s += sums[i][threadIdx.x];
  }
  dx[row * ld + c] = static_cast<uint16_t>(to16<kBf16>(s * control->range[1]));
}

// ------------------------------------------------------------------------------------------------ host

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Where everything lies in the workspace.
struct Space {
  size_t total = 0;
  size_t take(size_t bytes) {
    const size_t at = total;
    total += (bytes + 255) / 256 * 256;
    return at;
  }
};

struct Layout {
  Space space;
  size_t control, info, column, weight, start, has, packed, at_target, partial;      // forward
  size_t gap, inverse, grad, bias, acc, split, split_bytes;                          // backward
  int64_t ldp, slots, ldg, ld_acc, plane;      // plane 0: dx is not cut into planes
  Pieces pieces;
  int planes;
  bool gathered;
};

// Whether the label's logit is a product of its own: one row of w each, or, column-major, a 32-byte sector an element, which
// only few rows can pay (7355 x 3520 x 8144: 270 of 1700 us).
bool labels_apart(const ixk_linear_loss_desc& d) { return d.w_order == IXK_ROW_MAJOR || d.rows <= kDirectRows; }
int64_t starts_of(int64_t vocab) { return (vocab + kStartUnit - 1) / kStartUnit; }

Layout layout_for(const ixk_linear_loss_desc& d, bool backward) {
  Layout l{};
  const int64_t N = d.rows, D = d.hidden, V = d.vocab, K = std::max<int64_t>(d.entries, 1);
  l.gathered = backward || N > kDirectRows;
  l.control = l.space.take(sizeof(Control));
  if (d.entries > 0) {
    l.column = l.space.take(4 * N * K);
    l.weight = l.space.take(4 * N * K);
    l.start = l.space.take(sizeof(uint16_t) * N * starts_of(V));
    l.has = l.space.take(4 * N);
  }
  l.ldp = round_up(D, kPitchUnit);
  if (l.gathered) {
    l.info = l.space.take(sizeof(RowInfo) * N);
    l.packed = l.space.take(2 * N * l.ldp);
  }
  if (!backward) {
    if (d.entries > 0 || !labels_apart(d)) l.at_target = l.space.take(4 * N * K);
    l.slots = stat_slots(N, V);
    l.partial = l.space.take(sizeof(float2) * l.slots * N);
    return l;
  }
  if (d.entries == 0 && labels_apart(d)) l.gap = l.space.take(4 * N);
  l.inverse = l.space.take(4 * N);
  l.pieces = pieces_for(N, V);
  l.ldg = round_up(l.pieces.columns, kPitchUnit);
  l.grad = l.space.take(2 * round_up(N, 256) * l.ldg);
  l.bias = l.space.take(4 * l.pieces.bias_partials());
  l.ld_acc = round_up(D, kPitchUnit / 2);
  if (N > kDirectRows) {
    l.plane = N * l.ld_acc;
    l.planes = static_cast<int>(std::clamp<int64_t>(kPlaneBytes / (4 * l.plane), 1, kMaxPlanes));
    l.acc = l.space.take(4 * l.plane * l.planes);
  } else if (l.pieces.count == 1) {      // (planes of the kernel for few rows: dense)
    l.ld_acc = D;
    l.plane = N * D;
    l.planes = gemm::stream_splits(N, D, V, 2, kSplitBytes);
    l.acc = l.space.take(4 * l.plane * l.planes);
  } else {
    l.acc = l.space.take(4 * N * l.ld_acc);
    l.split_bytes = std::min(gemm::problem_workspace_bytes(N, D, l.pieces.columns), kSplitBytes);
    l.split = l.space.take(l.split_bytes);
  }
  return l;
}

int check(const ixk_linear_loss_desc* d, const char* name, bool distill, bool backward, const void* x, const void* w, const void* bias,
          const void* index, const void* teacher) {
  const std::string who = std::string(name) + ": ";
  if (d == nullptr) return fail(IXK_INVALID_ARGUMENT, who + "desc is NULL");
  if (d->reserved != 0) return fail(IXK_INVALID_ARGUMENT, who + "desc.reserved must be 0");
  if (d->dtype != IXK_BF16 && d->dtype != IXK_F16) return fail(IXK_UNIMPLEMENTED, who + "dtype must be BF16 or F16");
  if (d->rows < 0 || d->hidden <= 0 || d->vocab <= 0) return fail(IXK_INVALID_ARGUMENT, who + "negative rows, or no hidden size or vocabulary");
  if (d->rows > (1 << 24) || d->hidden > (1 << 20) || d->vocab > (1 << 24))
    return fail(IXK_UNIMPLEMENTED, who + "more than 2^24 rows or columns, or a hidden size above 2^20");
  for (int order : {d->w_order, d->dw_order})
    if (order != IXK_ROW_MAJOR && order != IXK_COL_MAJOR)
      return fail(IXK_INVALID_ARGUMENT, who + "w_order and dw_order must be 0 (row-major) or 1 (column-major)");
  if (d->index_bytes != 4 && d->index_bytes != 8) return fail(IXK_INVALID_ARGUMENT, who + "index_bytes must be 4 or 8");
  if (!(d->scale > 0.0f) || !std::isfinite(d->scale))
    return fail(IXK_INVALID_ARGUMENT, who + (distill ? "temperature must be positive and finite" : "the logits' scale must be positive and finite"));
  const int64_t w_inner = d->w_order == IXK_ROW_MAJOR ? d->hidden : d->vocab, dw_inner = d->dw_order == IXK_ROW_MAJOR ? d->hidden : d->vocab;
  if (d->x_stride < d->hidden || d->w_stride < w_inner || (backward && (d->dx_stride < d->hidden || d->dw_stride < dw_inner)))
    return fail(IXK_INVALID_ARGUMENT, who + "a stride is smaller than the contiguous dimension");
  if (distill) {
    if (d->entries < 1) return fail(IXK_INVALID_ARGUMENT, who + "entries must be at least 1");
    if (d->entries > kMaxEntries) return fail(IXK_UNIMPLEMENTED, who + "more than 256 entries per row");
    if (d->teacher_dtype != IXK_BF16 && d->teacher_dtype != IXK_F16 && d->teacher_dtype != IXK_F32)
      return fail(IXK_UNIMPLEMENTED, who + "teacher_dtype must be BF16, F16 or F32");
    if (d->index_stride < d->entries || d->teacher_stride < d->entries)
      return fail(IXK_INVALID_ARGUMENT, who + "a row of entries is longer than its stride");
  } else if (d->entries != 0) {
    return fail(IXK_INVALID_ARGUMENT, who + "entries must be 0");
  }
  if (d->rows > 0 && (x == nullptr || w == nullptr || index == nullptr || (distill && teacher == nullptr)))
    return fail(IXK_INVALID_ARGUMENT, who + "a required pointer is NULL");
  if (!aligned(x, 16) || !aligned(w, 16)) return fail(IXK_INVALID_ARGUMENT, who + "x and weight must be 16-byte aligned (TMA)");
  if (d->x_stride % 8 != 0 || d->w_stride % 8 != 0)
    return fail(IXK_UNIMPLEMENTED, who + "the strides of x and weight must be multiples of 8 elements (TMA)");
  if (!aligned(bias, 2) || !aligned(index, d->index_bytes) || (distill && !aligned(teacher, d->teacher_dtype == IXK_F32 ? 4 : 2)))
    return fail(IXK_INVALID_ARGUMENT, who + "a pointer is not aligned to its element size");
  return IXK_OK;
}

int check_space(const char* name, const Layout& l, const void* workspace, size_t bytes) {
  if (workspace == nullptr || !aligned(workspace, 256) || bytes < l.space.total)
    return fail(IXK_WORKSPACE_TOO_SMALL, std::string(name) + ": need " + std::to_string(l.space.total) + " bytes of 256-byte aligned scratch");
  return IXK_OK;
}

// Logits' scale, gradient factor and loss factor: z = s (x w^T + b); cross entropy is that of softmax(z); distillation at
// temperature T is T^2 times the divergence at s = 1 / T.
struct Scales {
  float logits, grad, loss;
};
Scales scales_of(const ixk_linear_loss_desc& d, bool distill) {
  if (!distill) return Scales{d.scale, d.scale, 1.0f};
  return Scales{1.0f / d.scale, d.scale, d.scale * d.scale};
}

// The targets as the kernels take them; distillation's lists are made here.
int targets_of(const ixk_linear_loss_desc& d, const Layout& l, char* ws, const void* index, const void* teacher, cudaStream_t stream,
               Targets* t, HasTarget* has) {
  t->wide = d.index_bytes == 8;
  t->ignore_index = d.ignore_index;
  has->wide = t->wide;
  has->vocab = static_cast<int>(d.vocab);
  has->ignore_index = d.ignore_index;
  if (teacher == nullptr) {
    t->labels = has->labels = index;
    t->apart = labels_apart(d) ? 1 : 0;
    t->entries = 1;
    return IXK_OK;
  }
  t->entries = d.entries;
  Lists a{};
  a.index = index;
  a.teacher = teacher;
  a.index_stride = d.index_stride;
  a.teacher_stride = d.teacher_stride;
  a.wide = t->wide;
  a.teacher_dtype = d.teacher_dtype;
  a.rows = static_cast<int>(d.rows);
  a.entries = d.entries;
  a.vocab = static_cast<int>(d.vocab);
  a.inv_temperature = 1.0f / d.scale;
  t->column = a.column = reinterpret_cast<int*>(ws + l.column);
  t->weight = a.weight = reinterpret_cast<float*>(ws + l.weight);
  t->start = a.start = reinterpret_cast<uint16_t*>(ws + l.start);
  t->starts = a.starts = static_cast<int>(starts_of(d.vocab));
  has->has = a.has = reinterpret_cast<int*>(ws + l.has);
  const int64_t ctas = std::min<int64_t>((d.rows + kListWarps - 1) / kListWarps, 148 * 16);
  auto* fn = d.entries <= 32 ? lists_kernel<1> : d.entries <= 64 ? lists_kernel<2> : d.entries <= 128 ? lists_kernel<4> : lists_kernel<8>;
  return launch_overlapped(fn, dim3(static_cast<unsigned>(ctas)), dim3(32 * kListWarps), 0, stream, a);
}

// (w and bias: backward with labels apart, else nullptr)
int gather(const ixk_linear_loss_desc& d, const Layout& l, char* ws, const HasTarget& has, const void* x, float* loss, float* lse,
           const void* w, const void* bias, const float* lse_in, const float* grad_loss, const Scales& scales, bool want_dw, int sm_count,
           cudaStream_t stream) {
  const bool backward = loss == nullptr;
  Gather g{};
  g.has = has;
  g.x = static_cast<const uint16_t*>(x);
  g.packed = reinterpret_cast<uint16_t*>(ws + l.packed);
  g.ldx = d.x_stride;
  g.ldp = l.ldp;
  g.rows = static_cast<int>(d.rows);
  g.hidden = static_cast<int>(d.hidden);
  // (each CTA counts the rows in front of it: at most 1024 CTAs, or their number would count twice; 65536 x 256: 67 us, 153 with
  // 4096 CTAs, 58 with 256, which give back as much at 8192 x 4096)
  g.rows_per_cta = static_cast<int>(std::max<int64_t>(8, (d.rows + 1023) / 1024));
  g.control = reinterpret_cast<Control*>(ws + l.control);
  g.info = reinterpret_cast<RowInfo*>(ws + l.info);
  g.inverse = backward ? reinterpret_cast<int*>(ws + l.inverse) : nullptr;
  g.loss = loss;
  g.lse = lse;
  g.lse_in = lse_in;
  g.grad_loss = grad_loss;
  g.grad_stride = d.grad_loss_stride;
  g.factor = scales.grad;
  g.top = !backward ? 0.0f : d.dtype == IXK_F16 ? 0x1p13f : 1.0f;
  if (backward && d.rows > kDirectRows) {
    g.dx_tiles_n = static_cast<int>((d.hidden + gemm::kTwoTile - 1) / gemm::kTwoTile);
    g.piece_slabs = static_cast<int>((l.pieces.columns + kSlabRows - 1) / kSlabRows);
    g.dw_tiles = want_dw ? g.dx_tiles_n * static_cast<int>((l.pieces.columns + gemm::kTwoTile - 1) / gemm::kTwoTile) : 0;
    g.pairs = sm_count / 2;
    g.max_planes = l.planes;
  }
  const int64_t ctas = (d.rows + g.rows_per_cta - 1) / g.rows_per_cta;
  auto go = [&](auto* fn) { return launch_overlapped(fn, dim3(static_cast<unsigned>(ctas)), dim3(kGatherThreads), 0, stream, g); };
  if (w == nullptr) return go(gather_kernel<false, 0>);
  g.gap = reinterpret_cast<float*>(ws + l.gap);
  g.w = static_cast<const uint16_t*>(w);
  g.bias = static_cast<const uint16_t*>(bias);
  g.ldw = d.w_stride;
  g.w_column_major = d.w_order == IXK_COL_MAJOR ? 1 : 0;
  g.scale = scales.logits;
  return loss_shape(d.rows, [&](auto rows, auto threads) {
    constexpr int kShares = decltype(threads)::value / 32 / decltype(rows)::value;
    return go(d.dtype == IXK_BF16 ? gather_kernel<true, kShares> : gather_kernel<false, kShares>);
  });
}

Pass pass_of(const ixk_linear_loss_desc& d, const Scales& s, const void* x, int64_t ldx, const void* w, const void* bias, const Targets& t) {
  Pass p{};
  p.dtype = d.dtype;
  p.w_column_major = d.w_order == IXK_COL_MAJOR;
  p.rows = d.rows;
  p.hidden = d.hidden;
  p.vocab = d.vocab;
  p.x = x;
  p.ldx = ldx;
  p.w = w;
  p.ldw = d.w_stride;
  p.bias = bias;
  p.scale = s.logits;
  p.first = 0;
  p.count = d.vocab;
  p.targets = t;
  return p;
}

int forward(const char* name, const ixk_linear_loss_desc* d, bool distill, const void* x, const void* w, const void* bias,
            const void* index, const void* teacher, float* loss, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(d, name, distill, false, x, w, bias, index, teacher);
  if (rc != IXK_OK) return rc;
  if (d->rows > 0 && (loss == nullptr || lse == nullptr)) return fail(IXK_INVALID_ARGUMENT, std::string(name) + ": loss and lse must be non-NULL");
  if (!aligned(loss, 4) || !aligned(lse, 4)) return fail(IXK_INVALID_ARGUMENT, std::string(name) + ": loss and lse must be 4-byte aligned");
  if (d->rows == 0) return IXK_OK;
  const Layout l = layout_for(*d, false);
  if ((rc = check_space(name, l, workspace, workspace_bytes)) != IXK_OK) return rc;
  DeviceInfo dev;
  if ((rc = get_device_info(&dev)) != IXK_OK) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const Scales scales = scales_of(*d, distill);
  Targets t{};
  HasTarget has{};
  if ((rc = targets_of(*d, l, ws, index, teacher, s, &t, &has)) != IXK_OK) return rc;
  Pass p = pass_of(*d, scales, x, d->x_stride, w, bias, t);
  if (l.gathered) {
    if ((rc = gather(*d, l, ws, has, x, loss, lse, nullptr, nullptr, nullptr, nullptr, scales, false, dev.sm_count, s)) != IXK_OK) return rc;
    p.x = ws + l.packed;
    p.ldx = l.ldp;
    p.active_rows = &reinterpret_cast<const Control*>(ws + l.control)->active;
    p.info = reinterpret_cast<const RowInfo*>(ws + l.info);
  }
  p.partial = reinterpret_cast<float2*>(ws + l.partial);
  p.at_target = reinterpret_cast<float*>(ws + l.at_target);
  if ((rc = launch_stats(p, dev, s)) != IXK_OK) return rc;
  Loss a{};
  a.has = has;
  a.partial = p.partial;
  a.at_target = p.at_target;
  a.weight = t.weight;
  a.active = p.active_rows;
  a.info = p.info;
  a.rows = static_cast<int>(d->rows);
  a.slots = static_cast<int>(l.slots);
  a.entries = t.entries;
  a.factor = scales.loss;
  a.loss = loss;
  a.lse = lse;
  a.apart = t.apart;
  a.x = static_cast<const uint16_t*>(p.x);
  a.ldx = p.ldx;
  a.w = static_cast<const uint16_t*>(w);
  a.ldw = d->w_stride;
  a.w_column_major = p.w_column_major ? 1 : 0;
  a.bias = static_cast<const uint16_t*>(bias);
  a.hidden = static_cast<int>(d->hidden);
  a.scale = scales.logits;
  return loss_shape(d->rows, [&](auto rows, auto threads) -> int {
    constexpr int kRows = decltype(rows)::value, kThreads = decltype(threads)::value;
    auto* fn = d->dtype == IXK_BF16 ? loss_kernel<kRows, kThreads, true> : loss_kernel<kRows, kThreads, false>;
    return launch_overlapped(fn, dim3(static_cast<unsigned>((d->rows + kRows - 1) / kRows)), dim3(kThreads), 0, s, a);
  });
}

int backward(const char* name, const ixk_linear_loss_desc* d, bool distill, const void* x, const void* w, const void* bias,
             const void* index, const void* teacher, const float* lse, const float* grad_loss, void* dx, void* dw, void* dbias,
             void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(d, name, distill, true, x, w, bias, index, teacher);
  if (rc != IXK_OK) return rc;
  const std::string who = std::string(name) + ": ";
  if (d->rows > 0 && (lse == nullptr || grad_loss == nullptr)) return fail(IXK_INVALID_ARGUMENT, who + "lse and grad_loss must be non-NULL");
  if (dbias != nullptr && bias == nullptr) return fail(IXK_INVALID_ARGUMENT, who + "dbias without a bias");
  if (!aligned(lse, 4) || !aligned(grad_loss, 4) || !aligned(dx, 2) || !aligned(dw, 2) || !aligned(dbias, 2))
    return fail(IXK_INVALID_ARGUMENT, who + "a pointer is not aligned to its element size");
  if (d->grad_loss_stride < 0) return fail(IXK_INVALID_ARGUMENT, who + "grad_loss_stride must not be negative");
  DeviceInfo dev;
  auto s = static_cast<cudaStream_t>(stream);
  if (d->rows == 0) {      // sums over no rows
    if ((rc = get_device_info(&dev)) != IXK_OK) return rc;
    const bool row_major = d->dw_order == IXK_ROW_MAJOR;
    if (dw != nullptr)
      IXK_CUDA_OK(cudaMemset2DAsync(dw, d->dw_stride * 2, 0, (row_major ? d->hidden : d->vocab) * 2, row_major ? d->vocab : d->hidden, s));
    if (dbias != nullptr) IXK_CUDA_OK(cudaMemsetAsync(dbias, 0, d->vocab * 2, s));
    return IXK_OK;
  }
  const Layout l = layout_for(*d, true);
  if ((rc = check_space(name, l, workspace, workspace_bytes)) != IXK_OK) return rc;
  if ((rc = get_device_info(&dev)) != IXK_OK) return rc;
  char* ws = static_cast<char*>(workspace);
  const Scales scales = scales_of(*d, distill);
  const bool bf16 = d->dtype == IXK_BF16;
  Targets t{};
  HasTarget has{};
  if ((rc = targets_of(*d, l, ws, index, teacher, s, &t, &has)) != IXK_OK) return rc;
  if ((rc = gather(*d, l, ws, has, x, nullptr, nullptr, t.apart ? w : nullptr, bias, lse, grad_loss, scales, dw != nullptr, dev.sm_count, s)) != IXK_OK)
    return rc;
  if (t.apart) t.gap = reinterpret_cast<const float*>(ws + l.gap);
  Pass p = pass_of(*d, scales, ws + l.packed, l.ldp, w, bias, t);
  const Control* control = reinterpret_cast<const Control*>(ws + l.control);
  p.active_rows = &control->active;
  p.info = reinterpret_cast<const RowInfo*>(ws + l.info);
  p.range = control->range;
  p.grad = ws + l.grad;
  p.ldg = l.ldg;
  float* acc = reinterpret_cast<float*>(ws + l.acc);

  gemm::Problem common;
  common.kind = gemm::kKindF16;
  common.ab_dtype = d->dtype;
  common.a_fmt = common.b_fmt = bf16 ? 1u : 0u;
  common.bias_dtype = d->dtype;
  for (int64_t first = 0; first < d->vocab; first += l.pieces.columns) {
    p.first = first;
    p.count = l.pieces.columns_of(first);
    if ((rc = launch_grad(p, dev, s)) != IXK_OK) return rc;
    gemm::Problem both[2] = {common, common};
    if (dx != nullptr) {       // dx += G w
      gemm::Problem& g = both[0];
      g.M = d->rows;
      g.N = d->hidden;
      g.K = p.count;
      g.a = p.grad;
      g.lda = l.ldg;
      const bool row_major = d->w_order == IXK_ROW_MAJOR;
      g.b = static_cast<const uint16_t*>(w) + (row_major ? first * d->w_stride : first);
      g.ldb = d->w_stride;
      g.b_mn_major = row_major;
      g.d = acc;
      g.c = acc;
      g.ldd = g.ldc = l.ld_acc;
      g.d_batch_stride = g.c_batch_stride = l.plane;
      if (d->rows > kDirectRows) g.batch = l.planes;
      g.out_dtype = IXK_F32;
      g.beta = first == 0 ? 0.0f : 1.0f;
    }
    if (dw != nullptr) {       // dw[v, :] = sum over rows of G[row, v] x[row, :], or its transpose
      gemm::Problem& g = both[1];
      const bool row_major = d->dw_order == IXK_ROW_MAJOR;
      g.M = row_major ? p.count : d->hidden;
      g.N = row_major ? d->hidden : p.count;
      g.K = d->rows;
      g.a = row_major ? p.grad : p.x;
      g.lda = row_major ? l.ldg : l.ldp;
      g.b = row_major ? p.x : p.grad;
      g.ldb = row_major ? l.ldp : l.ldg;
      g.a_mn_major = g.b_mn_major = true;
      g.d = static_cast<uint16_t*>(dw) + (row_major ? first * d->dw_stride : first);
      g.ldd = g.ldc = d->dw_stride;
      g.out_dtype = d->dtype;
      g.acc_scale_dev = p.range + 1;
    }
    if (both[1].M > 0) both[1].k_limit = p.active_rows;
    if (d->rows <= kDirectRows && both[0].M > 0) {      // one row block: dx is a stream of the weights
      const gemm::Problem& g = both[0];
      rc = l.plane == 0 ? gemm::run_problem(g, ws + l.split, l.split_bytes, dev, s)
                        : gemm::launch_stream(g, l.planes, l.planes > 1 ? acc : nullptr, dev, s);
      if (rc != IXK_OK) return rc;
      both[0].M = 0;
    }
    if (both[0].M > 0) both[0].m_limit = p.active_rows;
    if ((rc = gemm::launch_two(both, &control->plane_slabs, dev, s)) != IXK_OK) return rc;
    if (dbias != nullptr) {
      const unsigned blocks = static_cast<unsigned>((p.count + kBiasCols - 1) / kBiasCols), parts = static_cast<unsigned>(l.pieces.bias_parts);
      float* partial = reinterpret_cast<float*>(ws + l.bias);
      auto* out = static_cast<uint16_t*>(dbias) + first;
      const bool few = d->rows <= kFewBiasRows;
      auto* fn = few ? (bf16 ? bias_kernel<true, kFewGroups> : bias_kernel<false, kFewGroups>)
                     : (bf16 ? bias_kernel<true, kBiasGroups> : bias_kernel<false, kBiasGroups>);
      rc = launch_overlapped(fn, dim3(blocks, parts), dim3(32 * (few ? kFewGroups : kBiasGroups)), 0, s,
                             static_cast<const uint16_t*>(p.grad), l.ldg, control, static_cast<int>(p.count), partial, out);
      if (rc == IXK_OK && parts > 1)
        rc = launch_overlapped(bf16 ? bias_sum_kernel<true> : bias_sum_kernel<false>, dim3(static_cast<unsigned>((p.count + 127) / 128)), dim3(128), 0, s,
                               static_cast<const float*>(partial), static_cast<int>(parts), control, static_cast<int>(p.count), out);
      if (rc != IXK_OK) return rc;
    }
  }
  if (dx == nullptr) return IXK_OK;
  const int* inverse = reinterpret_cast<const int*>(ws + l.inverse);
  if (d->rows <= kDirectRows)
    return launch_overlapped(bf16 ? scatter_few_kernel<true> : scatter_few_kernel<false>,
                             dim3(static_cast<unsigned>(d->rows), static_cast<unsigned>((d->hidden + kFewCols - 1) / kFewCols)), dim3(32 * kFewPlaneGroups), 0, s,
                             static_cast<const float*>(acc), l.ld_acc, l.plane, std::max(l.planes, 1), inverse, control, static_cast<int>(d->hidden),
                             static_cast<uint16_t*>(dx), d->dx_stride);
  const int vec = aligned(dx, 16) && d->dx_stride % 8 == 0;
  // (a row of less than one vector has a warp too, for its single elements)
  const int width = static_cast<int>(std::clamp<int64_t>(round_up(vec ? d->hidden / 8 : d->hidden, 32), 32, 256));
  return launch_overlapped(bf16 ? scatter_kernel<true> : scatter_kernel<false>, dim3(static_cast<unsigned>((d->rows + 256 / width - 1) / (256 / width))),
                           dim3(256), 0, s, static_cast<const float*>(acc), l.ld_acc, l.plane, inverse, control, static_cast<int>(d->rows),
                           static_cast<int>(d->hidden), vec, width, static_cast<uint16_t*>(dx), d->dx_stride);
}

}  // namespace
}  // namespace head
}  // namespace ixk

extern "C" {

int ixk_linear_xent_fwd(const ixk_linear_loss_desc* desc, const void* x, const void* weight, const void* bias, const void* labels,
                        float* loss, float* lse, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  IXK_API_RANGE("ixk_linear_xent_fwd");
  ixk::clear_error();
  return ixk::head::forward("linear_xent_fwd", desc, false, x, weight, bias, labels, nullptr, loss, lse, workspace, workspace_bytes, cuda_stream);
}

int ixk_linear_xent_bwd(const ixk_linear_loss_desc* desc, const void* x, const void* weight, const void* bias, const void* labels,
                        const float* lse, const float* grad_loss, void* dx, void* dweight, void* dbias, void* workspace,
                        size_t workspace_bytes, void* cuda_stream) {
  IXK_API_RANGE("ixk_linear_xent_bwd");
  ixk::clear_error();
  return ixk::head::backward("linear_xent_bwd", desc, false, x, weight, bias, labels, nullptr, lse, grad_loss, dx, dweight, dbias, workspace,
                             workspace_bytes, cuda_stream);
}

int ixk_linear_distill_fwd(const ixk_linear_loss_desc* desc, const void* x, const void* weight, const void* bias, const void* index,
                           const void* teacher, float* loss, float* lse, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  IXK_API_RANGE("ixk_linear_distill_fwd");
  ixk::clear_error();
  return ixk::head::forward("linear_distill_fwd", desc, true, x, weight, bias, index, teacher, loss, lse, workspace, workspace_bytes, cuda_stream);
}

int ixk_linear_distill_bwd(const ixk_linear_loss_desc* desc, const void* x, const void* weight, const void* bias, const void* index,
                           const void* teacher, const float* lse, const float* grad_loss, void* dx, void* dweight, void* dbias,
                           void* workspace, size_t workspace_bytes, void* cuda_stream) {
  IXK_API_RANGE("ixk_linear_distill_bwd");
  ixk::clear_error();
  return ixk::head::backward("linear_distill_bwd", desc, true, x, weight, bias, index, teacher, lse, grad_loss, dx, dweight, dbias, workspace,
                             workspace_bytes, cuda_stream);
}

size_t ixk_linear_loss_workspace_bytes(const ixk_linear_loss_desc* desc, int backward) {
  if (desc == nullptr || desc->rows <= 0 || desc->hidden <= 0 || desc->vocab <= 0 || desc->entries < 0 || desc->rows > (1 << 24) ||
      desc->hidden > (1 << 20) || desc->vocab > (1 << 24) || desc->entries > ixk::head::kMaxEntries)
    return 0;
  return ixk::head::layout_for(*desc, backward != 0).space.total;
}

}  // extern "C"
