// Row norms for training: LayerNorm and RMSNorm with gain, gain_offset and shift, the forward pass keeping each row's
// statistics and the backward pass with the sums over the rows that gain and shift need.
//
//   xh = (x - mean) rstd          (RMS: mean = 0)        y  = xh (offset + gain) + shift
//   h  = gy (offset + gain)                              dx = rstd (h - [mean h] - xh mean(h xh))
//   dgain = sum over rows of gy xh                       dshift = sum over rows of gy
//
// Every element is read once and written once: the bound is HBM, 2 R C elements forward, 3 R C backward.
//
// A row belongs to a group of threads (a warp for short rows, a CTA else) and stays in their registers between its
// statistics and its result.  CTAs are persistent: a thread has the same columns in every row, so gain and shift are read
// once, and the columns' sums over the CTA's rows grow in its registers (fp32) instead of passing through memory.  They
// leave as one row of partials per CTA, which a second kernel adds up in a fixed order: the result does not depend on
// which CTA was faster.  The next row's loads are asked for before this row's statistics are waited for.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "host_common.h"
#include "ptx.cuh"

namespace ixk {
namespace norm {

namespace {

constexpr int kMaxThreads = 1024;
constexpr int kMaxElems = 16;             // elements of a row per thread
constexpr int64_t kMaxCols = kMaxThreads * kMaxElems;
constexpr int kAssumedSms = 148;          // (the workspace query runs without a device)
constexpr int kThreadsPerSm = 1024;       // what 64 registers a thread leave room for
constexpr int kSumCols = 32, kSumParts = 32;

// kVec elements of type T as they lie in memory.
template <typename T, int kVec>
using Raw = std::conditional_t<kVec * sizeof(T) == 16, uint4, std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>>;

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
template <typename T, int kVec>
__device__ __forceinline__ void unpack(const Raw<T, kVec>& raw, float (&f)[kVec]) {
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int j = 0; j < kVec; ++j) f[j] = to_float<T>(e[j]);
}
template <typename T, int kVec>
__device__ __forceinline__ Raw<T, kVec> pack(const float (&f)[kVec]) {
  Raw<T, kVec> raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int j = 0; j < kVec; ++j) e[j] = from_float<T>(f[j]);
  return raw;
}
__device__ __forceinline__ float load_param(const void* p, int64_t i, int dtype) {
  if (dtype == IXK_F32) return static_cast<const float*>(p)[i];
  if (dtype == IXK_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

struct Args {
  const void *x, *gain, *shift, *gy;
  void* out;                    // y or dx
  float *mean, *rstd;
  float *part_gain, *part_shift;   // [parts][cols], nullptr: not wanted
  int64_t rows, ldx, ldg, ldo;
  int cols, rms, param_dtype;
  float eps, gain_offset, inv_cols;
};

// The sums of kCount values over the row's threads, in every one of them.  kWarp: the row is a warp's; else a CTA's, and
// consecutive calls take the two halves of the scratch in turn, so that one barrier per call is enough.
template <bool kWarp, int kCount>
__device__ __forceinline__ void row_sums(float (&v)[kCount], float* scratch, int& turn) {
#pragma unroll
  for (int c = 0; c < kCount; ++c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[c] += __shfl_xor_sync(0xffffffffu, v[c], o);
  }
  if constexpr (!kWarp) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    float* s = scratch + turn * (2 * 32);
    turn ^= 1;
    if (lane == 0) {
#pragma unroll
      for (int c = 0; c < kCount; ++c) s[c * 32 + warp] = v[c];
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kCount; ++c) {
      float t = lane < warps ? s[c * 32 + lane] : 0.0f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      v[c] = t;
    }
  }
}

// A thread's kPer vectors of a row: vector i is number thread + i * threads of the row.
template <typename T, int kVec, int kPer>
struct Piece {
  Raw<T, kVec> raw[kPer];
  __device__ __forceinline__ void load(const void* base, int64_t row, int64_t ld, int thread, int threads, int nvec) {
    const T* p = static_cast<const T*>(base) + row * ld;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = thread + i * threads;
      if (v < nvec) raw[i] = *reinterpret_cast<const Raw<T, kVec>*>(p + static_cast<int64_t>(v) * kVec);
      else raw[i] = Raw<T, kVec>{};
    }
  }
};

template <typename T, int kVec, int kPer, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 256 : kMaxThreads, 1) row_norm_fwd_kernel(const Args a) {
  __shared__ float scratch[2 * 2 * 32];
  const int threads = kWarp ? 32 : blockDim.x, thread = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int64_t groups = kWarp ? static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5) : gridDim.x;
  int64_t row = kWarp ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int nvec = a.cols / kVec;
  int turn = 0;
  ptx::grid_dependency_sync();
  float scale[kPer * kVec], shift[kPer * kVec];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int c = (thread + i * threads) * kVec + j;
      scale[i * kVec + j] = a.gain != nullptr && c < a.cols ? a.gain_offset + load_param(a.gain, c, a.param_dtype) : 1.0f;
      shift[i * kVec + j] = a.shift != nullptr && c < a.cols ? load_param(a.shift, c, a.param_dtype) : 0.0f;
    }
  }
  Piece<T, kVec, kPer> next;
  if (row < a.rows) next.load(a.x, row, a.ldx, thread, threads, nvec);
  for (; row < a.rows; row += groups) {
    const Piece<T, kVec, kPer> cur = next;
    if (row + groups < a.rows) next.load(a.x, row + groups, a.ldx, thread, threads, nvec);
    float s[1] = {0.0f};
    float mean = 0.0f;
    if (!a.rms) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        float f[kVec];
        unpack<T, kVec>(cur.raw[i], f);
#pragma unroll
        for (int j = 0; j < kVec; ++j) s[0] += f[j];
      }
      row_sums<kWarp, 1>(s, scratch, turn);
      mean = s[0] * a.inv_cols;
      s[0] = 0.0f;
    }
    // (the squares of what is left of the mean, not the mean of the squares: no cancellation)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      float f[kVec];
      unpack<T, kVec>(cur.raw[i], f);
      if (thread + i * threads < nvec) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) s[0] = fmaf(f[j] - mean, f[j] - mean, s[0]);
      }
    }
    row_sums<kWarp, 1>(s, scratch, turn);
    const float rstd = rsqrtf(fmaf(s[0], a.inv_cols, a.eps));
    T* out = static_cast<T*>(a.out) + row * a.ldo;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = thread + i * threads;
      if (v < nvec) {
        float f[kVec];
        unpack<T, kVec>(cur.raw[i], f);
#pragma unroll
        for (int j = 0; j < kVec; ++j) f[j] = fmaf((f[j] - mean) * rstd, scale[i * kVec + j], shift[i * kVec + j]);
        *reinterpret_cast<Raw<T, kVec>*>(out + static_cast<int64_t>(v) * kVec) = pack<T, kVec>(f);
      }
    }
    if (thread == 0) {
      if (a.mean != nullptr) a.mean[row] = mean;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
  }
}

template <typename T, int kVec, int kPer, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 256 : kMaxThreads, 1) row_norm_bwd_kernel(const Args a) {
  __shared__ float scratch[2 * 2 * 32];
  extern __shared__ float sums[];    // kWarp: [2][cols]
  const int threads = kWarp ? 32 : blockDim.x, thread = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int64_t groups = kWarp ? static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5) : gridDim.x;
  int64_t row = kWarp ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int nvec = a.cols / kVec;
  int turn = 0;
  ptx::grid_dependency_sync();
  float scale[kPer * kVec], dgain[kPer * kVec], dshift[kPer * kVec];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int c = (thread + i * threads) * kVec + j;
      scale[i * kVec + j] = a.gain != nullptr && c < a.cols ? a.gain_offset + load_param(a.gain, c, a.param_dtype) : 1.0f;
      dgain[i * kVec + j] = dshift[i * kVec + j] = 0.0f;
    }
  }
  Piece<T, kVec, kPer> next_x, next_g;
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t r) {
    next_x.load(a.x, r, a.ldx, thread, threads, nvec);
    next_g.load(a.gy, r, a.ldg, thread, threads, nvec);
    next_mean = a.rms ? 0.0f : a.mean[r];
    next_rstd = a.rstd[r];
  };
  if (row < a.rows) fetch(row);
  for (; row < a.rows; row += groups) {
    const Piece<T, kVec, kPer> cur_x = next_x, cur_g = next_g;
    const float mean = next_mean, rstd = next_rstd;
    if (row + groups < a.rows) fetch(row + groups);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      float x[kVec], g[kVec];
      unpack<T, kVec>(cur_x.raw[i], x);
      unpack<T, kVec>(cur_g.raw[i], g);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {     // (behind the row's end g is 0)
        const float xh = (x[j] - mean) * rstd, h = g[j] * scale[i * kVec + j];
        dgain[i * kVec + j] = fmaf(g[j], xh, dgain[i * kVec + j]);
        dshift[i * kVec + j] += g[j];
        s[0] = fmaf(h, xh, s[0]);
        s[1] += h;
      }
    }
    row_sums<kWarp, 2>(s, scratch, turn);
    const float c1 = s[0] * a.inv_cols, c0 = a.rms ? 0.0f : s[1] * a.inv_cols;
    T* out = static_cast<T*>(a.out) + row * a.ldo;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = thread + i * threads;
      if (v < nvec) {
        float x[kVec], g[kVec];
        unpack<T, kVec>(cur_x.raw[i], x);
        unpack<T, kVec>(cur_g.raw[i], g);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const float xh = (x[j] - mean) * rstd, h = g[j] * scale[i * kVec + j];
          x[j] = rstd * (h - fmaf(xh, c1, c0));
        }
        *reinterpret_cast<Raw<T, kVec>*>(out + static_cast<int64_t>(v) * kVec) = pack<T, kVec>(x);
      }
    }
  }
  if (a.part_gain == nullptr && a.part_shift == nullptr) return;
  if constexpr (kWarp) {     // the CTA's warps add up one after the other
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
      if (static_cast<int>(threadIdx.x >> 5) == w) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const int c = (thread + i * threads) * kVec + j;
            if (c < a.cols) {
              sums[c] = (w == 0 ? 0.0f : sums[c]) + dgain[i * kVec + j];
              sums[a.cols + c] = (w == 0 ? 0.0f : sums[a.cols + c]) + dshift[i * kVec + j];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      if (a.part_gain != nullptr) a.part_gain[static_cast<int64_t>(blockIdx.x) * a.cols + c] = sums[c];
      if (a.part_shift != nullptr) a.part_shift[static_cast<int64_t>(blockIdx.x) * a.cols + c] = sums[a.cols + c];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const int c = (thread + i * threads) * kVec + j;
        if (c < a.cols) {
          if (a.part_gain != nullptr) a.part_gain[static_cast<int64_t>(blockIdx.x) * a.cols + c] = dgain[i * kVec + j];
          if (a.part_shift != nullptr) a.part_shift[static_cast<int64_t>(blockIdx.x) * a.cols + c] = dshift[i * kVec + j];
        }
      }
    }
  }
}

// dgain (blockIdx.y 0) and dshift (1): the CTAs' rows of partials added up, 32 columns per CTA.
__global__ void __launch_bounds__(kSumCols* kSumParts) row_norm_sum_kernel(const float* part_gain, const float* part_shift, int parts,
                                                                          int cols, void* dgain, void* dshift, int dtype) {
  ptx::grid_dependency_sync();
  __shared__ float s[kSumParts][kSumCols + 1];
  const float* part = blockIdx.y == 0 ? part_gain : part_shift;
  void* out = blockIdx.y == 0 ? dgain : dshift;
  if (out == nullptr) return;
  const int lane = threadIdx.x % kSumCols, p0 = threadIdx.x / kSumCols, c = blockIdx.x * kSumCols + lane;
  float t = 0.0f;
  if (c < cols) {
#pragma unroll 4
    for (int p = p0; p < parts; p += kSumParts) t += part[static_cast<int64_t>(p) * cols + c];
  }
  s[p0][lane] = t;
  __syncthreads();
  // (column p0 now, its partial sums across the lanes)
  t = s[lane][p0];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int col = blockIdx.x * kSumCols + p0;
  if (lane == 0 && col < cols) {
    if (dtype == IXK_F32) static_cast<float*>(out)[col] = t;
    else if (dtype == IXK_BF16) static_cast<__nv_bfloat16*>(out)[col] = __float2bfloat16_rn(t);
    else static_cast<__half*>(out)[col] = __float2half_rn(t);
  }
}

// How a row is dealt out: vectors of 16 bytes where every row starts on one, else single elements.
struct Plan {
  int vec, per, threads, groups_per_cta;
  bool warp;
};
Plan plan_for(int64_t cols, int elem_bytes, bool aligned) {
  Plan p{};
  const int full = 16 / elem_bytes;
  p.vec = aligned && cols % full == 0 ? full : 1;
  const int64_t vecs = cols / p.vec;
  // a warp per row up to eight elements a thread
  if (vecs * p.vec <= 32 * 8) {
    p.warp = true;
    p.threads = 256;
    p.groups_per_cta = 8;
    p.per = static_cast<int>((vecs + 31) / 32);
  } else {
    p.groups_per_cta = 1;
    p.per = 1;
    while (p.per * p.vec < 8) p.per *= 2;                                         // eight elements a thread ...
    while (vecs > static_cast<int64_t>(kMaxThreads) * p.per) p.per *= 2;          // ... or sixteen
    p.threads = static_cast<int>((vecs + p.per - 1) / p.per + 31) / 32 * 32;
  }
  int per = 1;
  while (per < p.per) per *= 2;
  p.per = per;
  return p;
}
int64_t ctas_for(const Plan& p, int64_t rows) {
  const int64_t want = (rows + p.groups_per_cta - 1) / p.groups_per_cta;
  return std::min<int64_t>(want, static_cast<int64_t>(kAssumedSms) * std::max(1, kThreadsPerSm / p.threads));
}

template <typename T, bool kBwd>
int launch(const Plan& p, const Args& a, int64_t ctas, cudaStream_t stream) {
  const size_t smem = kBwd && p.warp ? 2 * sizeof(float) * a.cols : 0;
  auto go = [&](auto vec, auto per, auto warp) -> int {
    constexpr int kVec = decltype(vec)::value, kPer = decltype(per)::value;
    constexpr bool kWarp = decltype(warp)::value;
    if constexpr (kBwd) return launch_overlapped(row_norm_bwd_kernel<T, kVec, kPer, kWarp>, dim3(ctas), dim3(p.threads), smem, stream, a);
    else return launch_overlapped(row_norm_fwd_kernel<T, kVec, kPer, kWarp>, dim3(ctas), dim3(p.threads), smem, stream, a);
  };
  constexpr int kFull = 16 / sizeof(T);
#define IXK_NORM_CASE(V, P, W) \
  if (p.vec == V && p.per == P && p.warp == W) return go(std::integral_constant<int, V>{}, std::integral_constant<int, P>{}, std::bool_constant<W>{});
  IXK_NORM_CASE(kFull, 1, true)
  if constexpr (kFull == 4) { IXK_NORM_CASE(kFull, 2, true) }
  IXK_NORM_CASE(1, 1, true)
  IXK_NORM_CASE(1, 2, true)
  IXK_NORM_CASE(1, 4, true)
  IXK_NORM_CASE(1, 8, true)
  if constexpr (kFull == 8) { IXK_NORM_CASE(kFull, 1, false) }
  IXK_NORM_CASE(kFull, 2, false)
  if constexpr (kFull == 4) { IXK_NORM_CASE(kFull, 4, false) }
  IXK_NORM_CASE(1, 8, false)
  IXK_NORM_CASE(1, 16, false)
#undef IXK_NORM_CASE
  return fail(IXK_UNIMPLEMENTED, "row_norm: no kernel for this row");
}

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
int bytes_of(int dtype) { return dtype == IXK_F32 ? 4 : 2; }

int check(const ixk_row_norm_desc* d, const char* name) {
  const std::string who = std::string(name) + ": ";
  if (d == nullptr) return fail(IXK_INVALID_ARGUMENT, who + "desc is NULL");
  if (d->dtype != IXK_BF16 && d->dtype != IXK_F16 && d->dtype != IXK_F32)
    return fail(IXK_UNIMPLEMENTED, who + "dtype must be BF16, F16 or F32");
  if (d->param_dtype != d->dtype && d->param_dtype != IXK_F32)
    return fail(IXK_UNIMPLEMENTED, who + "gain and shift must have the rows' type or be F32");
  if (d->kind != IXK_NORM_LAYER && d->kind != IXK_NORM_RMS) return fail(IXK_INVALID_ARGUMENT, who + "unknown kind");
  if (d->reserved != 0) return fail(IXK_INVALID_ARGUMENT, who + "desc.reserved must be 0");
  if (d->rows < 0 || d->cols <= 0) return fail(IXK_INVALID_ARGUMENT, who + "negative rows or no columns");
  if (d->cols > kMaxCols) return fail(IXK_UNIMPLEMENTED, who + "rows longer than 16384 elements");
  if (d->rows > 0x7fffffff) return fail(IXK_UNIMPLEMENTED, who + "more than 2^31-1 rows");
  if (!(d->eps >= 0.0f)) return fail(IXK_INVALID_ARGUMENT, who + "eps must not be negative");
  return IXK_OK;
}

int fwd(const ixk_row_norm_desc* d, const void* x, const void* gain, const void* shift, void* y, float* mean, float* rstd,
        void* stream) {
  int rc = check(d, "row_norm_fwd");
  if (rc != IXK_OK) return rc;
  if (d->rows > 0 && (x == nullptr || y == nullptr)) return fail(IXK_INVALID_ARGUMENT, "row_norm_fwd: x and y must be non-NULL");
  if (d->x_stride < d->cols || d->y_stride < d->cols) return fail(IXK_INVALID_ARGUMENT, "row_norm_fwd: a row stride is smaller than the row");
  const int es = bytes_of(d->dtype), ps = bytes_of(d->param_dtype);
  if (!aligned(x, es) || !aligned(y, es) || !aligned(gain, ps) || !aligned(shift, ps) || !aligned(mean, 4) || !aligned(rstd, 4))
    return fail(IXK_INVALID_ARGUMENT, "row_norm_fwd: a pointer is not aligned to its element size");
  DeviceInfo info;
  if ((rc = get_device_info(&info)) != IXK_OK) return rc;
  if (d->rows == 0) return IXK_OK;
  const bool wide = aligned(x, 16) && aligned(y, 16) && d->x_stride * es % 16 == 0 && d->y_stride * es % 16 == 0;
  const Plan p = plan_for(d->cols, es, wide);
  Args a{};
  a.x = x;
  a.gain = gain;
  a.shift = shift;
  a.out = y;
  a.mean = d->kind == IXK_NORM_LAYER ? mean : nullptr;
  a.rstd = rstd;
  a.rows = d->rows;
  a.cols = static_cast<int>(d->cols);
  a.ldx = d->x_stride;
  a.ldo = d->y_stride;
  a.rms = d->kind == IXK_NORM_RMS;
  a.param_dtype = d->param_dtype;
  a.eps = d->eps;
  a.gain_offset = d->gain_offset;
  a.inv_cols = 1.0f / static_cast<float>(d->cols);
  const int64_t want = (d->rows + p.groups_per_cta - 1) / p.groups_per_cta;
  const int64_t ctas = std::min<int64_t>(want, static_cast<int64_t>(info.sm_count) * (2048 / p.threads));
  auto s = static_cast<cudaStream_t>(stream);
  if (d->dtype == IXK_F32) return launch<float, false>(p, a, ctas, s);
  if (d->dtype == IXK_BF16) return launch<__nv_bfloat16, false>(p, a, ctas, s);
  return launch<__half, false>(p, a, ctas, s);
}

// (the partials' CTAs must not depend on alignment, which the query does not know: the most that any plan has)
size_t part_bytes(const ixk_row_norm_desc* d) {
  const int es = bytes_of(d->dtype);
  const int64_t ctas = std::max(ctas_for(plan_for(d->cols, es, true), d->rows), ctas_for(plan_for(d->cols, es, false), d->rows));
  return static_cast<size_t>(ctas) * d->cols * sizeof(float);
}

int bwd(const ixk_row_norm_desc* d, const void* gy, const void* x, const void* gain, const float* mean, const float* rstd, void* dx,
        void* dgain, void* dshift, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(d, "row_norm_bwd");
  if (rc != IXK_OK) return rc;
  const bool layer = d->kind == IXK_NORM_LAYER;
  if (d->rows > 0 && (gy == nullptr || x == nullptr || rstd == nullptr || dx == nullptr || (layer && mean == nullptr)))
    return fail(IXK_INVALID_ARGUMENT, "row_norm_bwd: grad_y, x, the row statistics and dx must be non-NULL");
  if (dgain != nullptr && gain == nullptr) return fail(IXK_INVALID_ARGUMENT, "row_norm_bwd: dgain without a gain");
  if (d->x_stride < d->cols || d->grad_y_stride < d->cols || d->dx_stride < d->cols)
    return fail(IXK_INVALID_ARGUMENT, "row_norm_bwd: a row stride is smaller than the row");
  const int es = bytes_of(d->dtype), ps = bytes_of(d->param_dtype);
  if (!aligned(x, es) || !aligned(gy, es) || !aligned(dx, es) || !aligned(gain, ps) || !aligned(dgain, ps) || !aligned(dshift, ps) ||
      !aligned(mean, 4) || !aligned(rstd, 4))
    return fail(IXK_INVALID_ARGUMENT, "row_norm_bwd: a pointer is not aligned to its element size");
  const bool params = dgain != nullptr || dshift != nullptr;
  const size_t one = part_bytes(d), need = params ? 2 * one : 0;
  if (need > 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < need))
    return fail(IXK_WORKSPACE_TOO_SMALL, "row_norm_bwd: need " + std::to_string(need) + " bytes of 16-byte aligned scratch");
  DeviceInfo info;
  if ((rc = get_device_info(&info)) != IXK_OK) return rc;
  const bool wide = aligned(x, 16) && aligned(gy, 16) && aligned(dx, 16) && d->x_stride * es % 16 == 0 &&
                    d->grad_y_stride * es % 16 == 0 && d->dx_stride * es % 16 == 0;
  const Plan p = plan_for(d->cols, es, wide);
  const int64_t ctas = ctas_for(p, d->rows);
  Args a{};
  a.x = x;
  a.gy = gy;
  a.gain = gain;
  a.out = dx;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.part_gain = dgain != nullptr ? static_cast<float*>(workspace) : nullptr;
  a.part_shift = dshift != nullptr ? reinterpret_cast<float*>(static_cast<char*>(workspace) + one) : nullptr;
  a.rows = d->rows;
  a.cols = static_cast<int>(d->cols);
  a.ldx = d->x_stride;
  a.ldg = d->grad_y_stride;
  a.ldo = d->dx_stride;
  a.rms = !layer;
  a.param_dtype = d->param_dtype;
  a.gain_offset = d->gain_offset;
  a.inv_cols = 1.0f / static_cast<float>(d->cols);
  auto s = static_cast<cudaStream_t>(stream);
  if (d->rows > 0) {
    rc = d->dtype == IXK_F32 ? launch<float, true>(p, a, ctas, s)
         : d->dtype == IXK_BF16 ? launch<__nv_bfloat16, true>(p, a, ctas, s) : launch<__half, true>(p, a, ctas, s);
    if (rc != IXK_OK) return rc;
  }
  if (!params) return IXK_OK;
  return launch_overlapped(row_norm_sum_kernel, dim3(static_cast<unsigned>((d->cols + kSumCols - 1) / kSumCols), 2), dim3(kSumCols * kSumParts),
                           0, s, static_cast<const float*>(a.part_gain), static_cast<const float*>(a.part_shift), static_cast<int>(ctas), a.cols,
                           dgain, dshift, d->param_dtype);
}

}  // namespace
}  // namespace norm
}  // namespace ixk

extern "C" {

int ixk_row_norm_fwd(const ixk_row_norm_desc* desc, const void* x, const void* gain, const void* shift, void* y, float* mean,
                     float* rstd, void* cuda_stream) {
  IXK_API_RANGE("ixk_row_norm_fwd");
  ixk::clear_error();
  return ixk::norm::fwd(desc, x, gain, shift, y, mean, rstd, cuda_stream);
}

int ixk_row_norm_bwd(const ixk_row_norm_desc* desc, const void* grad_y, const void* x, const void* gain, const float* mean,
                     const float* rstd, void* dx, void* dgain, void* dshift, void* workspace, size_t workspace_bytes,
                     void* cuda_stream) {
  IXK_API_RANGE("ixk_row_norm_bwd");
  ixk::clear_error();
  return ixk::norm::bwd(desc, grad_y, x, gain, mean, rstd, dx, dgain, dshift, workspace, workspace_bytes, cuda_stream);
}

size_t ixk_row_norm_bwd_workspace_bytes(const ixk_row_norm_desc* desc) {
  if (desc == nullptr || desc->rows < 0 || desc->cols <= 0 || desc->cols > ixk::norm::kMaxCols) return 0;
  return 2 * ixk::norm::part_bytes(desc);
}

}  // extern "C"
