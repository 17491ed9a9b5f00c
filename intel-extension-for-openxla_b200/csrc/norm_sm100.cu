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
// leave as one row of partials per CTA or pair of CTAs, which a second kernel adds up in a fixed order: the result does not
// depend on which CTA was faster.  Statistics and sums are fp32, the variance is taken about the mean, and 1 / sqrt is the
// correctly rounded one: its error would be shared by all elements of a row.
//
// Which kernel a row takes (times: forward / backward with its sums, cold caches, one call waited for):
//   up to 256 columns, whole 16-byte vectors    row_norm_*_rows_kernel, several rows a warp      65536 x 256 bf16   22 /  32 us
//   257 .. 8192, or whole vectors or not        row_norm_*_ring_kernel, rows through a ring      8192 x 4096 bf16   35 /  50 us
//   up to 256 single elements, or above 8192    row_norm_*_kernel, a row a warp or a CTA         (512 threads of 16 columns are
//                                               the ring's limit; 5461 x 12288 bf16   74 / 190 us)
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
constexpr int kSumCols = 16, kSumParts = 16;

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
// The compiler may not keep what it unpacked of `raw` beyond this point: registers hold the row as it lies in memory, not
// twice as many floats.
__device__ __forceinline__ void forget(uint4& raw) { asm volatile("" : "+r"(raw.x), "+r"(raw.y), "+r"(raw.z), "+r"(raw.w)); }
__device__ __forceinline__ void forget(uint32_t& raw) { asm volatile("" : "+r"(raw)); }
__device__ __forceinline__ void forget(uint16_t& raw) { asm volatile("" : "+h"(raw)); }
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
  int gain_vec, shift_vec;      // gain and shift start on 16 bytes
  int stages;                   // of the ring, and a row's bytes in it
  uint32_t row_bytes;
  int* status_word;
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

// Rows that neither of the kernels below takes.  kAhead: parameters in registers, the next row's loads asked for before this
// row's statistics are waited for.  Otherwise a CTA's row, whose 1024 threads of 16 columns have 64 registers each: parameters
// in shared memory, one row at a time.  Ahead and not: 5461 rows of 12288 16-bit elements in whole vectors, backward, 189 and
// 202 us; of 12287, forward 275 and 214, backward 507 and 423; 3000 x 10000 fp32 in whole vectors, forward 70 and 82, backward
// 151 and 120.
template <typename T, int kVec, bool kWarp, bool kBwd>
constexpr bool kAhead = kWarp || (kVec > 1 && (sizeof(T) == 2 || !kBwd));
template <typename T, int kVec, int kPer, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 256 : kMaxThreads, 1) row_norm_fwd_kernel(const Args a) {
  __shared__ float scratch[2 * 2 * 32];
  extern __shared__ float params[];      // not ahead: scale and shift, [2][cols]
  constexpr bool kRegs = kAhead<T, kVec, kWarp, false>;
  const int threads = kWarp ? 32 : blockDim.x, thread = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int64_t groups = kWarp ? static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5) : gridDim.x;
  int64_t row = kWarp ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int nvec = a.cols / kVec;
  int turn = 0;
  ptx::grid_dependency_sync();
  float own_scale[kRegs ? kPer * kVec : 1], own_shift[kRegs ? kPer * kVec : 1];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int c = (thread + i * threads) * kVec + j;
      const float scale = a.gain != nullptr && c < a.cols ? a.gain_offset + load_param(a.gain, c, a.param_dtype) : 1.0f;
      const float shift = a.shift != nullptr && c < a.cols ? load_param(a.shift, c, a.param_dtype) : 0.0f;
      if constexpr (kRegs) {
        own_scale[i * kVec + j] = scale;
        own_shift[i * kVec + j] = shift;
      } else if (c < a.cols) {      // (read by this thread alone)
        params[c] = scale;
        params[a.cols + c] = shift;
      }
    }
  }
  Piece<T, kVec, kPer> next;
  if (kRegs && row < a.rows) next.load(a.x, row, a.ldx, thread, threads, nvec);
  for (; row < a.rows; row += groups) {
    if (!kRegs) next.load(a.x, row, a.ldx, thread, threads, nvec);
    Piece<T, kVec, kPer> cur = next;
    if (kRegs && row + groups < a.rows) next.load(a.x, row + groups, a.ldx, thread, threads, nvec);
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
    if constexpr (!kRegs) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) forget(cur.raw[i]);
    }
    const float rstd = __frsqrt_rn(fmaf(s[0], a.inv_cols, a.eps));
    T* out = static_cast<T*>(a.out) + row * a.ldo;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = thread + i * threads;
      if (v < nvec) {
        float f[kVec];
        unpack<T, kVec>(cur.raw[i], f);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          float scale, shift;
          if constexpr (kRegs) {
            scale = own_scale[i * kVec + j];
            shift = own_shift[i * kVec + j];
          } else {
            scale = params[v * kVec + j];
            shift = params[a.cols + v * kVec + j];
          }
          f[j] = fmaf((f[j] - mean) * rstd, scale, shift);
        }
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
  extern __shared__ float sums[];    // kWarp: [2][cols]; not ahead: the scale, [cols]
  const int threads = kWarp ? 32 : blockDim.x, thread = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int64_t groups = kWarp ? static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5) : gridDim.x;
  int64_t row = kWarp ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int nvec = a.cols / kVec;
  int turn = 0;
  ptx::grid_dependency_sync();
  constexpr bool kRegs = kAhead<T, kVec, kWarp, true>;
  float own_scale[kRegs ? kPer * kVec : 1], dgain[kPer * kVec], dshift[kPer * kVec];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int c = (thread + i * threads) * kVec + j;
      const float scale = a.gain != nullptr && c < a.cols ? a.gain_offset + load_param(a.gain, c, a.param_dtype) : 1.0f;
      if constexpr (kRegs) own_scale[i * kVec + j] = scale;
      else if (c < a.cols) sums[c] = scale;      // (read by this thread alone)
      dgain[i * kVec + j] = dshift[i * kVec + j] = 0.0f;
    }
  }
  auto scale_of = [&](int i, int j) {      // (behind the row's end g is 0)
    if constexpr (kRegs) return own_scale[i * kVec + j];
    else return thread + i * threads < nvec ? sums[(thread + i * threads) * kVec + j] : 0.0f;
  };
  Piece<T, kVec, kPer> next_x, next_g;
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t r) {
    next_x.load(a.x, r, a.ldx, thread, threads, nvec);
    next_g.load(a.gy, r, a.ldg, thread, threads, nvec);
    next_mean = a.rms ? 0.0f : a.mean[r];
    next_rstd = a.rstd[r];
  };
  if (kRegs && row < a.rows) fetch(row);
  for (; row < a.rows; row += groups) {
    if (!kRegs) fetch(row);
    Piece<T, kVec, kPer> cur_x = next_x, cur_g = next_g;
    const float mean = next_mean, rstd = next_rstd;
    if (kRegs && row + groups < a.rows) fetch(row + groups);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      float x[kVec], g[kVec];
      unpack<T, kVec>(cur_x.raw[i], x);
      unpack<T, kVec>(cur_g.raw[i], g);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {     // (behind the row's end g is 0)
        const float xh = (x[j] - mean) * rstd, h = g[j] * scale_of(i, j);
        dgain[i * kVec + j] = fmaf(g[j], xh, dgain[i * kVec + j]);
        dshift[i * kVec + j] += g[j];
        s[0] = fmaf(h, xh, s[0]);
        s[1] += h;
      }
    }
    row_sums<kWarp, 2>(s, scratch, turn);
    if constexpr (!kRegs) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        forget(cur_x.raw[i]);
        forget(cur_g.raw[i]);
      }
    }
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
          const float xh = (x[j] - mean) * rstd, h = g[j] * scale_of(i, j);
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

// Whole vectors are worked on as pairs of fp32 (fma.rn.f32x2 and its kin: half of the instructions, which bound these
// kernels, not memory, when every element is its own: 27 a element forward and 45 backward).
template <typename T>
constexpr int kPairs = 8 / sizeof(T);     // of a 16-byte vector
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& raw, uint64_t (&p)[kPairs<T>]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < kPairs<T>; ++j) {
    if constexpr (std::is_same_v<T, float>) {
      p[j] = ptx::f32x2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
    } else if constexpr (std::is_same_v<T, __half>) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      p[j] = ptx::f32x2(f.x, f.y);
    } else {
      p[j] = ptx::f32x2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack_pairs(const uint64_t (&p)[kPairs<T>]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < kPairs<T>; ++j) {
    float lo, hi;
    ptx::f32x2_split(p[j], lo, hi);
    if constexpr (std::is_same_v<T, float>) {
      w[2 * j] = __float_as_uint(lo);
      w[2 * j + 1] = __float_as_uint(hi);
    } else if constexpr (std::is_same_v<T, __half>) {
      const __half2 h = __floats2half2_rn(lo, hi);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T, int kN>
__device__ __forceinline__ void unpack_all(const uint4* raw, uint64_t (&p)[kN]) {
#pragma unroll
  for (int i = 0; i < kN / kPairs<T>; ++i) {
    uint64_t part[kPairs<T>];
    unpack_pairs<T>(raw[i], part);
#pragma unroll
    for (int j = 0; j < kPairs<T>; ++j) p[i * kPairs<T> + j] = part[j];
  }
}
__device__ __forceinline__ float pair_sum(uint64_t p) {
  float lo, hi;
  ptx::f32x2_split(p, lo, hi);
  return lo + hi;
}
// offset + parameters of type P, as pairs: the kN pairs from column c on (`none` without a parameter).
template <typename P, int kN>
__device__ __forceinline__ void load_params(const void* p, int c, bool vec, float offset, float none, uint64_t (&out)[kN]) {
  const uint64_t off = ptx::f32x2(offset, offset);
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < kN; ++j) out[j] = ptx::f32x2(none, none);
  } else if (vec) {      // (as many bytes as the parameters of a vector of columns have: 16 or 32)
    const P* at = static_cast<const P*>(p) + c;
#pragma unroll
    for (int j = 0; j < kN; j += kPairs<P>) {
      uint64_t part[kPairs<P>];
      unpack_pairs<P>(*reinterpret_cast<const uint4*>(at + 2 * j), part);
#pragma unroll
      for (int i = 0; i < kPairs<P>; ++i) out[j + i] = ptx::add2(part[i], off);
    }
  } else {
    const P* at = static_cast<const P*>(p) + c;
#pragma unroll
    for (int j = 0; j < kN; ++j) out[j] = ptx::add2(ptx::f32x2(to_float<P>(at[2 * j]), to_float<P>(at[2 * j + 1])), off);
  }
}
// The warp's sums of kCount values (a power of two), in every lane.  Halves of the lanes first take over halves of the values,
// so that 8 values take 9 shuffles and 8 to hand the sums back instead of 40.
template <int kCount>
__device__ __forceinline__ int value_of_lane(int lane) {
  return kCount == 8 ? lane >> 2 : kCount == 4 ? lane >> 3 : kCount == 2 ? lane >> 4 : 0;
}
template <int kCount>
__device__ __forceinline__ float warp_sum_of_lane(float (&v)[kCount]) {     // of value value_of_lane
  const int lane = threadIdx.x & 31;
  int o = 16;
#pragma unroll
  for (int n = kCount; n > 1; n /= 2, o /= 2) {
    const bool upper = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float keep = upper ? v[i + n / 2] : v[i], give = upper ? v[i] : v[i + n / 2];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
#pragma unroll
  for (; o > 0; o /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}
template <int kCount>
__device__ __forceinline__ void warp_sums(float (&v)[kCount]) {
  const float t = warp_sum_of_lane<kCount>(v);
#pragma unroll
  for (int c = 0; c < kCount; ++c) v[c] = __shfl_sync(0xffffffffu, t, c * (32 / kCount));
}
// The same over a CTA of at most 16 warps; `scratch` is not the one of the call before.
template <int kCount>
__device__ __forceinline__ void cta_sums(float (&v)[kCount], float (&scratch)[kCount][16]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  constexpr int kLanes = 32 / kCount;      // per value
  const float t = warp_sum_of_lane<kCount>(v);
  const int c = value_of_lane<kCount>(lane), at = lane % kLanes;
  if (at == 0) scratch[c][warp] = t;
  __syncthreads();
  float u = at < warps ? scratch[c][at] : 0.0f;
  if (kLanes < 16 && at + kLanes < warps) u += scratch[c][at + kLanes];
#pragma unroll
  for (int o = kLanes / 2; o > 0; o /= 2) u += __shfl_xor_sync(0xffffffffu, u, o);
#pragma unroll
  for (int i = 0; i < kCount; ++i) v[i] = __shfl_sync(0xffffffffu, u, i * kLanes);
}

// Forward, short rows (up to eight elements a lane): a warp has kRows rows at a time, all of their loads out at once and no
// barrier between warps.  65536 x 256 bf16: 16 us on the device, 67 MB at 4.2 TB/s, what a copy of that size gets between its
// start and its end (rows copied ahead into shared memory changed nothing).
template <typename T, typename P, int kPer, int kRows>
__global__ void __launch_bounds__(128) row_norm_fwd_rows_kernel(const Args a) {
  constexpr int kVec = 16 / sizeof(T), kN = kPairs<T>;
  ptx::grid_dependency_sync();
  const int lane = threadIdx.x & 31, nvec = a.cols / kVec;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t first = (static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5)) * kRows; first < a.rows; first += warps * kRows) {
    uint4 raw[kRows][kPer];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (first + r) * a.ldx);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int v = lane + 32 * i;
        raw[r][i] = first + r < a.rows && v < nvec ? x[v] : make_uint4(0, 0, 0, 0);
      }
    }
    float mean[kRows], s[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) mean[r] = 0.0f;
    if (!a.rms) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        uint64_t t = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          uint64_t f[kN];
          unpack_pairs<T>(raw[r][i], f);
#pragma unroll
          for (int j = 0; j < kN; ++j) t = ptx::add2(t, f[j]);
        }
        mean[r] = pair_sum(t);
      }
      warp_sums<kRows>(mean);
#pragma unroll
      for (int r = 0; r < kRows; ++r) mean[r] *= a.inv_cols;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const uint64_t minus = ptx::f32x2(-mean[r], -mean[r]);
      uint64_t t = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        forget(raw[r][i]);
        if (lane + 32 * i < nvec) {
          uint64_t f[kN];
          unpack_pairs<T>(raw[r][i], f);
#pragma unroll
          for (int j = 0; j < kN; ++j) {
            f[j] = ptx::add2(f[j], minus);
            t = ptx::fma2(f[j], f[j], t);
          }
        }
      }
      s[r] = pair_sum(t);
    }
    warp_sums<kRows>(s);
#pragma unroll
    for (int r = 0; r < kRows; ++r) s[r] = __frsqrt_rn(fmaf(s[r], a.inv_cols, a.eps));
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = lane + 32 * i;
      if (v < nvec) {
        uint64_t scale[kN], shift[kN];
        load_params<P, kN>(a.gain, v * kVec, a.gain_vec, a.gain_offset, 1.0f, scale);
        load_params<P, kN>(a.shift, v * kVec, a.shift_vec, 0.0f, 0.0f, shift);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          if (first + r < a.rows) {
            const uint64_t minus = ptx::f32x2(-mean[r], -mean[r]), rstd = ptx::f32x2(s[r], s[r]);
            uint64_t f[kN];
            forget(raw[r][i]);
            unpack_pairs<T>(raw[r][i], f);
#pragma unroll
            for (int j = 0; j < kN; ++j) f[j] = ptx::fma2(ptx::mul2(ptx::add2(f[j], minus), rstd), scale[j], shift[j]);
            reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (first + r) * a.ldo)[v] = pack_pairs<T>(f);
          }
        }
      }
    }
    if (lane < kRows && first + lane < a.rows) {
      float m = mean[0], q = s[0];
#pragma unroll
      for (int r = 1; r < kRows; ++r) {
        if (lane == r) {
          m = mean[r];
          q = s[r];
        }
      }
      if (a.mean != nullptr) a.mean[first + lane] = m;
      if (a.rstd != nullptr) a.rstd[first + lane] = q;
    }
  }
}

// What kN pairs of columns add to a row's two sums, mean(h xh) and mean(h), and to the columns' own.
template <typename T, int kN>
__device__ __forceinline__ void bwd_sums(const uint4* xr, const uint4* gr, float mean, float rstd, const uint64_t (&scale)[kN], uint64_t (&dgain)[kN],
                                         uint64_t (&dshift)[kN], uint64_t& hx, uint64_t& hs) {
  const uint64_t minus = ptx::f32x2(-mean, -mean), r2 = ptx::f32x2(rstd, rstd);
  uint64_t x[kN], g[kN];
  unpack_all<T, kN>(xr, x);
  unpack_all<T, kN>(gr, g);
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const uint64_t xh = ptx::mul2(ptx::add2(x[j], minus), r2), h = ptx::mul2(g[j], scale[j]);
    dgain[j] = ptx::fma2(g[j], xh, dgain[j]);
    dshift[j] = ptx::add2(dshift[j], g[j]);
    hx = ptx::fma2(h, xh, hx);
    hs = ptx::add2(hs, h);
  }
}
// dx of kN pairs: rstd (h - c0 - xh c1).
template <typename T, int kN>
__device__ __forceinline__ void bwd_dx(uint4* xr, uint4* gr, float mean, float rstd, const uint64_t (&scale)[kN], float c1, float c0,
                                       uint64_t (&x)[kN]) {
#pragma unroll
  for (int i = 0; i < kN / kPairs<T>; ++i) {
    forget(xr[i]);
    forget(gr[i]);
  }
  const uint64_t minus = ptx::f32x2(-mean, -mean), r2 = ptx::f32x2(rstd, rstd), m1 = ptx::f32x2(-c1, -c1), m0 = ptx::f32x2(-c0, -c0);
  uint64_t g[kN];
  unpack_all<T, kN>(xr, x);
  unpack_all<T, kN>(gr, g);
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const uint64_t xh = ptx::mul2(ptx::add2(x[j], minus), r2);
    x[j] = ptx::mul2(ptx::fma2(xh, m1, ptx::fma2(g[j], scale[j], m0)), r2);
  }
}
template <int kN>
__device__ __forceinline__ void put_pairs(float* out, const uint64_t (&p)[kN], bool add) {
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    float lo, hi;
    ptx::f32x2_split(p[j], lo, hi);
    out[2 * j] = add ? out[2 * j] + lo : lo;
    out[2 * j + 1] = add ? out[2 * j + 1] + hi : hi;
  }
}

// Backward, short rows (up to eight elements a lane): a warp has kRows rows at a time, a lane kPer vectors of columns and
// their sums.  65536 x 256 bf16: 24 us on the device, 100 MB at 4.2 TB/s, and 5 us for the sums.
template <typename T, typename P, int kPer, int kRows>
__global__ void __launch_bounds__(256) row_norm_bwd_rows_kernel(const Args a) {
  constexpr int kVec = 16 / sizeof(T), kN = kPairs<T>;
  extern __shared__ float sums[];    // [2][cols]
  ptx::grid_dependency_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nvec = a.cols / kVec;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  uint64_t scale[kPer][kN], dgain[kPer][kN], dshift[kPer][kN];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int v = lane + 32 * i;
    if (v < nvec) load_params<P, kN>(a.gain, v * kVec, a.gain_vec, a.gain_offset, 1.0f, scale[i]);
#pragma unroll
    for (int j = 0; j < kN; ++j) dgain[i][j] = dshift[i][j] = 0;
  }
  for (int64_t first = (static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp) * kRows; first < a.rows; first += warps * kRows) {
    uint4 xr[kRows][kPer], gr[kRows][kPer];
    float mean[kRows], rstd[kRows], s[2 * kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool there = first + r < a.rows;
      const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (first + r) * a.ldx);
      const uint4* g = reinterpret_cast<const uint4*>(static_cast<const T*>(a.gy) + (first + r) * a.ldg);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int v = lane + 32 * i;
        const bool in = there && v < nvec;
        xr[r][i] = in ? x[v] : make_uint4(0, 0, 0, 0);
        gr[r][i] = in ? g[v] : make_uint4(0, 0, 0, 0);
      }
      mean[r] = there && !a.rms ? a.mean[first + r] : 0.0f;
      rstd[r] = there ? a.rstd[first + r] : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      uint64_t hx = 0, hs = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 32 * i < nvec) bwd_sums<T, kN>(&xr[r][i], &gr[r][i], mean[r], rstd[r], scale[i], dgain[i], dshift[i], hx, hs);
      s[2 * r] = pair_sum(hx);
      s[2 * r + 1] = pair_sum(hs);
    }
    warp_sums<2 * kRows>(s);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float c1 = s[2 * r] * a.inv_cols, c0 = a.rms ? 0.0f : s[2 * r + 1] * a.inv_cols;
      uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (first + r) * a.ldo);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int v = lane + 32 * i;
        if (first + r < a.rows && v < nvec) {
          uint64_t dx[kN];
          bwd_dx<T, kN>(&xr[r][i], &gr[r][i], mean[r], rstd[r], scale[i], c1, c0, dx);
          out[v] = pack_pairs<T>(dx);
        }
      }
    }
  }
  if (a.part_gain == nullptr && a.part_shift == nullptr) return;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {     // the CTA's warps add up one after the other
    if (warp == w) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int v = lane + 32 * i;
        if (v < nvec) {
          put_pairs<kN>(sums + v * kVec, dgain[i], w > 0);
          put_pairs<kN>(sums + a.cols + v * kVec, dshift[i], w > 0);
        }
      }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
    if (a.part_gain != nullptr) a.part_gain[static_cast<int64_t>(blockIdx.x) * a.cols + c] = sums[c];
    if (a.part_shift != nullptr) a.part_shift[static_cast<int64_t>(blockIdx.x) * a.cols + c] = sums[a.cols + c];
  }
}

// Longer rows: a CTA takes kRows rows at a time out of a ring in shared memory that bulk copies keep full (about 190 KB under
// way an SM, which registers could not hold beside the parameters and the columns' sums), and one barrier serves the sums of
// all of them.  A thread has 16 columns: with eight, the sums across threads were a third of all instructions.  What bounds
// it is the chain of a batch (copy's arrival, sums, barrier, result) with two batches an SM to fill the gaps: 8192 x 4096 bf16
// LayerNorm 32 us on the device forward (134 MB at 4.2 TB/s), 43 backward (201 MB at 4.7 TB/s); three or four CTAs an SM have
// too few registers (37 us called, not 35), one row a batch pays its barriers alone.
// kWhole: rows start on 16 bytes and hold whole vectors; a thread has vectors of columns.  Otherwise a row's image in the ring
// keeps the row's place within 16 bytes, the copy brings every 16-byte piece that the row touches (of the first and the last
// row only those that lie wholly in it: nothing outside the tensor is read, and the rest comes element by element), and a
// thread has single columns, blockDim apart.
enum : int { kSiteRing = 701 };
constexpr int kRingBytes = 190 * 1024;
constexpr int kRingThreads = 512, kRingElems = 16, kRingPairs = kRingElems / 2;
constexpr int kMaxStages = 16;
constexpr int kCluster = 2;      // CTAs of the backward ring that add up their columns' sums (with four, clusters wait for places: 72 us, not 49)

// The ring of kTensors tensors' rows: stage s holds batch blockIdx + s * gridDim, then every stages-th one after it.
template <typename T, int kRows, int kTensors, bool kWhole>
struct Ring {
  uint8_t* data;        // [stages][kRows][kTensors][row_bytes]
  uint64_t* full;
  int* abort_flag;
  const void* from[kTensors];
  int64_t ld[kTensors];
  int rows, batches, cols;
  uint32_t row_bytes;   // in the ring
  int stages, stage;
  uint32_t phase;
  bool alive;
  int* status_word;

  __device__ __forceinline__ const T* row_of(int t, int row) const { return static_cast<const T*>(from[t]) + row * ld[t]; }
  __device__ __forceinline__ uint32_t stage_bytes() const { return kTensors * kRows * row_bytes; }
  __device__ __forceinline__ int rows_of(int batch) const { return min(kRows, rows - batch * kRows); }
  // The part of a row's image that the copy brings: [begin, end), bytes from the 16-byte boundary at or in front of the row.
  __device__ __forceinline__ void copied(int t, int row, uint32_t& begin, uint32_t& end) const {
    const uint32_t at = reinterpret_cast<uintptr_t>(row_of(t, row)) & 15u;
    begin = row == 0 ? (at + 15u) & ~15u : 0;
    end = (at + cols * static_cast<uint32_t>(sizeof(T)) + (row == rows - 1 ? 0u : 15u)) & ~15u;
  }
  __device__ __forceinline__ void fetch(int batch, int s) {      // one thread
    const int n = rows_of(batch);
    const uint32_t bar = ptx::smem_u32(&full[s]);
    const uint32_t dst = ptx::smem_u32(data) + s * stage_bytes();
    uint32_t bytes = kTensors * n * row_bytes, begin = 0, end = row_bytes;
    if constexpr (!kWhole) {
      bytes = 0;
      for (int i = 0; i < n * kTensors; ++i) {
        copied(i % kTensors, batch * kRows + i / kTensors, begin, end);
        bytes += end > begin ? end - begin : 0;
      }
    }
    ptx::mbar_expect_tx(bar, bytes);
    for (int r = 0; r < n; ++r) {
#pragma unroll
      for (int t = 0; t < kTensors; ++t) {
        const T* row = row_of(t, batch * kRows + r);
        if constexpr (!kWhole) copied(t, batch * kRows + r, begin, end);
        if (kWhole || end > begin)
          ptx::bulk_load_1d(dst + (r * kTensors + t) * row_bytes + begin,
                            reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(row) & ~uintptr_t(15)) + begin, end - begin, bar);
      }
    }
  }
  __device__ __forceinline__ void init() {
    if (threadIdx.x == 0) {
      *abort_flag = 0;
      for (int s = 0; s < stages; ++s) ptx::mbar_init(ptx::smem_u32(&full[s]), 1);
      ptx::fence_mbar_init();
    }
    __syncthreads();
  }
  __device__ __forceinline__ void start() {
    stage = 0;
    phase = 0;
    alive = true;
    if (threadIdx.x == 0)
      for (int s = 0; s < stages; ++s)
        if (batches - static_cast<int>(blockIdx.x) > s * static_cast<int>(gridDim.x)) fetch(blockIdx.x + s * gridDim.x, s);
  }
  // (a wait that gave up is not tried again: the loop runs out with what is in the ring)
  __device__ __forceinline__ const uint8_t* wait(int batch) {
    if (alive) alive = ptx::mbar_wait(ptx::smem_u32(&full[stage]), phase, ptx::AbortCtl{abort_flag, status_word}, kSiteRing);
    uint8_t* at = data + stage * stage_bytes();
    const int first = batch * kRows, last = first + rows_of(batch) - 1;
    if (!kWhole && (first == 0 || last == rows - 1)) {      // what the copies left out of the first and the last row
      for (int i = 0; i < 2 * kTensors; ++i) {
        const int t = i >> 1, row = i & 1 ? rows - 1 : 0;
        if (row < first || row > last) continue;
        uint32_t begin, end;
        copied(t, row, begin, end);
        const uint32_t start = reinterpret_cast<uintptr_t>(row_of(t, row)) & 15u;
        uint8_t* image = at + ((row - first) * kTensors + t) * row_bytes;
        for (int c = threadIdx.x; c < cols; c += blockDim.x) {
          const uint32_t p = start + c * static_cast<uint32_t>(sizeof(T));
          if (p < begin || p >= end) *reinterpret_cast<Raw<T, 1>*>(image + p) = reinterpret_cast<const volatile Raw<T, 1>*>(row_of(t, row))[c];
        }
      }
      __syncthreads();
    }
    return at;
  }
  // This thread's 16 columns of a row, zeros where there are none.
  __device__ __forceinline__ void read(const uint8_t* at, int t, int r, int batch, uint4 (&raw)[kRingPairs / kPairs<T>]) const {
    const uint8_t* image = at + (r * kTensors + t) * row_bytes;
    constexpr int kVec = 2 * kPairs<T>, kCount = kRingPairs / kPairs<T>;
    if constexpr (kWhole) {
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        raw[i] = v * kVec < cols ? reinterpret_cast<const uint4*>(image)[v] : make_uint4(0, 0, 0, 0);
      }
    } else {
      const Raw<T, 1>* row = reinterpret_cast<const Raw<T, 1>*>(image + (reinterpret_cast<uintptr_t>(row_of(t, batch * kRows + r)) & 15u));
      uint32_t words[kCount * 4];
#pragma unroll
      for (int e = 0; e < kRingElems; ++e) {
        const int c = threadIdx.x + e * blockDim.x;
        const uint32_t bits = c < cols ? row[c] : 0;
        if constexpr (sizeof(T) == 4) words[e] = bits;
        else if (e & 1) words[e / 2] |= bits << 16;
        else words[e / 2] = bits;
      }
#pragma unroll
      for (int i = 0; i < kCount; ++i) raw[i] = make_uint4(words[4 * i], words[4 * i + 1], words[4 * i + 2], words[4 * i + 3]);
    }
  }
  // Behind a barrier that every thread reached after its reads of the stage and a fence_proxy_async_smem.
  __device__ __forceinline__ void refill(int batch) {
    const int ahead = stages * gridDim.x;
    if (threadIdx.x == 0 && ahead < batches - batch) fetch(batch + ahead, stage);
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  __device__ __forceinline__ void finish() const {
    if (*abort_flag != 0) __nanosleep(2000000);      // copies still in flight land before their shared memory is released
  }
};

// The column of a thread's element e (pair e / 2): kWhole, element e % kVec of vector thread + (e / kVec) * threads.
template <typename T, bool kWhole>
__device__ __forceinline__ int column_of(int e) {
  constexpr int kVec = 2 * kPairs<T>;
  return kWhole ? (threadIdx.x + e / kVec * blockDim.x) * kVec + e % kVec : threadIdx.x + e * blockDim.x;
}
template <typename T, bool kWhole>
__device__ __forceinline__ void write_row(T* row, int cols, const uint64_t (&p)[kRingPairs]) {
  constexpr int kN = kPairs<T>;
  if constexpr (kWhole) {
#pragma unroll
    for (int i = 0; i < kRingPairs / kN; ++i) {
      uint64_t part[kN];
#pragma unroll
      for (int j = 0; j < kN; ++j) part[j] = p[i * kN + j];
      const int v = threadIdx.x + i * blockDim.x;
      if (v * 2 * kN < cols) reinterpret_cast<uint4*>(row)[v] = pack_pairs<T>(part);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kRingPairs; ++j) {
      float f[2];
      ptx::f32x2_split(p[j], f[0], f[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c = column_of<T, false>(2 * j + k);
        if (c < cols) row[c] = from_float<T>(f[k]);
      }
    }
  }
}
template <typename T, typename P, bool kWhole>
__device__ __forceinline__ void ring_params(const void* p, int cols, bool vec, float offset, float none, uint64_t (&out)[kRingPairs]) {
  constexpr int kN = kPairs<T>;
  if constexpr (kWhole) {
#pragma unroll
    for (int i = 0; i < kRingPairs / kN; ++i) {
      uint64_t part[kN] = {};
      const int c = column_of<T, true>(2 * kN * i);
      if (c < cols) load_params<P, kN>(p, c, vec, offset, none, part);
#pragma unroll
      for (int j = 0; j < kN; ++j) out[i * kN + j] = part[j];
    }
  } else {
    const P* at = static_cast<const P*>(p);
#pragma unroll
    for (int j = 0; j < kRingPairs; ++j) {      // (a column behind the last one is never used)
      const int c = min(column_of<T, false>(2 * j), cols - 1), d = min(column_of<T, false>(2 * j + 1), cols - 1);
      out[j] = p == nullptr ? ptx::f32x2(none, none) : ptx::f32x2(offset + to_float<P>(at[c]), offset + to_float<P>(at[d]));
    }
  }
}

template <typename T, typename P, int kRows, bool kWhole>
__global__ void __launch_bounds__(kRingThreads, 1) row_norm_fwd_ring_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t data[];
  __shared__ alignas(8) uint64_t full[kMaxStages];
  __shared__ float scratch[2][kRows][16];
  __shared__ int abort_flag;
  Ring<T, kRows, 1, kWhole> ring{data, full, &abort_flag, {a.x}, {a.ldx}, static_cast<int>(a.rows), static_cast<int>((a.rows + kRows - 1) / kRows),
                                 a.cols, a.row_bytes, a.stages};
  ring.status_word = a.status_word;
  ring.init();
  ptx::grid_dependency_sync();
  ring.start();
  uint64_t scale[kRingPairs], shift[kRingPairs];
  ring_params<T, P, kWhole>(a.gain, a.cols, a.gain_vec, a.gain_offset, 1.0f, scale);
  ring_params<T, P, kWhole>(a.shift, a.cols, a.shift_vec, 0.0f, 0.0f, shift);
  int turn = 0;
  for (int batch = blockIdx.x; batch < ring.batches; batch += gridDim.x) {      // (rows + gridDim * stages fits an int: check())
    const int there = ring.rows_of(batch);
    const uint8_t* at = ring.wait(batch);
    uint64_t x[kRows][kRingPairs];
    float mean[kRows], s[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      uint64_t t = 0;
      if (r < there) {
        uint4 raw[kRingPairs / kPairs<T>];
        ring.read(at, 0, r, batch, raw);
        unpack_all<T, kRingPairs>(raw, x[r]);
#pragma unroll
        for (int j = 0; j < kRingPairs; ++j) t = ptx::add2(t, x[r][j]);
      }
      mean[r] = pair_sum(t);
    }
    ptx::fence_proxy_async_smem();      // the reads above come before the copy that overwrites them
    if (a.rms) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) mean[r] = 0.0f;
    } else {
      cta_sums<kRows>(mean, scratch[turn ^ 1]);
#pragma unroll
      for (int r = 0; r < kRows; ++r) mean[r] *= a.inv_cols;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      uint64_t t = 0;
      if (r < there) {
        const uint64_t minus = ptx::f32x2(-mean[r], -mean[r]);
#pragma unroll
        for (int j = 0; j < kRingPairs; ++j) {
          x[r][j] = ptx::add2(x[r][j], minus);
          // (columns behind the row's end count nothing; whole vectors end together)
          if (kWhole ? column_of<T, true>(2 * j) < a.cols : column_of<T, false>(2 * j + 1) < a.cols) {
            t = ptx::fma2(x[r][j], x[r][j], t);
          } else if (!kWhole && column_of<T, false>(2 * j) < a.cols) {
            float lo, hi;
            ptx::f32x2_split(x[r][j], lo, hi);
            t = ptx::add2(t, ptx::f32x2(lo * lo, 0.0f));
          }
        }
      }
      s[r] = pair_sum(t);
    }
    cta_sums<kRows>(s, scratch[turn]);
    turn ^= a.rms;      // (LayerNorm's two sums alternate by themselves)
    ring.refill(batch);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r < there) {
        const int64_t row = static_cast<int64_t>(batch) * kRows + r;
        const float rstd = __frsqrt_rn(fmaf(s[r], a.inv_cols, a.eps));
        const uint64_t r2 = ptx::f32x2(rstd, rstd);
#pragma unroll
        for (int j = 0; j < kRingPairs; ++j) x[r][j] = ptx::fma2(ptx::mul2(x[r][j], r2), scale[j], shift[j]);
        write_row<T, kWhole>(static_cast<T*>(a.out) + row * a.ldo, a.cols, x[r]);
        if (threadIdx.x == 0) {
          if (a.mean != nullptr) a.mean[row] = mean[r];
          if (a.rstd != nullptr) a.rstd[row] = rstd;
        }
      }
    }
  }
  ring.finish();
}

template <typename T, typename P, int kRows, bool kWhole>
__global__ void __launch_bounds__(kRingThreads, 1) row_norm_bwd_ring_kernel(const Args a) {
  constexpr int kCount = kRingPairs / kPairs<T>;
  extern __shared__ __align__(16) uint8_t data[];
  __shared__ alignas(8) uint64_t full[kMaxStages];
  __shared__ float scratch[2][2 * kRows][16];
  __shared__ int abort_flag;
  Ring<T, kRows, 2, kWhole> ring{data, full, &abort_flag, {a.x, a.gy}, {a.ldx, a.ldg}, static_cast<int>(a.rows), static_cast<int>((a.rows + kRows - 1) / kRows),
                                 a.cols, a.row_bytes, a.stages};
  ring.status_word = a.status_word;
  ring.init();
  ptx::grid_dependency_sync();
  ring.start();
  uint64_t scale[kRingPairs], dgain[kRingPairs], dshift[kRingPairs];
  ring_params<T, P, kWhole>(a.gain, a.cols, a.gain_vec, a.gain_offset, 1.0f, scale);
#pragma unroll
  for (int j = 0; j < kRingPairs; ++j) dgain[j] = dshift[j] = 0;
  float next_mean[kRows], next_rstd[kRows];
  auto stats = [&](int batch) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool is = batch < ring.batches && r < ring.rows_of(batch);
      next_mean[r] = is && !a.rms ? a.mean[batch * kRows + r] : 0.0f;
      next_rstd[r] = is ? a.rstd[batch * kRows + r] : 0.0f;
    }
  };
  stats(blockIdx.x);
  int turn = 0;
  for (int batch = blockIdx.x; batch < ring.batches; batch += gridDim.x) {      // (rows + gridDim * stages fits an int: check())
    const int there = ring.rows_of(batch);
    float mean[kRows], rstd[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      mean[r] = next_mean[r];
      rstd[r] = next_rstd[r];
    }
    stats(batch + gridDim.x);
    const uint8_t* at = ring.wait(batch);
    uint4 xr[kRows][kCount], gr[kRows][kCount];
    float s[2 * kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      uint64_t hx = 0, hs = 0;
      if (r < there) {      // (behind the row's end grad_y reads 0)
        ring.read(at, 0, r, batch, xr[r]);
        ring.read(at, 1, r, batch, gr[r]);
        bwd_sums<T, kRingPairs>(xr[r], gr[r], mean[r], rstd[r], scale, dgain, dshift, hx, hs);
      }
      s[2 * r] = pair_sum(hx);
      s[2 * r + 1] = pair_sum(hs);
    }
    ptx::fence_proxy_async_smem();      // the reads above come before the copy that overwrites them
    cta_sums<2 * kRows>(s, scratch[turn]);
    turn ^= 1;
    ring.refill(batch);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r < there) {
        const float c1 = s[2 * r] * a.inv_cols, c0 = a.rms ? 0.0f : s[2 * r + 1] * a.inv_cols;
        uint64_t dx[kRingPairs];
        bwd_dx<T, kRingPairs>(xr[r], gr[r], mean[r], rstd[r], scale, c1, c0, dx);
        write_row<T, kWhole>(static_cast<T*>(a.out) + static_cast<int64_t>(batch * kRows + r) * a.ldo, a.cols, dx);
      }
    }
  }
  ring.finish();
  if (a.part_gain == nullptr && a.part_shift == nullptr) return;
  // The sums of a cluster's CTAs leave as one row: each CTA puts its own into the ring's memory and adds up a slice of the
  // columns over all of them.  (Written and read one by one they took 15 of 60 us at 8192 x 4096 bf16.)
  float* mine = reinterpret_cast<float*>(data);      // [2][columns up to a multiple of 4]
  const int pitch = (a.cols + 3) & ~3;
  __syncthreads();                                   // (the ring has been read)
#pragma unroll
  for (int j = 0; j < kRingPairs; ++j) {
    float f[2], g[2];
    ptx::f32x2_split(dgain[j], f[0], f[1]);
    ptx::f32x2_split(dshift[j], g[0], g[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = column_of<T, kWhole>(2 * j + k);
      if (c < a.cols) {
        mine[c] = f[k];
        mine[pitch + c] = g[k];
      }
    }
  }
  ptx::cluster_sync_all();
  const int slice = (pitch / 4 + kCluster - 1) / kCluster, rank = static_cast<int>(ptx::cluster_ctarank());
  const int begin = rank * slice, end = min(begin + slice, pitch / 4);
  const int64_t row = static_cast<int64_t>(blockIdx.x / kCluster) * a.cols;
  uint32_t at[kCluster];
#pragma unroll
  for (int r = 0; r < kCluster; ++r) at[r] = ptx::map_to_cta(ptx::smem_u32(mine), r);
  for (int q = begin + threadIdx.x; q < end; q += blockDim.x) {
    float4 part[2][kCluster];      // (all loads out before the first sum: a load from a neighbour takes long)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < kCluster; ++r) part[t][r] = ptx::ld_shared_cluster_f32x4(at[r] + 4 * (t * pitch + 4 * q));
    float* out[2] = {a.part_gain, a.part_shift};
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float f[4] = {part[t][0].x, part[t][0].y, part[t][0].z, part[t][0].w};
#pragma unroll
      for (int r = 1; r < kCluster; ++r) {
        f[0] += part[t][r].x;
        f[1] += part[t][r].y;
        f[2] += part[t][r].z;
        f[3] += part[t][r].w;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (out[t] != nullptr && 4 * q + k < a.cols) out[t][row + 4 * q + k] = f[k];
    }
  }
  ptx::cluster_sync_all();      // (nobody leaves while its memory is read)
}

// dgain (blockIdx.y 0) and dshift (1): the CTAs' rows of partials added up, kSumCols columns per CTA, every sixteenth row by a
// thread and the threads' sums in a tree: always the same order.  148 rows of 4096: 5 us, a launch and two reads' latency.
__global__ void __launch_bounds__(kSumCols* kSumParts) row_norm_sum_kernel(const float* part_gain, const float* part_shift, int parts,
                                                                          int cols, void* dgain, void* dshift, int dtype) {
  ptx::grid_dependency_sync();
  __shared__ float s[kSumParts][kSumCols];
  const float* part = blockIdx.y == 0 ? part_gain : part_shift;
  void* out = blockIdx.y == 0 ? dgain : dshift;
  if (out == nullptr) return;
  const int lane = threadIdx.x % kSumCols, p0 = threadIdx.x / kSumCols, c = blockIdx.x * kSumCols + lane;
  float t = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int p = p0; p < parts; p += kSumParts) t += part[static_cast<int64_t>(p) * cols + c];
  }
  s[p0][lane] = t;
  __syncthreads();
#pragma unroll
  for (int n = kSumParts / 2; n > 0; n /= 2) {
    if (p0 < n) s[p0][lane] += s[p0 + n][lane];
    __syncthreads();
  }
  if (p0 == 0 && c < cols) {
    t = s[0][lane];
    if (dtype == IXK_F32) static_cast<float*>(out)[c] = t;
    else if (dtype == IXK_BF16) static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(t);
    else static_cast<__half*>(out)[c] = __float2half_rn(t);
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
// Short rows (up to eight elements a lane of a warp) and those that the ring takes.
bool short_rows(int64_t cols) { return cols <= 32 * 8; }
bool vec_takes(int64_t cols, bool whole) { return cols <= kRingThreads * kRingElems && (whole || !short_rows(cols)); }
int ring_threads(int64_t cols) { return static_cast<int>((cols + kRingElems - 1) / kRingElems + 31) / 32 * 32; }
int ring_ctas_per_sm(int threads) { return std::clamp(kRingThreads / threads, 1, 8); }
// (a row that is not whole vectors keeps its place within 16 bytes)
int64_t ring_row_bytes(int64_t cols, int elem_bytes, bool whole) { return whole ? cols * elem_bytes : (cols * elem_bytes + 15) / 16 * 16 + 16; }
// Two rows a batch where every CTA gets two batches and the ring holds three of them.
int ring_rows(int64_t cols, int64_t rows, int elem_bytes, bool bwd) {
  const int ctas = ring_ctas_per_sm(ring_threads(cols));
  return rows >= 4 * kAssumedSms * ctas && 3 * (bwd ? 4 : 2) * ring_row_bytes(cols, elem_bytes, false) <= kRingBytes / ctas ? 2 : 1;
}
int64_t vec_ctas(int64_t cols, int64_t rows, int elem_bytes, bool bwd) {
  if (short_rows(cols)) {
    const int64_t warps = (rows + 3) / 4;      // (four rows of 16-bit elements a warp, or more)
    return bwd ? std::min<int64_t>((warps + 7) / 8, kAssumedSms * 2) : std::min<int64_t>((warps + 3) / 4, kAssumedSms * 8);
  }
  const int batch = ring_rows(cols, rows, elem_bytes, bwd);
  const int64_t ctas = std::min<int64_t>((rows + batch - 1) / batch, static_cast<int64_t>(kAssumedSms) * ring_ctas_per_sm(ring_threads(cols)));
  return bwd ? (ctas + kCluster - 1) / kCluster * kCluster : ctas;
}
int64_t ctas_for(const Plan& p, int64_t rows) {
  const int64_t want = (rows + p.groups_per_cta - 1) / p.groups_per_cta;
  return std::min<int64_t>(want, static_cast<int64_t>(kAssumedSms) * std::max(1, kThreadsPerSm / p.threads));
}

template <typename T, bool kBwd>
int launch(const Plan& p, const Args& a, int64_t ctas, cudaStream_t stream) {
  auto go = [&](auto vec, auto per, auto warp) -> int {
    constexpr int kVec = decltype(vec)::value, kPer = decltype(per)::value;
    constexpr bool kWarp = decltype(warp)::value;
    auto* fn = &row_norm_fwd_kernel<T, kVec, kPer, kWarp>;
    if constexpr (kBwd) fn = &row_norm_bwd_kernel<T, kVec, kPer, kWarp>;
    size_t smem = kBwd && kWarp ? 2 * sizeof(float) * a.cols : 0;
    if constexpr (!kAhead<T, kVec, kWarp, kBwd>) {
      smem = (kBwd ? 1 : 2) * sizeof(float) * a.cols;
      static thread_local int configured_device = -1;
      int dev = 0;
      IXK_CUDA_OK(cudaGetDevice(&dev));
      if (configured_device != dev) {
        IXK_CUDA_OK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(2 * sizeof(float) * kMaxCols)));
        configured_device = dev;
      }
    }
    return launch_overlapped(fn, dim3(ctas), dim3(p.threads), smem, stream, a);
  };
  constexpr int kFull = 16 / sizeof(T);
#define IXK_NORM_CASE(V, P, W) \
  if (p.vec == V && p.per == P && p.warp == W) return go(std::integral_constant<int, V>{}, std::integral_constant<int, P>{}, std::bool_constant<W>{});
  IXK_NORM_CASE(kFull, 16 / kFull, false)
  IXK_NORM_CASE(1, 1, true)
  IXK_NORM_CASE(1, 2, true)
  IXK_NORM_CASE(1, 4, true)
  IXK_NORM_CASE(1, 8, true)
  IXK_NORM_CASE(1, 16, false)
#undef IXK_NORM_CASE
  return fail(IXK_UNIMPLEMENTED, "row_norm: no kernel for this row");
}

// Short rows of whole vectors by the warp, longer rows of any kind by the ring.
template <typename T, typename P, bool kBwd>
int launch_vec(Args a, bool whole, int64_t ctas, cudaStream_t stream) {
  if (short_rows(a.cols)) {
    constexpr int kPer = sizeof(T) / 2;
    if constexpr (kBwd)
      return launch_overlapped(row_norm_bwd_rows_kernel<T, P, kPer, 4 / kPer>, dim3(static_cast<unsigned>(ctas)), dim3(256), 2 * sizeof(float) * a.cols, stream, a);
    else
      return launch_overlapped(row_norm_fwd_rows_kernel<T, P, kPer, 8 / kPer>, dim3(static_cast<unsigned>(ctas)), dim3(128), 0, stream, a);
  }
  auto go = [&](auto rows_tag, auto whole_tag) -> int {
    constexpr int kRows = decltype(rows_tag)::value;
    constexpr bool kWhole = decltype(whole_tag)::value;
    auto* fn = &row_norm_fwd_ring_kernel<T, P, kRows, kWhole>;
    if constexpr (kBwd) fn = &row_norm_bwd_ring_kernel<T, P, kRows, kWhole>;
    a.row_bytes = static_cast<uint32_t>(ring_row_bytes(a.cols, sizeof(T), kWhole));
    const int threads = ring_threads(a.cols), stage = (kBwd ? 2 : 1) * kRows * static_cast<int>(a.row_bytes);
    a.stages = std::min(kMaxStages, kRingBytes / ring_ctas_per_sm(threads) / stage);
    static thread_local int configured_device = -1;
    int dev = 0;
    IXK_CUDA_OK(cudaGetDevice(&dev));
    if (configured_device != dev) {
      IXK_CUDA_OK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes));
      configured_device = dev;
    }
    const size_t smem = std::max(static_cast<size_t>(a.stages) * stage, kBwd ? 2 * sizeof(float) * ((a.cols + 3) / 4 * 4) : 0);
    if constexpr (!kBwd) return launch_overlapped(fn, dim3(static_cast<unsigned>(ctas)), dim3(threads), smem, stream, a);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kCluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    IXK_CUDA_OK(cudaLaunchKernelEx(&cfg, fn, static_cast<const Args>(a)));
    count_launch();
    return IXK_OK;
  };
  const bool two = ring_rows(a.cols, a.rows, sizeof(T), kBwd) == 2;
  constexpr std::integral_constant<int, 1> kOne;
  constexpr std::integral_constant<int, 2> kTwo;
  if (whole) return two ? go(kTwo, std::true_type{}) : go(kOne, std::true_type{});
  return two ? go(kTwo, std::false_type{}) : go(kOne, std::false_type{});
}

// call(a value of the rows' type, one of the parameters')
template <typename Call>
int with_types(int dtype, int param_dtype, const Call& call) {
  if (dtype == IXK_F32) return call(float{}, float{});
  if (dtype == IXK_BF16) return param_dtype == IXK_F32 ? call(__nv_bfloat16{}, float{}) : call(__nv_bfloat16{}, __nv_bfloat16{});
  return param_dtype == IXK_F32 ? call(__half{}, float{}) : call(__half{}, __half{});
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
  if (d->rows > (1 << 30)) return fail(IXK_UNIMPLEMENTED, who + "more than 2^30 rows");
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
  a.gain_vec = aligned(gain, 16);
  a.shift_vec = aligned(shift, 16);
  a.status_word = info.status_word;
  const bool whole = wide && d->cols * es % 16 == 0;
  if (vec_takes(d->cols, whole))
    return with_types(d->dtype, d->param_dtype, [&](auto t, auto pt) {
      return launch_vec<decltype(t), decltype(pt), false>(a, whole, vec_ctas(d->cols, d->rows, es, false), static_cast<cudaStream_t>(stream));
    });
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
  const int64_t ctas = std::max({ctas_for(plan_for(d->cols, es, true), d->rows), ctas_for(plan_for(d->cols, es, false), d->rows),
                                 vec_ctas(d->cols, d->rows, es, true)});
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
  const bool whole = wide && d->cols * es % 16 == 0, vec = vec_takes(d->cols, whole);
  const int64_t ctas = vec ? vec_ctas(d->cols, d->rows, es, true) : ctas_for(p, d->rows);
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
  a.gain_vec = aligned(gain, 16);
  a.status_word = info.status_word;
  if (d->rows > 0 && vec) {
    rc = with_types(d->dtype, d->param_dtype, [&](auto t, auto pt) { return launch_vec<decltype(t), decltype(pt), true>(a, whole, ctas, s); });
    if (rc != IXK_OK) return rc;
  } else if (d->rows > 0) {
    rc = d->dtype == IXK_F32 ? launch<float, true>(p, a, ctas, s)
         : d->dtype == IXK_BF16 ? launch<__nv_bfloat16, true>(p, a, ctas, s) : launch<__half, true>(p, a, ctas, s);
    if (rc != IXK_OK) return rc;
  }
  if (!params) return IXK_OK;
  return launch_overlapped(row_norm_sum_kernel, dim3(static_cast<unsigned>((d->cols + kSumCols - 1) / kSumCols), 2), dim3(kSumCols * kSumParts),
                           0, s, static_cast<const float*>(a.part_gain), static_cast<const float*>(a.part_shift),
                           static_cast<int>(vec && !short_rows(d->cols) ? ctas / kCluster : ctas), a.cols,
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
