// RMSNorm of every query and key head and the position rotation in one pass, into a dense tensor or into the pages of a
// key/value cache, and the gradient.
//
// A head's H elements lie in G lanes of 8 (G = 8, 16 or 32), a warp holds 32 / G heads.  With r = 1 / sqrt(mean(x^2) + eps),
// w = gain_offset + gain and R the rotation by the token's angles:
//   y = R (x r w).  An element's pair lies in the same lane (interleaved) or in the lane H_rot / 16 away (half-split), whose
//   unscaled x comes by shuffle.  r is the head's, so y_i = r (a_i x_i + b_i x_pair), with a = w cos and b = -+ w_pair sin the
//   same for all heads of a token: made once per warp.
//   backward: g~ = R^T g, h = g~ w, dx = r (h - x r^2 mean(h x)), dgain = sum of g~ x r.
// Bound by HBM: every head read and written once (64 lanes' worth of arithmetic per 16 bytes stays under the memory's time).
// r is made again from x in the backward pass, which reads x anyway: nothing is kept.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "paged.h"
#include "ptx.cuh"

namespace ixk {
namespace qk {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBwdCtas = 148 * 4;

struct Args {
  int heads, kv_heads, rotary_chunks;   // 8-element chunks of a head that rotate
  int head_chunks;                      // and of the head
  int interleaved, wide_positions;
  int param_fp32;
  float eps, gain_offset, inv_size;
  int64_t tokens, places;
  int64_t q_strides[2], k_strides[2], v_strides[2], qo_strides[2], ko_strides[2], gq_strides[2], gk_strides[2];   // in elements
  const void *q, *k, *v, *gq, *gk, *q_gain, *k_gain;
  const float *cos_t, *sin_t;
  const void* positions;
  void *qo, *ko;                        // outputs, or dq and dk
  paged::CacheArgs cache;
  const int* slots;                     // nullptr: k to ko
  int q_segments, kv_segments, v_segments, rows_per_warp;   // forward: a warp's share of a token's heads
  float* partial;                       // backward: [CTA][2][256]
  int with_gains;
};

// Eight elements of a head as floats, and back with one rounding.
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  uint4 w;
  __device__ __forceinline__ void load(const void* base, int64_t element) { w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + element); }
  __device__ __forceinline__ void store(void* base, int64_t element) const { *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + element) = w; }
  __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(words[i] << 16);
      f[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    uint32_t words[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      words[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    w = make_uint4(words[0], words[1], words[2], words[3]);
  }
  __device__ __forceinline__ Vec from_lane(int lane) const {
    Vec v;
    v.w.x = __shfl_sync(0xffffffffu, w.x, lane);
    v.w.y = __shfl_sync(0xffffffffu, w.y, lane);
    v.w.z = __shfl_sync(0xffffffffu, w.z, lane);
    v.w.w = __shfl_sync(0xffffffffu, w.w, lane);
    return v;
  }
};
template <>
struct Vec<__half> : Vec<__nv_bfloat16> {
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&words[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    uint32_t words[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      words[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    w = make_uint4(words[0], words[1], words[2], words[3]);
  }
  __device__ __forceinline__ Vec from_lane(int lane) const {
    Vec v;
    static_cast<Vec<__nv_bfloat16>&>(v) = Vec<__nv_bfloat16>::from_lane(lane);
    return v;
  }
};
template <>
struct Vec<float> {
  float v[8];
  __device__ __forceinline__ void load(const void* base, int64_t element) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + element);
    const float4 a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  __device__ __forceinline__ void store(void* base, int64_t element) const {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + element);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = v[i];
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f[i];
  }
  __device__ __forceinline__ Vec from_lane(int lane) const {
    Vec r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = __shfl_sync(0xffffffffu, v[i], lane);
    return r;
  }
};

__device__ __forceinline__ int64_t position_of(const Args& a, int64_t token) {
  if (a.positions == nullptr) return token % a.places;
  return a.wide_positions ? static_cast<const int64_t*>(a.positions)[token] : static_cast<const int*>(a.positions)[token];
}

// gain_offset + gain of a lane's eight columns (chunk < head_chunks)
template <typename T>
__device__ __forceinline__ void load_weights(const Args& a, const void* gain, int chunk, bool there, float (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.0f;
  if (gain == nullptr || !there) return;
  if (a.param_fp32) {
    Vec<float> v;
    v.load(gain, chunk * 8);
    v.get(w);
  } else {
    Vec<T> v;
    v.load(gain, chunk * 8);
    v.get(w);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] += a.gain_offset;
}

// A lane's place in its head and the angles of its elements.
struct Turn {
  bool there;        // the lane holds elements of the head
  bool turns, second;   // they rotate; half-split: they are second of their pairs
  int pair_lane;     // half-split: where the others are (the lane itself where nothing rotates)
  int chunk;
};
template <int kLanes>
__device__ __forceinline__ Turn turn_of(const Args& a, int lane) {
  Turn t;
  t.chunk = lane & (kLanes - 1);
  t.there = t.chunk < a.head_chunks;
  t.turns = t.chunk < a.rotary_chunks;
  const int half = a.rotary_chunks >> 1;
  t.second = !a.interleaved && t.turns && t.chunk >= half;
  t.pair_lane = a.interleaved || !t.turns ? lane : t.second ? lane - half : lane + half;
  return t;
}
// c and s of the lane's eight elements: y_i = c_i u_i + s_i u_pair(i).  (Interleaved: the pair is the neighbour.)
__device__ __forceinline__ void load_angles(const Args& a, const Turn& t, int64_t place, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
  }
  if (!t.turns) return;
  const int half = a.rotary_chunks >> 1;
  if (a.interleaved) {
    const int64_t at = (place * a.rotary_chunks + t.chunk) * 4;
    const float4 cs = *reinterpret_cast<const float4*>(a.cos_t + at), sn = *reinterpret_cast<const float4*>(a.sin_t + at);
    const float cv[4] = {cs.x, cs.y, cs.z, cs.w}, sv[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[2 * i] = c[2 * i + 1] = cv[i];
      s[2 * i] = -sv[i];
      s[2 * i + 1] = sv[i];
    }
  } else {
    const int64_t at = (place * half + (t.second ? t.chunk - half : t.chunk)) * 8;
    Vec<float> cv, sv;
    cv.load(a.cos_t, at);
    sv.load(a.sin_t, at);
    cv.get(c);
    sv.get(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = t.second ? s[i] : -s[i];
  }
}

template <int kLanes>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The elements that pair with a lane's eight.
template <typename T>
__device__ __forceinline__ void pairs_of(const Args& a, const Vec<T>& v, const float (&x)[8], int pair_lane, float (&p)[8]) {
  if (a.interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = x[i ^ 1];
  } else {
    v.from_lane(pair_lane).get(p);
  }
}

constexpr int kUnroll = 4;   // heads of a lane in flight

template <typename T, int kLanes>
__global__ void __launch_bounds__(kThreads) forward_kernel(const __grid_constant__ Args a) {
  ptx::grid_dependency_sync();
  constexpr int kGroups = 32 / kLanes;
  const int lane = threadIdx.x & 31;
  const int segments = a.q_segments + a.kv_segments + a.v_segments;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t token = w / segments;
  if (token >= a.tokens) return;
  int segment = static_cast<int>(w - token * segments);
  const int64_t place = position_of(a, token);
  if (place < 0 || place >= a.places) return;
  const bool is_q = segment < a.q_segments;
  const bool is_v = segment >= a.q_segments + a.kv_segments;
  if (!is_q) segment -= is_v ? a.q_segments + a.kv_segments : a.q_segments;
  const int heads = is_q ? a.heads : a.kv_heads;
  const int head0 = segment * a.rows_per_warp, head1 = min(head0 + a.rows_per_warp, heads);
  const Turn t = turn_of<kLanes>(a, lane);

  const void* in = is_q ? a.q : is_v ? a.v : a.k;
  const int64_t in_head = is_q ? a.q_strides[1] : is_v ? a.v_strides[1] : a.k_strides[1];
  const int64_t in_at = token * (is_q ? a.q_strides[0] : is_v ? a.v_strides[0] : a.k_strides[0]) + t.chunk * 8;
  void* out;
  int64_t out_head, out_at;
  if (is_q || a.slots == nullptr) {
    out = is_q ? a.qo : a.ko;
    out_head = is_q ? a.qo_strides[1] : a.ko_strides[1];
    out_at = token * (is_q ? a.qo_strides[0] : a.ko_strides[0]) + t.chunk * 8;
  } else {
    const int slot = a.slots[token];
    const unsigned page = static_cast<unsigned>(slot) / static_cast<unsigned>(a.cache.page_size);
    if (slot < 0 || page >= static_cast<unsigned>(a.cache.pages)) return;
    const int in_page = slot - static_cast<int>(page) * a.cache.page_size;
    const paged::CacheArgs& c = a.cache;
    out = is_v ? c.v : c.k;
    out_head = (is_v ? c.v_head : c.k_head) * 8;
    out_at = (is_v ? page * c.v_page + in_page * c.v_token : page * c.k_page + in_page * c.k_token) * 8 + t.chunk * 8;
  }
  if (is_v) {
    for (int h0 = head0 + lane / kLanes; h0 < head1; h0 += kGroups * kUnroll) {
      Vec<T> x[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (h0 + u * kGroups < head1 && t.there) x[u].load(in, in_at + (h0 + u * kGroups) * in_head);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (h0 + u * kGroups < head1 && t.there) x[u].store(out, out_at + (h0 + u * kGroups) * out_head);
    }
    return;
  }
  float c[8], s[8];
  load_angles(a, t, place, c, s);
  {
    float g[8], gp[8];
    load_weights<T>(a, is_q ? a.q_gain : a.k_gain, t.chunk, t.there, g);
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) gp[i] = g[i ^ 1];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) gp[i] = __shfl_sync(0xffffffffu, g[i], t.pair_lane);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] *= g[i];
      s[i] *= gp[i];
    }
  }
  for (int h0 = head0; h0 < head1; h0 += kGroups * kUnroll) {     // (uniform in the warp: shuffles)
    const int mine = h0 + lane / kLanes;
    Vec<T> x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      x[u].zero();
      if (mine + u * kGroups < head1 && t.there) x[u].load(in, in_at + (mine + u * kGroups) * in_head);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (h0 + u * kGroups >= head1) break;
      float f[8], p[8];
      x[u].get(f);
      float sq = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sq = fmaf(f[i], f[i], sq);
      const float r = rsqrtf(head_sum<kLanes>(sq) * a.inv_size + a.eps);
      pairs_of<T>(a, x[u], f, t.pair_lane, p);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = r * fmaf(f[i], c[i], t.turns ? p[i] * s[i] : 0.0f);
      if (mine + u * kGroups < head1 && t.there) {
        x[u].set(f);
        x[u].store(out, out_at + (mine + u * kGroups) * out_head);
      }
    }
  }
}

// A CTA's warps walk the tokens; each lane sums the gains' gradients of its eight columns in registers, q's and k's apart,
// then the CTA's lanes of the same columns are added in order and leave as one row of partial sums.
template <typename T, int kLanes>
__global__ void __launch_bounds__(kThreads) backward_kernel(const __grid_constant__ Args a) {
  ptx::grid_dependency_sync();
  constexpr int kGroups = 32 / kLanes;
  constexpr int kUnroll = 2;
  __shared__ float sums[kWarps * kGroups][kLanes * 8 + 4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Turn t = turn_of<kLanes>(a, lane);
  float acc[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[0][i] = acc[1][i] = 0.0f;
  const int segments = a.q_segments + a.kv_segments;
  const int64_t units = a.tokens * segments;
  auto heads_of = [&](auto k_tag, int64_t token, int segment, const float (&c)[8], const float (&s)[8], bool valid) {
    constexpr int which = decltype(k_tag)::value;
    const void* x_in = which ? a.k : a.q;
    const void* g_in = which ? a.gk : a.gq;
    void* out = which ? a.ko : a.qo;
    const int64_t* xs = which ? a.k_strides : a.q_strides;
    const int64_t* gs = which ? a.gk_strides : a.gq_strides;
    const int64_t* os = which ? a.ko_strides : a.qo_strides;
    const int heads = which ? a.kv_heads : a.heads;
    const int head0 = segment * a.rows_per_warp, head1 = min(head0 + a.rows_per_warp, heads);
    const int64_t x_at = token * xs[0] + t.chunk * 8, g_at = token * gs[0] + t.chunk * 8, o_at = token * os[0] + t.chunk * 8;
    float wgt[8];
    load_weights<T>(a, which ? a.k_gain : a.q_gain, t.chunk, t.there, wgt);
    for (int h0 = head0; h0 < head1; h0 += kGroups * kUnroll) {
      const int mine = h0 + lane / kLanes;
      Vec<T> x[kUnroll], g[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        x[u].zero();
        g[u].zero();
        if (valid && mine + u * kGroups < head1 && t.there) {
          x[u].load(x_in, x_at + (mine + u * kGroups) * xs[1]);
          g[u].load(g_in, g_at + (mine + u * kGroups) * gs[1]);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (h0 + u * kGroups >= head1) break;
        const bool mine_there = mine + u * kGroups < head1 && t.there;
        float f[8], h[8], p[8];
        x[u].get(f);
        g[u].get(h);
        pairs_of<T>(a, g[u], h, t.pair_lane, p);
        float sq = 0.0f, hx = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h[i] = fmaf(h[i], c[i], t.turns ? -p[i] * s[i] : 0.0f);      // turned back
          sq = fmaf(f[i], f[i], sq);
          hx = fmaf(h[i] * wgt[i], f[i], hx);
        }
        const float square = head_sum<kLanes>(sq);
        // (0 for a row that is left out: with eps 0 its root would be infinite)
        const float r = valid && mine + u * kGroups < head1 ? rsqrtf(square * a.inv_size + a.eps) : 0.0f;
        const float m = head_sum<kLanes>(hx) * a.inv_size * r * r;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[which][i] = fmaf(h[i] * r, f[i], acc[which][i]);
          h[i] = r * (h[i] * wgt[i] - f[i] * m);
        }
        if (mine_there) {
          g[u].set(h);
          g[u].store(out, o_at + (mine + u * kGroups) * os[1]);
        }
      }
    }
  };
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + warp; unit < units; unit += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t token = unit / segments;
    const int segment = static_cast<int>(unit - token * segments);
    const int64_t place = position_of(a, token);
    const bool valid = place >= 0 && place < a.places;
    float c[8], s[8];
    load_angles(a, t, valid ? place : 0, c, s);
    if (segment < a.q_segments) heads_of(std::integral_constant<int, 0>{}, token, segment, c, s, valid);
    else heads_of(std::integral_constant<int, 1>{}, token, segment - a.q_segments, c, s, valid);
  }
  if (!a.with_gains) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
    float* row = sums[warp * kGroups + lane / kLanes] + t.chunk * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) row[i] = acc[which][i];
    __syncthreads();
    if (threadIdx.x < kLanes * 8) {
      float v = 0.0f;
#pragma unroll 4
      for (int i = 0; i < kWarps * kGroups; ++i) v += sums[i][threadIdx.x];
      a.partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * 256 + threadIdx.x] = v;
    }
  }
}

// The CTAs' rows of partial sums added up: 32 columns a CTA, 32 threads a column, then a tree over them.
template <typename T>
__global__ void __launch_bounds__(1024) gains_kernel(const float* partial, int rows, int size, void* dq_gain, void* dk_gain, int param_fp32) {
  ptx::grid_dependency_sync();
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = (size + 31) / 32;
  const int which = blockIdx.x / blocks, column = (blockIdx.x - which * blocks) * 32 + lane;
  float v = 0.0f;
  if (column < size)
    for (int r = warp; r < rows; r += 32) v += partial[(static_cast<int64_t>(r) * 2 + which) * 256 + column];
  part[lane][warp] = v;
  __syncthreads();
  v = part[warp][lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  void* out = which ? dk_gain : dq_gain;
  const int c = (blockIdx.x - which * blocks) * 32 + warp;
  if (lane == 0 && c < size && out != nullptr) {
    if (param_fp32) static_cast<float*>(out)[c] = v;
    else static_cast<T*>(out)[c] = static_cast<T>(v);
  }
}

int check(const ixk_qk_desc* d, const char* who) {
  const std::string at(who);
  if (d == nullptr) return fail(IXK_INVALID_ARGUMENT, at + ": desc is NULL");
  if (d->dtype != IXK_BF16 && d->dtype != IXK_F16 && d->dtype != IXK_F32) return fail(IXK_UNIMPLEMENTED, at + ": dtype must be BF16, F16 or F32");
  if (d->param_dtype != d->dtype && d->param_dtype != IXK_F32) return fail(IXK_UNIMPLEMENTED, at + ": gains must have dtype or be F32");
  if (d->tokens < 0 || d->heads < 1 || d->kv_heads < 1 || d->places < 1)
    return fail(IXK_INVALID_ARGUMENT, at + ": heads and places must be positive, tokens not negative");
  if (d->head_size < 8 || d->head_size % 8 != 0 || d->head_size > 256)
    return fail(IXK_UNIMPLEMENTED, at + ": head_size must be a multiple of 8, at most 256");
  if (d->rotary_dim < 1 || d->rotary_dim > d->head_size || d->rotary_dim % (d->interleaved ? 8 : 16) != 0)
    return fail(IXK_INVALID_ARGUMENT, at + ": rotary_dim must be a multiple of 16 (interleaved: 8) elements, at most head_size");
  if (d->position_bytes != 4 && d->position_bytes != 8) return fail(IXK_INVALID_ARGUMENT, at + ": position_bytes must be 4 or 8");
  if (!(d->eps >= 0.0f) || d->gain_offset != d->gain_offset) return fail(IXK_INVALID_ARGUMENT, at + ": eps must not be negative or NaN");
  if (d->heads > 65536 || d->kv_heads > 65536 || d->tokens > 0x7fffffff) return fail(IXK_UNIMPLEMENTED, at + ": too many heads or tokens");
  return IXK_OK;
}
// Strides of a tensor: multiples of eight elements; of one that is written, rows must not overlap.
int check_strides(const int64_t (&s)[2], int64_t tokens, int64_t heads, int size, bool written, const char* who, const char* name) {
  const std::string at = std::string(who) + ": " + name;
  if (s[0] % 8 != 0 || s[1] % 8 != 0) return fail(IXK_INVALID_ARGUMENT, at + ": strides must be multiples of 8 elements");
  if (s[0] < 0 || s[1] < 0) return fail(IXK_INVALID_ARGUMENT, at + ": negative stride");
  if (written && ((tokens > 1 && s[0] < size) || (heads > 1 && s[1] < size))) return fail(IXK_INVALID_ARGUMENT, at + ": rows overlap");
  return IXK_OK;
}

Args base_args(const ixk_qk_desc* d) {
  Args a{};
  a.heads = d->heads;
  a.kv_heads = d->kv_heads;
  a.head_chunks = d->head_size / 8;
  a.rotary_chunks = d->rotary_dim / 8;
  a.interleaved = d->interleaved != 0;
  a.wide_positions = d->position_bytes == 8;
  a.param_fp32 = d->param_dtype == IXK_F32;
  a.eps = d->eps;
  a.gain_offset = d->gain_offset;
  a.inv_size = 1.0f / static_cast<float>(d->head_size);
  a.tokens = d->tokens;
  a.places = d->places;
  for (int i = 0; i < 2; ++i) {
    a.q_strides[i] = d->q_strides[i];
    a.k_strides[i] = d->k_strides[i];
    a.v_strides[i] = d->v_strides[i];
    a.qo_strides[i] = d->q_out_strides[i];
    a.ko_strides[i] = d->k_out_strides[i];
    a.gq_strides[i] = d->gq_strides[i];
    a.gk_strides[i] = d->gk_strides[i];
  }
  return a;
}

int lanes_for(int head_size) { return head_size <= 64 ? 8 : head_size <= 128 ? 16 : 32; }

// Heads that a warp takes: four loads a lane and more where there are tokens enough to fill the GPU, fewer where not.
void split_heads(Args* a, int lanes, int sm_count) {
  const int groups = 32 / lanes;
  int rows = groups * 8;
  while (rows > groups) {
    const int64_t warps = a->tokens * ((a->heads + rows - 1) / rows + (a->kv_heads + rows - 1) / rows);
    if (warps >= static_cast<int64_t>(sm_count) * 32) break;
    rows /= 2;
  }
  a->rows_per_warp = rows;
  a->q_segments = (a->heads + rows - 1) / rows;
  a->kv_segments = (a->kv_heads + rows - 1) / rows;
  a->v_segments = 0;
}

template <template <typename, int> class Launcher, typename... More>
int dispatch(int dtype, int lanes, const More&... more) {
  auto with = [&](auto tag) {
    using T = decltype(tag);
    return lanes == 8 ? Launcher<T, 8>::run(more...) : lanes == 16 ? Launcher<T, 16>::run(more...) : Launcher<T, 32>::run(more...);
  };
  if (dtype == IXK_BF16) return with(__nv_bfloat16{});
  if (dtype == IXK_F16) return with(__half{});
  return with(float{});
}
template <typename T, int kLanes>
struct Forward {
  static int run(const Args& a, unsigned grid, cudaStream_t s) { return launch_overlapped(forward_kernel<T, kLanes>, dim3(grid), dim3(kThreads), 0, s, a); }
};
template <typename T, int kLanes>
struct Backward {
  static int run(const Args& a, unsigned grid, cudaStream_t s) { return launch_overlapped(backward_kernel<T, kLanes>, dim3(grid), dim3(kThreads), 0, s, a); }
};

int64_t backward_ctas(const Args& a) {
  const int64_t units = a.tokens * (a.q_segments + a.kv_segments);
  return std::max<int64_t>(1, std::min<int64_t>((units + kWarps - 1) / kWarps, kMaxBwdCtas));
}

}  // namespace
}  // namespace qk
}  // namespace ixk

using namespace ixk;
using ixk::paged::aligned16;

extern "C" {

int ixk_qk_norm_rotary_fwd(const ixk_qk_desc* d, const void* q, const void* k, const void* v, const void* q_gain, const void* k_gain,
                           const float* cos_table, const float* sin_table, const void* positions, void* q_out, void* k_out,
                           const ixk_paged_cache* cache, const int32_t* slots, void* k_pages, void* v_pages, void* cuda_stream) {
  IXK_API_RANGE("ixk_qk_norm_rotary_fwd");
  clear_error();
  const char* who = "qk_norm_rotary";
  if (int st = qk::check(d, who)) return st;
  const bool paged = cache != nullptr;
  if (paged) {
    if (int st = paged::check_cache(cache, k_pages, v_pages, who)) return st;
    if (cache->dtype != d->dtype || cache->heads != d->kv_heads || cache->head_size != d->head_size)
      return fail(IXK_INVALID_ARGUMENT, "qk_norm_rotary: the cache's type, heads or head_size are not those of k and v");
  }
  if (d->tokens > 0 && (q == nullptr || k == nullptr || cos_table == nullptr || sin_table == nullptr || q_out == nullptr ||
                        (paged ? v == nullptr || slots == nullptr : k_out == nullptr)))
    return fail(IXK_INVALID_ARGUMENT, "qk_norm_rotary: null argument");
  if (int st = qk::check_strides(d->q_strides, d->tokens, d->heads, d->head_size, false, who, "q")) return st;
  if (int st = qk::check_strides(d->k_strides, d->tokens, d->kv_heads, d->head_size, false, who, "k")) return st;
  if (int st = qk::check_strides(d->q_out_strides, d->tokens, d->heads, d->head_size, true, who, "q_out")) return st;
  if (paged) {
    if (int st = qk::check_strides(d->v_strides, d->tokens, d->kv_heads, d->head_size, false, who, "v")) return st;
  } else if (int st = qk::check_strides(d->k_out_strides, d->tokens, d->kv_heads, d->head_size, true, who, "k_out")) {
    return st;
  }
  for (const void* p : {q, k, v, q_gain, k_gain, static_cast<const void*>(cos_table), static_cast<const void*>(sin_table),
                        static_cast<const void*>(q_out), static_cast<const void*>(k_out)})
    if (!aligned16(p)) return fail(IXK_INVALID_ARGUMENT, "qk_norm_rotary: pointers must be 16-byte aligned");
  DeviceInfo info;
  if (int st = get_device_info(&info)) return st;
  if (d->tokens == 0) return IXK_OK;
  qk::Args a = qk::base_args(d);
  a.q = q, a.k = k, a.v = v, a.q_gain = q_gain, a.k_gain = k_gain, a.cos_t = cos_table, a.sin_t = sin_table, a.positions = positions;
  a.qo = q_out, a.ko = k_out;
  const int lanes = qk::lanes_for(d->head_size);
  qk::split_heads(&a, lanes, info.sm_count);
  if (paged) {
    a.cache = paged::cache_args(cache, k_pages, v_pages);
    a.slots = slots;
    a.v_segments = a.kv_segments;
  }
  const int64_t warps = a.tokens * (a.q_segments + a.kv_segments + a.v_segments);
  const int64_t grid = (warps + qk::kWarps - 1) / qk::kWarps;
  if (grid > 0x7fffffff) return fail(IXK_UNIMPLEMENTED, "qk_norm_rotary: too many tokens and heads");
  return qk::dispatch<qk::Forward>(d->dtype, lanes, a, static_cast<unsigned>(grid), static_cast<cudaStream_t>(cuda_stream));
}

size_t ixk_qk_norm_rotary_bwd_workspace_bytes(const ixk_qk_desc* d) {
  if (qk::check(d, "qk_norm_rotary") != IXK_OK) return 0;
  qk::Args a = qk::base_args(d);
  qk::split_heads(&a, qk::lanes_for(d->head_size), 148);
  return static_cast<size_t>(qk::backward_ctas(a)) * 2 * 256 * sizeof(float);
}

int ixk_qk_norm_rotary_bwd(const ixk_qk_desc* d, const void* grad_q, const void* grad_k, const void* q, const void* k, const void* q_gain,
                           const void* k_gain, const float* cos_table, const float* sin_table, const void* positions, void* dq, void* dk,
                           void* dq_gain, void* dk_gain, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  IXK_API_RANGE("ixk_qk_norm_rotary_bwd");
  clear_error();
  const char* who = "qk_norm_rotary backward";
  if (int st = qk::check(d, who)) return st;
  if (d->tokens > 0 && (grad_q == nullptr || grad_k == nullptr || q == nullptr || k == nullptr || cos_table == nullptr || sin_table == nullptr ||
                        dq == nullptr || dk == nullptr))
    return fail(IXK_INVALID_ARGUMENT, "qk_norm_rotary backward: null argument");
  if (int st = qk::check_strides(d->q_strides, d->tokens, d->heads, d->head_size, false, who, "q")) return st;
  if (int st = qk::check_strides(d->k_strides, d->tokens, d->kv_heads, d->head_size, false, who, "k")) return st;
  if (int st = qk::check_strides(d->gq_strides, d->tokens, d->heads, d->head_size, false, who, "grad_q")) return st;
  if (int st = qk::check_strides(d->gk_strides, d->tokens, d->kv_heads, d->head_size, false, who, "grad_k")) return st;
  if (int st = qk::check_strides(d->q_out_strides, d->tokens, d->heads, d->head_size, true, who, "dq")) return st;
  if (int st = qk::check_strides(d->k_out_strides, d->tokens, d->kv_heads, d->head_size, true, who, "dk")) return st;
  for (const void* p : {grad_q, grad_k, q, k, q_gain, k_gain, static_cast<const void*>(cos_table), static_cast<const void*>(sin_table),
                        static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(workspace)})
    if (!aligned16(p)) return fail(IXK_INVALID_ARGUMENT, "qk_norm_rotary backward: pointers must be 16-byte aligned");
  const bool gains = dq_gain != nullptr || dk_gain != nullptr;
  if (gains && (workspace == nullptr || workspace_bytes < ixk_qk_norm_rotary_bwd_workspace_bytes(d)))
    return fail(IXK_WORKSPACE_TOO_SMALL, "qk_norm_rotary backward: workspace_bytes is below ixk_qk_norm_rotary_bwd_workspace_bytes");
  DeviceInfo info;
  if (int st = get_device_info(&info)) return st;
  if (d->tokens == 0 && !gains) return IXK_OK;
  qk::Args a = qk::base_args(d);
  a.q = q, a.k = k, a.gq = grad_q, a.gk = grad_k, a.q_gain = q_gain, a.k_gain = k_gain, a.cos_t = cos_table, a.sin_t = sin_table;
  a.positions = positions, a.qo = dq, a.ko = dk;
  a.partial = static_cast<float*>(workspace);
  a.with_gains = gains;
  const int lanes = qk::lanes_for(d->head_size);
  qk::split_heads(&a, lanes, 148);
  const int ctas = static_cast<int>(qk::backward_ctas(a));
  auto s = static_cast<cudaStream_t>(cuda_stream);
  if (int st = qk::dispatch<qk::Backward>(d->dtype, lanes, a, static_cast<unsigned>(ctas), s)) return st;
  if (!gains) return IXK_OK;
  const dim3 grid(2 * ((d->head_size + 31) / 32));
  const float* partial = a.partial;
  if (d->dtype == IXK_F16 && !a.param_fp32)
    return launch_overlapped(qk::gains_kernel<__half>, grid, dim3(1024), 0, s, partial, ctas, d->head_size, dq_gain, dk_gain, a.param_fp32);
  return launch_overlapped(qk::gains_kernel<__nv_bfloat16>, grid, dim3(1024), 0, s, partial, ctas, d->head_size, dq_gain, dk_gain, a.param_fp32);
}

}  // extern "C"
