// RMSNorm of every query and key head and the position rotation in one pass, into a dense tensor or into the pages of a
// key/value cache, and the gradient.
//
// A head's H elements lie in G lanes of 16 (G = 4, 8 or 16), a warp holds 32 / G heads.  A lane has two chunks of 8 that turn into
// each other (half-split), or any two (interleaved pairs lie inside a chunk; what does not turn), so no element is needed by two
// lanes.  With r = 1 / sqrt(mean(x^2) + eps), w = gain_offset + gain and R the rotation by the token's angles:
//   y = R (x r w):  y_i = r (a_i x_i + b_i x_pair), with a = w cos and b = -+ w_pair sin the same for all heads of a token.
//   backward: g~ = R^T g, h = g~ w, dx = r (h - x r^2 mean(h x)), dgain = sum of g~ x r.
// r is made again from x in the backward pass, which reads x anyway: nothing is kept.
//
// Bound by HBM: every head read and written once.  A warp takes a token (or, where tokens are few, a part of its heads), a few heads a
// lane at a time, and asks for the next ones before it computes those it has; what a token needs once (angles, slot, addresses)
// is shared by all of its heads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "paged.h"
#include "ptx.cuh"

namespace ixk {
namespace qk {

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kForwardCtas = 4;       // on an SM: 128 registers a thread
constexpr int kBackwardCtas = 4;
constexpr int kMaxBwdCtas = 148 * kBackwardCtas;
// Heads of a lane at a time.
template <typename T>
constexpr int kForwardHeads = sizeof(T) == 2 ? 2 : 1;
constexpr int kBackwardHeads = 1;
// Segments of a warp in shared memory or on their way there.
template <typename T>
constexpr int kBackwardStages = sizeof(T) == 2 ? 4 : 2;
constexpr int kForwardStages = 3;

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
  int q_segments, kv_segments, segments;     // stretches of a token's heads: queries, then keys, then values
  int turns, parts;                     // tokens of every warp; warps that share the segments of a token of the last turn
  int64_t rest;                         // tokens of the last turn
  float* partial;                       // backward: [CTA][2][256]
  int with_gains;
};

// Eight elements of a head as four pairs of floats (two operations an instruction on a pair), and back with one rounding.
struct Pairs {
  uint64_t v[4];
};
__device__ __forceinline__ Pairs mul(const Pairs& a, const Pairs& b) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = ptx::mul2(a.v[i], b.v[i]);
  return r;
}
__device__ __forceinline__ Pairs mul(const Pairs& a, float b) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = ptx::mul2(a.v[i], ptx::f32x2(b, b));
  return r;
}
__device__ __forceinline__ Pairs fma(const Pairs& a, const Pairs& b, const Pairs& c) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = ptx::fma2(a.v[i], b.v[i], c.v[i]);
  return r;
}
__device__ __forceinline__ Pairs fma(const Pairs& a, float b, const Pairs& c) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = ptx::fma2(a.v[i], ptx::f32x2(b, b), c.v[i]);
  return r;
}
// The sum of the products.
__device__ __forceinline__ float dot(const Pairs& a, const Pairs& b) {
  uint64_t s = ptx::mul2(a.v[0], b.v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) s = ptx::fma2(a.v[i], b.v[i], s);
  float lo, hi;
  ptx::f32x2_split(s, lo, hi);
  return lo + hi;
}
// Every element's neighbour.
__device__ __forceinline__ Pairs swapped(const Pairs& a) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    ptx::f32x2_split(a.v[i], lo, hi);
    r.v[i] = ptx::f32x2(hi, lo);
  }
  return r;
}

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  uint4 w;
  __device__ __forceinline__ void load(const void* base, int64_t element) { w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + element); }
  __device__ __forceinline__ void store(void* base, int64_t element) const { *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + element) = w; }
  __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void from_shared(const uint4* at) { w = at[0]; }
  __device__ __forceinline__ Pairs get() const {
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    Pairs r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = ptx::f32x2(__uint_as_float(words[i] << 16), __uint_as_float(words[i] & 0xffff0000u));
    return r;
  }
  __device__ __forceinline__ void set(const Pairs& f) {
    uint32_t words[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      ptx::f32x2_split(f.v[i], lo, hi);
      const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
      words[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    w = make_uint4(words[0], words[1], words[2], words[3]);
  }
};
template <>
struct Vec<__half> : Vec<__nv_bfloat16> {
  __device__ __forceinline__ Pairs get() const {
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    Pairs r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&words[i]));
      r.v[i] = ptx::f32x2(p.x, p.y);
    }
    return r;
  }
  __device__ __forceinline__ void set(const Pairs& f) {
    uint32_t words[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      ptx::f32x2_split(f.v[i], lo, hi);
      const __half2 h = __floats2half2_rn(lo, hi);
      words[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    w = make_uint4(words[0], words[1], words[2], words[3]);
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
    float* p = static_cast<float*>(base) + element;
    if ((reinterpret_cast<uintptr_t>(p) & 31u) == 0) {        // (strides are multiples of 32 bytes: all of a tensor's, or none)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
                   "f"(v[5]), "f"(v[6]), "f"(v[7])
                   : "memory");
      return;
    }
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  }
  __device__ __forceinline__ void from_shared(const uint4* at) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 w = at[i * kThreads];
      v[4 * i] = __uint_as_float(w.x), v[4 * i + 1] = __uint_as_float(w.y), v[4 * i + 2] = __uint_as_float(w.z), v[4 * i + 3] = __uint_as_float(w.w);
    }
  }
  __device__ __forceinline__ Pairs get() const {
    Pairs r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = ptx::f32x2(v[2 * i], v[2 * i + 1]);
    return r;
  }
  __device__ __forceinline__ void set(const Pairs& f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) ptx::f32x2_split(f.v[i], v[2 * i], v[2 * i + 1]);
  }
};

// Eight elements on their way to a thread's own places in shared memory (zeros where it has none): nobody else reads them, so the
// thread's own wait is all there is to wait for.  fp32: two copies, each of half of every 32-byte sector, the second out of L1 (with
// stores of whole sectors: 8192 tokens of 16 + 4 heads of 128 forward 42.6 -> 30.3 us, backward 69.5 -> 51.3).
template <typename T>
__device__ __forceinline__ void copy_vec(uint4* to, const T* from, bool there) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
    if constexpr (sizeof(T) == 4) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(to + i * kThreads)), "l"(from + (there ? i * 16 / static_cast<int>(sizeof(T)) : 0)),
                   "r"(there ? 16 : 0)
                   : "memory");
    } else {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(to + i * kThreads)), "l"(from + (there ? i * 16 / static_cast<int>(sizeof(T)) : 0)),
                   "r"(there ? 16 : 0)
                   : "memory");
    }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// gain_offset + gain of eight columns, 1 without a gain
template <typename T>
__device__ __forceinline__ Pairs load_weights(const Args& a, const void* gain, int first, bool there) {
  Pairs w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w.v[i] = ptx::f32x2(1.0f, 1.0f);
  if (gain == nullptr || !there) return w;
  if (a.param_fp32) {
    Vec<float> v;
    v.load(gain, first);
    w = v.get();
  } else {
    Vec<T> v;
    v.load(gain, first);
    w = v.get();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w.v[i] = ptx::add2(w.v[i], ptx::f32x2(a.gain_offset, a.gain_offset));
  return w;
}

template <typename T>
__device__ __forceinline__ float weight_of(const Args& a, const void* gain, int column) {
  if (gain == nullptr || column >= a.head_chunks * 8) return 1.0f;
  return a.gain_offset + (a.param_fp32 ? static_cast<const float*>(gain)[column] : static_cast<float>(static_cast<const T*>(gain)[column]));
}
__device__ __forceinline__ Pairs eight(const float* at) {
  const float4 x = reinterpret_cast<const float4*>(at)[0], y = reinterpret_cast<const float4*>(at)[1];
  Pairs r;
  r.v[0] = ptx::f32x2(x.x, x.y), r.v[1] = ptx::f32x2(x.z, x.w), r.v[2] = ptx::f32x2(y.x, y.y), r.v[3] = ptx::f32x2(y.z, y.w);
  return r;
}

// Chunks that do not turn have no other element's product, not even 0 times it, which is no number where the element is an infinity.
// kWhole: heads that turn from end to end have no such chunks (these selects cost 8192 tokens of 16 + 4 heads of 128 17.7 -> 18.5 us).
template <bool kWhole>
__device__ __forceinline__ Pairs only(const Pairs& a, bool turns) {
  if constexpr (kWhole) return a;
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = turns ? a.v[i] : 0ull;
  return r;
}

// A lane's place in its head: its two chunks (behind the head's last: none).  The lanes' first chunks lie side by side, and the
// second ones, so that a copy or store of the warp is of whole 32-byte sectors.  (Two neighbouring chunks a lane cost interleaved heads
// twice the trips to L2: 8192 tokens of 16 + 4 heads of 128 forward 22.9 -> 16.4 us, backward 40.5 -> 28.9.)
struct Place {
  int a, b;          // first elements
  bool has_a, has_b, turns;
  bool turns_a, turns_b;         // the chunks' elements turn, into each other's or (interleaved) into their neighbours
};
template <int kLanes>
__device__ __forceinline__ Place place_of(const Args& a, int lane) {
  const int i = lane & (kLanes - 1), half = a.interleaved ? 0 : a.rotary_chunks >> 1;
  Place p;
  p.turns = i < half;                                       // (half-split: into each other; what does not turn begins at 2 half)
  const int first = p.turns ? i : half + i, second = p.turns ? i + half : kLanes + i;
  p.a = first * 8;
  p.b = second * 8;
  p.has_a = first < a.head_chunks;
  p.has_b = second < a.head_chunks;
  p.turns_a = a.interleaved ? first < a.rotary_chunks : p.turns;
  p.turns_b = a.interleaved ? second < a.rotary_chunks : p.turns;
  return p;
}

__device__ __forceinline__ int64_t position_of(const Args& a, int64_t token) {
  if (a.positions == nullptr) return token % a.places;
  return a.wide_positions ? static_cast<const int64_t*>(a.positions)[token] : static_cast<const int*>(a.positions)[token];
}
// A lane's cosines and sines: half-split, of its eight pairs; interleaved, of the four pairs of each of its chunks.  What does not
// turn has 1 and 0.
struct Angles {
  float c[8], s[8];
};
template <bool kHalf>
__device__ __forceinline__ Angles load_angles(const Args& a, const Place& p, int64_t place) {
  Angles g;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    g.c[i] = 1.0f;
    g.s[i] = 0.0f;
  }
  if (kHalf && !p.turns) return g;
  const float* c = a.cos_t + place * (a.rotary_chunks * 4);
  const float* s = a.sin_t + place * (a.rotary_chunks * 4);
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const int first = i == 0 ? p.a : p.b;
    if (!kHalf && first >= a.rotary_chunks * 8) continue;
    const int at = kHalf ? p.a + i : first >> 1;
    const float4 cv = *reinterpret_cast<const float4*>(c + at), sv = *reinterpret_cast<const float4*>(s + at);
    g.c[i] = cv.x, g.c[i + 1] = cv.y, g.c[i + 2] = cv.z, g.c[i + 3] = cv.w;
    g.s[i] = sv.x, g.s[i + 1] = sv.y, g.s[i + 2] = sv.z, g.s[i + 3] = sv.w;
  }
  return g;
}
// What a lane's elements are multiplied with: y_i = c_i u_i + s_i u_pair(i).
struct Turn {
  Pairs ca, sa, cb, sb;
};
template <bool kHalf, bool kBack>
__device__ __forceinline__ Turn turn_of(const Angles& g) {
  Turn t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (kHalf) {
      const float s0 = kBack ? -g.s[2 * i] : g.s[2 * i], s1 = kBack ? -g.s[2 * i + 1] : g.s[2 * i + 1];
      t.ca.v[i] = t.cb.v[i] = ptx::f32x2(g.c[2 * i], g.c[2 * i + 1]);
      t.sa.v[i] = ptx::f32x2(-s0, -s1);
      t.sb.v[i] = ptx::f32x2(s0, s1);
    } else {
      const float s0 = kBack ? -g.s[i] : g.s[i], s1 = kBack ? -g.s[4 + i] : g.s[4 + i];
      t.ca.v[i] = ptx::f32x2(g.c[i], g.c[i]);
      t.sa.v[i] = ptx::f32x2(-s0, s0);
      t.cb.v[i] = ptx::f32x2(g.c[4 + i], g.c[4 + i]);
      t.sb.v[i] = ptx::f32x2(-s1, s1);
    }
  }
  return t;
}
// The turn backwards, without weights: half-split, of both chunks by the same angles.
template <bool kHalf, bool kWhole>
struct BackTurn;
template <bool kWhole>
struct BackTurn<true, kWhole> {
  Pairs c, s;
  bool turns;
  __device__ __forceinline__ BackTurn(const Angles& g, const Place& p) : turns(p.turns) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c.v[i] = ptx::f32x2(g.c[2 * i], g.c[2 * i + 1]);
      s.v[i] = ptx::f32x2(g.s[2 * i], g.s[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void operator()(const Pairs& xa, const Pairs& xb, Pairs* ya, Pairs* yb) const {
    Pairs across = mul(only<kWhole>(xa, turns), s);
#pragma unroll
    for (int i = 0; i < 4; ++i) across.v[i] ^= 0x8000000080000000ull;
    *ya = fma(xa, c, mul(only<kWhole>(xb, turns), s));
    *yb = fma(xb, c, across);
  }
};
template <bool kWhole>
struct BackTurn<false, kWhole> {
  Turn t;
  bool turns_a, turns_b;
  __device__ __forceinline__ BackTurn(const Angles& g, const Place& p) : t(turn_of<false, true>(g)), turns_a(p.turns_a), turns_b(p.turns_b) {}
  __device__ __forceinline__ void operator()(const Pairs& xa, const Pairs& xb, Pairs* ya, Pairs* yb) const {
    *ya = fma(xa, t.ca, mul(only<kWhole>(swapped(xa), turns_a), t.sa));
    *yb = fma(xb, t.cb, mul(only<kWhole>(swapped(xb), turns_b), t.sb));
  }
};
template <bool kHalf, bool kWhole>
__device__ __forceinline__ void turn(const Turn& t, const Place& p, const Pairs& xa, const Pairs& xb, Pairs* ya, Pairs* yb) {
  *ya = fma(xa, t.ca, mul(only<kWhole>(kHalf ? xb : swapped(xa), p.turns_a), t.sa));
  *yb = fma(xb, t.cb, mul(only<kWhole>(kHalf ? xa : swapped(xb), p.turns_b), t.sb));
}

template <int kLanes>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A warp's tokens: first, first + step ... in `turns` turns, then, in a last one, segments [seg0, seg1) of the token `last`.
struct Share {
  int64_t first, step, last;
  int turns, seg0, seg1;
  __device__ __forceinline__ int64_t token(int turn) const { return turn < turns ? first + turn * step : last; }
};
__device__ __forceinline__ Share share_of(const Args& a) {
  const unsigned warp = blockIdx.x * kWarps + (threadIdx.x >> 5), parts = a.parts;      // (a token's warps are neighbours)
  const unsigned mine = warp / parts;
  const int part = static_cast<int>(warp - mine * parts);
  Share s;
  s.first = warp;
  s.step = gridDim.x * kWarps;
  s.turns = a.turns;
  s.last = a.turns * s.step + mine;
  s.seg0 = part * a.segments / a.parts;
  s.seg1 = mine < a.rest ? (part + 1) * a.segments / a.parts : 0;
  return s;
}

// All tokens' heads of one kind: a warp walks over its tokens and their segments of this kind (in the last turn [seg0, seg1)), the
// next segments' heads (the next token's, behind the last) on their way to shared memory meanwhile.
enum : int { kQueries = 0, kKeys = 1, kValues = 2 };
template <typename T, int kLanes, bool kHalf, bool kWhole, int kKind>
__device__ __forceinline__ void forward_kind(const Args& a, const Place& p, const Share& share, int seg0, int seg1, uint4* ring) {
  const int turns = share.turns + (seg0 < seg1 ? 1 : 0);
  if (turns == 0) return;
  constexpr int kGroups = 32 / kLanes, kHeads = kForwardHeads<T>, kRows = kGroups * kHeads;
  const int lane = threadIdx.x & 31;
  const T* in = static_cast<const T*>(kKind == kQueries ? a.q : kKind == kKeys ? a.k : a.v);
  const int64_t* strides = kKind == kQueries ? a.q_strides : kKind == kKeys ? a.k_strides : a.v_strides;
  const int heads = kKind == kQueries ? a.heads : a.kv_heads, segments = kKind == kQueries ? a.q_segments : a.kv_segments;
  constexpr int kVec = sizeof(T) / 2 * kThreads;        // places of eight elements
  // the segment that is asked for next, and its stage
  int64_t ahead_token = share.token(0);
  int ahead_turn = 0, ahead_seg = share.turns > 0 ? 0 : seg0, ahead = 0;
  auto ask = [&]() {
    if (ahead_turn < turns) {
      const int head = ahead_seg * kRows + lane / kLanes;
      const T* x = in + ahead_token * strides[0] + head * strides[1];
      uint4* to = ring + ahead * (2 * kHeads * kVec);
#pragma unroll
      for (int i = 0; i < kHeads; ++i, x += kGroups * strides[1]) {
        const bool there = head + i * kGroups < heads;
        copy_vec(to + (2 * i) * kVec, there && p.has_a ? x + p.a : in, there && p.has_a);
        copy_vec(to + (2 * i + 1) * kVec, there && p.has_b ? x + p.b : in, there && p.has_b);
      }
      if (++ahead_seg == (ahead_turn < share.turns ? segments : seg1)) {
        ++ahead_turn;
        ahead_seg = ahead_turn < share.turns ? 0 : seg0;
        ahead_token = share.token(ahead_turn);
      }
    }
    copies_commit();
    if (++ahead == kForwardStages) ahead = 0;
  };
#pragma unroll
  for (int i = 0; i < kForwardStages - 1; ++i) ask();
  int stage = 0;
  int64_t place = position_of(a, share.token(0));
  for (int i_turn = 0; i_turn < turns; ++i_turn) {
    const int64_t token = share.token(i_turn);
    int seg = i_turn < share.turns ? 0 : seg0;
    const int seg_end = i_turn < share.turns ? segments : seg1;
    const bool valid = place >= 0 && place < a.places;
    const int slot = kKind != kQueries && a.slots != nullptr ? a.slots[token] : 0;
    Turn t;
    if (kKind != kValues) {
      t = turn_of<kHalf, false>(load_angles<kHalf>(a, p, valid ? place : 0));
      const void* gain = kKind == kQueries ? a.q_gain : a.k_gain;
      const Pairs wa = load_weights<T>(a, gain, p.a, p.has_a), wb = load_weights<T>(a, gain, p.b, p.has_b);
      t.ca = mul(t.ca, wa);
      t.cb = mul(t.cb, wb);
      t.sa = only<kWhole>(mul(t.sa, kHalf ? wb : swapped(wa)), p.turns_a);
      t.sb = only<kWhole>(mul(t.sb, kHalf ? wa : swapped(wb)), p.turns_b);
    }
    if (i_turn + 1 < turns) place = position_of(a, share.token(i_turn + 1));
    T* y = static_cast<T*>(kKind == kQueries ? a.qo : a.ko);
    int64_t y_head = kKind == kQueries ? a.qo_strides[1] : a.ko_strides[1], y_token = token * (kKind == kQueries ? a.qo_strides[0] : a.ko_strides[0]);
    bool written = valid;
    if (kKind != kQueries && a.slots != nullptr) {
      const paged::CacheArgs& c = a.cache;
      const unsigned page = static_cast<unsigned>(slot) / static_cast<unsigned>(c.page_size);
      const int in_page = slot - static_cast<int>(page) * c.page_size;
      written = valid && slot >= 0 && page < static_cast<unsigned>(c.pages);
      y = reinterpret_cast<T*>(kKind == kKeys ? c.k : c.v);
      y_head = (kKind == kKeys ? c.k_head : c.v_head) * 8;
      y_token = (kKind == kKeys ? page * c.k_page + in_page * c.k_token : page * c.v_page + in_page * c.v_token) * 8;
    }
    int head = seg * kRows + lane / kLanes;
    y += y_token + head * y_head;
    y_head *= kGroups;
    for (; seg < seg_end; ++seg, head += kRows) {
      copies_wait<kForwardStages - 2>();
      Vec<T> xa[kHeads], xb[kHeads];
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        xa[i].from_shared(ring + (stage * 2 * kHeads + 2 * i) * kVec);
        xb[i].from_shared(ring + (stage * 2 * kHeads + 2 * i + 1) * kVec);
      }
      if (++stage == kForwardStages) stage = 0;
      ask();                                                 // into the stage that the segment before this one was read from
#pragma unroll
      for (int i = 0; i < kHeads; ++i, y += y_head) {
        if (seg * kRows + i * kGroups >= heads) break;       // (uniform in the warp: shuffles)
        if (kKind != kValues) {
          const Pairs fa = xa[i].get(), fb = xb[i].get();
          const float r = rsqrtf(head_sum<kLanes>(dot(fa, fa) + dot(fb, fb)) * a.inv_size + a.eps);
          Pairs ya, yb;
          turn<kHalf, kWhole>(t, p, fa, fb, &ya, &yb);
          xa[i].set(mul(ya, r));
          xb[i].set(mul(yb, r));
        }
        if (written && head + i * kGroups < heads) {
          if (p.has_a) xa[i].store(y, p.a);
          if (p.has_b) xb[i].store(y, p.b);
        }
      }
    }
  }
  copies_wait<0>();
}
template <typename T, int kLanes, bool kHalf, bool kWhole>
__global__ void __launch_bounds__(kThreads, kForwardCtas) forward_kernel(const __grid_constant__ Args a) {
  ptx::grid_dependency_sync();
  const Place p = place_of<kLanes>(a, threadIdx.x & 31);
  const Share share = share_of(a);
  __shared__ uint4 ring[kForwardStages * 2 * kForwardHeads<T> * (sizeof(T) / 2) * kThreads];
  uint4* mine = ring + threadIdx.x;
  const int first_k = a.q_segments, first_v = first_k + a.kv_segments;
  forward_kind<T, kLanes, kHalf, kWhole, kQueries>(a, p, share, share.seg0, min(share.seg1, first_k), mine);
  forward_kind<T, kLanes, kHalf, kWhole, kKeys>(a, p, share, max(share.seg0 - first_k, 0), min(share.seg1, first_v) - first_k, mine);
  if (a.slots != nullptr) forward_kind<T, kLanes, kHalf, kWhole, kValues>(a, p, share, max(share.seg0 - first_v, 0), share.seg1 - first_v, mine);
}

// The same for the gradients; each lane sums the gains' gradients of its columns in registers over all tokens of its warp, then the
// lanes of the same columns are added, the CTA's warps in order, and leave as one row of partial sums.  The weights stay in shared
// memory, 16 registers a lane less: what 128 could not hold went to memory in the inner loop, 137 -> 128 us forward and backward.
template <typename T, int kLanes, bool kHalf, bool kWhole, int kKind>
__device__ __forceinline__ void backward_kind(const Args& a, const Place& p, const Share& share, int seg0, int seg1, uint4* ring, const float* weights, float* row) {
  constexpr int kGroups = 32 / kLanes, kHeads = kBackwardHeads, kRows = kGroups * kHeads;
  const int lane = threadIdx.x & 31;
  Pairs acc_a, acc_b;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc_a.v[i] = acc_b.v[i] = 0;
  const int turns = share.turns + (seg0 < seg1 ? 1 : 0);
  if (turns > 0) {
    const T* x_in = static_cast<const T*>(kKind == kQueries ? a.q : a.k);
    const T* g_in = static_cast<const T*>(kKind == kQueries ? a.gq : a.gk);
    T* out = static_cast<T*>(kKind == kQueries ? a.qo : a.ko);
    const int64_t* xs = kKind == kQueries ? a.q_strides : a.k_strides;
    const int64_t* gs = kKind == kQueries ? a.gq_strides : a.gk_strides;
    const int64_t* os = kKind == kQueries ? a.qo_strides : a.ko_strides;
    const int heads = kKind == kQueries ? a.heads : a.kv_heads, segments = kKind == kQueries ? a.q_segments : a.kv_segments;
    constexpr int kVec = sizeof(T) / 2 * kThreads, kStages = kBackwardStages<T>;
    const int64_t o_step = kGroups * os[1];
    struct Heads {
      Vec<T> xa, xb, ga, gb;
    };
    int64_t ahead_token = share.token(0);
    int ahead_turn = 0, ahead_seg = share.turns > 0 ? 0 : seg0, ahead = 0;
    auto ask = [&]() {
      if (ahead_turn < turns) {
        const int head = ahead_seg * kRows + lane / kLanes;
        const T* x = x_in + ahead_token * xs[0] + head * xs[1];
        const T* g = g_in + ahead_token * gs[0] + head * gs[1];
        uint4* to = ring + ahead * (4 * kHeads * kVec);
#pragma unroll
        for (int i = 0; i < kHeads; ++i, x += kGroups * xs[1], g += kGroups * gs[1], to += 4 * kVec) {
          const bool has_a = head + i * kGroups < heads && p.has_a, has_b = head + i * kGroups < heads && p.has_b;
          copy_vec(to, has_a ? x + p.a : x_in, has_a);
          copy_vec(to + kVec, has_b ? x + p.b : x_in, has_b);
          copy_vec(to + 2 * kVec, has_a ? g + p.a : g_in, has_a);
          copy_vec(to + 3 * kVec, has_b ? g + p.b : g_in, has_b);
        }
        if (++ahead_seg == (ahead_turn < share.turns ? segments : seg1)) {
          ++ahead_turn;
          ahead_seg = ahead_turn < share.turns ? 0 : seg0;
          ahead_token = share.token(ahead_turn);
        }
      }
      copies_commit();
      if (++ahead == kStages) ahead = 0;
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) ask();
    int stage = 0;
    int64_t place = position_of(a, share.token(0));
    for (int i_turn = 0; i_turn < turns; ++i_turn) {
      const int64_t token = share.token(i_turn);
      int seg = i_turn < share.turns ? 0 : seg0;
      const int seg_end = i_turn < share.turns ? segments : seg1;
      const bool valid = place >= 0 && place < a.places;
      const BackTurn<kHalf, kWhole> turn_back(load_angles<kHalf>(a, p, valid ? place : 0), p);
      if (i_turn + 1 < turns) place = position_of(a, share.token(i_turn + 1));
      int head = seg * kRows + lane / kLanes;
      T* o = out + token * os[0] + head * os[1];
      for (; seg < seg_end; ++seg, head += kRows) {
        copies_wait<kStages - 2>();
        Heads now[kHeads];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          const uint4* from = ring + (stage * kHeads + i) * 4 * kVec;
          now[i].xa.from_shared(from), now[i].xb.from_shared(from + kVec), now[i].ga.from_shared(from + 2 * kVec), now[i].gb.from_shared(from + 3 * kVec);
        }
        if (++stage == kStages) stage = 0;
        ask();
#pragma unroll
        for (int i = 0; i < kHeads; ++i, o += o_step) {
          if (seg * kRows + i * kGroups >= heads) break;                  // (uniform in the warp: shuffles)
          const Pairs fa = now[i].xa.get(), fb = now[i].xb.get();
          Pairs ha, hb;
          turn_back(now[i].ga.get(), now[i].gb.get(), &ha, &hb);
          const Pairs ua = mul(ha, eight(weights + p.a)), ub = mul(hb, eight(weights + p.b));
          const float square = head_sum<kLanes>(dot(fa, fa) + dot(fb, fb)), along = head_sum<kLanes>(dot(ua, fa) + dot(ub, fb));
          const float r = rsqrtf(square * a.inv_size + a.eps);
          if (head + i * kGroups >= heads) continue;
          if (valid) {
            const float m = -along * a.inv_size * r * r;
            acc_a = fma(mul(ha, r), fa, acc_a);
            acc_b = fma(mul(hb, r), fb, acc_b);
            now[i].ga.set(mul(fma(fa, m, ua), r));
            now[i].gb.set(mul(fma(fb, m, ub), r));
          } else {
            now[i].ga.zero();        // (a token that was left out, whatever it holds)
            now[i].gb.zero();
          }
          if (p.has_a) now[i].ga.store(o, p.a);
          if (p.has_b) now[i].gb.store(o, p.b);
        }
      }
    }
    copies_wait<0>();
  }
  if (!a.with_gains) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[4];
    ptx::f32x2_split(acc_a.v[i], x[0], x[1]);
    ptx::f32x2_split(acc_b.v[i], x[2], x[3]);
#pragma unroll
    for (int o = kLanes; o < 32; o *= 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += __shfl_xor_sync(0xffffffffu, x[e], o);
    }
    if (lane < kLanes && p.has_a) *reinterpret_cast<float2*>(row + p.a + 2 * i) = make_float2(x[0], x[1]);
    if (lane < kLanes && p.has_b) *reinterpret_cast<float2*>(row + p.b + 2 * i) = make_float2(x[2], x[3]);
  }
}
template <typename T, int kLanes, bool kHalf, bool kWhole>
__global__ void __launch_bounds__(kThreads, kBackwardCtas) backward_kernel(const __grid_constant__ Args a) {
  ptx::grid_dependency_sync();
  __shared__ __align__(16) float sums[2][kWarps][kLanes * 16];
  __shared__ uint4 ring[kBackwardStages<T> * 4 * kBackwardHeads * (sizeof(T) / 2) * kThreads];
  __shared__ __align__(16) float weights[2][kLanes * 16];       // gain_offset + gain, of queries and of keys
  for (int i = threadIdx.x; i < 2 * kLanes * 16; i += kThreads) {
    const int kind = i / (kLanes * 16), column = i - kind * (kLanes * 16);
    weights[kind][column] = weight_of<T>(a, kind ? a.k_gain : a.q_gain, column);
  }
  __syncthreads();
  const Place p = place_of<kLanes>(a, threadIdx.x & 31);
  const Share share = share_of(a);
  backward_kind<T, kLanes, kHalf, kWhole, kQueries>(a, p, share, share.seg0, min(share.seg1, a.q_segments), ring + threadIdx.x, weights[0], sums[0][threadIdx.x >> 5]);
  backward_kind<T, kLanes, kHalf, kWhole, kKeys>(a, p, share, max(share.seg0 - a.q_segments, 0), share.seg1 - a.q_segments, ring + threadIdx.x, weights[1], sums[1][threadIdx.x >> 5]);
  if (!a.with_gains) return;
  __syncthreads();           // (the only one: a CTA's warps may have unlike numbers of queries and of keys)
  for (int i = threadIdx.x; i < 2 * a.head_chunks * 8; i += kThreads) {
    const int kind = i >= a.head_chunks * 8, column = i - kind * a.head_chunks * 8;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += sums[kind][w][column];
    a.partial[(static_cast<int64_t>(blockIdx.x) * 2 + kind) * 256 + column] = v;
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
  constexpr int kAtOnce = 10;          // loads in flight (592 rows: two turns)
  for (int r0 = warp; r0 < rows; r0 += 32 * kAtOnce) {
    float x[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int r = r0 + 32 * i;
      x[i] = column < size && r < rows ? partial[(static_cast<int64_t>(r) * 2 + which) * 256 + column] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) v += x[i];
  }
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
// Strides of a tensor: multiples of eight elements; of one that is written, rows must not overlap (what else must not: shared_memory).
int check_strides(const int64_t (&s)[2], int64_t tokens, int64_t heads, int size, bool written, const char* who, const char* name) {
  const std::string at = std::string(who) + ": " + name;
  if (s[0] % 8 != 0 || s[1] % 8 != 0) return fail(IXK_INVALID_ARGUMENT, at + ": strides must be multiples of 8 elements");
  if (s[0] < 0 || s[1] < 0) return fail(IXK_INVALID_ARGUMENT, at + ": negative stride");
  if (written && ((tokens > 1 && s[0] < size) || (heads > 1 && s[1] < size))) return fail(IXK_INVALID_ARGUMENT, at + ": rows overlap");
  return IXK_OK;
}

// The memory of a call's tensors.
int element(const ixk_qk_desc* d) { return d->dtype == IXK_F32 ? 4 : 2; }
paged::Operand heads_of(const ixk_qk_desc* d, const void* p, const int64_t (&s)[2], int64_t heads) {
  return paged::Operand(p, d->head_size * element(d), {d->tokens, heads}, s, element(d));
}
paged::Operand gain_of(const ixk_qk_desc* d, const void* p) { return paged::Operand(p, d->head_size * (d->param_dtype == IXK_F32 ? 4 : 2)); }
paged::Operand table_of(const ixk_qk_desc* d, const float* p) {
  const int64_t row = d->rotary_dim * 2;
  return paged::Operand(p, row, {d->places}, &row, 1);
}
paged::Operand positions_of(const ixk_qk_desc* d, const void* p) { return paged::Operand(p, d->tokens * d->position_bytes); }
int shared(const char* name, const char* who) {
  return name == nullptr ? IXK_OK : fail(IXK_INVALID_ARGUMENT, std::string(who) + ": " + name + " shares memory with another operand or with itself");
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

int lanes_for(int head_size) { return head_size <= 64 ? 4 : head_size <= 128 ? 8 : 16; }

// The segments of a token (of `rows` heads), and how tokens go over as many warps as are on the GPU at one time: whole turns of a
// token a warp, then a last one in which several warps share a token if there are enough (8192 tokens of 16 + 16 heads of 256, 3.46
// turns: forward 51.4 -> 48.4 us; all tokens in two parts, 6.92 turns, were slower than 4 whole ones).  Equal runs of segments
// instead, whatever their kind, leave warps with nothing but keys, of which a token has few: 68 -> 96 us for 16384 tokens of 32 + 8 heads.
int64_t split(Args* a, int rows, bool with_v, int64_t most) {
  a->q_segments = (a->heads + rows - 1) / rows;
  a->kv_segments = (a->kv_heads + rows - 1) / rows;
  a->segments = a->q_segments + a->kv_segments * (with_v ? 2 : 1);
  const int64_t warps = most * kWarps;
  a->turns = static_cast<int>(a->tokens / warps);
  a->rest = a->tokens - a->turns * warps;
  a->parts = a->rest == 0 ? 1 : static_cast<int>(std::min<int64_t>(a->segments, warps / a->rest));
  return a->turns > 0 ? most : std::max<int64_t>(1, (a->tokens * a->parts + kWarps - 1) / kWarps);
}
int forward_heads(int dtype) { return dtype == IXK_F32 ? kForwardHeads<float> : kForwardHeads<__half>; }

template <template <typename, int> class Launcher, typename... More>
int dispatch(int dtype, int lanes, const More&... more) {
  auto with = [&](auto tag) {
    using T = decltype(tag);
    return lanes == 4 ? Launcher<T, 4>::run(more...) : lanes == 8 ? Launcher<T, 8>::run(more...) : Launcher<T, 16>::run(more...);
  };
  if (dtype == IXK_BF16) return with(__nv_bfloat16{});
  if (dtype == IXK_F16) return with(__half{});
  return with(float{});
}
template <typename T, int kLanes>
struct Forward {
  static int run(const Args& a, unsigned grid, cudaStream_t s) {
    const bool whole = a.rotary_chunks == a.head_chunks;
    const auto kernel = a.interleaved ? whole ? forward_kernel<T, kLanes, false, true> : forward_kernel<T, kLanes, false, false>
                                      : whole ? forward_kernel<T, kLanes, true, true> : forward_kernel<T, kLanes, true, false>;
    return launch_overlapped(kernel, dim3(grid), dim3(kThreads), 0, s, a);
  }
};
template <typename T, int kLanes>
struct Backward {
  static int run(const Args& a, unsigned grid, cudaStream_t s) {
    const bool whole = a.rotary_chunks == a.head_chunks;
    const auto kernel = a.interleaved ? whole ? backward_kernel<T, kLanes, false, true> : backward_kernel<T, kLanes, false, false>
                                      : whole ? backward_kernel<T, kLanes, true, true> : backward_kernel<T, kLanes, true, false>;
    return launch_overlapped(kernel, dim3(grid), dim3(kThreads), 0, s, a);
  }
};

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
  if (d->tokens > 0) {
    const paged::Operand mq = qk::heads_of(d, q, d->q_strides, d->heads), mk = qk::heads_of(d, k, d->k_strides, d->kv_heads),
                         mqo = qk::heads_of(d, q_out, d->q_out_strides, d->heads), gains[2] = {qk::gain_of(d, q_gain), qk::gain_of(d, k_gain)},
                         tables[2] = {qk::table_of(d, cos_table), qk::table_of(d, sin_table)}, mp = qk::positions_of(d, positions);
    if (paged) {
      const paged::Operand mv = qk::heads_of(d, v, d->v_strides, d->kv_heads), ms(slots, d->tokens * 4), kp = paged::key_pages(cache, k_pages),
                           vp = paged::value_pages(cache, v_pages);
      if (int st = qk::shared(paged::shared_memory({{"q_out", &mqo, &mq, nullptr}, {"k_pages", &kp, nullptr, nullptr}, {"v_pages", &vp, nullptr, nullptr}},
                                                   {&mq, &mk, &mv, &gains[0], &gains[1], &tables[0], &tables[1], &mp, &ms}),
                              who))
        return st;
    } else {
      const paged::Operand mko = qk::heads_of(d, k_out, d->k_out_strides, d->kv_heads);
      if (int st = qk::shared(paged::shared_memory({{"q_out", &mqo, &mq, nullptr}, {"k_out", &mko, &mk, nullptr}},
                                                   {&mq, &mk, &gains[0], &gains[1], &tables[0], &tables[1], &mp}),
                              who))
        return st;
    }
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
  if (paged) {
    a.cache = paged::cache_args(cache, k_pages, v_pages);
    a.slots = slots;
  }
  const int64_t grid = qk::split(&a, 32 / lanes * qk::forward_heads(d->dtype), paged, static_cast<int64_t>(info.sm_count) * qk::kForwardCtas);
  return qk::dispatch<qk::Forward>(d->dtype, lanes, a, static_cast<unsigned>(grid), static_cast<cudaStream_t>(cuda_stream));
}

size_t ixk_qk_norm_rotary_bwd_workspace_bytes(const ixk_qk_desc* d) {
  if (qk::check(d, "qk_norm_rotary") != IXK_OK) return 0;
  qk::Args a = qk::base_args(d);
  return static_cast<size_t>(qk::split(&a, 32 / qk::lanes_for(d->head_size) * qk::kBackwardHeads, false, qk::kMaxBwdCtas)) * 2 * 256 * sizeof(float);
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
  {
    const paged::Operand mq = qk::heads_of(d, q, d->q_strides, d->heads), mk = qk::heads_of(d, k, d->k_strides, d->kv_heads),
                         mgq = qk::heads_of(d, grad_q, d->gq_strides, d->heads), mgk = qk::heads_of(d, grad_k, d->gk_strides, d->kv_heads),
                         mdq = qk::heads_of(d, dq, d->q_out_strides, d->heads), mdk = qk::heads_of(d, dk, d->k_out_strides, d->kv_heads),
                         in[2] = {qk::gain_of(d, q_gain), qk::gain_of(d, k_gain)}, out[2] = {qk::gain_of(d, dq_gain), qk::gain_of(d, dk_gain)},
                         tables[2] = {qk::table_of(d, cos_table), qk::table_of(d, sin_table)}, mp = qk::positions_of(d, positions),
                         scratch(gains ? workspace : nullptr, static_cast<int64_t>(ixk_qk_norm_rotary_bwd_workspace_bytes(d)));
    // (a gain's gradient in the gain's place: written when the gain has been read)
    if (int st = qk::shared(paged::shared_memory({{"dq", &mdq, &mq, &mgq}, {"dk", &mdk, &mk, &mgk}, {"dq_gain", &out[0], &in[0], nullptr},
                                                  {"dk_gain", &out[1], &in[1], nullptr}, {"the workspace", &scratch, nullptr, nullptr}},
                                                 {&mq, &mk, &mgq, &mgk, &in[0], &in[1], &tables[0], &tables[1], &mp}),
                            who))
      return st;
  }
  DeviceInfo info;
  if (int st = get_device_info(&info)) return st;
  if (d->tokens == 0 && !gains) return IXK_OK;
  qk::Args a = qk::base_args(d);
  a.q = q, a.k = k, a.gq = grad_q, a.gk = grad_k, a.q_gain = q_gain, a.k_gain = k_gain, a.cos_t = cos_table, a.sin_t = sin_table;
  a.positions = positions, a.qo = dq, a.ko = dk;
  a.partial = static_cast<float*>(workspace);
  a.with_gains = gains;
  const int lanes = qk::lanes_for(d->head_size);
  const int ctas = static_cast<int>(qk::split(&a, 32 / lanes * qk::kBackwardHeads, false, qk::kMaxBwdCtas));
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
