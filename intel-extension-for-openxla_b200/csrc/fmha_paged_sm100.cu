// Attention of a step's new rows (a tree of drafted tokens, a chain, or one token a request) over a paged key/value cache.
//
//   o = sum_t p_t v_t / sum_t p_t,   p_t = exp(head_scale q.k_t)   over the keys that a row sees
//
// The G query heads of a key head and a request's new tokens are the rows of one tile of 128: every key and value is read
// once for all of them.  A unit of work is 64 keys of one tile (request, key head, block of tokens); all units of the call, in
// that order, are cut into equal runs, one for every worker, whatever the requests' lengths are.  A worker is a CTA; up to head
// size 128 there are two on an SM, so that one's products run beside the other's exponentials.
//
//   warps 0-3   softmax: a thread owns a row (a lane of tensor memory); then the row's result
//   warp 4      copies: Q, K_0, K_1, V_0, K_2, V_1 ... of the run through a ring of 64-key slots, page by page
//   warp 5      tcgen05.mma: S_g+1 = Q K_g+1^T into one of two buffers, then O += P_g V_g (P from tensor memory)
//
// Bound by HBM: 64 keys of K and V take H * 256 bytes, 1340 cycles of an SM's share of the bandwidth at H = 128, the two products
// 640 (the tile is padded to 128 rows), the softmax about 1000 and beside those of the other worker.
// Weights are taken of a reference point near the running maximum, which is raised when that has moved by more than 2^8 (fp16: 2^4), so O
// is seldom rescaled.  P is rounded to nearest, and the row is divided by the sum of the rounded values, so that a row with one
// large weight loses nothing; the log-sum-exp is taken of the sum of the fp32 ones.  That rounding puts O 0.0021 to 0.0025 (bf16)
// from 64 bits, where its own rounding alone is 0.0017 (fp16 2.7e-4, 2.1e-4).  P as two 16-bit parts is as good as fp32, but takes
// half as many products again (64 trees of 16 55.4 -> 58.7 us, ragged ones at head size 256 69 -> 77, prompts 18 %), and a
// lower part of 0 or below it makes of an infinite value no number.  fp16 has few exponents: there the reference
// point lies 2^11 below the maximum, so that the largest weights are 2^11 to 2^15 and those down to 2^-25 of them normal numbers
// (with 1 to 2^8, thousands of keys at 2^-25 of the largest added up to nothing); smaller ones are off by 2^-36 of it at most.
//
// A tile whose units all lie in one run is written out; otherwise its parts go to scratch in fp32, and the second kernel joins
// them.  A worker has at most two: the end of a tile that an earlier worker began, and the beginning of one that goes on.
//
// Units that reach behind the keys that all rows of a tile see (a request's committed tokens, and without a mask the new ones in front
// of the tile's) see masks, bit by bit, and the stale rest of its last page.  There the softmax warps go through V in shared
// memory first: rows behind the end become zeros, and of drafts every NaN and infinity, since 0 * NaN would reach rows that do not
// see the draft; rows that do see it get them back at the end (`odd_values`).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "paged.h"
#include "ptx.cuh"

namespace ixk {
namespace fmha_paged {

namespace {

constexpr int kRows = 128;            // rows of a tile (= TMEM lanes)
constexpr int kKeys = 64;             // keys of a unit
constexpr int kChunkElems = 64;       // 16-bit elements of a 128-byte swizzle row
constexpr int kThreads = 192;         // 224 where V has a copy warp of its own
constexpr int kCopyWarp = 4;
constexpr int kMmaWarp = 5;
constexpr int kCopyVWarp = 6;
constexpr int kSoftmaxThreads = 128;
constexpr int kTable = 56;            // requests whose numbers a worker holds in shared memory
constexpr int kTileCost = 3;          // what a tile costs beside its units (Q, masks, results)
constexpr int kMinUnits = 2;          // shortest run: with one, the parts to join cost more than the second unit (5 rows, 705 keys: 11.9, 12.4 us)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Where the reference point of a row's weights lies below its maximum when it is set, and how far the maximum may then rise (log2 units).
template <bool kBf16>
constexpr float kBelowMaximum = kBf16 ? 0.0f : 11.0f;
template <bool kBf16>
constexpr float kRise = kBf16 ? 8.0f : 4.0f;

enum : int { kSiteLoadQ = 801, kSiteLoadKV = 802, kSiteMmaQ = 803, kSiteMmaKV = 804, kSiteMmaP = 805, kSiteMmaO = 806, kSiteSoftmaxS = 807,
             kSiteSoftmaxO = 808, kSiteSoftmaxV = 809, kSiteAlign = 810 };

template <int kHeadDim>
struct Cfg {
  static constexpr int kChunks = kHeadDim / kChunkElems;
  static constexpr int kQChunkBytes = kRows * 128;
  static constexpr int kKvChunkBytes = kKeys * 128;
  static constexpr int kQBytes = kChunks * kQChunkBytes;
  static constexpr int kSlotBytes = kChunks * kKvChunkBytes;
  static constexpr int kWorkers = kHeadDim <= 128 ? 2 : 1;        // on an SM
  // A copy of a page's 64 columns costs its warp about 100 cycles: 32 a unit of K and as many of V in pages of 8 tokens and heads of less
  // than 256 columns (or apart from one another, so that none holds more), more than the 2700 that the unit's bytes take.
  static constexpr bool kTwoCopyWarps = kHeadDim == 256;
  static constexpr int kAllThreads = kTwoCopyWarps ? kThreads + 32 : kThreads;
  static constexpr int kSlots = kHeadDim == 64 ? 8 : 5;
  static constexpr int kTmemColumns = kHeadDim <= 128 ? 256 : 512;
  static constexpr int kTmemO = 2 * kKeys;                        // S in two buffers of 64 columns
  static constexpr int kTailBytes = 8 * (10 + 2 * kSlots) + 32 + 8 * 12 + kTable * 12;
  static constexpr int kSmemBytes = kQBytes + kSlots * kSlotBytes + kTailBytes;
  static_assert(kSmemBytes <= (kWorkers == 2 ? 115712 : 232448), "shared memory budget");
  static_assert(kTmemO + kHeadDim <= kTmemColumns, "TMEM budget");
};

struct Args {
  int requests, heads, kv_heads, group, head_size;
  int block_tokens;           // tokens of a tile: 128 / group
  int rows_in;                // rows of q
  int columns, page_shift, pages;
  int cap;                    // keys that a table row can hold
  float scale_log2;           // > 0, so that the maximum can be taken of the raw products
  int negate;                 // the scale is negative: S = -Q.K^T
  int64_t table_stride, mask_stride;
  int mask_words;
  const int *table, *lengths, *row_start, *granted, *mask;
  const uint16_t* v;          // (odd values of drafts)
  int64_t v_strides[3];       // page, token, head
  uint16_t* out;
  int64_t o_strides[2];
  int out_sectors;            // out's rows start on 32-byte boundaries and hold whole 32-byte sectors
  float* lse;
  int* status_word;
  int part_rows;              // rows of a part in scratch
  // Split tiles: first row, first head, rows, parts + (worker << 16).  By the worker that began it and did not finish it ([workers]; 0
  // parts: none), or, where tiles are few, by tile ([requests][kv_heads][tile_blocks]; 0 parts: whole).
  int4* meta;
  int tile_blocks;            // 0: by worker
  int workers;
  float* part_o;              // [2 * workers][kHeadDim / 4][part_rows][4]: a warp's rows side by side
  float4* part_stat;          // [2 * workers][part_rows]: reference point (log2), sum, sum of rounded weights
};

// A request's numbers, cut to what its buffers hold.
struct Request {
  int length, rows, row0;     // committed tokens, new rows, first row
};
__device__ __forceinline__ Request load_request(const Args& a, int b) {
  Request r;
  const int start = a.row_start[b], n = a.granted[b];
  r.length = min(max(a.lengths[b], 0), a.cap);
  r.row0 = start;
  r.rows = start < 0 || start >= a.rows_in ? 0 : max(min(n, a.rows_in - start), 0);
  return r;
}
// (rarely called: kept out of the walks' code)
__device__ __noinline__ Request far_request(const Args& a, int b) { return load_request(a, b); }
// Keys and 64-key units of the block of tokens that starts at token t0.
__device__ __forceinline__ int block_keys(const Args& a, const Request& r, int t0) {
  const int seen = a.mask != nullptr ? r.rows : min(r.rows, t0 + a.block_tokens);
  return static_cast<int>(min(static_cast<long long>(r.length) + seen, static_cast<long long>(a.cap)));
}
__device__ __forceinline__ int block_units(const Args& a, const Request& r, int t0) { return (block_keys(a, r, t0) + kKeys - 1) / kKeys; }
// What one key head of a request costs: its units, and kTileCost for every tile.
__device__ __forceinline__ long long head_cost(const Args& a, const Request& r) {
  if (r.rows <= 0) return 0;
  if (r.rows <= a.block_tokens) return block_units(a, r, 0) + kTileCost;
  long long sum = 0;
  for (int t0 = 0; t0 < r.rows; t0 += a.block_tokens) sum += block_units(a, r, t0) + kTileCost;
  return sum;
}

// A worker's walk over its run, a stretch of the costs of all tiles one behind the other.  A tile's costs begin with kTileCost
// that stand for its start and end; the worker in whose run these end begins it.
struct Walk {
  int b, kv_head, t0;
  Request req;
  int first, unit, end;       // units of the tile: the run's first, the present one, behind the run's last
  int units;                  // of the whole tile
  long long budget;           // the run's end, from the tile's start on
  bool live;
  const int* table;           // the run's first requests in shared memory
  int table_base, table_count;

  __device__ __forceinline__ Request request(const Args& a, int i) const {
    const int k = i - table_base;
    if (k >= 0 && k < table_count) return Request{table[3 * k], table[3 * k + 1], table[3 * k + 2]};
    return far_request(a, i);
  }
  // The tile at (b, kv_head, t0), whose first `from` costs lie before the run.
  __device__ __forceinline__ void enter(const Args& a, int from) {
    units = block_units(a, req, t0);
    first = unit = max(from - kTileCost, 0);
    end = static_cast<int>(max(min(static_cast<long long>(units), budget - kTileCost), 0LL));
  }
  __device__ __forceinline__ void next_tile(const Args& a) {
    budget -= units + kTileCost;
    if (budget <= kTileCost) {        // (the next tile's first unit is another worker's, or there is none)
      live = false;
      return;
    }
    t0 += a.block_tokens;
    if (t0 >= req.rows) {
      t0 = 0;
      if (++kv_head == a.kv_heads) {
        kv_head = 0;
        do {
          if (++b >= a.requests) {
            live = false;
            return;
          }
          req = request(a, b);
        } while (req.rows == 0);
      }
    }
    enter(a, 0);
  }
  // `offset`: of the run's start in request start_b; `count`: its costs
  __device__ __forceinline__ void begin(const Args& a, int start_b, long long offset, long long count) {
    b = start_b;
    live = count > 0;
    if (!live) return;
    req = request(a, b);
    const long long per_head = head_cost(a, req);
    kv_head = offset < per_head ? 0
              : (offset >> 31) == 0 ? static_cast<int>(static_cast<unsigned>(offset) / static_cast<unsigned>(per_head))
                                    : static_cast<int>(offset / per_head);
    long long rest = offset - kv_head * per_head;
    t0 = 0;
    for (long long cost; rest >= (cost = block_units(a, req, t0) + kTileCost); t0 += a.block_tokens) rest -= cost;
    budget = rest + count;
    enter(a, static_cast<int>(rest));
    if (unit >= end) next_tile(a);
  }
  __device__ __forceinline__ bool done() const { return !live; }
  __device__ __forceinline__ bool starts() const { return unit == first; }
  __device__ __forceinline__ bool ends() const { return unit + 1 == end; }                     // the tile's last unit of this run
  __device__ __forceinline__ bool last() const { return ends() && budget - (units + kTileCost) <= kTileCost; }
  __device__ __forceinline__ void next(const Args& a) {
    if (++unit >= end) next_tile(a);
  }
};

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 32 bytes, 32-byte aligned: a whole sector, where a lane's 16 would be half of one.
__device__ __forceinline__ void store_sector(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
               "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Issued by one elected lane of a converged warp; descriptors as (lo, hi) halves, the high one a constant.
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, e;\n\t"
      ".reg .b64 da, db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, e;\n\t"
      ".reg .b64 db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Which of keys [k0, k0 + 64) a row sees, as bits: committed ones, and drafts by its mask or, without one, up to itself.  Of a unit
// with keys behind those that all rows see (so length - k0 < 64).  `words`: the row's mask, its first two words in m0 and m1.
__device__ __forceinline__ uint64_t visible_keys(const Args& a, const Request& r, const int* words, uint32_t m0, uint32_t m1, int token, int k0) {
  auto below = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull; };
  const int committed = r.length - k0, end = min(r.rows, a.cap - r.length) + committed;
  uint64_t bits = below(committed);
  if (words == nullptr) {
    bits |= below(min(committed + token + 1, end));
  } else {
    // drafts d0 .. d0 + 63 stand at keys k0 .. (d0 < 0: the first of them at key k0 - d0)
    const int d0 = -committed;
    const int w0 = d0 >> 5, shift = d0 & 31;       // (rounded down)
    auto word = [&](int w) {
      if (w == 0) return m0;
      if (w == 1) return m1;
      return w > 1 && w < a.mask_words ? static_cast<uint32_t>(words[w]) : 0u;
    };
    const uint32_t x = word(w0), y = word(w0 + 1), z = word(w0 + 2);
    const uint32_t lo = __funnelshift_r(x, y, shift), hi = __funnelshift_r(y, z, shift);
    bits |= (static_cast<uint64_t>(hi) << 32 | lo) & below(end);
  }
  return bits;
}

// 0 as long as all numbers were finite: each times 0, added up.
template <bool kBf16>
__device__ __forceinline__ uint32_t finite_test(uint32_t acc, uint32_t w) {
  if constexpr (kBf16) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w), __floats2bfloat162_rn(0.0f, 0.0f), *reinterpret_cast<const __nv_bfloat162*>(&acc));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&w), __floats2half2_rn(0.0f, 0.0f), *reinterpret_cast<const __half2*>(&acc));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// The rare case, kept out of the way: a stretch of V in shared memory with its NaN and infinities made zeros.
__device__ __noinline__ void clear_odd_values(uint4* v, int begin, int pieces, int stride, int first, int pitch, uint32_t expo) {
  for (int n = first; n < pieces; n += stride) {
    const int i = ((begin + n) >> 6) * pitch + ((begin + n) & 63);
    const uint4 w = v[i];
    uint32_t words[4] = {w.x, w.y, w.z, w.w};
    for (int e = 0; e < 4; ++e) {
      if ((words[e] & expo) == expo) words[e] &= 0xffff0000u;
      if ((words[e] >> 16 & expo) == expo) words[e] &= 0x0000ffffu;
    }
    v[i] = make_uint4(words[0], words[1], words[2], words[3]);
  }
}
// ... and the other end of it: rows that were written without them get the odd values of the drafts [d0, d1) that they see, out of memory
// again.  `out`: a row itself, or `part`: its part in scratch.  All lanes of a warp call it; `row_ok`: those that have a row.  A
// lane looks for odd values in one of 32 drafts; then the rows add up those that they see, 8 columns at a time, and change these once.
template <bool kBf16>
__device__ __noinline__ void add_odd_values(const Args& a, int length, int b, int kv_head, bool row_ok, int token, int q_row, int d0, int d1, uint16_t* out,
                                            float* part, int64_t part_pitch) {
  constexpr uint32_t kExponent = kBf16 ? 0x7f80u : 0x7c00u;
  const int lane = threadIdx.x & 31, pieces = a.head_size / 8;
  for (; d0 < d1; d0 += 32) {
    const uint4* mine = nullptr;
    uint32_t test = 0;
    if (d0 + lane < d1) {
      const int k = length + d0 + lane, page = a.table[b * a.table_stride + (k >> a.page_shift)];
      if (static_cast<unsigned>(page) < static_cast<unsigned>(a.pages)) {
        mine = reinterpret_cast<const uint4*>(a.v + page * a.v_strides[0] + (k & ((1 << a.page_shift) - 1)) * a.v_strides[1] + kv_head * a.v_strides[2]);
#pragma unroll 8
        for (int i = 0; i < pieces; ++i) {
          const uint4 w = mine[i];
          test = finite_test<kBf16>(finite_test<kBf16>(finite_test<kBf16>(finite_test<kBf16>(test, w.x), w.y), w.z), w.w);
        }
      }
    }
    const uint32_t found = __ballot_sync(0xffffffffu, (test & 0x7fff7fffu) != 0);
    if (found == 0) continue;
    uint32_t sees = 0;         // of the 32 drafts, by this lane's row
    if (row_ok && a.mask == nullptr) {
      const int n = token + 1 - d0;
      sees = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
    } else if (row_ok) {
      const int* words = a.mask + q_row * a.mask_stride;
      const int w = d0 >> 5;
      sees = __funnelshift_r(w < a.mask_words ? words[w] : 0, w + 1 < a.mask_words ? words[w + 1] : 0, d0 & 31);
    }
    for (int c = 0; c < pieces; ++c) {
      float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      for (uint32_t left = found; left != 0; left &= left - 1) {
        const int i = __ffs(left) - 1;
        const uint4* v = reinterpret_cast<const uint4*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), i));
        if (!(sees >> i & 1u)) continue;
        const uint4 w = v[c];
        const uint32_t held[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t bits = held[e >> 1] >> 16 * (e & 1) & 0xffffu;
          if ((bits & kExponent) == kExponent) sum[e] += unpack2<kBf16>(bits).x;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (sum[e] == 0.0f) continue;
        const int i = c * 8 + e;
        if (part != nullptr) part[(i >> 2) * part_pitch + (i & 3)] += sum[e];
        else out[i] = static_cast<uint16_t>(pack2<kBf16>(unpack2<kBf16>(out[i]).x + sum[e], 0.0f) & 0xffffu);
      }
    }
  }
}

// kLse: the sum of the unrounded weights is wanted as well.  (Without it an instruction of eight in the inner loop is gone: 512 requests of 10 to
// 300 keys 54.7 -> 50.9 us.)
// kGroups: small pages.  A copy brings 8 keys, all 64-column chunks of them, and a slot is [8-key group][chunk][8 keys]; otherwise a copy
// brings a page's (at most 64) keys of one chunk, and a slot is [chunk][keys].  Copies are what a unit waits for where there are more
// than 8 of K or of V: 48 requests of 300 to 12000 keys in pages of 8 at head size 128 70 -> 57 us, at 256 88 -> 75.
template <int kHeadDim, bool kBf16, bool kLse, bool kGroups>
__global__ void __launch_bounds__(Cfg<kHeadDim>::kAllThreads, Cfg<kHeadDim>::kWorkers)
fmha_paged_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                  const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ Args args) {
  using C = Cfg<kHeadDim>;
  constexpr int kSlots = C::kSlots;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t q_smem = ptx::smem_u32(smem);
  const uint32_t kv_smem = q_smem + C::kQBytes;
  const uint32_t bar_base = kv_smem + kSlots * C::kSlotBytes;
  const uint32_t q_full = bar_base, q_empty = bar_base + 8, o_free = bar_base + 16;
  // (by buffer: what a thread waits for is then never two phases ahead of what it knows to have passed)
  auto s_full = [&](int i) { return bar_base + 8u * (3 + i); };
  auto p_full = [&](int i) { return bar_base + 8u * (5 + i); };
  auto pv_done = [&](int i) { return bar_base + 8u * (7 + i); };
  auto kv_full = [&](int s) { return bar_base + 8u * (9 + s); };
  auto kv_empty = [&](int s) { return bar_base + 8u * (9 + kSlots + s); };
  uint8_t* tail = smem + C::kQBytes + kSlots * C::kSlotBytes + 8 * (10 + 2 * kSlots);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(tail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 4);
  volatile int* odd_values = reinterpret_cast<volatile int*>(tail + 8);      // [3] by tile
  int* start_request = reinterpret_cast<int*>(tail + 20);
  long long* start_offset = reinterpret_cast<long long*>(tail + 24);
  long long* sums = reinterpret_cast<long long*>(tail + 32);                 // [6]
  long long* other_sums = sums + 6;                                          // [6]
  int* table = reinterpret_cast<int*>(tail + 32 + 8 * 12);                   // [kTable][3]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ptx::AbortCtl ctl{abort_flag, args.status_word};
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    odd_values[0] = odd_values[1] = odd_values[2] = 0;
    ptx::mbar_init(q_full, 1);
    ptx::mbar_init(q_empty, 1);
    ptx::mbar_init(o_free, kSoftmaxThreads);
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(s_full(i), 1);
      ptx::mbar_init(p_full(i), kSoftmaxThreads);
      ptx::mbar_init(pv_done(i), 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      ptx::mbar_init(kv_full(s), 1);
      ptx::mbar_init(kv_empty(s), 1);
    }
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmap_q);
    ptx::prefetch_tmap(&tmap_k);
    ptx::prefetch_tmap(&tmap_v);
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), C::kTmemColumns);
    ptx::tmem_relinquish();
  }
  ptx::grid_dependency_sync();

  // (the page table on its way to L2, a line a thread: who reads which of it is not known yet)
  {
    const int64_t lines = ((args.requests - 1) * args.table_stride + args.columns + 31) / 32;
    const int64_t line = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (line < lines) asm volatile("prefetch.global.L2 [%0];" ::"l"(args.table + min(line * 32, (args.requests - 1) * args.table_stride + args.columns - 1)));
  }
  // ---- the run: its length from the costs of all requests, its start from their sums
  Request mine{0, 0, 0};
  auto cost_of = [&](const Request& r) { return head_cost(args, r) * args.kv_heads; };
  const bool scans = threadIdx.x < kThreads;
  if (scans && static_cast<int>(threadIdx.x) < args.requests) mine = load_request(args, threadIdx.x);
  const long long my_cost = cost_of(mine);
  auto prefix = [&](long long v) {     // inclusive, in the warp; the warp's sum to `sums`
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    if (lane == 31 && scans) sums[warp] = v;
    return v;
  };
  long long upto = prefix(my_cost);
  long long others = 0;                // of the requests behind the first kThreads
  for (int b = threadIdx.x + kThreads; scans && b < args.requests; b += kThreads) others += cost_of(load_request(args, b));
  if (args.requests > kThreads) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) others += __shfl_xor_sync(0xffffffffu, others, o);
    if (lane == 0 && scans) other_sums[warp] = others;
  }
  auto keep = [&](int i, const Request& r) {
    table[3 * i] = r.length;
    table[3 * i + 1] = r.rows;
    table[3 * i + 2] = r.row0;
  };
  const bool few = args.requests <= kTable;
  if (few && static_cast<int>(threadIdx.x) < args.requests) keep(threadIdx.x, mine);
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) upto += sums[w];
    total += sums[w];
  }
  long long before = total;            // costs of the requests that the scan has been over
  if (args.requests > kThreads)
    for (int w = 0; w < kThreads / 32; ++w) total += other_sums[w];
  const unsigned grid = gridDim.x;
  long long run = (total >> 31) == 0 ? (static_cast<unsigned>(total) + grid - 1u) / grid : (total + grid - 1) / grid;
  run = max(run, static_cast<long long>(kMinUnits));
  const long long start = run * blockIdx.x;
  const bool aligned = (q_smem & 1023u) == 0;
  if (!aligned && threadIdx.x == 0) atomicCAS(args.status_word, 0, kSiteAlign);
  const long long count = aligned ? max(min(run, total - start), 0LL) : 0LL;
  if (count > 0) {
    if (start >= upto - my_cost && start < upto) {
      *start_request = threadIdx.x;
      *start_offset = start - (upto - my_cost);
    }
    for (int b0 = kThreads; before <= start; b0 += kThreads) {      // (the same in all threads; start < total)
      const int b = b0 + static_cast<int>(threadIdx.x);
      const long long cost = scans && b < args.requests ? cost_of(load_request(args, b)) : 0;
      __syncthreads();
      upto = prefix(cost) + before;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) upto += sums[w];
        before += sums[w];
      }
      if (start >= upto - cost && start < upto) {
        *start_request = b;
        *start_offset = start - (upto - cost);
      }
    }
    __syncthreads();
    if (!few) {
      const int i = *start_request + static_cast<int>(threadIdx.x);
      if (threadIdx.x < kTable && i < args.requests) keep(threadIdx.x, load_request(args, i));
      __syncthreads();
    }
  }
  Walk walk;
  walk.table = table;
  walk.table_base = count > 0 && !few ? *start_request : 0;
  walk.table_count = min(kTable, args.requests - walk.table_base);
  walk.begin(args, count > 0 ? *start_request : 0, count > 0 ? *start_offset : 0, count);

  auto load_q = [&](const Walk& at) {
    ptx::mbar_expect_tx(q_full, static_cast<uint32_t>(C::kChunks * args.group * args.block_tokens * 128));
#pragma unroll
    for (int c = 0; c < C::kChunks; ++c)
      ptx::tma_load_3d(q_smem + c * C::kQChunkBytes, &tmap_q, q_full, c * kChunkElems, at.kv_head * args.group, at.req.row0 + at.t0);
  };
  if (warp == kCopyWarp || (C::kTwoCopyWarps && warp == kCopyVWarp)) {
    // ------------------------------------------------------------------ copies: a page's 64 columns at a time
    const int box_keys = kGroups ? 8 : min(kKeys, 1 << args.page_shift);
    const int pieces = kKeys / box_keys;
    const int piece = kGroups ? lane : lane / C::kChunks, chunk = kGroups ? 0 : lane - piece * C::kChunks;
    const int to = piece * box_keys * 128 * (kGroups ? C::kChunks : 1) + chunk * C::kKvChunkBytes;
    // Keys and values that one tile reads leave L2 first: books, page table, Q and the parts in scratch stay (64 trees of 16 over 1024 to
    // 4096 keys 62.9 -> 57.3 us, 24 ragged ones at head size 256 73 -> 69.3).
    const uint64_t once = ptx::l2_evict_first(), again = ptx::l2_evict_normal();
    bool alive = true;
    auto wait = [&](uint32_t bar, uint32_t parity, int site) {
      if (alive && !ptx::mbar_wait(bar, parity, ctl, site)) alive = false;
      alive = __all_sync(0xffffffffu, alive);
      return alive;
    };
    // A unit's page numbers, a lane each.  (Pages behind the last key are not looked up: their rows are zeros, as those of a page
    // number outside the cache.)
    auto pages_of = [&](const Walk& at) {
      const int k0 = at.unit * kKeys + piece * box_keys;
      int page = args.pages;
      if (piece < pieces && k0 < at.req.length + min(at.req.rows, args.cap - at.req.length)) {
        page = args.table[at.b * args.table_stride + (k0 >> args.page_shift)];
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(args.pages)) page = args.pages;
      }
      return page;
    };
    // `load`: its place in the sequence K_0, K_1, V_0, K_2, V_1 ...
    auto load_unit = [&](const Walk& at, uint32_t load, int page, const CUtensorMap* map) {
      const int slot = load % kSlots;
      if (!wait(kv_empty(slot), ((load / kSlots) & 1u) ^ 1u, kSiteLoadKV)) return;
      if (lane == 0) ptx::mbar_expect_tx(kv_full(slot), C::kSlotBytes);
      __syncwarp();
      if (piece < pieces) {
        const int in_page = (at.unit * kKeys + (kGroups ? piece * box_keys : 0)) & ((1 << args.page_shift) - 1);
        ptx::tma_load_4d(kv_smem + slot * C::kSlotBytes + to, map, kv_full(slot), chunk * kChunkElems, kGroups ? in_page : at.kv_head,
                         kGroups ? at.kv_head * C::kChunks : in_page, page, at.req.rows > args.block_tokens ? again : once);
      }
    };
    Walk k_walk = walk, v_walk = walk;
    uint32_t tiles = 1, k_units = 0, v_units = 0;       // (the first tile's Q: by the warp of the products)
    int next_pages = 0, pages0 = 0, pages1 = 0;
    auto load_k = [&]() {
      load_unit(k_walk, k_units < 2 ? k_units : 2 * k_units - 1, next_pages, &tmap_k);
      // a new tile: Q, once the products of the one before have read theirs (behind its first keys, which then are on their way already)
      if (alive && k_units > 0 && k_walk.starts()) {
        if (!wait(q_empty, (tiles & 1u) ^ 1u, kSiteLoadQ)) return;
        ++tiles;
        if (lane == 0) load_q(k_walk);
        __syncwarp();
      }
      // (in one warp V follows K by two units at most)
      if (k_units == v_units) pages0 = next_pages;
      else pages1 = next_pages;
      ++k_units;
      k_walk.next(args);
      if (!k_walk.done()) next_pages = pages_of(k_walk);     // on its way while the ring is full
    };
    auto load_v = [&](int page) {
      load_unit(v_walk, v_walk.last() ? 2 * v_units + 1 : 2 * v_units + 2, page, &tmap_v);
      ++v_units;
      v_walk.next(args);
    };
    if (!walk.done()) pages0 = next_pages = pages_of(walk);
    if (C::kTwoCopyWarps && warp == kCopyVWarp) {
      while (alive && !v_walk.done()) {
        load_v(pages0);
        if (!v_walk.done()) pages0 = pages_of(v_walk);
      }
    } else {
      if (!k_walk.done()) load_k();
      while (alive && (C::kTwoCopyWarps ? !k_walk.done() : !v_walk.done())) {
        if (!k_walk.done()) load_k();
        if (!C::kTwoCopyWarps && alive) {
          load_v(pages0);
          pages0 = pages1;
        }
      }
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------------ products (all lanes; one elected per instruction)
    // The first tile's Q, while the copy warp looks up pages.
    if (lane == 0 && !walk.done()) load_q(walk);
    __syncwarp();
    constexpr uint32_t fmt = kBf16 ? 1u : 0u;
    const uint32_t idesc_s = ptx::umma_idesc(fmt, fmt, 0, 0, kRows, kKeys) | (args.negate ? 1u << 13 : 0u);      // (bit 13: A negated)
    const uint32_t idesc_o = ptx::umma_idesc(fmt, fmt, 0, 1, kRows, kHeadDim);
    const uint32_t kv_chunk = kGroups ? 1024u : C::kKvChunkBytes, kv_group = kGroups ? C::kChunks * 1024u : 1024u;
    const uint64_t qmajor = ptx::umma_smem_desc(0, 16, 1024);
    const uint64_t kmajor = ptx::umma_smem_desc(0, 16, kv_group);
    const uint64_t mnmajor = ptx::umma_smem_desc(0, kv_chunk, kv_group);
    const uint32_t q_lo = static_cast<uint32_t>(qmajor), q_hi = static_cast<uint32_t>(qmajor >> 32);
    const uint32_t k_lo = static_cast<uint32_t>(kmajor), k_hi = static_cast<uint32_t>(kmajor >> 32);
    const uint32_t v_lo = static_cast<uint32_t>(mnmajor), v_hi = static_cast<uint32_t>(mnmajor >> 32);
    bool alive = true;
    auto wait = [&](uint32_t bar, uint32_t parity, int site) {
      if (alive && !ptx::mbar_wait(bar, parity, ctl, site)) alive = false;
      alive = __all_sync(0xffffffffu, alive);
      return alive;
    };
    uint32_t slot = 0, slot_parity = 0;
    auto advance = [&]() {
      if (++slot == static_cast<uint32_t>(kSlots)) {
        slot = 0;
        slot_parity ^= 1u;
      }
    };
    Walk s_walk = walk, o_walk = walk;
    uint32_t s_units = 0, o_units = 0, q_parity = 0, o_parity = 1;
    auto issue_s = [&]() {
      if (s_walk.starts()) {
        if (!wait(q_full, q_parity, kSiteMmaQ)) return;
        q_parity ^= 1u;
      }
      if (!wait(kv_full(slot), slot_parity, kSiteMmaKV)) return;
      ptx::tc_fence_after_sync();
      const uint32_t d = tmem_base + (s_units & 1u) * kKeys;
      const uint32_t qa = q_lo + (q_smem >> 4), kb = k_lo + ((kv_smem + slot * C::kSlotBytes) >> 4);
#pragma unroll
      for (int ks = 0; ks < kHeadDim / 16; ++ks)
        mma_ss(d, qa + (((ks >> 2) * C::kQChunkBytes + (ks & 3) * 32) >> 4), q_hi, kb + (((ks >> 2) * kv_chunk + (ks & 3) * 32) >> 4), k_hi,
               idesc_s, ks != 0 ? 1u : 0u);
      ptx::umma_commit_elect(s_full(s_units & 1u));
      ptx::umma_commit_elect(kv_empty(slot));
      if (s_walk.ends()) ptx::umma_commit_elect(q_empty);
      advance();
      ++s_units;
      s_walk.next(args);
    };
    if (!s_walk.done()) issue_s();
    while (alive && !o_walk.done()) {
      if (!s_walk.done()) issue_s();
      if (!alive) break;
      // O of the tile before must have been read out
      if (o_walk.starts()) {
        if (!wait(o_free, o_parity, kSiteMmaO)) break;
        o_parity ^= 1u;
      }
      if (!wait(kv_full(slot), slot_parity, kSiteMmaKV)) break;
      if (!wait(p_full(o_units & 1u), (o_units >> 1) & 1u, kSiteMmaP)) break;
      ptx::tc_fence_after_sync();
      const uint32_t a = tmem_base + (o_units & 1u) * kKeys, d = tmem_base + C::kTmemO;
      const uint32_t vb = v_lo + ((kv_smem + slot * C::kSlotBytes) >> 4);
#pragma unroll
      for (int ks = 0; ks < kKeys / 16; ++ks)
        mma_ts(d, a + ks * 8, vb + ((ks * 2 * kv_group) >> 4), v_hi, idesc_o, (!o_walk.starts() || ks != 0) ? 1u : 0u);
      ptx::umma_commit_elect(pv_done(o_units & 1u));
      ptx::umma_commit_elect(kv_empty(slot));
      advance();
      ++o_units;
      o_walk.next(args);
    }
  } else {
    // ------------------------------------------------------------------ softmax and results
    const int row = warp * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t o_addr = tmem_base + lane_addr + C::kTmemO;
    const int row_token = row / args.group, row_head = row - row_token * args.group;
    uint32_t g = 0, tiles = 0;
    bool alive = true;
    // (A warp's lanes go on together or give up together: what follows has them all, in votes and in accesses to tensor memory.)
    auto wait = [&](uint32_t bar, uint32_t parity, int site) {
      alive = ptx::mbar_wait_warp(bar, parity, ctl, site);
      return alive;
    };
    int4 begun = make_int4(0, 0, 0, 0);       // the tile that this worker leaves to others: none so far
    while (alive && !walk.done()) {
      const Request req = walk.req;
      const int token = walk.t0 + row_token;
      const bool row_ok = row_token < args.block_tokens && token < req.rows;
      const bool warp_ok = __any_sync(0xffffffffu, row_ok);
      const int q_row = req.row0 + token;
      const int keys_end = req.length + min(req.rows, args.cap - req.length);
      const int first_unit = walk.unit;
      // the keys in front of this one are seen by all rows of the tile
      const int common = req.length + (args.mask != nullptr ? 0 : min(walk.t0, args.cap - req.length));
      // the row's mask, asked for long before it is needed
      const int* words = args.mask != nullptr ? args.mask + q_row * args.mask_stride : nullptr;
      uint32_t m0 = 0, m1 = 0;
      if (words != nullptr && row_ok) {
        m0 = words[0];
        if (args.mask_words > 1) m1 = words[1];
      }
      float m_run = -INFINITY, l_run = 0.0f, r_run = 0.0f;     // reference point, sum, sum of the rounded weights
      bool more = true;
      for (; more; ++g) {
        const int buf = g & 1u;
        const int k0 = walk.unit * kKeys;
        const bool masked = k0 + kKeys > common;
        const uint32_t s_addr = tmem_base + lane_addr + buf * kKeys;
        if (!wait(s_full(buf), (g >> 1) & 1u, kSiteSoftmaxS)) break;
        ptx::tc_fence_after_sync();
        if (warp_ok) {
          uint32_t r[2][32];
          ptx::tmem_ld_32x32(s_addr, r[0]);
          ptx::tmem_ld_32x32(s_addr + 32, r[1]);
          ptx::tmem_ld_wait();
          const float mult = args.scale_log2;
          bool seen1 = true;        // some row of the warp sees keys of the second half
          if (masked) {
            const uint64_t bits = row_ok ? visible_keys(args, req, words, m0, m1, token, k0) : 0ull;
            const uint32_t lo = static_cast<uint32_t>(bits), hi = static_cast<uint32_t>(bits >> 32);
            seen1 = __any_sync(0xffffffffu, hi != 0u);
            if (!__all_sync(0xffffffffu, lo == 0xffffffffu)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(lo >> i & 1u)) r[0][i] = 0xff800000u;
            }
            if (!__all_sync(0xffffffffu, hi == 0xffffffffu)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(hi >> i & 1u)) r[1][i] = 0xff800000u;
            }
          }
          float mx[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) mx[e] = ptx::max3(__uint_as_float(r[0][2 * e]), __uint_as_float(r[0][2 * e + 1]), __uint_as_float(r[0][16 + 2 * e]));
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            mx[e] = ptx::max3(mx[e], __uint_as_float(r[0][17 + 2 * e]), __uint_as_float(r[1][2 * e]));
            mx[e] = ptx::max3(mx[e], __uint_as_float(r[1][2 * e + 1]), __uint_as_float(r[1][16 + 2 * e]));
            mx[e] = fmaxf(mx[e], __uint_as_float(r[1][17 + 2 * e]));
          }
          const float top = fmaxf(fmaxf(ptx::max3(mx[0], mx[1], mx[2]), mx[3]), fmaxf(ptx::max3(mx[4], mx[5], mx[6]), mx[7])) * mult;
          float alpha = 1.0f;
          if (row_ok && top - m_run > kBelowMaximum<kBf16> + kRise<kBf16>) {     // also where the row has seen nothing so far
            const float to = top - kBelowMaximum<kBf16>;
            alpha = ptx::ex2_approx(m_run - to);
            m_run = to;
          }
          __syncwarp();          // (what follows accesses tensor memory with all lanes)
          if (walk.unit != first_unit && __any_sync(0xffffffffu, alpha != 1.0f)) {
            // (S of this unit was issued behind P.V of the unit before the last: only the last one's may still run)
            if (!wait(pv_done((g - 1) & 1u), ((g - 1) >> 1) & 1u, kSiteSoftmaxO)) break;
            ptx::tc_fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < kHeadDim / 32; ++c) {
              uint32_t o[32];
              ptx::tmem_ld_32x32(o_addr + c * 32, o);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              ptx::tmem_st_32x32(o_addr + c * 32, o);
            }
          }
          const float m_use = m_run == -INFINITY ? 0.0f : m_run;
          const uint64_t mult2 = ptx::f32x2(mult, mult), minus2 = ptx::f32x2(-m_use, -m_use);
          uint64_t total2 = ptx::f32x2(0.0f, 0.0f), round2 = total2;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t packed[16];
            if (c == 1 && !seen1) {
#pragma unroll
              for (int i = 0; i < 16; ++i) packed[i] = 0u;
              ptx::tmem_st_32x16(s_addr + c * 16, packed);
              break;
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float x0, x1;
              ptx::f32x2_split(ptx::fma2(ptx::f32x2(__uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1])), mult2, minus2), x0, x1);
              x0 = ptx::ex2_approx(x0);
              x1 = ptx::ex2_approx(x1);
              if constexpr (kLse) total2 = ptx::add2(total2, ptx::f32x2(x0, x1));
              packed[i >> 1] = pack2<kBf16>(x0, x1);
              const float2 rounded = unpack2<kBf16>(packed[i >> 1]);
              round2 = ptx::add2(round2, ptx::f32x2(rounded.x, rounded.y));
            }
            ptx::tmem_st_32x16(s_addr + c * 16, packed);
          }
          float t0, t1;
          if constexpr (kLse) {
            ptx::f32x2_split(total2, t0, t1);
            l_run = l_run * alpha + (t0 + t1);
          }
          ptx::f32x2_split(round2, t0, t1);
          r_run = r_run * alpha + (t0 + t1);
          ptx::tmem_st_wait();
        }
        if (masked) {
          // V behind the last key, and values of drafts that are no numbers
          const uint32_t load = walk.last() ? 2 * g + 1 : 2 * g + 2;
          if (!wait(kv_full(load % kSlots), (load / kSlots) & 1u, kSiteSoftmaxV)) break;
          uint4* v = reinterpret_cast<uint4*>(smem + C::kQBytes + (load % kSlots) * C::kSlotBytes);     // (16-byte pieces: a key is 8 in a chunk)
          const int d0 = max(common - k0, 0), d1 = min(keys_end - k0, kKeys);
          // (whole pages behind the last key were never copied: zeros already)
          const int stale = (min(((keys_end - 1) >> args.page_shift << args.page_shift) + (1 << args.page_shift) - k0, kKeys) - d1) * 8;
          const int drafts = (d1 - d0) * 8;
          const int pitch = kGroups ? C::kChunks * 64 : 64, chunk = kGroups ? 64 : kKeys * 8;
          auto piece = [&](int c, int i) -> uint4& { return kGroups ? v[c * chunk + (i >> 6) * pitch + (i & 63)] : v[c * chunk + i]; };
          uint32_t test = 0;
#pragma unroll 1
          for (int i = row; i < drafts; i += kSoftmaxThreads) {
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c) {
              const uint4 w = piece(c, d0 * 8 + i);
              test = finite_test<kBf16>(finite_test<kBf16>(finite_test<kBf16>(finite_test<kBf16>(test, w.x), w.y), w.z), w.w);
            }
          }
#pragma unroll 1
          for (int i = row; i < stale; i += kSoftmaxThreads) {
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c) piece(c, d1 * 8 + i) = make_uint4(0, 0, 0, 0);
          }
          if ((test & 0x7fff7fffu) != 0) {      // (this thread's own pieces)
            for (int c = 0; c < C::kChunks; ++c) clear_odd_values(v + c * chunk, d0 * 8, drafts, kSoftmaxThreads, row, pitch, kBf16 ? 0x7f80u : 0x7c00u);
            odd_values[tiles % 3] = 1;
          }
          ptx::fence_proxy_async_smem();
        }
        more = !walk.ends();
        // The flag of the tile after this one: last used two tiles ago, by nobody any more once all threads are in this one.
        if (!more && row == 0) odd_values[(tiles + 1) % 3] = 0;
        ptx::tc_fence_before_sync();
        ptx::mbar_arrive(p_full(buf));
        if (more) walk.next(args);
      }
      if (!alive) break;
      if (!wait(pv_done((g - 1) & 1u), ((g - 1) >> 1) & 1u, kSiteSoftmaxO)) break;
      ptx::tc_fence_after_sync();
      const bool odd = odd_values[tiles % 3] != 0;
      ++tiles;
      const bool whole = first_unit == 0 && walk.end == walk.units;
      const int head = walk.kv_head * args.group + row_head;
      int64_t part = 2 * static_cast<int64_t>(blockIdx.x);
      if (whole && args.tile_blocks != 0 && row == 0)
        args.meta[(walk.b * args.kv_heads + walk.kv_head) * args.tile_blocks + walk.t0 / args.block_tokens] = make_int4(0, 0, 0, 0);
      if (!whole && first_unit == 0) {
        ++part;
        // (the workers behind this one have runs of `run`)
        const long long after = walk.units + kTileCost - walk.budget;
        begun = make_int4(req.row0 + walk.t0, walk.kv_head * args.group, min(args.block_tokens, req.rows - walk.t0) * args.group,
                          static_cast<int>((after + run - 1) / run + 1) | static_cast<int>(blockIdx.x) << 16);
        if (args.tile_blocks != 0 && row == 0)
          args.meta[(walk.b * args.kv_heads + walk.kv_head) * args.tile_blocks + walk.t0 / args.block_tokens] = begun;
      }
      if (warp_ok) {
        // (nothing seen: its products are sums of 0 times numbers)
        const float inv_l = r_run == 0.0f ? 0.0f : __fdividef(1.0f, r_run);
        const uint64_t inv2 = ptx::f32x2(inv_l, inv_l);
        uint16_t* out_row = args.out + q_row * args.o_strides[0] + head * args.o_strides[1];
        float* part_row = args.part_o + (part * (kHeadDim / 4) * args.part_rows + row) * 4;
        const int64_t part_pitch = static_cast<int64_t>(args.part_rows) * 4;
#pragma unroll 1
        for (int c0 = 0; c0 < kHeadDim; c0 += 64) {
          uint32_t o[64];
          __syncwarp();
          ptx::tmem_ld_32x32(o_addr + c0, *reinterpret_cast<uint32_t(*)[32]>(o));
          ptx::tmem_ld_32x32(o_addr + c0 + 32, *reinterpret_cast<uint32_t(*)[32]>(o + 32));
          ptx::tmem_ld_wait();
          if (!row_ok) continue;
          if (whole) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float x, y;
              ptx::f32x2_split(ptx::mul2(ptx::f32x2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), inv2), x, y);
              o[i] = pack2<kBf16>(x, y);
            }
            if (args.out_sectors) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (c0 + e * 16 < args.head_size)
                  store_sector(out_row + c0 + e * 16, {o[8 * e], o[8 * e + 1], o[8 * e + 2], o[8 * e + 3], o[8 * e + 4], o[8 * e + 5], o[8 * e + 6],
                                                       o[8 * e + 7]});
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (c0 + e * 8 < args.head_size)
                  reinterpret_cast<uint4*>(out_row + c0)[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              *reinterpret_cast<uint4*>(part_row + (c0 / 4 + e) * part_pitch) = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
        if (row_ok) {
          if (!whole) args.part_stat[part * args.part_rows + row] = make_float4(m_run, l_run, r_run, 0.0f);
          else if (kLse)
            args.lse[static_cast<int64_t>(q_row) * args.heads + head] = l_run == 0.0f ? -INFINITY : (m_run + log2f(l_run)) * kLn2;
        }
        if (odd) {
          __syncwarp();
          add_odd_values<kBf16>(args, req.length, walk.b, walk.kv_head, row_ok, token, q_row, max(first_unit * kKeys, common) - req.length,
                                min(walk.end * kKeys, keys_end) - req.length, out_row, whole ? nullptr : part_row, part_pitch);
        }
      }
      ptx::tc_fence_before_sync();
      ptx::mbar_arrive(o_free);
      walk.next(args);
    }
    if (threadIdx.x == 0 && args.tile_blocks == 0) args.meta[blockIdx.x] = begun;
  }

  if (*abort_flag != 0) __nanosleep(2000000);
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, C::kTmemColumns);
  }
}

// Joins the parts of the tiles that several workers did.  With the parts' reference points m_i and sums l_i, M = max m_i:
//   o = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i
// Worker w's own part is at 2 w + 1, those of the workers behind it at 2 (w + i).  A thread takes 16 columns of a row, a warp 32 rows
// of these columns, as the parts lie in memory.  Bound by trips to memory: what it needs of the tile is one load, then
// two or four parts' numbers and values are asked for together.
constexpr int kJoinRows = 32;
constexpr int kJoinWarps = 8;         // that share the parts, where there are many
// A row's 16 columns, or what some of the parts add to them.
struct Joined {
  float top = -INFINITY, sum = 0.0f, rounded = 0.0f;
  float o[16] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
};
// Parts first, first + step, ... below `end`, kCount of them asked for together.
template <int kHeadDim, int kCount>
__device__ __forceinline__ void add_parts(const Args& a, int worker, int row, int column, int first, int step, int end, Joined* j) {
  float4 stat[kCount], v[kCount][4];
#pragma unroll
  for (int i = 0; i < kCount; ++i) {
    stat[i] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[i][e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int part = first + i * step;
    if (part < end) {
      const int64_t p = 2 * (static_cast<int64_t>(worker) + part) + (part == 0 ? 1 : 0);
      stat[i] = a.part_stat[p * a.part_rows + row];
      const float* src = a.part_o + (p * (kHeadDim / 4) * a.part_rows + row) * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = *reinterpret_cast<const float4*>(src + (column / 4 + e) * static_cast<int64_t>(a.part_rows) * 4);
    }
  }
  float m = j->top;
#pragma unroll
  for (int i = 0; i < kCount; ++i) m = fmaxf(m, stat[i].x);
  const float use = m == -INFINITY ? 0.0f : m;
  const float old = ptx::ex2_approx(j->top - use);       // (0 before the first part that saw anything)
  j->top = m;
  j->sum *= old;
  j->rounded *= old;
#pragma unroll
  for (int e = 0; e < 16; ++e) j->o[e] *= old;
#pragma unroll
  for (int i = 0; i < kCount; ++i) {
    const float weight = ptx::ex2_approx(stat[i].x - use);      // a part that saw nothing: 0, and nothing in it
    j->sum = fmaf(weight, stat[i].y, j->sum);
    j->rounded = fmaf(weight, stat[i].z, j->rounded);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      j->o[4 * e] = fmaf(weight, v[i][e].x, j->o[4 * e]);
      j->o[4 * e + 1] = fmaf(weight, v[i][e].y, j->o[4 * e + 1]);
      j->o[4 * e + 2] = fmaf(weight, v[i][e].z, j->o[4 * e + 2]);
      j->o[4 * e + 3] = fmaf(weight, v[i][e].w, j->o[4 * e + 3]);
    }
  }
}
template <int kHeadDim, bool kBf16>
__global__ void __launch_bounds__(kHeadDim * 2) fmha_paged_join_kernel(const __grid_constant__ Args a) {
  ptx::grid_dependency_sync();
  const int4 tile = a.meta[blockIdx.x];
  const int parts = tile.w & 0xffff;
  const int row = blockIdx.y * kJoinRows + (threadIdx.x & 31), column = (threadIdx.x >> 5) * 16;
  if (parts == 0 || row >= tile.z || column >= a.head_size) return;
  Joined j;
  for (int i0 = 0; i0 < parts; i0 += 2) add_parts<kHeadDim, 2>(a, blockIdx.x, row, column, i0, 1, parts, &j);
  const int token = row / a.group;
  const int64_t q_row = tile.x + token, head = tile.y + row - token * a.group;
  const float inv = 1.0f / j.rounded;
  uint16_t* out = a.out + q_row * a.o_strides[0] + head * a.o_strides[1] + column;
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = j.rounded == 0.0f ? 0u : pack2<kBf16>(j.o[2 * e] * inv, j.o[2 * e + 1] * inv);
  if (a.out_sectors) {
    store_sector(out, w);
  } else {
    reinterpret_cast<uint4*>(out)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    if (column + 8 < a.head_size) reinterpret_cast<uint4*>(out)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
  if (column == 0 && a.lse != nullptr) a.lse[q_row * a.heads + head] = j.sum == 0.0f ? -INFINITY : (j.top + log2f(j.sum)) * kLn2;
}
// The same for few tiles of many parts: a CTA takes 16 columns of 32 rows of one, its warps share the parts.
template <int kHeadDim, bool kBf16>
__global__ void __launch_bounds__(kJoinWarps * 32) fmha_paged_join_many_kernel(const __grid_constant__ Args a) {
  ptx::grid_dependency_sync();
  __shared__ float of_warp[kJoinWarps][19][33];
  const int named = a.meta[blockIdx.x].w, parts = named & 0xffff, worker = named >> 16;
  const int row0 = blockIdx.y * kJoinRows, column = blockIdx.z * 16, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // The tile's numbers are made again: in the place of one that this call does not have stands an earlier call's.
  const int head_tile = static_cast<int>(blockIdx.x) / a.tile_blocks, t0 = (static_cast<int>(blockIdx.x) - head_tile * a.tile_blocks) * a.block_tokens;
  const int b = head_tile / a.kv_heads, head0 = (head_tile - b * a.kv_heads) * a.group;
  const Request req = load_request(a, b);
  const int rows = min(a.block_tokens, req.rows - t0) * a.group;
  if (rows <= row0 || parts == 0 || worker < 0 || worker + parts > a.workers || column >= a.head_size) return;
  Joined j;
  if (row0 + lane < rows)
    for (int i0 = warp; i0 < parts; i0 += 4 * kJoinWarps) add_parts<kHeadDim, 4>(a, worker, row0 + lane, column, i0, kJoinWarps, parts, &j);
  of_warp[warp][0][lane] = j.top;
  of_warp[warp][1][lane] = j.sum;
  of_warp[warp][2][lane] = j.rounded;
#pragma unroll
  for (int e = 0; e < 16; ++e) of_warp[warp][3 + e][lane] = j.o[e];
  __syncthreads();
  // two columns of a row a thread
  const int row = threadIdx.x >> 3, pair = (threadIdx.x & 7) * 2;
  if (row0 + row >= rows || column + pair >= a.head_size) return;
  float top = -INFINITY, sum = 0.0f, rounded = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, of_warp[w][0][row]);
  const float use = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    const float weight = ptx::ex2_approx(of_warp[w][0][row] - use);
    sum = fmaf(weight, of_warp[w][1][row], sum);
    rounded = fmaf(weight, of_warp[w][2][row], rounded);
    x = fmaf(weight, of_warp[w][3 + pair][row], x);
    y = fmaf(weight, of_warp[w][4 + pair][row], y);
  }
  const int token = (row0 + row) / a.group;
  const int64_t q_row = req.row0 + t0 + token, head = head0 + row0 + row - token * a.group;
  const float inv = 1.0f / rounded;
  *reinterpret_cast<uint32_t*>(a.out + q_row * a.o_strides[0] + head * a.o_strides[1] + column + pair) =
      rounded == 0.0f ? 0u : pack2<kBf16>(x * inv, y * inv);
  if (column + pair == 0 && a.lse != nullptr) a.lse[q_row * a.heads + head] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

int head_dim(int head_size) { return head_size <= 64 ? 64 : head_size <= 128 ? 128 : 256; }
int workers(int dim, int sm_count) { return sm_count * (dim <= 128 ? 2 : 1); }

struct Scratch {
  size_t meta, stat, o, total;
  int part_rows;
};
Scratch scratch_of(const ixk_fmha_paged_desc* d, const ixk_paged_cache* c, int sm_count) {
  const int dim = head_dim(c->head_size), w = workers(dim, sm_count);
  const int group = std::max(d->heads / std::max(c->heads, 1), 1);
  const int64_t tokens = std::max<int64_t>(std::min<int64_t>(std::max(kRows / group, 1), d->rows), 0);
  Scratch s;
  s.part_rows = static_cast<int>(tokens * group);
  s.meta = 0;
  s.stat = (static_cast<size_t>(w) * sizeof(int4) + 255) / 256 * 256;
  s.o = s.stat + (static_cast<size_t>(2 * w) * s.part_rows * sizeof(float4) + 255) / 256 * 256;
  s.total = s.o + static_cast<size_t>(2 * w) * s.part_rows * dim * sizeof(float);
  return s;
}

int check(const ixk_fmha_paged_desc* d, const ixk_paged_cache* c) {
  if (d == nullptr || c == nullptr) return fail(IXK_INVALID_ARGUMENT, "fmha_paged: desc or cache is NULL");
  if (d->reserved != 0) return fail(IXK_INVALID_ARGUMENT, "fmha_paged: desc.reserved must be 0");
  if (d->requests < 0 || d->rows < 0 || d->columns < 1 || d->heads < 1 || c->heads < 1 || d->mask_words < 0)
    return fail(IXK_INVALID_ARGUMENT, "fmha_paged: negative size, or no heads or table columns");
  if (c->head_size < 8 || c->head_size % 8 != 0 || c->head_size > 256)
    return fail(IXK_UNIMPLEMENTED, "fmha_paged: head_size must be a multiple of 8, at most 256");
  if (d->heads % c->heads != 0) return fail(IXK_INVALID_ARGUMENT, "fmha_paged: heads must be a multiple of the cache's heads");
  if (d->heads / c->heads > kRows) return fail(IXK_UNIMPLEMENTED, "fmha_paged: more than 128 query heads to a key head");
  if (c->page_size < 8 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) != 0)
    return fail(IXK_UNIMPLEMENTED, "fmha_paged: page_size must be 8, 16, 32, 64, 128 or 256");
  if (!std::isfinite(d->head_scale * kLog2e)) return fail(IXK_INVALID_ARGUMENT, "fmha_paged: head_scale is not finite");
  // (the kernel's counts run past these by a CTA's threads)
  if (d->rows > 0x7fffffff - 256 || d->requests > 0x7fffffff - 65536 || static_cast<int64_t>(d->columns) * c->page_size > 0x7fffffff - 256)
    return fail(IXK_UNIMPLEMENTED, "fmha_paged: 2^31 rows, requests, or keys of a request, or more");
  return IXK_OK;
}

template <int kHeadDim, bool kBf16, bool kLse, bool kGroups>
int launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const Args& a, int device, int sm_count, cudaStream_t stream) {
  using C = Cfg<kHeadDim>;
  static std::atomic<uint64_t> allowed{0};      // devices on which the kernel may use its shared memory
  const uint64_t bit = 1ull << (device & 63);
  if ((allowed.load(std::memory_order_relaxed) & bit) == 0) {
    IXK_CUDA_OK(cudaFuncSetAttribute(fmha_paged_kernel<kHeadDim, kBf16, kLse, kGroups>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  const int w = workers(kHeadDim, sm_count);
  if (int st = launch_overlapped(fmha_paged_kernel<kHeadDim, kBf16, kLse, kGroups>, dim3(w), dim3(C::kAllThreads), C::kSmemBytes, stream, q, k, v, a)) return st;
  const unsigned blocks = static_cast<unsigned>((a.part_rows + kJoinRows - 1) / kJoinRows);
  if (a.tile_blocks != 0)
    return launch_overlapped(fmha_paged_join_many_kernel<kHeadDim, kBf16>, dim3(static_cast<unsigned>(a.requests) * a.kv_heads * a.tile_blocks, blocks, kHeadDim / 16),
                             dim3(kJoinWarps * 32), 0, stream, a);
  return launch_overlapped(fmha_paged_join_kernel<kHeadDim, kBf16>, dim3(w, blocks), dim3(kHeadDim * 2), 0, stream, a);
}

}  // namespace
}  // namespace fmha_paged
}  // namespace ixk

using namespace ixk;

extern "C" {

size_t ixk_fmha_paged_fwd_workspace_bytes(const ixk_fmha_paged_desc* desc, const ixk_paged_cache* cache) {
  if (fmha_paged::check(desc, cache) != IXK_OK) return 0;
  return fmha_paged::scratch_of(desc, cache, 148).total;
}

int ixk_fmha_paged_fwd(const ixk_fmha_paged_desc* d, const ixk_paged_cache* c, const void* q, const void* k_pages, const void* v_pages,
                       const int32_t* page_table, const int32_t* lengths, const int32_t* row_start, const int32_t* granted,
                       const int32_t* mask, void* out, float* lse, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  IXK_API_RANGE("ixk_fmha_paged_fwd");
  clear_error();
  if (int st = fmha_paged::check(d, c)) return st;
  if (int st = paged::check_cache(c, k_pages, v_pages, "fmha_paged")) return st;
  if (d->requests > 0 && d->rows > 0 &&
      (q == nullptr || out == nullptr || page_table == nullptr || lengths == nullptr || row_start == nullptr || granted == nullptr))
    return fail(IXK_INVALID_ARGUMENT, "fmha_paged: null argument");
  if (!paged::aligned16(q) || !paged::aligned16(out) || !paged::aligned16(workspace))
    return fail(IXK_INVALID_ARGUMENT, "fmha_paged: q, out and workspace must be 16-byte aligned");
  if (d->requests > 1 && d->table_stride < d->columns) return fail(IXK_INVALID_ARGUMENT, "fmha_paged: rows of the page table overlap");
  if (mask != nullptr && (d->mask_words < 1 || (d->rows > 1 && d->mask_stride < d->mask_words)))
    return fail(IXK_INVALID_ARGUMENT, "fmha_paged: mask must have words, and rows that do not overlap");
  for (int i = 0; i < 2; ++i) {
    const int64_t extent = i == 0 ? d->rows : d->heads;
    if (d->q_strides[i] % 8 != 0 || d->o_strides[i] % 8 != 0)
      return fail(IXK_UNIMPLEMENTED, "fmha_paged: q and out strides must be multiples of 8 elements (16 bytes)");
    if (extent > 1 && (d->q_strides[i] < c->head_size || d->o_strides[i] < c->head_size))
      return fail(IXK_INVALID_ARGUMENT, "fmha_paged: rows of q or out overlap");
  }
  if (d->requests > 0 && d->rows > 0) {
    const int64_t rows = d->rows, requests = d->requests;
    const paged::Operand mq(q, c->head_size * 2, {rows, d->heads}, d->q_strides, 2), mo(out, c->head_size * 2, {rows, d->heads}, d->o_strides, 2),
        kp = paged::key_pages(c, k_pages), vp = paged::value_pages(c, v_pages), table(page_table, paged::rows_extent(requests, d->table_stride, d->columns) * 4),
        books[3] = {{lengths, requests * 4}, {row_start, (requests + 1) * 4}, {granted, requests * 4}},
        bits(mask, paged::rows_extent(rows, d->mask_stride, d->mask_words) * 4), ml(lse, rows * d->heads * 4),
        scratch(workspace, static_cast<int64_t>(std::min(workspace_bytes, fmha_paged::scratch_of(d, c, 148).total)));
    if (const char* name = paged::shared_memory({{"out", &mo, &mq, nullptr}, {"lse", &ml, nullptr, nullptr}, {"the workspace", &scratch, nullptr, nullptr}},
                                                {&mq, &kp, &vp, &table, &books[0], &books[1], &books[2], &bits}))
      return fail(IXK_INVALID_ARGUMENT, std::string("fmha_paged: ") + name + " shares memory with another operand or with itself");
  }
  DeviceInfo info;
  if (int st = get_device_info(&info)) return st;
  if (d->requests == 0 || d->rows == 0) return IXK_OK;
  if (info.sm_count > 148) info.sm_count = 148;        // (what the workspace was asked for)
  const fmha_paged::Scratch scratch = fmha_paged::scratch_of(d, c, info.sm_count);
  if (workspace == nullptr || workspace_bytes < scratch.total)
    return fail(IXK_WORKSPACE_TOO_SMALL, "fmha_paged: workspace_bytes is below ixk_fmha_paged_fwd_workspace_bytes");

  fmha_paged::Args a{};
  a.requests = d->requests;
  a.heads = d->heads;
  a.kv_heads = c->heads;
  a.group = d->heads / c->heads;
  a.head_size = c->head_size;
  a.block_tokens = fmha_paged::kRows / a.group;
  a.rows_in = static_cast<int>(d->rows);
  a.columns = d->columns;
  a.page_shift = __builtin_ctz(static_cast<unsigned>(c->page_size));
  a.pages = c->pages;
  a.cap = d->columns * c->page_size;
  const uint32_t chunks = static_cast<uint32_t>(c->head_size / fmha_paged::kChunkElems);
  const bool by_groups = c->head_size == fmha_paged::head_dim(c->head_size) && c->page_size < fmha_paged::kKeys && fmha_paged::kKeys / c->page_size * chunks > 8 &&
                (c->heads == 1 || (c->k_strides[3] == c->head_size && c->v_strides[3] == c->head_size));
  a.negate = d->head_scale < 0.0f;
  // (0: all weights alike; a tiny one, since masked scores are -inf)
  a.scale_log2 = d->head_scale == 0.0f ? 1e-30f : std::fabs(d->head_scale) * fmha_paged::kLog2e;
  a.table_stride = d->table_stride;
  a.mask_stride = d->mask_stride;
  a.mask_words = d->mask_words;
  a.table = page_table, a.lengths = lengths, a.row_start = row_start, a.granted = granted, a.mask = mask;
  a.v = static_cast<const uint16_t*>(v_pages);
  for (int i = 0; i < 3; ++i) a.v_strides[i] = c->v_strides[i + 1];
  a.out = static_cast<uint16_t*>(out);
  for (int i = 0; i < 2; ++i) a.o_strides[i] = d->o_strides[i];
  a.out_sectors = (reinterpret_cast<uintptr_t>(out) & 31u) == 0 && c->head_size % 16 == 0 && d->o_strides[0] % 16 == 0 && d->o_strides[1] % 16 == 0;
  a.lse = lse;
  a.status_word = info.status_word;
  a.part_rows = scratch.part_rows;
  a.workers = fmha_paged::workers(fmha_paged::head_dim(c->head_size), info.sm_count);
  // Tiles of two parts and more (if they are of about one length): several warps share the parts of one in the join (one request, us:
  // 8000 keys 27.4 -> 13.8, 60000 keys 49 -> 33; 4 trees of 16 over 4000 keys 21 -> 17.8).
  const int64_t blocks = (d->rows + a.block_tokens - 1) / a.block_tokens, tiles = static_cast<int64_t>(d->requests) * c->heads * blocks;
  a.tile_blocks = tiles * 2 <= a.workers ? static_cast<int>(blocks) : 0;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.meta = reinterpret_cast<int4*>(ws + scratch.meta);
  a.part_stat = reinterpret_cast<float4*>(ws + scratch.stat);
  a.part_o = reinterpret_cast<float*>(ws + scratch.o);

  const CUtensorMapDataType type = c->dtype == IXK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  // (the stride of a dimension of one entry is never used: any that a map takes)
  auto bytes = [](int64_t stride, int64_t extent) { return static_cast<uint64_t>(extent > 1 ? stride * 2 : 512); };
  CUtensorMap mq, mk, mv;
  TmapSpec sq{type, 3, {static_cast<uint64_t>(c->head_size), static_cast<uint64_t>(d->heads), static_cast<uint64_t>(d->rows)},
              {bytes(d->q_strides[1], d->heads), bytes(d->q_strides[0], d->rows)},
              {fmha_paged::kChunkElems, static_cast<uint32_t>(a.group), static_cast<uint32_t>(a.block_tokens)}, true};
  if (int st = encode_tmap(&mq, q, sq)) return st;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i == 0 ? c->k_strides : c->v_strides;
    const uint32_t keys = static_cast<uint32_t>(std::min(c->page_size, fmha_paged::kKeys));
    TmapSpec sk{type, 4,
                {static_cast<uint64_t>(c->head_size), static_cast<uint64_t>(c->heads), static_cast<uint64_t>(c->page_size), static_cast<uint64_t>(c->pages)},
                {bytes(s[3], c->heads), bytes(s[2], c->page_size), bytes(s[1], c->pages)},
                {fmha_paged::kChunkElems, 1, keys, 1}, true};
    if (by_groups)       // all chunks of all heads of a token behind one another
      sk = TmapSpec{type, 4,
                    {fmha_paged::kChunkElems, static_cast<uint64_t>(c->page_size), static_cast<uint64_t>(c->heads) * chunks, static_cast<uint64_t>(c->pages)},
                    {bytes(s[2], c->page_size), fmha_paged::kChunkElems * 2, bytes(s[1], c->pages)},
                    {fmha_paged::kChunkElems, 8, chunks, 1}, true};
    if (int st = encode_tmap(i == 0 ? &mk : &mv, i == 0 ? k_pages : v_pages, sk)) return st;
  }
  auto s = static_cast<cudaStream_t>(cuda_stream);
  const int dim = fmha_paged::head_dim(c->head_size);
  auto with = [&](auto bf16, auto with_lse) {
    constexpr bool kBf16 = decltype(bf16)::value, kLse = decltype(with_lse)::value;
    if (dim == 64) return fmha_paged::launch<64, kBf16, kLse, false>(mq, mk, mv, a, info.device, info.sm_count, s);
    if (dim == 128)
      return by_groups ? fmha_paged::launch<128, kBf16, kLse, true>(mq, mk, mv, a, info.device, info.sm_count, s)
                       : fmha_paged::launch<128, kBf16, kLse, false>(mq, mk, mv, a, info.device, info.sm_count, s);
    return by_groups ? fmha_paged::launch<256, kBf16, kLse, true>(mq, mk, mv, a, info.device, info.sm_count, s)
                     : fmha_paged::launch<256, kBf16, kLse, false>(mq, mk, mv, a, info.device, info.sm_count, s);
  };
  const std::true_type yes;
  const std::false_type no;
  if (lse != nullptr) return c->dtype == IXK_BF16 ? with(yes, yes) : with(no, yes);
  return c->dtype == IXK_BF16 ? with(yes, no) : with(no, no);
}

}  // extern "C"
