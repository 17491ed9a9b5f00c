// The logits of a vocabulary head, z = scale (x w^T + bias), made tile by tile on the tensor cores and never stored: each tile
// is turned, where it lies in tensor memory, into what the loss or its gradient needs of it.
//
//   statistics   per row the running maximum and sum of exponentials (base 2: t = z log2 e, one fused multiply-add), and
//                z at the row's targets; a label's column can be left out (the tensor cores cut what an addition shifts out
//                instead of rounding it: a logit of 10 loses 4e-5 over 4096 products, and the label's is the one that the
//                loss is made of, so the loss kernel makes it again in fp32 where that is a row of w to read)
//   gradient     G = g (softmax(z) - target weights), g relative to the batch's largest, rounded once to the 16-bit operand
//                of the two products that follow (dx = G w, dw = G^T x): a rounding error of at most 2^-8 or 2^-11 of each
//                entry, as of any activation gradient, independent from entry to entry.  p - 1 of a label apart is handed in, made
//                of the same fp32 logit as lse; the other targets' p - q is made of the logits that lse was made of, chunk of K by
//                chunk: where the model is sure of a token, or agrees with its teacher, the logit's own error would be as large
//
// Both are 2 N D V flops on the tensor cores, which bound them from hidden sizes of about 600 on: 2048 x 4096 x 51200 532 and
// 530 us alone, 1.61 PFLOP/s, and as much as the power limit leaves of that in a row of such calls.  Below, the epilogue does:
// reading tensor memory (16 bytes a cycle and quarter of an SM) and V N exponentials (16 a cycle and SM) take 2048 cycles each
// of a tile's 4400 at 6000 x 160 x 30000, 111 us.  Few rows are a stream of w: 16 x 4096 x 51200 72 us, 5.8 TB/s.
// CTA pairs work on 256 x 256 tiles (cta_group::2: half of w's tile per CTA),
// or, where that leaves pairs without one, single CTAs on 128 rows and as many columns as give every SM an equal share.
// A unit of work is a row block and a strip of consecutive column tiles, whose statistics stay in registers.
//
//   warp 0      TMA producer: slabs of 64 hidden elements of x and w into a ring (128-byte swizzle)
//   warp 1      tcgen05.mma issuer (even CTA of a pair), accumulators double-buffered in tensor memory
//   warps 2-9   epilogue: two warps per 32 rows, taking groups of 64 columns in turn; a thread is a row
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>

#include "head_loss.h"
#include "ptx.cuh"

namespace ixk {
namespace head {

namespace {

constexpr int kBlockM = 128;
constexpr int kSlabElems = 64;
constexpr int kSlabBytes = 128;
constexpr int kUmmaK = 16;
constexpr int kMaxTileN = 256;
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 32 * (2 + kEpilogueWarps);
constexpr int kTmemCols = 2 * kMaxTileN;
constexpr int kRingBytes = 192 * 1024;
constexpr int kMaxStages = 32;
constexpr int kBoxBytes = 32 * 128;                       // a warp's 32 rows x 64 16-bit (or 32 fp32) columns
constexpr int kBarrierBytes = 8 * (2 * kMaxStages + 4) + 8;
constexpr int kSmemBytes = kRingBytes + kEpilogueWarps * kBoxBytes + kBarrierBytes + 1024;
static_assert(kSmemBytes <= 232448, "shared memory budget");
constexpr int kGroupM = 8;      // row blocks that share a column strip in L2
constexpr int kAssumedSms = 148;
constexpr int kMaxStrip = 8;
constexpr float kLog2E = 1.4426950408889634f;
// Slabs of K that the tensor cores add up before the statistics' warps take over: their sums cut what an addition shifts out
// (4e-6 of a logit over K = 4096, always towards zero), the warps' fp32 additions round.  Every chunk is read out of tensor
// memory, which holds up the next one's products, and its sums' registers spill (264 to 328 bytes a thread).  4096 x 4096 x 32768,
// statistics: without chunks 646 us, of 24 slabs 664, of 16 671; the lse of logits of about 10, its label not apart, is off by
// 2.6e-5, 8e-6 and 6e-6, apart (few rows too) by 3.3e-6, 1.1e-6 and 0.9e-6.  A tile's chunks are of equal length, at most this.
constexpr int kChunkSlabs = 24;
// The gradient takes the same chunks where its targets' entries come from the tile (7355 x 3520 x 8144 column-major, forward and
// backward: 1224 -> 1253 us).
enum class Mode { kStats, kStatsChunks, kGrad, kGradChunks };     // statistics of one chunk, of several; gradient the same
enum : int { kSiteProducer = 601, kSiteFull = 602, kSiteAcc = 603, kSiteEpilogue = 604 };

struct Args {
  int rows, slabs, first, count;        // columns [first, first + count)
  int tiles_n, tile_n, strip, strips;
  int stages, stage_bytes, a_bytes, b_boxes, chunk_slabs;
  int w_mn_major;
  uint32_t idesc;
  const int* active_rows;
  const RowInfo* info;
  const void* bias;
  int bf16, bias_vec_ok;
  float scale, scale2;                  // of the logits; times log2 e
  Targets targets;
  float2* partial;
  float* at_target;
  const float* range;
  int* status_word;
};

__device__ __forceinline__ float2 unpack2(uint32_t w, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// v[i] += bias[c + i] for i < count (the same 32 values in every lane).
__device__ __forceinline__ void add_bias(const Args& a, int c, int count, float (&v)[32]) {
  const uint16_t* b = static_cast<const uint16_t*>(a.bias) + c;
  if (a.bias_vec_ok && count == 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 w = reinterpret_cast<const uint4*>(b)[i];
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2(words[j], a.bf16);
        v[8 * i + 2 * j] += f.x;
        v[8 * i + 2 * j + 1] += f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < count) v[i] += unpack2(b[i], a.bf16).x;
  }
}

// A thread's row of its warp's box as 32 floats: 16-byte pieces exchanged by the row, so that the warp's accesses to one
// piece of every row meet all banks.
__device__ __forceinline__ uint32_t box_addr(uint32_t box, int lane, int i) {
  return box + static_cast<uint32_t>(lane * 128 + (((i >> 2) ^ (lane & 7)) << 4) + (i & 3) * 4);
}
__device__ __forceinline__ void box_put(uint32_t box, int lane, const float (&v)[32]) {
#pragma unroll
  for (int g = 0; g < 8; ++g)
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(box_addr(box, lane, 4 * g)), "f"(v[4 * g]), "f"(v[4 * g + 1]),
                 "f"(v[4 * g + 2]), "f"(v[4 * g + 3])
                 : "memory");
}
__device__ __forceinline__ void box_get(uint32_t box, int lane, float (&v)[32]) {
#pragma unroll
  for (int g = 0; g < 8; ++g)
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v[4 * g]), "=f"(v[4 * g + 1]), "=f"(v[4 * g + 2]), "=f"(v[4 * g + 3])
                 : "r"(box_addr(box, lane, 4 * g))
                 : "memory");
}
__device__ __forceinline__ float box_read(uint32_t addr) {
  float f;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(addr) : "memory");
  return f;
}
__device__ __forceinline__ void box_write(uint32_t addr, float f) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(f) : "memory");
}

// A row's walk through its targets in ascending order.
struct Walk {
  const int* column;
  int entries, at, next, after;     // the columns of targets `at` and at + 1 (asked for a step ahead of its use)
  __device__ __forceinline__ void step() {
    ++at;
    next = after;
    after = at + 1 < entries ? column[at + 1] : kNoColumn;
  }
};
__device__ __forceinline__ Walk start_walk(const Targets& t, const RowInfo& info, bool active, int from) {
  Walk w{nullptr, 1, 0, kNoColumn, kNoColumn};
  if (!active) return w;
  if (t.labels != nullptr) {
    if (info.label >= from) w.next = info.label;
    return w;
  }
  w.column = t.column + static_cast<int64_t>(info.row) * t.entries;
  w.entries = t.entries;
  w.at = t.start[static_cast<int64_t>(info.row) * t.starts + from / kStartUnit];
  w.next = w.at < t.entries ? w.column[w.at] : kNoColumn;
  w.after = w.at + 1 < t.entries ? w.column[w.at + 1] : kNoColumn;
  while (w.next < from) w.step();
  return w;
}

template <bool kPair, Mode kMode>
__global__ void __launch_bounds__(kThreads, 1)
head_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
            const __grid_constant__ CUtensorMap tmap_g, const Args args) {
  constexpr bool kGrad = kMode == Mode::kGrad || kMode == Mode::kGradChunks, kChunks = kMode == Mode::kStatsChunks || kMode == Mode::kGradChunks;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
  const uint32_t box_base = smem_base + kRingBytes;
  const uint32_t bar_base = box_base + kEpilogueWarps * kBoxBytes;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kMaxStages + s); };
  auto acc_full_bar = [&](int b) { return bar_base + 8u * (2 * kMaxStages + b); };
  auto acc_empty_bar = [&](int b) { return bar_base + 8u * (2 * kMaxStages + 2 + b); };
  uint8_t* tail = smem_gen + kRingBytes + kEpilogueWarps * kBoxBytes + 8 * (2 * kMaxStages + 4);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(tail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? ptx::cluster_ctarank() : 0;
  ptx::AbortCtl ctl{abort_flag, args.status_word};

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kMaxStages; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(acc_full_bar(b), 1);
      ptx::mbar_init(acc_empty_bar(b), (kPair ? 2 : 1) * 32 * kEpilogueWarps);
    }
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmap_x);
    ptx::prefetch_tmap(&tmap_w);
    if (kGrad) ptx::prefetch_tmap(&tmap_g);
  }
  __syncthreads();
  if constexpr (kPair) ptx::cluster_sync_all();   // both CTAs' barriers exist before anyone arrives on them remotely
  if (warp == 1) {                                // (cta_group::2: one warp of each CTA)
    const uint32_t slot = ptx::smem_u32(const_cast<uint32_t*>(tmem_slot));
    if constexpr (kPair) {
      ptx::tmem_alloc_pair(slot, kTmemCols);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(slot, kTmemCols);
      ptx::tmem_relinquish();
    }
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if constexpr (kPair) ptx::cluster_sync_all();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  ptx::grid_dependency_sync();

  // (an empty batch still makes one row block, of zeros, for the products that read whole slabs of rows)
  const int active_rows = args.active_rows != nullptr ? min(*args.active_rows, args.rows) : args.rows;
  constexpr int kTileM = (kPair ? 2 : 1) * kBlockM;
  const int tiles_m = max((active_rows + kTileM - 1) / kTileM, 1);
  const int num_units = tiles_m * args.strips;
  const int worker = kPair ? blockIdx.x >> 1 : blockIdx.x, workers = kPair ? gridDim.x >> 1 : gridDim.x;
  // Units of a band of row blocks, strip by strip: the CTAs at work share few strips of w and few blocks of x in L2.
  const ptx::FastDiv by_band(kGroupM * args.strips), by_last((tiles_m - 1) % kGroupM + 1);
  auto unit_at = [&](int u, int& bm, int& n_begin, int& n_end) {
    int r, in, strip;
    const int first_m = by_band.div(u, r) * kGroupM;
    if (tiles_m - first_m >= kGroupM) {
      strip = r / kGroupM;
      in = r % kGroupM;
    } else {
      strip = by_last.div(r, in);
    }
    bm = first_m + in;
    n_begin = strip * args.strip;
    n_end = min(n_begin + args.strip, args.tiles_n);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    int stage = 0;
    uint32_t phase = 0;
    bool alive = true;
    const uint32_t cta_bytes = static_cast<uint32_t>(args.a_bytes + (args.w_mn_major ? args.b_boxes * kSlabElems : kPair ? args.tile_n / 2 : args.tile_n) * kSlabBytes);
    for (int u = worker; u < num_units && alive; u += workers) {
      int bm, n_begin, n_end;
      unit_at(u, bm, n_begin, n_end);
      const int m0 = (kPair ? bm * 2 + static_cast<int>(rank) : bm) * kBlockM;
      for (int n = n_begin; n < n_end && alive; ++n) {
        const int v0 = args.first + n * args.tile_n + (kPair ? static_cast<int>(rank) * (args.tile_n / 2) : 0);
        for (int kb = 0; kb < args.slabs; ++kb) {
          if (!ptx::mbar_wait(empty_bar(stage), phase ^ 1u, ctl, kSiteProducer)) {
            alive = false;
            break;
          }
          const uint32_t a_dst = smem_base + stage * args.stage_bytes;
          const uint32_t b_dst = a_dst + args.a_bytes;
          const int k0 = kb * kSlabElems;
          if (ptx::elect_one()) {
            if constexpr (kPair) {   // both CTAs' copies are counted on the even CTA's barrier
              const uint32_t bar = ptx::map_to_cta(full_bar(stage), 0);
              if (rank == 0) ptx::mbar_expect_tx(full_bar(stage), 2 * cta_bytes);
              ptx::tma_load_3d_pair(a_dst, &tmap_x, bar, k0, m0, 0);
              if (args.w_mn_major) {
                for (int i = 0; i < args.b_boxes; ++i)
                  ptx::tma_load_3d_pair(b_dst + i * (kSlabElems * kSlabBytes), &tmap_w, bar, v0 + i * kSlabElems, k0, 0);
              } else {
                ptx::tma_load_3d_pair(b_dst, &tmap_w, bar, k0, v0, 0);
              }
            } else {
              const uint32_t bar = full_bar(stage);
              ptx::mbar_expect_tx(bar, cta_bytes);
              ptx::tma_load_3d(a_dst, &tmap_x, bar, k0, m0, 0);
              if (args.w_mn_major) {
                for (int i = 0; i < args.b_boxes; ++i)
                  ptx::tma_load_3d(b_dst + i * (kSlabElems * kSlabBytes), &tmap_w, bar, v0 + i * kSlabElems, k0, 0);
              } else {
                ptx::tma_load_3d(b_dst, &tmap_w, bar, k0, v0, 0);
              }
            }
          }
          __syncwarp();
          if (++stage == args.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------ MMA issuer (for both CTAs of a pair)
    int stage = 0, buf = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool alive = true;
    const uint32_t b_lbo = args.w_mn_major ? kSlabElems * kSlabBytes : 16;
    const uint32_t b_kstep = args.w_mn_major ? kUmmaK * kSlabBytes : 32;
    for (int u = worker; u < num_units && alive; u += workers) {
      int bm, n_begin, n_end;
      unit_at(u, bm, n_begin, n_end);
      // (accumulators are handed over tile by tile, or chunk by chunk of one)
      const int chunks = kChunks ? (args.slabs + args.chunk_slabs - 1) / args.chunk_slabs : 1;
      for (int i = 0; i < (n_end - n_begin) * chunks && alive; ++i) {
        if (!ptx::mbar_wait(acc_empty_bar(buf), acc_phase ^ 1u, ctl, kSiteAcc)) {
          alive = false;
          break;
        }
        ptx::tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + buf * kMaxTileN;
        const int slabs = kChunks ? min(args.chunk_slabs, args.slabs - i % chunks * args.chunk_slabs) : args.slabs;
        for (int kb = 0; kb < slabs; ++kb) {
          if (!ptx::mbar_wait(full_bar(stage), phase, ctl, kSiteFull)) {
            alive = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t a_src = smem_base + stage * args.stage_bytes;
          const uint32_t b_src = a_src + args.a_bytes;
#pragma unroll
          for (int ks = 0; ks < kSlabElems / kUmmaK; ++ks) {
            const uint64_t da = ptx::umma_smem_desc(a_src + ks * 32, 16, 1024);
            const uint64_t db = ptx::umma_smem_desc(b_src + ks * b_kstep, b_lbo, 1024);
            if constexpr (kPair) ptx::umma_ss_pair_elect<ptx::kKindF16>(d_tmem, da, db, args.idesc, (kb | ks) != 0 ? 1u : 0u);
            else ptx::umma_ss_elect<ptx::kKindF16>(d_tmem, da, db, args.idesc, (kb | ks) != 0 ? 1u : 0u);
          }
          if constexpr (kPair) ptx::umma_commit_pair_elect(empty_bar(stage));
          else ptx::umma_commit_elect(empty_bar(stage));
          if (++stage == args.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!alive) break;
        if constexpr (kPair) ptx::umma_commit_pair_elect(acc_full_bar(buf));
        else ptx::umma_commit_elect(acc_full_bar(buf));
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1u;
      }
    }
  } else if (warp >= 2) {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;           // TMEM lanes [32 quarter, 32 quarter + 32) belong to this warp
    const int half = (warp - 2) >> 2;       // which groups of 64 columns
    const uint32_t box = box_base + static_cast<uint32_t>((warp - 2) * kBoxBytes);
    const uint32_t acc_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const bool bf16 = args.bf16 != 0;
    const float s2 = args.scale2;
    int buf = 0;
    uint32_t acc_phase = 0;
    bool alive = true;
    const float range = kGrad ? *args.range : 1.0f;
    int warp_row = 0, n_begin = 0, n_end = 0;
    RowInfo info{0, kNoColumn, 0.0f, 0.0f};
    // a unit's place, and what is to be known of this thread's row (asked for a unit ahead of its use)
    auto look = [&](int u, int& first_row, int& from, int& to, RowInfo& i) {
      int bm;
      unit_at(u, bm, from, to);
      first_row = (kPair ? bm * 2 + static_cast<int>(rank) : bm) * kBlockM + quarter * 32;
      const int row = first_row + lane;
      if (row >= active_rows) return;
      if (args.info != nullptr) {
        const int4 v = *reinterpret_cast<const int4*>(args.info + row);
        i = RowInfo{v.x, v.y, __int_as_float(v.z), __int_as_float(v.w)};
      } else {
        i.row = row;
        if (args.targets.labels != nullptr) {
          const int64_t label = args.targets.wide ? static_cast<const int64_t*>(args.targets.labels)[row] : static_cast<const int*>(args.targets.labels)[row];
          // (a label outside the vocabulary is in no tile)
          i.label = label != args.targets.ignore_index && label >= 0 && label < kNoColumn ? static_cast<int>(label) : kNoColumn;
        }
      }
    };
    if (worker < num_units) look(worker, warp_row, n_begin, n_end, info);
    int next_row = 0, next_begin = 0, next_end = 0;
    RowInfo next_info = info;
    for (int u = worker; u < num_units && alive; u += workers, warp_row = next_row, n_begin = next_begin, n_end = next_end, info = next_info) {
      if (u + workers < num_units) look(u + workers, next_row, next_begin, next_end, next_info);
      const int row = warp_row + lane;
      const bool active = row < active_rows;
      const int64_t orig = info.row;
      Walk walk = start_walk(args.targets, info, active, args.first + n_begin * args.tile_n);
      float top = -FLT_MAX, sum = 0.0f;     // statistics so far: t <= top, sum of 2^(t - top)
      const float lse2 = info.lse2, coef = info.coef * range;
      // (the products read the gradient's rows up to the end of a slab, or of the only row block: zeros)
      const bool work = !kGrad ? warp_row < active_rows
                               : args.rows <= kDirectRows || warp_row < (active_rows + kSlabElems - 1) / kSlabElems * kSlabElems;
      // 32 columns of the tile from c0 on, `count` of them in the vocabulary, into the row's statistics
      auto take = [&](float (&v)[32], int col, int count) {
        const int col_end = col + count;
        if (args.bias != nullptr) add_bias(args, col, count, v);
        const bool hit = __any_sync(0xffffffffu, walk.next < col_end);
        if (hit) {
          box_put(box, lane, v);
          while (walk.next < col_end) {
            if (walk.next >= col) {
              const uint32_t addr = box_addr(box, lane, walk.next - col);
              // (a label apart stays out of the sum: the loss adds it, from a product of its own)
              if (args.targets.apart) box_write(addr, -INFINITY);
              else args.at_target[orig * walk.entries + walk.at] = box_read(addr) * args.scale;
            }
            walk.step();
          }
          if (args.targets.apart) box_get(box, lane, v);
        }
        if (count < 32) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i >= count) v[i] = -INFINITY;
        }
        float m = v[0];
#pragma unroll
        for (int i = 1; i < 31; i += 2) m = ptx::max3(m, v[i], v[i + 1]);
        m = fmaxf(m, v[31]);
        // (finite, whatever the logits: an infinite one makes the sum infinite, not undefined)
        const float new_top = fminf(fmaxf(top, m * s2), FLT_MAX);
        sum *= ptx::ex2_approx(top - new_top);
        top = new_top;
        const uint64_t scale_pair = ptx::f32x2(s2, s2), top_pair = ptx::f32x2(-top, -top);
        uint64_t part0 = ptx::f32x2(0.0f, 0.0f), part1 = part0;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float e0, e1, e2, e3;
          ptx::f32x2_split(ptx::fma2(ptx::f32x2(v[i], v[i + 1]), scale_pair, top_pair), e0, e1);
          ptx::f32x2_split(ptx::fma2(ptx::f32x2(v[i + 2], v[i + 3]), scale_pair, top_pair), e2, e3);
          part0 = ptx::add2(part0, ptx::f32x2(ptx::ex2_approx(e0), ptx::ex2_approx(e1)));
          part1 = ptx::add2(part1, ptx::f32x2(ptx::ex2_approx(e2), ptx::ex2_approx(e3)));
        }
        float a, b;
        ptx::f32x2_split(ptx::add2(part0, part1), a, b);
        sum += a + b;
      };
      // the same columns as 16-bit entries of the gradient
      auto gradient = [&](float (&v)[32], int col, int count, uint32_t* words) {
        const int col_end = col + count;
        if (args.bias != nullptr) add_bias(args, col, count, v);
        const bool hit = __any_sync(0xffffffffu, walk.next < col_end);
        const uint64_t scale_pair = ptx::f32x2(s2, s2), lse_pair = ptx::f32x2(-lse2, -lse2);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float e0, e1;
          ptx::f32x2_split(ptx::fma2(ptx::f32x2(v[i], v[i + 1]), scale_pair, lse_pair), e0, e1);
          v[i] = ptx::ex2_approx(e0) * coef;
          v[i + 1] = ptx::ex2_approx(e1) * coef;
        }
        if (hit) {
          box_put(box, lane, v);
          while (walk.next < col_end) {
            if (walk.next >= col) {
              const uint32_t addr = box_addr(box, lane, walk.next - col);
              if (args.targets.apart) {
                box_write(addr, coef * args.targets.gap[row]);
              } else {
                const float weight = args.targets.labels != nullptr ? 1.0f : args.targets.weight[orig * walk.entries + walk.at];
                box_write(addr, box_read(addr) - coef * weight);
              }
            }
            walk.step();
          }
          box_get(box, lane, v);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) words[i] = active ? pack2(v[2 * i], v[2 * i + 1], bf16) : 0u;
      };
      // 64 columns of them on their way, through this warp's box
      auto box_free = [&] {      // (the store before this one has read it)
        if (lane == 0) ptx::bulk_wait_group_read<0>();
        __syncwarp();
      };
      auto leave = [&](const uint32_t (&words)[32], int column) {
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const uint32_t addr = box + static_cast<uint32_t>(lane * 128 + ((g ^ (lane & 7)) << 4));
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(words[4 * g]), "r"(words[4 * g + 1]),
                       "r"(words[4 * g + 2]), "r"(words[4 * g + 3])
                       : "memory");
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          ptx::tma_store_3d(&tmap_g, box, column, warp_row, 0);
          ptx::bulk_commit_group();
        }
      };
      for (int n = n_begin; n < n_end; ++n) {
        const int n0 = n * args.tile_n, limit = min(args.tile_n, args.count - n0);
        if constexpr (kChunks) {
          // the tile's logits chunk of K by chunk, in registers: this warp's two groups of 64 columns
          float acc[2][64];
          for (int first = 0; first < args.slabs && alive; first += args.chunk_slabs) {
            alive = ptx::mbar_wait(acc_full_bar(buf), acc_phase, ctl, kSiteEpilogue);
            if (!alive) break;
            ptx::tc_fence_after_sync();
            if (work) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int c0 = half * 64 + (q >> 1) * 128 + (q & 1) * 32;
                if (c0 < limit) {      // warp-uniform
                  uint32_t r[32];
                  ptx::tmem_ld_32x32(acc_lane + buf * kMaxTileN + c0, r);
                  ptx::tmem_ld_wait();
#pragma unroll
                  for (int i = 0; i < 32; ++i) {
                    float& sum_of = acc[q >> 1][(q & 1) * 32 + i];
                    sum_of = __uint_as_float(r[i]) + (first == 0 ? 0.0f : sum_of);
                  }
                }
              }
            }
            ptx::tc_fence_before_sync();
            if (kPair && rank == 1) ptx::mbar_arrive_cluster_tmem(acc_empty_bar(buf), 0);
            else ptx::mbar_arrive(acc_empty_bar(buf));
            buf ^= 1;
            if (buf == 0) acc_phase ^= 1u;
          }
          if (!alive) break;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int g0 = half * 64 + g * 128;
            if (!work || g0 >= limit) continue;
            uint32_t words[32];
            if constexpr (kGrad) box_free();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c0 = g0 + 32 * h, count = min(32, limit - c0);
              float v[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = acc[g][32 * h + i];
              if constexpr (kGrad) {
                if (count > 0) {
                  gradient(v, args.first + n0 + c0, count, words + 16 * h);
                } else {
#pragma unroll
                  for (int i = 0; i < 16; ++i) words[16 * h + i] = 0u;
                }
              } else if (count > 0) {
                take(v, args.first + n0 + c0, count);
              }
            }
            if constexpr (kGrad) leave(words, n0 + g0);
          }
          continue;
        }
        if (!ptx::mbar_wait(acc_full_bar(buf), acc_phase, ctl, kSiteEpilogue)) {
          alive = false;
          break;
        }
        ptx::tc_fence_after_sync();
        const uint32_t acc = acc_lane + buf * kMaxTileN;
        if (work) {
#pragma unroll 1
          for (int g0 = half * 64; g0 < limit; g0 += 128) {
            uint32_t words[32];
            if constexpr (kGrad) box_free();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c0 = g0 + 32 * h, count = min(32, limit - c0);
              if (count > 0) {           // warp-uniform
                uint32_t r[32];
                float v[32];
                ptx::tmem_ld_32x32(acc + c0, r);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
                if constexpr (!kGrad) take(v, args.first + n0 + c0, count);
                else gradient(v, args.first + n0 + c0, count, words + 16 * h);
              } else if constexpr (kGrad) {
#pragma unroll
                for (int i = 0; i < 16; ++i) words[16 * h + i] = 0u;
              }
            }
            if constexpr (kGrad) leave(words, n0 + g0);
          }
        }
        ptx::tc_fence_before_sync();
        if (kPair && rank == 1) ptx::mbar_arrive_cluster_tmem(acc_empty_bar(buf), 0);
        else ptx::mbar_arrive(acc_empty_bar(buf));
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1u;
      }
      if constexpr (!kGrad) {
        if (alive && active)
          args.partial[static_cast<int64_t>(2 * (n_begin / args.strip) + half) * args.rows + row] = make_float2(top, sum);
      }
    }
    if (kGrad && lane == 0) ptx::bulk_wait_group<0>();   // the boxes must outlive the stores that read them
  }

  // Teardown.  On the abort path give copies still in flight time to land before their shared memory is released; neither
  // CTA of a pair leaves while the other can still read its shared memory or arrive on its barriers.
  if (*abort_flag != 0) __nanosleep(2000000);
  ptx::tc_fence_before_sync();
  __syncthreads();
  if constexpr (kPair) ptx::cluster_sync_all();
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    if constexpr (kPair) ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
    else ptx::tmem_dealloc(tmem_base, kTmemCols);
  }
  if constexpr (kPair) ptx::cluster_sync_all();
}

struct Tiling {
  bool pair;
  int tile_n, tiles_n, strip, strips;
};

// 256 x 256 tiles on CTA pairs once every pair has one (narrower ones where that fills the last of few rounds); else row blocks
// of 128 and column tiles that are as wide as a whole number of rounds of all SMs allows, in steps of `unit` columns.
Tiling tiling_for(int64_t rows, int64_t columns, int unit) {
  Tiling t{};
  const int64_t pairs = kAssumedSms / 2, pair_rows = (rows + 255) / 256, wide = (columns + kMaxTileN - 1) / kMaxTileN;
  t.pair = rows > kBlockM && pair_rows * wide >= pairs;
  t.strip = 1;
  if (t.pair) {
    // (a tile of w columns takes about w + 16 columns' time; the gradient's boxes are 64 columns, a CTA's half 16)
    t.tile_n = kMaxTileN;
    auto time = [&](int w) { return (pair_rows * ((columns + w - 1) / w) + pairs - 1) / pairs * (w + 16); };
    for (int w = kMaxTileN; w >= 192; w -= std::max(unit, 32))
      if (time(w) * 100 < time(t.tile_n) * 98) t.tile_n = w;
    const int64_t wide = (columns + t.tile_n - 1) / t.tile_n;
    t.tiles_n = static_cast<int>(wide);
    // the longest strip that does not lengthen the longest pair's share by more than 1 %
    auto rounds = [&](int strip) { return (pair_rows * ((wide + strip - 1) / strip) + pairs - 1) / pairs * strip; };
    for (int s = 2; s <= kMaxStrip; s *= 2)
      if (rounds(s) * 100 <= rounds(1) * 101) t.strip = s;
  } else {
    const int64_t blocks = (rows + kBlockM - 1) / kBlockM;
    const int64_t tiles = (blocks * wide + kAssumedSms - 1) / kAssumedSms * kAssumedSms;     // of whole rounds
    const int64_t per_block = std::max<int64_t>(tiles / blocks, 1);
    const int64_t width = (columns + per_block - 1) / per_block;
    t.tile_n = static_cast<int>(std::min<int64_t>(std::max<int64_t>((width + unit - 1) / unit * unit, 32), kMaxTileN));
    t.tiles_n = static_cast<int>((columns + t.tile_n - 1) / t.tile_n);
  }
  t.strips = (t.tiles_n + t.strip - 1) / t.strip;
  return t;
}

constexpr int kStatUnit = 16, kGradUnit = 64;   // (the gradient leaves in boxes of 64 columns)

template <bool kGrad>
int launch(const Pass& p, const DeviceInfo& dev, cudaStream_t stream) {
  const Tiling t = tiling_for(p.rows, p.count, kGrad ? kGradUnit : kStatUnit);
  const int a_rows = t.pair ? kBlockM : static_cast<int>(std::min<int64_t>(kBlockM, (p.rows + 7) / 8 * 8));
  const int b_rows = t.pair ? t.tile_n / 2 : t.tile_n;
  const CUtensorMapDataType dt = p.dtype == IXK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto map = [&](CUtensorMap* out, const void* base, int64_t inner, int64_t outer, int64_t ld, int box_inner, int box_outer) {
    TmapSpec s{};
    s.dtype = dt;
    s.rank = 3;
    s.swizzle128 = true;
    s.dims[0] = inner;
    s.dims[1] = outer;
    s.dims[2] = 1;
    s.strides_bytes[0] = static_cast<uint64_t>(ld) * 2;
    s.strides_bytes[1] = s.strides_bytes[0] * outer;
    s.box[0] = box_inner;
    s.box[1] = box_outer;
    s.box[2] = 1;
    return encode_tmap(out, base, s);
  };
  CUtensorMap tx, tw, tg;
  int rc = map(&tx, p.x, p.hidden, p.rows, p.ldx, kSlabElems, a_rows);
  if (rc != IXK_OK) return rc;
  rc = p.w_column_major ? map(&tw, p.w, p.vocab, p.hidden, p.ldw, kSlabElems, kSlabElems)
                        : map(&tw, p.w, p.hidden, p.vocab, p.ldw, kSlabElems, b_rows);
  if (rc != IXK_OK) return rc;
  tg = tx;
  if (kGrad && (rc = map(&tg, p.grad, p.count, (p.rows + 255) / 256 * 256, p.ldg, 64, 32)) != IXK_OK) return rc;

  Args a{};
  a.rows = static_cast<int>(p.rows);
  a.slabs = static_cast<int>((p.hidden + kSlabElems - 1) / kSlabElems);
  const int chunks = (a.slabs + kChunkSlabs - 1) / kChunkSlabs;
  a.chunk_slabs = (a.slabs + chunks - 1) / chunks;
  a.first = static_cast<int>(p.first);
  a.count = static_cast<int>(p.count);
  a.tiles_n = t.tiles_n;
  a.tile_n = t.tile_n;
  a.strip = t.strip;
  a.strips = t.strips;
  a.w_mn_major = p.w_column_major ? 1 : 0;
  a.a_bytes = a_rows * kSlabBytes;
  a.b_boxes = (b_rows + kSlabElems - 1) / kSlabElems;
  // (stages start on the swizzle's 1024 bytes; an MN-major w takes whole boxes of 64 columns)
  a.stage_bytes = (a.a_bytes + (p.w_column_major ? a.b_boxes * kSlabElems : b_rows) * kSlabBytes + 1023) / 1024 * 1024;
  // (the MMA reads 128 rows of x whatever their number: the last stage ends that far before the ring does)
  a.stages = std::min(kMaxStages, (kRingBytes - (kBlockM * kSlabBytes - a.a_bytes)) / a.stage_bytes);
  const uint32_t fmt = p.dtype == IXK_BF16 ? 1u : 0u;
  a.idesc = ptx::umma_idesc(fmt, fmt, 0, a.w_mn_major, t.pair ? 2 * kBlockM : kBlockM, t.tile_n);
  a.active_rows = p.active_rows;
  a.info = p.info;
  a.bias = p.bias;
  a.bf16 = p.dtype == IXK_BF16 ? 1 : 0;
  a.bias_vec_ok = p.bias != nullptr && (reinterpret_cast<uintptr_t>(p.bias) & 15u) == 0;
  a.scale = p.scale;
  a.scale2 = p.scale * kLog2E;
  a.targets = p.targets;
  a.partial = p.partial;
  a.at_target = p.at_target;
  a.range = p.range;
  a.status_word = dev.status_word;

  const int64_t tile_rows = t.pair ? 2 * kBlockM : kBlockM;
  const int64_t units = (p.rows + tile_rows - 1) / tile_rows * t.strips;
  auto go = [&](auto pair_tag, auto mode_tag) -> int {
    constexpr bool kPair = decltype(pair_tag)::value;
    constexpr Mode kMode = decltype(mode_tag)::value;
    auto* fn = &head_kernel<kPair, kMode>;
    static thread_local int configured_device = -1;
    if (configured_device != dev.device) {
      IXK_CUDA_OK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
      configured_device = dev.device;
    }
    const int workers = static_cast<int>(std::min<int64_t>(units, kPair ? dev.sm_count / 2 : dev.sm_count));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((kPair ? 2 : 1) * workers);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kPair ? 2 : 1;
    IXK_CUDA_OK(cudaLaunchKernelEx(&cfg, fn, tx, tw, tg, a));
    count_launch();
    return IXK_OK;
  };
  using std::integral_constant;
  constexpr integral_constant<Mode, kGrad ? Mode::kGrad : Mode::kStats> kOne;
  constexpr integral_constant<Mode, kGrad ? Mode::kGradChunks : Mode::kStatsChunks> kMany;
  // (a gradient with labels apart has its small differences from elsewhere)
  if (a.slabs > a.chunk_slabs && !(kGrad && a.targets.apart)) return t.pair ? go(std::true_type{}, kMany) : go(std::false_type{}, kMany);
  return t.pair ? go(std::true_type{}, kOne) : go(std::false_type{}, kOne);
}

}  // namespace

int stat_slots(int64_t rows, int64_t vocab) { return 2 * tiling_for(rows, vocab, kStatUnit).strips; }
int launch_stats(const Pass& p, const DeviceInfo& dev, cudaStream_t stream) { return launch<false>(p, dev, stream); }
int launch_grad(const Pass& p, const DeviceInfo& dev, cudaStream_t stream) { return launch<true>(p, dev, stream); }

}  // namespace head
}  // namespace ixk
