// The bookkeeping of a paged key/value cache on the GPU: pages for new tokens and the maps of a packed batch
// (ixk_paged_extend), and what follows a verification (ixk_paged_keep): the accepted drafts' keys and values close up,
// lengths grow, unused pages go back.
//
// Both rest on prefix sums over the requests.  With L_b tokens in the cache, n_b new ones and pages of S tokens:
//   have = ceil(L/S), want = ceil((L+n)/S), need = want - have; start_b = sum of n, first_b = sum of need, over the requests
// before b; the i-th page taken is free_pages[count - 1 - i], place have + i - first_b of its request's table row.  Which
// request a row or a page belongs to is then a binary search in the sums, which lie in shared memory.
#include <algorithm>

#include "paged.h"
#include "ptx.cuh"

namespace ixk {
namespace paged {

namespace {

constexpr int kThreads = 1024;        // of a block that does the sums; 256 where requests and rows are few
constexpr int kFewThreads = 256;
constexpr int kMaxRequests = 16384;   // 9 bytes a request in shared memory
constexpr int kMaxPath = 1024;

// Exclusive prefix sum over the block of one number a thread; `total`: of all.
__device__ __forceinline__ long long block_scan(long long v, long long* scratch, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  __syncthreads();          // (the scratch may still be read from the scan before)
  if (lane == 31) scratch[warp] = sum;
  __syncthreads();
  long long w = lane < static_cast<int>(blockDim.x >> 5) ? scratch[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += up;
  }
  const long long before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  *total = __shfl_sync(0xffffffffu, w, 31);
  return sum - v + (warp > 0 ? before : 0);
}

// The request whose range [sums[b], sums[b + 1]) holds `at`; sums ascend, sums[0] <= at < sums[n].
__device__ __forceinline__ int owner(const int* sums, int n, int at) {
  int lo = 0, hi = n;       // sums[lo] <= at < sums[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= at) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int pages_for(int tokens, int page_size) {
  return static_cast<int>((static_cast<unsigned>(tokens) + static_cast<unsigned>(page_size) - 1u) / static_cast<unsigned>(page_size));
}

struct ExtendArgs {
  int requests, page_size, pages, columns, rows;
  int in_place;                        // the count: the CTAs are a cluster
  int64_t table_stride;
  const int *lengths, *new_tokens, *free_pages, *free_count;
  int *page_table, *free_count_out, *granted, *row_start, *request, *position, *slot;
};

// Latency-bound: 20 bytes a request and 12 a row.  Every CTA makes the sums over all requests for itself (a few microseconds of loads
// less than a second launch would cost) and writes its share of rows and pages: a row a thread.  Where the count is updated in
// place, its CTAs are one cluster, and the update waits for all of them to have read it.
__global__ void __launch_bounds__(kThreads) extend_kernel(const __grid_constant__ ExtendArgs a) {
  extern __shared__ __align__(16) int smem[];
  __shared__ long long scratch[32];
  __shared__ int taken_max[32];
  int* start = smem;                                    // [B + 1]
  int* first = smem + a.requests + 1;                   // [B + 1]
  uint8_t* fits = reinterpret_cast<uint8_t*>(first + a.requests + 1);
  ptx::grid_dependency_sync();
  const int B = a.requests, threads = blockDim.x;
  const int per = (B + threads - 1) / threads;
  const int b0 = min(static_cast<int>(threadIdx.x) * per, B), b1 = min(b0 + per, B);
  const int available = min(max(*a.free_count, 0), a.pages);

  long long rows = 0, total;
  for (int b = b0; b < b1; ++b) {
    const int n = max(a.new_tokens[b], 0);
    start[b] = n;
    first[b] = a.lengths[b];
    rows += n;
  }
  long long row = block_scan(rows, scratch, &total);
  const int total_rows = static_cast<int>(min(total, static_cast<long long>(a.rows)));
  long long need = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = start[b], L = first[b];
    start[b] = static_cast<int>(min(row, static_cast<long long>(a.rows)));
    row += n;
    const bool ok = L >= 0 && static_cast<long long>(L) + n <= static_cast<long long>(a.columns) * a.page_size && row <= a.rows;
    fits[b] = ok;
    const int mine = ok ? pages_for(L + n, a.page_size) - pages_for(L, a.page_size) : 0;
    first[b] = mine;
    need += mine;
  }
  long long page = block_scan(need, scratch, &total);
  int served_pages = 0;
  for (int b = b0; b < b1; ++b) {
    const int mine = first[b];
    first[b] = static_cast<int>(min(page, 0x7fffffffLL));
    page += mine;
    if (fits[b] && mine > 0) {
      if (page <= available) served_pages = static_cast<int>(page);    // (ascending: the last one served counts)
      else fits[b] = 0;
    }
  }
  if (threadIdx.x == 0) {
    start[B] = total_rows;
    first[B] = static_cast<int>(min(total, 0x7fffffffLL));
  }
  // pages taken = the largest sum that was served
  int taken = __reduce_max_sync(0xffffffffu, served_pages);
  if ((threadIdx.x & 31) == 0) taken_max[threadIdx.x >> 5] = taken;
  __syncthreads();
  taken = __reduce_max_sync(0xffffffffu, static_cast<int>(threadIdx.x & 31) < (threads >> 5) ? taken_max[threadIdx.x & 31] : 0);

  // (Without a sign: rows and pages may be 2^31 less a little, and a thread's last index lies a stride behind them.)
  const unsigned stride = gridDim.x * threads, me = blockIdx.x * threads + threadIdx.x;
  for (int b = static_cast<int>(me); b <= B; b += static_cast<int>(stride)) {
    a.row_start[b] = start[b];
    if (b < B) a.granted[b] = fits[b] ? max(a.new_tokens[b], 0) : 0;
  }
  for (unsigned at = me; at < static_cast<unsigned>(taken); at += stride) {
    const int i = static_cast<int>(at);
    const int b = owner(first, B, i);
    a.page_table[b * a.table_stride + pages_for(a.lengths[b], a.page_size) + i - first[b]] = a.free_pages[available - 1 - i];
  }
  for (unsigned at = me; at < static_cast<unsigned>(a.rows); at += stride) {
    const int r = static_cast<int>(at);
    int request = -1, position = -1, slot = -1;
    if (r < total_rows) {
      const int b = owner(start, B, r);
      if (fits[b]) {
        const int L = a.lengths[b], have = pages_for(L, a.page_size);
        request = b;
        position = L + (r - start[b]);
        const int place = static_cast<int>(static_cast<unsigned>(position) / static_cast<unsigned>(a.page_size));
        const int p = place < have ? a.page_table[b * a.table_stride + place] : a.free_pages[available - 1 - (first[b] + place - have)];
        if (static_cast<unsigned>(p) < static_cast<unsigned>(a.pages)) slot = p * a.page_size + position - place * a.page_size;
      }
    }
    a.request[r] = request;
    a.position[r] = position;
    a.slot[r] = slot;
  }
  if (a.in_place && gridDim.x > 1) ptx::cluster_sync_all();
  else __syncthreads();
  if (me == 0) *a.free_count_out = available - taken;
}

struct KeepArgs {
  int requests, page_size, pages, columns;
  int64_t table_stride, path_stride;
  int path_columns;
  const int *lengths, *granted, *kept, *path, *page_table, *free_count;
  int *free_pages, *free_count_out, *lengths_out;
  CacheArgs cache;
  int vecs_per_head, heads, vecs;      // 16-byte vectors of a token: of a head; of K and V of all layers
  int chunks;                          // CTAs a request
};

// What a request keeps: the valid part of its path.
__device__ __forceinline__ void keep_range(const KeepArgs& a, int b, int* L, int* n, int* kept) {
  *L = max(a.lengths[b], 0);
  *n = max(a.granted[b], 0);
  *kept = min(a.kept[b], *n);
}
// Entries of the path that count, of the first `kept`: as long as they ascend and stay below n.
__device__ __forceinline__ bool path_entry_ok(const int* path, int j, int n) {
  return path[j] < n && path[j] > (j > 0 ? path[j - 1] : -1);
}

// The books: new lengths, and the pages above them back onto the free list.
__device__ void keep_books(const KeepArgs& a, int* smem) {
  __shared__ long long scratch[32];
  int* first = smem;                   // [B + 1]
  int* low = smem + a.requests + 1;    // [B]
  const int B = a.requests;
  const int threads = blockDim.x, per = (B + threads - 1) / threads;
  const int b0 = min(static_cast<int>(threadIdx.x) * per, B), b1 = min(b0 + per, B);
  const int count = min(max(*a.free_count, 0), a.pages);
  long long mine = 0, total;
  if (a.path != nullptr) {             // how much of a request's path counts: all entries of all requests, eight of a thread's at a time
    for (int b = threadIdx.x; b < B; b += threads) {
      int L, n, kept;
      keep_range(a, b, &L, &n, &kept);
      low[b] = min(kept, a.path_columns);
      first[b] = n;
    }
    __syncthreads();
    const int entries = B * a.path_columns;
    for (int e0 = threadIdx.x; e0 < entries; e0 += 8 * threads) {
      int now[8], before[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i * threads;
        now[i] = 0;
        before[i] = -1;
        if (e < entries) {
          const int b = e / a.path_columns, j = e - b * a.path_columns;
          const int* path = a.path + b * a.path_stride + j;
          now[i] = path[0];
          if (j > 0) before[i] = path[-1];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i * threads;
        if (e >= entries) break;
        const int b = e / a.path_columns, j = e - b * a.path_columns;
        if (now[i] >= first[b] || now[i] <= before[i]) atomicMin(&low[b], j);      // (the smallest, whoever comes first)
      }
    }
    __syncthreads();
  }
  for (int b = b0; b < b1; ++b) {
    int L, n, kept;
    keep_range(a, b, &L, &n, &kept);
    if (a.path != nullptr) kept = low[b];
    const long long most = static_cast<long long>(a.columns) * a.page_size;
    const int high_tokens = static_cast<int>(min(static_cast<long long>(L) + n, most));
    const int after = kept < 0 ? 0 : static_cast<int>(min(static_cast<long long>(L) + kept, most));
    low[b] = pages_for(after, a.page_size);
    first[b] = pages_for(high_tokens, a.page_size) - low[b];
    mine += first[b];
    a.lengths_out[b] = after;          // (nobody else reads this request's length)
  }
  long long sum = block_scan(mine, scratch, &total);
  for (int b = b0; b < b1; ++b) {
    const int c = first[b];
    first[b] = static_cast<int>(min(sum, 0x7fffffffLL));
    sum += c;
  }
  const int back = static_cast<int>(min(total, static_cast<long long>(a.pages - count)));
  if (threadIdx.x == 0) first[B] = static_cast<int>(min(total, 0x7fffffffLL));
  __syncthreads();
  for (unsigned at = threadIdx.x; at < static_cast<unsigned>(back); at += threads) {      // (as in extend_kernel)
    const int i = static_cast<int>(at), b = owner(first, B, i);
    a.free_pages[count + i] = a.page_table[b * a.table_stride + low[b] + i - first[b]];
  }
  if (threadIdx.x == 0) *a.free_count_out = count + back;
}

// The moves: a thread takes one 16-byte vector of a token (a layer, K or V, a head, a place in it) and walks the path in
// order, four entries at a time: four loads, then four stores.  An entry's source is never below its target, so a
// source read in its turn, or earlier, has not been written by a target before it.
constexpr int kMoveThreads = 256;
constexpr int kMoveCtas = 6;           // on an SM
constexpr int kBatch = 4;

// A position's page and its place there; page -1: none.
__device__ __forceinline__ int2 place_of(const KeepArgs& a, const int* table, long long position) {
  if (position >= static_cast<long long>(a.columns) * a.page_size) return make_int2(-1, 0);
  const int column = static_cast<int>(static_cast<unsigned>(position) / static_cast<unsigned>(a.page_size));
  const int page = table[column];
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.cache.pages)) return make_int2(-1, 0);
  return make_int2(page, static_cast<int>(position) - column * a.page_size);
}

__device__ void keep_moves(const KeepArgs& a, int* smem, int block) {
  __shared__ int valid;
  const int b = block / a.chunks, chunk = block - b * a.chunks;
  int L, n, kept;
  keep_range(a, b, &L, &n, &kept);
  kept = min(kept, a.path_columns);
  if (kept <= 0) return;
  const int* path = a.path + b * a.path_stride;
  const int* table = a.page_table + b * a.table_stride;
  int4* moves = reinterpret_cast<int4*>(smem);       // [path_columns]: from (page, place) to (page, place); page -1: nothing moves
  if (threadIdx.x == 0) valid = kept;
  __syncthreads();
  for (int j = threadIdx.x; j < kept; j += blockDim.x) {
    if (!path_entry_ok(path, j, n)) atomicMin(&valid, j);
    int2 from = make_int2(-1, 0), to = make_int2(-1, 0);
    if (path[j] > j) {
      from = place_of(a, table, static_cast<long long>(L) + path[j]);
      to = place_of(a, table, static_cast<long long>(L) + j);
    }
    moves[j] = make_int4(to.x < 0 ? -1 : from.x, from.y, to.x, to.y);
  }
  __syncthreads();
  kept = valid;
  for (int vec = chunk * blockDim.x + threadIdx.x; vec < a.vecs; vec += a.chunks * blockDim.x) {
    int rest = vec;
    const int in_head = rest % a.vecs_per_head;
    rest /= a.vecs_per_head;
    const int head = rest % a.heads;
    rest /= a.heads;
    const bool is_v = rest & 1;
    const int layer = rest >> 1;
    const CacheArgs& c = a.cache;
    uint4* base = is_v ? c.v + layer * c.v_layer + head * c.v_head + in_head : c.k + layer * c.k_layer + head * c.k_head + in_head;
    const int64_t page_stride = is_v ? c.v_page : c.k_page, token_stride = is_v ? c.v_token : c.k_token;
    for (int j0 = 0; j0 < kept; j0 += kBatch) {
      uint4 held[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (j0 + i >= kept) break;
        const int4 m = moves[j0 + i];
        if (m.x >= 0) held[i] = base[m.x * page_stride + m.y * token_stride];
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (j0 + i >= kept) break;
        const int4 m = moves[j0 + i];
        if (m.x >= 0) base[m.z * page_stride + m.w * token_stride] = held[i];
      }
    }
  }
}

__global__ void __launch_bounds__(kThreads) keep_books_kernel(const __grid_constant__ KeepArgs a) {
  extern __shared__ __align__(16) int smem[];
  ptx::grid_dependency_sync();
  keep_books(a, smem);
}
// The moves, and with_books beside them, in CTA 0, the books.  (Where the new lengths go over the old ones, which the moves read,
// the books wait for a launch of their own.)
__global__ void __launch_bounds__(kMoveThreads, kMoveCtas) keep_moves_kernel(const __grid_constant__ KeepArgs a, int with_books) {
  extern __shared__ __align__(16) int smem[];
  ptx::grid_dependency_sync();
  if (with_books && blockIdx.x == 0) keep_books(a, smem);
  else keep_moves(a, smem, static_cast<int>(blockIdx.x) - with_books);
}

int check_pool(const ixk_page_pool* p, const char* who) {
  const std::string at(who);
  if (p == nullptr) return fail(IXK_INVALID_ARGUMENT, at + ": pool is NULL");
  if (p->page_size < 1 || p->pages < 1 || p->columns < 1 || p->requests < 0)
    return fail(IXK_INVALID_ARGUMENT, at + ": page_size, pages and columns must be positive, requests not negative");
  if (p->requests > 1 && p->table_stride < p->columns) return fail(IXK_INVALID_ARGUMENT, at + ": rows of the page table overlap");
  if (static_cast<int64_t>(p->page_size) * p->pages > 0x7fffffff || static_cast<int64_t>(p->page_size) * p->columns > 0x7fffffff)
    return fail(IXK_UNIMPLEMENTED, at + ": 2^31 tokens or more in the cache or in a table row");
  if (p->requests > kMaxRequests) return fail(IXK_UNIMPLEMENTED, at + ": more than 16384 requests");
  return IXK_OK;
}

}  // namespace
}  // namespace paged
}  // namespace ixk

using namespace ixk;

extern "C" {

int ixk_paged_extend(const ixk_page_pool* pool, const int32_t* lengths, const int32_t* new_tokens, int32_t* page_table,
                     const int32_t* free_pages, const int32_t* free_count, int32_t* free_count_out, int32_t* granted,
                     int32_t* row_start, int64_t rows, int32_t* request, int32_t* position, int32_t* slot, void* cuda_stream) {
  IXK_API_RANGE("ixk_paged_extend");
  clear_error();
  if (int st = paged::check_pool(pool, "paged_extend")) return st;
  if (rows < 0) return fail(IXK_INVALID_ARGUMENT, "paged_extend: rows is negative");
  if (rows > 0x7fffffff - 65536) return fail(IXK_UNIMPLEMENTED, "paged_extend: 2^31 rows or more");
  if (free_pages == nullptr || free_count == nullptr || free_count_out == nullptr || row_start == nullptr ||
      (pool->requests > 0 && (lengths == nullptr || new_tokens == nullptr || page_table == nullptr || granted == nullptr)) ||
      (rows > 0 && (request == nullptr || position == nullptr || slot == nullptr)))
    return fail(IXK_INVALID_ARGUMENT, "paged_extend: null argument");
  const int64_t requests = pool->requests;
  if (paged::ints_overlap({{lengths, requests, false, nullptr}, {new_tokens, requests, false, nullptr}, {free_pages, pool->pages, false, nullptr},
                           {free_count, 1, false, nullptr}, {page_table, paged::rows_extent(requests, pool->table_stride, pool->columns), true, nullptr},
                           {free_count_out, 1, true, free_count}, {granted, requests, true, nullptr}, {row_start, requests + 1, true, nullptr},
                           {request, rows, true, nullptr}, {position, rows, true, nullptr}, {slot, rows, true, nullptr}}))
    return fail(IXK_INVALID_ARGUMENT, "paged_extend: an output shares memory with an input or another output");
  DeviceInfo info;
  if (int st = get_device_info(&info)) return st;
  const bool in_place = free_count_out == free_count;
  paged::ExtendArgs a{pool->requests, pool->page_size, pool->pages, pool->columns, static_cast<int>(rows), in_place, pool->table_stride,
                      lengths, new_tokens, free_pages, free_count, page_table, free_count_out, granted, row_start, request, position, slot};
  const size_t smem = (static_cast<size_t>(pool->requests) + 1) * 8 + pool->requests;
  if (smem > 48 * 1024)
    IXK_CUDA_OK(cudaFuncSetAttribute(paged::extend_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  const bool few = pool->requests <= paged::kFewThreads && rows <= 2 * paged::kFewThreads;
  const int threads = few ? paged::kFewThreads : paged::kThreads;
  // a row a thread; in place up to a cluster of eight
  const int64_t want = std::max<int64_t>(1, (std::max<int64_t>(rows, pool->requests) + threads - 1) / threads);
  unsigned ctas = static_cast<unsigned>(std::min<int64_t>(want, info.sm_count));
  if (in_place) {
    ctas = 1;
    while (ctas < 8 && ctas < want) ctas *= 2;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(cuda_stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = in_place && ctas > 1 ? 2 : 1;
  IXK_CUDA_OK(cudaLaunchKernelEx(&cfg, paged::extend_kernel, a));
  count_launch();
  return IXK_OK;
}

int ixk_paged_keep(const ixk_page_pool* pool, const int32_t* lengths, const int32_t* granted, const int32_t* kept,
                   const int32_t* path, int64_t path_columns, int64_t path_stride, const int32_t* page_table,
                   int32_t* free_pages, const int32_t* free_count, int32_t* free_count_out, int32_t* lengths_out,
                   const ixk_paged_cache* cache, void* k, void* v, void* cuda_stream) {
  IXK_API_RANGE("ixk_paged_keep");
  clear_error();
  if (int st = paged::check_pool(pool, "paged_keep")) return st;
  if (free_pages == nullptr || free_count == nullptr || free_count_out == nullptr ||
      (pool->requests > 0 && (lengths == nullptr || granted == nullptr || kept == nullptr || page_table == nullptr || lengths_out == nullptr)))
    return fail(IXK_INVALID_ARGUMENT, "paged_keep: null argument");
  if ((path == nullptr) != (cache == nullptr)) return fail(IXK_INVALID_ARGUMENT, "paged_keep: a path needs the cache whose tokens move, and only then");
  if (path != nullptr) {
    if (path_columns < 1 || (pool->requests > 1 && path_stride < path_columns))
      return fail(IXK_INVALID_ARGUMENT, "paged_keep: path must have columns, and rows that do not overlap");
    if (path_columns > paged::kMaxPath) return fail(IXK_UNIMPLEMENTED, "paged_keep: paths of more than 1024 entries");
    if (int st = paged::check_cache(cache, k, v, "paged_keep")) return st;
    if (cache->page_size != pool->page_size || cache->pages != pool->pages)
      return fail(IXK_INVALID_ARGUMENT, "paged_keep: pool and cache differ in pages or page_size");
    const paged::Operand kp = paged::key_pages(cache, k), vp = paged::value_pages(cache, v);
    const int64_t requests = pool->requests, table = paged::rows_extent(requests, pool->table_stride, pool->columns) * 4,
                  paths = paged::rows_extent(requests, path_stride, path_columns) * 4;
    const paged::Operand books[] = {{lengths, requests * 4}, {granted, requests * 4}, {kept, requests * 4}, {path, paths}, {page_table, table},
                                    {free_pages, pool->pages * static_cast<int64_t>(4)}, {free_count, 4}, {free_count_out, 4}, {lengths_out, requests * 4}};
    if (const char* name = paged::shared_memory({{"k", &kp, nullptr, nullptr}, {"v", &vp, nullptr, nullptr}},
                                                {&books[0], &books[1], &books[2], &books[3], &books[4], &books[5], &books[6], &books[7], &books[8]}))
      return fail(IXK_INVALID_ARGUMENT, std::string("paged_keep: ") + name + " of the cache shares memory with another operand or with itself");
  }
  const int64_t requests = pool->requests;
  if (paged::ints_overlap({{lengths, requests, false, nullptr}, {granted, requests, false, nullptr}, {kept, requests, false, nullptr},
                           {path, paged::rows_extent(path == nullptr ? 0 : requests, path_stride, path_columns), false, nullptr},
                           {page_table, paged::rows_extent(requests, pool->table_stride, pool->columns), false, nullptr}, {free_pages, pool->pages, true, nullptr},
                           {free_count, 1, false, nullptr}, {free_count_out, 1, true, free_count}, {lengths_out, requests, true, lengths}}))
    return fail(IXK_INVALID_ARGUMENT, "paged_keep: what it writes shares memory with something else (lengths_out may be lengths, free_count_out free_count)");
  DeviceInfo info;
  if (int st = get_device_info(&info)) return st;
  paged::KeepArgs a{};
  a.requests = pool->requests;
  a.page_size = pool->page_size;
  a.pages = pool->pages;
  a.columns = pool->columns;
  a.table_stride = pool->table_stride;
  a.path_stride = path_stride;
  a.path_columns = static_cast<int>(path_columns);
  a.lengths = lengths;
  a.granted = granted;
  a.kept = kept;
  a.path = path;
  a.page_table = page_table;
  a.free_count = free_count;
  a.free_pages = free_pages;
  a.free_count_out = free_count_out;
  a.lengths_out = lengths_out;
  auto s = static_cast<cudaStream_t>(cuda_stream);
  if (path != nullptr && pool->requests > 0) {
    a.cache = paged::cache_args(cache, k, v);
    a.vecs_per_head = cache->head_size / 8;
    a.heads = cache->heads;
    const int64_t vecs = static_cast<int64_t>(a.vecs_per_head) * a.heads * 2 * cache->layers;
    if (vecs > 0x3fffffff) return fail(IXK_UNIMPLEMENTED, "paged_keep: too many layers and heads");
    a.vecs = static_cast<int>(vecs);
    // CTAs a request: as many as are on the GPU at one time, if there is work for them
    const int64_t resident = static_cast<int64_t>(info.sm_count) * paged::kMoveCtas;
    a.chunks = static_cast<int>(std::max<int64_t>(1, std::min((vecs + paged::kMoveThreads - 1) / paged::kMoveThreads, resident / a.requests)));
    const size_t for_path = static_cast<size_t>(path_columns) * 16, for_books = (static_cast<size_t>(pool->requests) * 2 + 1) * 4;
    const int with_books = lengths_out != lengths && pool->requests <= 1024 ? 1 : 0;
    if (int st = launch_overlapped(paged::keep_moves_kernel, dim3(static_cast<unsigned>(a.requests) * a.chunks + with_books), dim3(paged::kMoveThreads),
                                   with_books ? std::max(for_path, for_books) : for_path, s, a, with_books))
      return st;
    if (with_books) return IXK_OK;
  }
  const size_t smem = (static_cast<size_t>(pool->requests) * 2 + 1) * 4;
  if (smem > 48 * 1024)
    IXK_CUDA_OK(cudaFuncSetAttribute(paged::keep_books_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  return launch_overlapped(paged::keep_books_kernel, dim3(1), dim3(pool->requests <= paged::kFewThreads ? paged::kFewThreads : paged::kThreads), smem, s, a);
}

}  // extern "C"
