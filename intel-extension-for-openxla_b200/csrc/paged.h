// Checks and addresses shared by the calls on a paged key/value cache.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "host_common.h"

namespace ixk {
namespace paged {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A call's int32 arrays: what it writes may share memory with nothing else of it, but an array that it updates in place (`with`).
struct Ints {
  const int32_t* p;
  int64_t count;
  bool written;
  const int32_t* with;
};
inline bool ints_overlap(std::initializer_list<Ints> all) {
  for (const Ints* a = all.begin(); a != all.end(); ++a) {
    if (!a->written || a->p == nullptr || a->count <= 0) continue;
    for (const Ints* b = all.begin(); b != all.end(); ++b) {
      if (b == a || b->p == nullptr || b->count <= 0 || (a->with == b->p && a->p == b->p)) continue;
      if (a->p < b->p + b->count && b->p < a->p + a->count) return true;
    }
  }
  return false;
}
inline int64_t rows_extent(int64_t rows, int64_t stride, int64_t columns) { return rows < 1 ? 0 : (rows - 1) * stride + columns; }

// The memory of an operand: runs of `run` bytes at `p` + sum of index_i * stride_i bytes, 0 <= index_i < extent_i.  None where there is no
// pointer or an extent is 0.  Strides are not negative.
struct Operand {
  uintptr_t p = 0;
  int64_t run = 0;
  int dims = 0;
  int64_t extent[4], stride[4];
  uint64_t reach = 0;                 // from the first byte to behind the last, 2^62 at most

  Operand(const void* at, int64_t bytes) : p(reinterpret_cast<uintptr_t>(at)), run(at == nullptr ? 0 : bytes), reach(run > 0 ? run : 0) {}
  Operand(const void* at, int64_t bytes, std::initializer_list<int64_t> extents, const int64_t* strides, int element) : Operand(at, bytes) {
    int i = 0;
    for (const int64_t n : extents) {
      if (n <= 0) run = 0;
      if (n > 1) {
        extent[dims] = n;
        stride[dims++] = strides[i] * element;
        constexpr uint64_t kMost = 1ull << 62;
        uint64_t more;
        if (__builtin_mul_overflow(static_cast<uint64_t>(n - 1), static_cast<uint64_t>(stride[dims - 1]), &more) || (reach += std::min(more, kMost)) > kMost) reach = kMost;
      }
      ++i;
    }
  }
  bool none() const { return run <= 0; }
  // In the same place, laid out the same way.
  bool is(const Operand& o) const {
    if (p != o.p || run != o.run || dims != o.dims) return false;
    for (int i = 0; i < dims; ++i)
      if (extent[i] != o.extent[i] || stride[i] != o.stride[i]) return false;
    return true;
  }
};
// Is there a sum of n_i * stride_i, lo_i <= n_i <= hi_i, above `low` and below `high`?  (And not of zeros alone, where these do not count.)
// From the largest stride down: of strides that enclose one another, as tensors have them, two or three n_i each can do.  Answers
// yes where it would have to try too many.
struct Steps {
  int count = 0, tries = 2000;
  int64_t stride[8];
  __int128 lo[8], hi[8];
  void add(int64_t s, int64_t from, int64_t to) {
    int i = 0;
    while (i < count && stride[i] > s) ++i;
    if (i < count && stride[i] == s) {
      lo[i] += from;
      hi[i] += to;
      return;
    }
    for (int k = count++; k > i; --k) stride[k] = stride[k - 1], lo[k] = lo[k - 1], hi[k] = hi[k - 1];
    stride[i] = s, lo[i] = from, hi[i] = to;
  }
  bool reaches(__int128 low, __int128 high, bool zeros_count, int i = 0) {
    if (--tries < 0) return true;
    if (i == count) return zeros_count && low < 0 && 0 < high;
    if (stride[i] == 0) {      // (all that are left: any n_i)
      return low < 0 && 0 < high && (zeros_count || hi[i] > lo[i]);
    }
    __int128 least = 0, most = 0;
    for (int k = i + 1; k < count; ++k) least += lo[k] * stride[k], most += hi[k] * stride[k];
    // n * stride + rest in (low, high) for some rest in [least, most]
    auto up = [&](__int128 v) { return v >= 0 ? v / stride[i] + 1 : -(-v / stride[i]) + (-v % stride[i] == 0 ? 1 : 0); };      // least n with n * stride > v
    const __int128 from = std::max(lo[i], up(low - most)), to = std::min(hi[i], -up(-(high - least)));
    for (__int128 n = from; n <= to; ++n) {
      const __int128 v = n * stride[i];
      if (reaches(low - v, high - v, zeros_count || n != 0, i + 1)) return true;
    }
    return false;
  }
};
// Do two operands share memory?
inline bool meet(const Operand& a, const Operand& b) {
  if (a.none() || b.none()) return false;
  if (b.p >= a.p ? b.p - a.p >= a.reach : a.p - b.p >= b.reach) return false;
  const __int128 apart = static_cast<__int128>(b.p) - static_cast<__int128>(a.p);
  Steps s;
  for (int i = 0; i < a.dims; ++i) s.add(a.stride[i], 0, a.extent[i] - 1);
  for (int i = 0; i < b.dims; ++i) s.add(b.stride[i], -(b.extent[i] - 1), 0);
  return s.reaches(apart - a.run, apart + b.run, true);
}
// Does an operand share memory with itself?
inline bool folds(const Operand& a) {
  if (a.none()) return false;
  uint64_t span = static_cast<uint64_t>(a.run);        // as most tensors lie: each dimension around those behind it
  int i = a.dims;
  while (i > 0 && static_cast<uint64_t>(a.stride[i - 1]) >= span && span < 1ull << 62) {
    --i;
    uint64_t more;
    span = __builtin_mul_overflow(static_cast<uint64_t>(a.extent[i] - 1), static_cast<uint64_t>(a.stride[i]), &more) ? ~0ull : span + std::min<uint64_t>(more, 1ull << 62);
  }
  if (i == 0) return false;
  Steps s;
  for (int i = 0; i < a.dims; ++i) s.add(a.stride[i], -(a.extent[i] - 1), a.extent[i] - 1);
  return s.count < a.dims || s.reaches(-a.run, a.run, false);      // (two of one stride: their indices can be exchanged)
}
// What a call writes may share memory with nothing else of it, but with the operand that it may be in the place of (`with`, `or_with`).
struct Written {
  const char* name;
  const Operand* what;
  const Operand* with;
  const Operand* or_with;
};
// The first of `written` that shares memory, nullptr if none does.
inline const char* shared_memory(std::initializer_list<Written> written, std::initializer_list<const Operand*> read) {
  for (const Written& w : written) {
    if (folds(*w.what)) return w.name;
    for (const Written& o : written)
      if (&o != &w && meet(*w.what, *o.what)) return w.name;
    for (const Operand* r : read)
      if (!((r == w.with || r == w.or_with) && w.what->is(*r)) && meet(*w.what, *r)) return w.name;
  }
  return nullptr;
}
inline Operand key_pages(const ixk_paged_cache* c, const void* k) {
  return Operand(k, c->head_size * 2, {c->layers, c->pages, c->page_size, c->heads}, c->k_strides, 2);
}
inline Operand value_pages(const ixk_paged_cache* c, const void* v) {
  return Operand(v, c->head_size * 2, {c->layers, c->pages, c->page_size, c->heads}, c->v_strides, 2);
}

// What the kernels need of a cache to find a token's row: strides in 16-byte vectors.
struct CacheArgs {
  uint4 *k, *v;
  int page_size, pages;
  int64_t k_layer, k_page, k_token, k_head;
  int64_t v_layer, v_page, v_token, v_head;
};

inline int check_cache(const ixk_paged_cache* c, const void* k, const void* v, const char* who) {
  const std::string at(who);
  if (c->dtype != IXK_BF16 && c->dtype != IXK_F16) return fail(IXK_UNIMPLEMENTED, at + ": the cache must be BF16 or F16");
  if (c->page_size < 1 || c->pages < 1 || c->heads < 1 || c->head_size < 1 || c->layers < 1)
    return fail(IXK_INVALID_ARGUMENT, at + ": cache sizes must be positive");
  if (static_cast<int64_t>(c->page_size) * c->pages > 0x7fffffff) return fail(IXK_UNIMPLEMENTED, at + ": a cache of 2^31 tokens or more");
  if (c->head_size % 8 != 0 || c->head_size > 256)
    return fail(IXK_UNIMPLEMENTED, at + ": head_size must be a multiple of 8, at most 256");
  const int64_t extent[4] = {c->layers, c->pages, c->page_size, c->heads};
  for (int i = 0; i < 4; ++i) {
    for (const int64_t s : {c->k_strides[i], c->v_strides[i]}) {
      if (s % 8 != 0) return fail(IXK_UNIMPLEMENTED, at + ": cache strides must be multiples of 8 elements (16 bytes)");
      if (extent[i] > 1 && s < c->head_size)
        return fail(IXK_INVALID_ARGUMENT, at + ": cache strides must be at least a head's size (rows would overlap)");
    }
  }
  if (k == nullptr || v == nullptr) return fail(IXK_INVALID_ARGUMENT, at + ": k and v of the cache must be non-NULL");
  if (!aligned16(k) || !aligned16(v)) return fail(IXK_INVALID_ARGUMENT, at + ": k and v of the cache must be 16-byte aligned");
  return IXK_OK;
}

inline CacheArgs cache_args(const ixk_paged_cache* c, void* k, void* v) {
  return CacheArgs{static_cast<uint4*>(k), static_cast<uint4*>(v), c->page_size, c->pages,
                   c->k_strides[0] / 8, c->k_strides[1] / 8, c->k_strides[2] / 8, c->k_strides[3] / 8,
                   c->v_strides[0] / 8, c->v_strides[1] / 8, c->v_strides[2] / 8, c->v_strides[3] / 8};
}

}  // namespace paged
}  // namespace ixk
