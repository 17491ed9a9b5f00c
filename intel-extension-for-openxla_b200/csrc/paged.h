// Checks and addresses shared by the calls on a paged key/value cache.
#pragma once

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
