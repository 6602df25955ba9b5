// operators.h - what the C entries of the paged-cache operators share: checks
// of arguments, the context's device, a cache's strides in bytes.
#pragma once

#include <climits>
#include <cmath>
#include <cstdlib>
#include <string>
#include <utility>

#include "attention.h"
#include "capi.h"
#include "runtime.h"

namespace relx {

inline void need(bool ok, const char *what) {
  if (!ok)
    throw Error("invalid_argument", what);
}

inline void layout(bool ok, const char *what) {
  if (!ok)
    throw Error("unsupported_layout", what);
}

inline int element_type(int64_t kind, int64_t bits) {
  if (kind == 0 && bits == 32)
    return kF32;
  if (kind == 0 && bits == 16)
    return kF16;
  if (kind == 1 && bits == 16)
    return kBF16;
  if (kind == 2 && bits == 8)
    return kI8;
  throw Error("unsupported_layout", "element type (kind " + std::to_string(kind) + ", " +
                                        std::to_string(bits) + " bits)");
}

inline bool fits32(int64_t v) { return v >= 0 && v <= INT32_MAX; }

inline void launched(hipError_t e, const char *what) {
  if (e != hipSuccess)
    throw Error("backend_failure", std::string(what) + ": " + hipGetErrorString(e));
}

// Runs `fn` with the context's device current, if the context takes calls.
// Not under its mutex, which transfers hold until the GPU has done them: these
// calls use nothing that it guards.
template <class F> inline void on_context(relx_ctx *ctx, F &&fn) {
  need(ctx != nullptr, "null context");
  if (ctx->ctx->closed || ctx->ctx->quarantined)
    throw Error("resources_closed", "context is closed or quarantined");
  DeviceScope scope(ctx->ctx->device);
  fn();
}

inline hipStream_t stream_of(uint64_t s) { return reinterpret_cast<hipStream_t>(s); }

// Whether elements of [n1, n2, dim] with these strides share a place.
inline bool overlap(int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t dim) {
  using Wide = __int128;
  s1 = n1 > 1 ? std::abs(s1) : 0;
  s2 = n2 > 1 ? std::abs(s2) : 0;
  if (s1 > s2) {
    std::swap(n1, n2);
    std::swap(s1, s2);
  }
  if ((n1 > 1 && s1 < dim) || (n2 > 1 && s2 < dim))
    return true;
  if (n1 <= 1 || n2 <= 1)
    return false;
  // the larger steps that end inside the smaller ones' reach: hardly ever any
  const Wide reach = static_cast<Wide>(n1 - 1) * s1;
  for (int64_t i = 1; i < n2 && static_cast<Wide>(i) * s2 < reach + dim; ++i) {
    const Wide at = static_cast<Wide>(i) * s2, below = at / s1; // the steps next to it
    if ((below < n1 && at - below * s1 < dim) || (below + 1 < n1 && (below + 1) * s1 - at < dim))
      return true;
  }
  return false;
}

// A result that several threads would write in one place is refused.
inline void writable(const relx_heads *h, int64_t rows, int64_t heads, int64_t dim) {
  need(!h || rows == 0 || heads == 0 || !overlap(rows, h->row, heads, h->head, dim), "a result's elements overlap");
}

inline Heads heads_of(const relx_heads *h, bool used, const char *what) {
  need(!used || (h && h->data), what);
  return used ? Heads{static_cast<char *>(h->data), h->row, h->head} : Heads{};
}

struct CacheBytes {
  int64_t key_page, key_slot, key_head, value_page, value_slot, value_head;
  int type;
};

inline CacheBytes cache_bytes(const relx_cache &c) {
  CacheBytes b;
  b.type = element_type(c.kind, c.bits);
  need(c.pages >= 0 && fits32(c.pages) && c.page >= 1 && fits32(c.page) && c.kv_heads >= 0, "cache: sizes");
  layout(c.page * c.pages <= INT32_MAX, "cache: more than 2^31 - 1 slots");
  need(c.pages == 0 || c.kv_heads == 0 || (c.keys && c.values), "cache: null keys or values");
  need(b.type != kI8 || c.kv_heads == 0 || (c.key_scale && c.value_scale), "cache: an int8 cache has a scale a head");
  need(c.key_page >= 0 && c.key_slot >= 0 && c.key_head >= 0 && c.value_page >= 0 && c.value_slot >= 0 &&
           c.value_head >= 0,
       "cache: negative strides");
  const int64_t w = b.type == kI8 ? 1 : b.type == kF32 ? 4 : 2;
  b.key_page = c.key_page * w;
  b.key_slot = c.key_slot * w;
  b.key_head = c.key_head * w;
  b.value_page = c.value_page * w;
  b.value_slot = c.value_slot * w;
  b.value_head = c.value_head * w;
  return b;
}

} // namespace relx
