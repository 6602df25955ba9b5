// window.cpp - C entry points of attention with a window and first tokens that
// stay, and of caches with a scale a block (include/relx.h).
#include <climits>
#include <cmath>

#include "attention.h"
#include "operators.h"

namespace relx {
namespace {

constexpr int64_t kMost = int64_t{1} << 30; // of a window and of first tokens: everything

// Scales of blocks that fit the cache. `kv_heads` and `pages` are checked.
void check_scales(const relx_block_scales &s, const relx_cache &c) {
  layout(c.kind == 2 && c.bits == 8, "blocks: scales go with an int8 cache");
  layout(s.block >= 16 && s.block % 16 == 0 && c.page % s.block == 0,
         "blocks: a block is a multiple of 16 tokens and divides the page");
  need(s.page >= 0 && s.block_stride >= 0 && s.head >= 0, "blocks: negative strides");
  need(c.pages == 0 || c.kv_heads == 0 || (s.key_scale && s.value_scale), "blocks: null scales");
  need(s.page <= INT32_MAX && s.block_stride <= INT32_MAX && s.head <= INT32_MAX, "blocks: strides");
}

// Whether pieces of `dim` elements, [n1, n2, n3] with these strides, lie apart in
// every two of the dimensions.
bool apart3(int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t n3, int64_t s3, int64_t dim) {
  return !overlap(n1, s1, n2, s2, dim) && !overlap(n1, s1, n3, s3, dim) && !overlap(n2, s2, n3, s3, dim);
}

BlockArgs block_args(const relx_block_append_args &p, int &type) {
  type = element_type(p.kind, p.bits);
  layout(type != kI8, "append: f32, f16 or bf16 keys and values");
  const relx_cache &c = p.cache;
  layout(c.kind == 2 && c.bits == 8, "append: blocks are of an int8 cache");
  relx_cache checked = c; // scales a head are not read
  checked.key_scale = p.scales.key_scale;
  checked.value_scale = p.scales.value_scale;
  const CacheBytes b = cache_bytes(checked);
  check_scales(p.scales, c);
  need(fits32(p.rows) && fits32(p.requests) && fits32(p.columns), "append: a size is negative or beyond 2^31 - 1");
  layout(c.kv_heads <= 65535, "append: more than 65535 heads");
  layout(c.dim >= 1 && c.dim <= 512, "append: head sizes up to 512");
  layout(p.columns == 0 || p.columns <= kMost / c.page, "append: a table of more than 2^30 tokens");
  // a workgroup of 256 threads for each number of a block, and 2^32 threads a dimension
  layout(p.rows / p.scales.block + 2 * p.requests + 1 < (int64_t{1} << 24), "append: more than 2^24 - 1 blocks");
  const bool used = p.rows > 0 && p.requests > 0 && c.kv_heads > 0;
  need(!used || (p.cached && p.starts), "append: null lengths");
  need(!used || p.columns == 0 || p.table, "append: null table");
  need(!used || c.pages == 0 ||
           (apart3(c.pages, c.key_page, c.page, c.key_slot, c.kv_heads, c.key_head, c.dim) &&
            apart3(c.pages, c.value_page, c.page, c.value_slot, c.kv_heads, c.value_head, c.dim)),
       "append: the cache's elements overlap");
  need(!used || c.pages == 0 ||
           apart3(c.pages, p.scales.page, c.page / p.scales.block, p.scales.block_stride, c.kv_heads, p.scales.head, 1),
       "append: the scales overlap");
  BlockArgs a{};
  a.x[0] = heads_of(&p.k, used, "append: null keys");
  a.x[1] = heads_of(&p.v, used, "append: null values");
  a.cache[0] = static_cast<char *>(c.keys);
  a.cache[1] = static_cast<char *>(c.values);
  a.page_stride[0] = b.key_page;
  a.page_stride[1] = b.value_page;
  a.slot_stride[0] = b.key_slot;
  a.slot_stride[1] = b.value_slot;
  a.head_stride[0] = b.key_head;
  a.head_stride[1] = b.value_head;
  a.scale[0] = p.scales.key_scale;
  a.scale[1] = p.scales.value_scale;
  a.scale_page = p.scales.page;
  a.scale_block = p.scales.block_stride;
  a.scale_head = p.scales.head;
  a.table = p.table;
  a.table_row = p.table_row;
  a.cached = p.cached;
  a.starts = p.starts;
  a.page = make_div(c.page);
  a.block = make_div(p.scales.block);
  a.rows = static_cast<int32_t>(used ? p.rows : 0);
  a.requests = static_cast<int32_t>(p.requests);
  a.columns = static_cast<int32_t>(p.columns);
  a.pages = static_cast<int32_t>(c.pages);
  a.kv_heads = static_cast<int32_t>(c.kv_heads);
  a.dim = static_cast<int32_t>(c.dim);
  return a;
}

} // namespace
} // namespace relx

extern "C" {

int relx_block_append(relx_ctx *ctx, const relx_block_append_args *args, uint64_t stream, relx_err *err) {
  return guarded(err, [&] {
    relx::need(args != nullptr, "null arguments");
    int type;
    const relx::BlockArgs a = relx::block_args(*args, type);
    relx::on_context(ctx, [&] {
      if (a.rows > 0 && a.pages > 0 && a.columns > 0)
        relx::launched(relx::blocks_launch(a, type, relx::stream_of(stream)), "block append");
    });
  });
}

int relx_tree_attention_view(relx_ctx *ctx, const relx_tree_attention_args *args, const relx_cache_view *view,
                             uint64_t stream, relx_err *err) {
  return guarded(err, [&] {
    relx::need(args && view, "null arguments");
    relx::need(view->window >= 0 && view->sinks >= 0, "attention: a negative window or number of first tokens");
    relx::layout(view->window == 0 || !args->mask || view->window / 64 >= args->words,
                 "attention: a window holds the trees of a mask, 64 tokens a word");
    relx_tree_attention_args p = *args;
    const bool blocks = view->scales.block != 0;
    if (blocks) {
      p.cache.key_scale = view->scales.key_scale;
      p.cache.value_scale = view->scales.value_scale;
    }
    relx::AttendPlan plan;
    int type;
    bool i8;
    relx::AttendArgs a = relx::attend_args(p, plan, type, i8);
    a.window = static_cast<int32_t>(view->window == 0 ? relx::kMost : std::min(view->window, relx::kMost));
    a.sinks = static_cast<int32_t>(std::min(view->sinks, relx::kMost));
    a.block = a.page; // a scale a head: of every block
    a.scale_page = a.scale_block = 0;
    a.scale_head = sizeof(float);
    if (blocks) {
      const relx_block_scales &s = view->scales;
      relx::check_scales(s, p.cache);
      // a lane's distance from the head's first scale is held in 32 bits
      relx::layout(static_cast<__int128>(p.cache.pages) * s.page + (p.cache.page / s.block) * s.block_stride < (int64_t{1} << 30),
                   "blocks: scales further apart than 4 GiB");
      a.block = relx::make_div(s.block);
      a.scale_page = static_cast<uint32_t>(s.page * 4);
      a.scale_block = static_cast<uint32_t>(s.block_stride * 4);
      a.scale_head = s.head * 4;
    }
    relx::attend_room(a, plan, p);
    relx::on_context(ctx, [&] {
      if (a.rows == 0)
        return;
      const hipStream_t on = relx::stream_of(stream);
      relx::launched(type == relx::kF16 ? i8 ? relx::attend_launch_f16_blocks(a, plan, on)
                                             : relx::attend_launch_f16_window(a, plan, on)
                     : i8               ? relx::attend_launch_bf16_blocks(a, plan, on)
                                        : relx::attend_launch_bf16_window(a, plan, on),
                     "attention");
    });
  });
}

} // extern "C"
