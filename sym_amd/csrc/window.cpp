// window.cpp - C entry points of attention with a window and first tokens that
// stay, and of caches with a scale a block (include/relx.h).
#include <climits>
#include <cmath>

#include "attention.h"
#include "operators.h"
#include "window.h"

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

// ------------------------------------------------------------ packed sequences

constexpr int kTileRows = 128, kMostSinks = 256;

// Rows that are read in pieces of 16 bytes, tiles of them from one address.
Heads rows_of(const relx_heads *h, bool used, int64_t rows, int64_t heads, const char *what) {
  const Heads x = heads_of(h, used, what);
  if (!used)
    return x;
  need(x.row >= 0 && x.head >= 0, "window attention: negative strides");
  layout((rows <= 1 || (x.row % 8 == 0 && x.row <= (int64_t{1} << 24))) && (heads <= 1 || x.head % 8 == 0) &&
             reinterpret_cast<uintptr_t>(x.data) % 16 == 0,
         "window attention: rows and heads at 16-byte addresses, rows at most 2^24 elements apart");
  return x;
}

WindowArgs window_args(const relx_window_args &p, int &type) {
  type = element_type(p.kind, p.bits);
  layout(type == kF16 || type == kBF16, "window attention: f16 or bf16 heads");
  need(fits32(p.rows) && fits32(p.sequences), "window attention: a size is negative or beyond 2^31 - 1");
  need(p.heads >= 1 && p.kv_heads >= 1 && p.heads % p.kv_heads == 0,
       "window attention: query heads are a multiple of the key heads");
  layout(p.heads <= 65535, "window attention: more than 65535 heads");
  layout(p.dim >= 8 && p.dim <= 128 && p.dim % 8 == 0, "window attention: head sizes are multiples of 8 up to 128");
  layout(p.rows <= kMost / 2, "window attention: more than 2^29 rows");
  need(p.window >= 0 && p.sinks >= 0, "window attention: a negative window or number of first tokens");
  const int64_t window = p.window == 0 ? kMost : std::min(p.window, kMost);
  const int64_t sinks = window >= p.rows ? 0 : p.sinks; // of a window that no row leaves: none apart
  layout(sinks <= kMostSinks, "window attention: more than 256 first tokens");
  const float scale = static_cast<float>(p.scale * 1.4426950408889634);
  need(std::isfinite(scale), "window attention: scale");
  need(p.rows == 0 || p.starts, "window attention: null starts");
  WindowArgs a{};
  a.starts = p.starts;
  a.lse = p.lse;
  a.rows = static_cast<int32_t>(p.rows);
  a.sequences = static_cast<int32_t>(p.sequences);
  a.heads = static_cast<int32_t>(p.heads);
  a.kv_heads = static_cast<int32_t>(p.kv_heads);
  a.dim = static_cast<int32_t>(p.dim);
  a.window = static_cast<int32_t>(window);
  a.sinks = static_cast<int32_t>(sinks);
  // By a scale below 2^-64 no score within f16's and bf16's usual range reaches a
  // bit of a weight: then 2^-64, by which the kernels divide.
  a.scale = std::fabs(scale) < 0x1p-64f ? std::copysign(0x1p-64f, scale) : scale;
  a.plain_scale = static_cast<float>(p.scale);
  const int64_t group = p.heads / p.kv_heads, parts = (group + 15) / 16, heads = (group + parts - 1) / parts;
  a.parts = static_cast<int32_t>((group + heads - 1) / heads);
  a.tile_heads = make_div(heads);
  a.tile_tokens = make_div(kTileRows / heads);
  // Keys of a workgroup in the backward pass: where there are few tiles of 128 of
  // all heads, 32. us of the whole backward with 32 and with 128, four query heads a
  // key head, window 512:
  //   heads of 128    17 tiles: 83, 168    136: 136, 188    260: 288, 340    520: 498, 493
  //   heads of 64     17 tiles: 58, 127    136: 76, 134     520: 252, 295
  // and longer, eight query heads, window 2048: 130 tiles of 128: 893, 953, 260: 1328,
  // 1158; four, window 1024: 1032 tiles of 64: 702, 706, 2056: 1425, 1358.
  const int64_t tiles = (p.rows / 128 + p.sequences) * p.kv_heads;
  a.key_tokens = make_div(tiles < (p.dim <= 64 ? 1024 : 256) ? 32 : 128);
  a.first_blocks = (a.sinks + 31) / 32;
  // half as many workgroups again as run at a time with heads of 64, three times as
  // many as run with wider ones, by shared memory
  const int64_t first = p.rows * p.kv_heads * std::max(a.first_blocks, 1) / 768;
  a.first_tokens = make_div(std::min<int64_t>(std::max<int64_t>((first + 31) / 32 * 32, 128), 4096));
  // Of rows that add to first tokens from outside their windows: only sequences
  // longer than the window have any, and there may be fewer of those than sequences.
  a.longer = make_div(std::min(window, p.rows) + 1);
  const auto pieces = [&](const FastDiv &size, int64_t sequences, int64_t heads_of_piece) {
    const int64_t n = p.rows / size.d + sequences + 2;
    // a workgroup of 256 threads for each, and 2^32 threads a dimension
    layout(n * heads_of_piece < (int64_t{1} << 24) - 8, "window attention: more than 2^24 - 8 tiles of rows and heads");
    return static_cast<int32_t>(n);
  };
  a.row_pieces = pieces(a.tile_tokens, p.sequences, p.kv_heads * a.parts);
  // Unless windows are as narrow, it is the first rows of a sequence that see few.
  const int64_t few = (kFew + a.tile_tokens.d - 1) / a.tile_tokens.d;
  a.few_pieces = window + sinks > kFew && p.sequences * few < a.row_pieces ? static_cast<int32_t>(few) : 0;
  a.key_pieces = pieces(a.key_tokens, p.sequences, p.kv_heads);
  a.first_pieces = pieces(a.first_tokens, std::min<int64_t>(p.sequences, p.rows / a.longer.d), p.kv_heads * std::max(a.first_blocks, 1));
  return a;
}

int64_t window_width(const WindowArgs &a) { return a.dim <= 64 ? 64 : 128; }
size_t stats_floats(const WindowArgs &a) { return (static_cast<size_t>(a.heads) * a.rows * 2 + 3) / 4 * 4; }
size_t window_workspace(const WindowArgs &a) {
  const size_t first = a.sinks ? static_cast<size_t>(a.first_pieces) * a.kv_heads * a.sinks * 2 * window_width(a) : 0;
  return (stats_floats(a) + first) * sizeof(float);
}

hipError_t window_launch(const WindowArgs &a, bool back, int type, hipStream_t s) {
  return type == kF16 ? window_launch_f16(a, back, s) : window_launch_bf16(a, back, s);
}

} // namespace
} // namespace relx

extern "C" {

int relx_window_attention(relx_ctx *ctx, const relx_window_args *args, uint64_t stream, relx_err *err) {
  return guarded(err, [&] {
    relx::need(args != nullptr, "null arguments");
    int type;
    relx::WindowArgs a = relx::window_args(*args, type);
    const bool used = a.rows > 0;
    a.q = relx::rows_of(&args->q, used, a.rows, a.heads, "window attention: null queries");
    a.k = relx::rows_of(&args->k, used, a.rows, a.kv_heads, "window attention: null keys");
    a.v = relx::rows_of(&args->v, used, a.rows, a.kv_heads, "window attention: null values");
    a.o = relx::rows_of(&args->out, used, a.rows, a.heads, "window attention: null result");
    relx::writable(&args->out, a.rows, a.heads, a.dim);
    relx::on_context(ctx, [&] {
      if (used)
        relx::launched(relx::window_launch(a, false, type, relx::stream_of(stream)), "window attention");
    });
  });
}

int relx_window_attention_workspace(const relx_window_args *args, size_t *bytes, relx_err *err) {
  return guarded(err, [&] {
    relx::need(args && bytes, "null arguments");
    relx_window_args p = *args;
    p.starts = reinterpret_cast<const int32_t *>(&p); // not read: only sizes count
    int type;
    *bytes = relx::window_workspace(relx::window_args(p, type));
  });
}

int relx_window_attention_backward(relx_ctx *ctx, const relx_window_args *args, const relx_heads *out_grad,
                                   const relx_heads *q_grad, const relx_heads *k_grad, const relx_heads *v_grad,
                                   void *workspace, size_t workspace_bytes, uint64_t stream, relx_err *err) {
  return guarded(err, [&] {
    relx::need(args != nullptr, "null arguments");
    int type;
    relx::WindowArgs a = relx::window_args(*args, type);
    const bool used = a.rows > 0;
    a.q = relx::rows_of(&args->q, used, a.rows, a.heads, "window attention: null queries");
    a.k = relx::rows_of(&args->k, used, a.rows, a.kv_heads, "window attention: null keys");
    a.v = relx::rows_of(&args->v, used, a.rows, a.kv_heads, "window attention: null values");
    a.o = relx::rows_of(&args->out, used, a.rows, a.heads, "window attention: null result");
    a.dout = relx::rows_of(out_grad, used, a.rows, a.heads, "window attention: null result's gradient");
    a.dq = relx::rows_of(q_grad, used, a.rows, a.heads, "window attention: null query gradient");
    a.dk = relx::rows_of(k_grad, used, a.rows, a.kv_heads, "window attention: null key gradient");
    a.dv = relx::rows_of(v_grad, used, a.rows, a.kv_heads, "window attention: null value gradient");
    relx::writable(q_grad, a.rows, a.heads, a.dim);
    relx::writable(k_grad, a.rows, a.kv_heads, a.dim);
    relx::writable(v_grad, a.rows, a.kv_heads, a.dim);
    relx::need(!used || a.lse, "window attention: the backward takes lse");
    const size_t want = relx::window_workspace(a);
    if (used && (workspace_bytes < want || !workspace))
      throw relx::Error("insufficient_capacity", "workspace holds " + std::to_string(workspace_bytes) +
                                                     " bytes, the call takes " + std::to_string(want));
    relx::need(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "window attention: workspace alignment");
    a.stats = static_cast<float *>(workspace);
    a.first_sums = a.stats + relx::stats_floats(a);
    relx::on_context(ctx, [&] {
      if (used)
        relx::launched(relx::window_launch(a, true, type, relx::stream_of(stream)), "window attention, backward");
    });
  });
}

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
    // Workgroups of 256 rows have no place here: two of 128 in their place, us for 8
    // requests of 48 tokens (192 rows) over up to 8192 int8 ones 87 against 107, of
    // 64 (256 rows) 93 against 100 and, up to 32768, 294 against 294; chunks of 512
    // tokens with a window of 2048 131 against 138, over 16 bits 113 against 118.
    if (plan.rows == 256) {
      plan.rows = 128;
      plan.workgroups = a.workgroups = relx::kMostWorkgroups;
      a.once = false;
    }
    // A table of up to 512 tokens: items are not cut, and nothing is left to join. us in
    // a graph, whole and cut, 8 key heads of 128, four rows each:
    //   bf16   1 request of 60 tokens 9.6, 11.5   of 440 13.1, 12.7   64 of up to 440 26.3, 40.3   256: 94, 120
    //   int8   7.9, 9.8   10.9, 10.8   15.9, 19.3   256: 42.5, 48.5 (four heads at a time)
    // and calls from Python 2 less than that, which the second launch took.
    plan.whole = plan.rows == 16 && plan.async && p.columns * p.cache.page <= 512;
    // Four int8 heads at a time, a wave each, where a token's heads lie closer together
    // than a head's tokens: 64 requests of up to 8192 tokens of 8 key heads, four rows
    // each, us with heads of 128: 135 against 153, of 80: 153 against 202, of 64: 97
    // against 131; of up to 512: 19.4 against 23.4; one of 100000: 48 against 51. Eight
    // of up to 1000 have too little for it (18.4 against 15.7): so not where the table
    // holds less than 2^17 tokens of all heads, nor for whole items that the card holds
    // at once (64 requests of up to 250 tokens: 21.0 against 11.7; 256: 25.5, 37.9).
    const int64_t kv = p.cache.kv_heads, tokens = p.columns * p.cache.page;
    const bool much = plan.whole ? p.requests * kv > relx::kMostWorkgroups : p.requests * tokens >= (1 << 17) / kv;
    plan.quads = i8 && much && plan.async && plan.rows == 16 && plan.width <= 128 && kv % 4 == 0 &&
                 (p.rows + p.requests - 1) / std::max<int64_t>(p.requests, 1) * (p.heads / kv) <= 4 &&
                 p.cache.key_head < p.cache.key_slot && p.cache.value_head < p.cache.value_slot;
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
