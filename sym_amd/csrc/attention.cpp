// attention.cpp - C entry points of the paged-cache operators: argument
// checks, what the kernels take, launches (include/relx.h).
#include "attention.h"

#include <climits>
#include <cmath>
#include <cstdlib>
#include <utility>

#include "capi.h"
#include "runtime.h"

namespace relx {
namespace {

void need(bool ok, const char *what) {
  if (!ok)
    throw Error("invalid_argument", what);
}

void layout(bool ok, const char *what) {
  if (!ok)
    throw Error("unsupported_layout", what);
}

int element_type(int64_t kind, int64_t bits) {
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

bool fits32(int64_t v) { return v >= 0 && v <= INT32_MAX; }

void launched(hipError_t e, const char *what) {
  if (e != hipSuccess)
    throw Error("backend_failure", std::string(what) + ": " + hipGetErrorString(e));
}

// Runs `fn` with the context's device current, if the context takes calls.
// Not under its mutex, which transfers hold until the GPU has done them: these
// calls use nothing that it guards.
template <class F> void on_context(relx_ctx *ctx, F &&fn) {
  need(ctx != nullptr, "null context");
  if (ctx->ctx->closed || ctx->ctx->quarantined)
    throw Error("resources_closed", "context is closed or quarantined");
  DeviceScope scope(ctx->ctx->device);
  fn();
}

hipStream_t stream_of(uint64_t s) { return reinterpret_cast<hipStream_t>(s); }

// Whether elements of [n1, n2, dim] with these strides share a place.
bool overlap(int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t dim) {
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
void writable(const relx_heads *h, int64_t rows, int64_t heads, int64_t dim) {
  need(!h || rows == 0 || heads == 0 || !overlap(rows, h->row, heads, h->head, dim), "a result's elements overlap");
}

// ------------------------------------------------------------ block tables

TablesArgs tables_args(const relx_block_tables_args &p) {
  need(fits32(p.requests) && fits32(p.columns) && fits32(p.rows) && fits32(p.words) && p.free_count >= 0,
       "block tables: a size is negative or beyond 2^31 - 1");
  need(p.page >= 1 && p.page <= INT32_MAX, "block tables: page size");
  need(p.starts && p.taken, "block tables: null starts or taken");
  need(p.requests == 0 || (p.cached && p.fresh), "block tables: null lengths");
  need(p.requests == 0 || p.columns == 0 || p.table, "block tables: null table");
  need(p.table_row >= p.columns || p.requests <= 1, "block tables: table rows overlap");
  need(p.free_count == 0 || p.free_pages, "block tables: null page list");
  need(p.rows == 0 || (p.slots && p.positions), "block tables: null slots or positions");
  // a list of no parents may have no address
  need(p.rows == 0 || (p.parents != nullptr) == (p.words > 0), "block tables: a mask goes with parents");
  need(!p.parents || p.rows == 0 || p.mask, "block tables: null mask");
  TablesArgs a{};
  a.cached = p.cached;
  a.fresh = p.fresh;
  a.table = p.table;
  a.table_row = p.table_row;
  a.free_pages = p.free_pages;
  a.free_count = p.free_count;
  a.parents = p.parents;
  a.starts = p.starts;
  a.slots = p.slots;
  a.positions = p.positions;
  a.mask = p.mask;
  a.taken = p.taken;
  a.page = make_div(p.page);
  a.requests = static_cast<int32_t>(p.requests);
  a.columns = static_cast<int32_t>(p.columns);
  a.rows = static_cast<int32_t>(p.rows);
  a.words = static_cast<int32_t>(p.words);
  return a;
}

// --------------------------------------------------------- norm and rotation

constexpr int64_t kMostDim = 512;

// The sizes of a call and its block of heads per wave.
RotateArgs rotate_args(const relx_rotation &r, int &type) {
  type = element_type(r.kind, r.bits);
  layout(type != kI8, "norm and rotation: f32, f16 or bf16 heads");
  need(fits32(r.rows) && r.heads >= 0 && r.kv_heads >= 0, "norm and rotation: a size is negative or beyond 2^31 - 1");
  layout(r.heads <= 65535 && r.kv_heads <= 65535, "norm and rotation: more than 65535 heads");
  layout(r.dim >= 1 && r.dim <= kMostDim, "norm and rotation: head sizes up to 512");
  need(r.rotary >= 0 && r.rotary <= r.dim && r.rotary % 2 == 0,
       "norm and rotation: an even number of elements within the head turns");
  need(r.angles >= 0 && fits32(r.angles), "norm and rotation: angles");
  need(r.rows == 0 || r.positions, "norm and rotation: null positions");
  need(r.rotary == 0 || r.angles == 0 || (r.cos && r.sin), "norm and rotation: null cos or sin");
  need(std::isfinite(r.eps) && r.eps >= 0, "norm and rotation: eps");
  RotateArgs a{};
  a.weight[0] = r.q_weight;
  a.weight[1] = r.k_weight;
  if (r.q_weight || r.k_weight) {
    a.weight_type = element_type(r.weight_kind, r.weight_bits);
    layout(a.weight_type != kI8, "norm and rotation: f32, f16 or bf16 weights");
  }
  a.positions = r.positions;
  a.cos = r.cos;
  a.sin = r.sin;
  a.rows = static_cast<int32_t>(r.rows);
  a.heads[0] = static_cast<int32_t>(r.heads);
  a.heads[1] = static_cast<int32_t>(r.kv_heads);
  a.dim = static_cast<int32_t>(r.dim);
  a.rotary = static_cast<int32_t>(r.rotary);
  a.angles = static_cast<int32_t>(r.angles);
  a.pairs = r.pairs != 0;
  a.eps = static_cast<float>(r.eps);
  a.inv_dim = 1.0f / static_cast<float>(r.dim);
  // A wave's heads at a time, twice where there are more of them: 32768 rows of 40
  // heads of 128 forward took 136 us in a trace so, 167 without, 133 to 158 with
  // four times.
  const int at_once = 64 / rotate_lanes(a.dim);
  a.chunk_heads = std::max(a.heads[0], a.heads[1]) > at_once ? 2 * at_once : at_once;
  for (int k = 0; k < 2; ++k)
    a.chunks[k] = (a.heads[k] + a.chunk_heads - 1) / a.chunk_heads;
  return a;
}

// Blocks of heads are the launch's second dimension.
void fits_launch(const RotateArgs &a) {
  layout(a.chunks[0] + a.chunks[1] + a.chunks[2] <= 65535, "norm and rotation: more than 65535 blocks of heads");
}

Heads heads_of(const relx_heads *h, bool used, const char *what) {
  need(!used || (h && h->data), what);
  return used ? Heads{static_cast<char *>(h->data), h->row, h->head} : Heads{};
}

size_t rotate_partial(const RotateArgs &a) {
  const int64_t chunks = a.chunks[0] + a.chunks[1];
  if (a.rows == 0 || chunks == 0)
    return 0;
  return static_cast<size_t>(rotate_blocks(kRotateBackward, a.rows, chunks) * chunks * a.dim) *
         sizeof(float);
}

// ------------------------------------------------------------ paged caches

struct CacheBytes {
  int64_t key_page, key_slot, key_head, value_page, value_slot, value_head;
  int type;
};

CacheBytes cache_bytes(const relx_cache &c) {
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

// ------------------------------------------------------------ attention

AttendArgs attend_args(const relx_tree_attention_args &p, AttendPlan &plan, int &type, bool &i8) {
  type = element_type(p.kind, p.bits);
  layout(type == kF16 || type == kBF16, "attention: f16 or bf16 queries");
  const CacheBytes c = cache_bytes(p.cache);
  i8 = c.type == kI8;
  layout(i8 || c.type == type, "attention: a cache of the queries' type or int8");
  need(fits32(p.rows) && fits32(p.requests) && fits32(p.columns) && fits32(p.words),
       "attention: a size is negative or beyond 2^31 - 1");
  // the join has a block of 512 threads for each, and 2^32 threads a dimension
  layout(p.requests < (int64_t{1} << 23) - 1, "attention: more than 2^23 - 2 requests");
  const int64_t kv = p.cache.kv_heads, dim = p.cache.dim;
  need(p.heads >= 1 && kv >= 1 && p.heads % kv == 0, "attention: query heads are a multiple of the key heads");
  layout(p.heads <= 65535, "attention: more than 65535 heads");
  layout(dim >= 8 && dim <= 256 && dim % 8 == 0, "attention: head sizes are multiples of 8 up to 256");
  layout(p.columns == 0 || p.columns <= (int64_t{1} << 30) / p.cache.page, "attention: a table of more than 2^30 tokens");
  layout(p.rows <= INT32_MAX / p.heads, "attention: more than 2^31 - 1 rows of heads");
  const float scale = static_cast<float>(p.scale * 1.4426950408889634);
  need(std::isfinite(scale), "attention: scale");
  need(p.rows == 0 || (p.q.data && p.out.data), "attention: null queries or result");
  writable(&p.out, p.rows, p.heads, dim);
  need(p.requests == 0 || (p.cached && p.starts), "attention: null lengths");
  need(p.requests == 0 || p.columns == 0 || p.table, "attention: null table");
  need(!p.mask || p.words >= 1, "attention: a mask has words");
  AttendArgs a{};
  a.q = static_cast<const char *>(p.q.data);
  a.q_row = p.q.row;
  a.q_head = p.q.head;
  a.out = static_cast<char *>(p.out.data);
  a.out_row = p.out.row;
  a.out_head = p.out.head;
  a.keys = static_cast<const char *>(p.cache.keys);
  a.values = static_cast<const char *>(p.cache.values);
  a.key_page = c.key_page;
  a.key_slot = c.key_slot;
  a.key_head = c.key_head;
  a.value_page = c.value_page;
  a.value_slot = c.value_slot;
  a.value_head = c.value_head;
  a.key_scale = p.cache.key_scale;
  a.value_scale = p.cache.value_scale;
  a.table = p.table;
  a.table_row = p.table_row;
  a.cached = p.cached;
  a.starts = p.starts;
  a.mask = p.mask;
  a.lse = p.lse;
  a.page = make_div(p.cache.page);
  a.group = make_div(p.heads / kv);
  a.rows = static_cast<int32_t>(p.rows);
  a.requests = static_cast<int32_t>(p.requests);
  a.heads = static_cast<int32_t>(p.heads);
  a.kv_heads = static_cast<int32_t>(kv);
  a.dim = static_cast<int32_t>(dim);
  a.pages = static_cast<int32_t>(p.cache.pages);
  a.columns = static_cast<int32_t>(p.columns);
  a.words = static_cast<int32_t>(p.words);
  a.scale = scale;
  plan = attend_plan(p.rows, p.requests, p.heads / kv, dim, p.cache.page);
  // a lane's distance inside a tile of 16 tokens is held in 32 bits
  if (a.key_slot > INT32_MAX / 32 || a.value_slot > INT32_MAX / 32)
    plan.even = false;
  const int64_t at = reinterpret_cast<int64_t>(a.keys) | reinterpret_cast<int64_t>(a.values) | a.key_page | a.key_slot |
                     a.key_head | a.value_page | a.value_slot | a.value_head;
  // Tiles that go to shared memory by themselves against tiles through registers:
  // 8 requests of 256 rows over up to 32768 tokens 276 us against 357, one of 52
  // rows over 131072 106 against 172, 64 int8 requests of one 259 against 431.
  plan.async = plan.even && (at | dim * (i8 ? 1 : 2)) % 16 == 0;
  if (plan.rows == 16)
    plan.workgroups = turn_workgroups(plan.width, i8, plan.async);
  a.workgroups = plan.workgroups;
  // Then keys and values go past the caches: 52 rows over 131072 tokens 106 us
  // against 120, 128 rows of 8 requests over up to 32768 182 to 189 against 209, 64
  // int8 requests of one row, whose kernel always does, 247 against 278. Where other
  // tiles read them too: 461 against 434 (512 tokens of 8 requests, up to 8192).
  a.once = p.requests > 0 && (p.rows + p.requests - 1) / p.requests * (p.heads / kv) <= plan.rows;
  return a;
}

} // namespace

AttendPlan attend_plan(int64_t rows, int64_t requests, int64_t group, int64_t dim, int64_t page) {
  AttendPlan p{};
  p.width = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  p.even = page % 16 == 0;
  // Query rows of a key head in an even batch. More rows of a workgroup read a
  // tile less often and leave fewer waves to read ahead; a row that is not there
  // costs what one that is does. 8 requests of up to 32768 tokens, 8 key heads
  // of 128, bf16, us by rows of an item:
  //   256 rows each   64: 598   128: 367   256: 270
  //   128 rows        64: 340   128: 173   256: 195
  //   64 rows         16: 440   64: 169   128: 174
  //   16 rows         16: 171   64: 176; 64 int8 requests of one row: 16: 254, 64: 423
  const int64_t q = requests > 0 ? (rows + requests - 1) / requests * group : 0;
  p.rows = q <= 16 ? 16 : q <= 64 || p.width == 256 ? 64 : q <= 128 ? 128 : 256;
  p.workgroups = p.rows == 256 ? kMostWorkgroups / 2 : kMostWorkgroups;
  return p;
}

size_t attend_part_rows(const AttendPlan &p) {
  // 256 rows always run half of the workgroups; 16 may, by the cache's addresses
  return static_cast<size_t>(p.rows == 256 ? kMostWorkgroups / 2 : kMostWorkgroups) * 2 * static_cast<size_t>(p.rows);
}

size_t attend_workspace(const AttendPlan &p, int64_t requests) {
  const size_t rows = attend_part_rows(p);
  return rows * static_cast<size_t>(p.width + 2) * sizeof(float) +
         (static_cast<size_t>(requests) + 1) * sizeof(int64_t);
}

hipError_t attend_launch(const AttendArgs &a, const AttendPlan &p, int type, bool i8, hipStream_t s) {
  if (type == kF16)
    return i8 ? attend_launch_f16_i8(a, p, s) : attend_launch_f16(a, p, s);
  return i8 ? attend_launch_bf16_i8(a, p, s) : attend_launch_bf16(a, p, s);
}

} // namespace relx

extern "C" {

int relx_block_tables(relx_ctx *ctx, const relx_block_tables_args *args, uint64_t stream,
                      relx_err *err) {
  return guarded(err, [&] {
    relx::need(args != nullptr, "null arguments");
    const relx::TablesArgs a = relx::tables_args(*args);
    relx::on_context(ctx, [&] {
      relx::launched(relx::tables_launch(a, relx::stream_of(stream)), "block tables");
    });
  });
}

int relx_norm_rotate(relx_ctx *ctx, const relx_rotation *rot, const relx_heads *q,
                     const relx_heads *k, const relx_heads *q_out, const relx_heads *k_out,
                     uint64_t stream, relx_err *err) {
  return guarded(err, [&] {
    relx::need(rot != nullptr, "null arguments");
    int type;
    relx::RotateArgs a = relx::rotate_args(*rot, type);
    relx::fits_launch(a);
    const bool uq = a.rows && a.heads[0], uk = a.rows && a.heads[1];
    a.x[0] = relx::heads_of(q, uq, "norm and rotation: null queries");
    a.x[1] = relx::heads_of(k, uk, "norm and rotation: null keys");
    relx::writable(q_out, a.rows, a.heads[0], a.dim);
    relx::writable(k_out, a.rows, a.heads[1], a.dim);
    a.y[0] = relx::heads_of(q_out, uq, "norm and rotation: null query result");
    a.y[1] = relx::heads_of(k_out, uk, "norm and rotation: null key result");
    relx::on_context(ctx, [&] {
      if (uq || uk)
        relx::launched(relx::rotate_launch(a, relx::kRotateForward, type, relx::stream_of(stream)),
                       "norm and rotation");
    });
  });
}

int relx_norm_rotate_workspace(const relx_rotation *rot, size_t *bytes, relx_err *err) {
  return guarded(err, [&] {
    relx::need(rot && bytes, "null arguments");
    int type;
    *bytes = relx::rotate_partial(relx::rotate_args(*rot, type));
  });
}

int relx_norm_rotate_backward(relx_ctx *ctx, const relx_rotation *rot, const relx_heads *dq,
                              const relx_heads *dk, const relx_heads *q, const relx_heads *k,
                              const relx_heads *q_grad, const relx_heads *k_grad,
                              float *q_weight_grad, float *k_weight_grad, void *workspace,
                              size_t workspace_bytes, uint64_t stream, relx_err *err) {
  return guarded(err, [&] {
    relx::need(rot != nullptr, "null arguments");
    int type;
    relx::RotateArgs a = relx::rotate_args(*rot, type);
    relx::fits_launch(a);
    const bool uq = a.rows && a.heads[0], uk = a.rows && a.heads[1];
    a.x[0] = relx::heads_of(q, uq, "norm and rotation: null queries");
    a.x[1] = relx::heads_of(k, uk, "norm and rotation: null keys");
    a.dz[0] = relx::heads_of(dq, uq, "norm and rotation: null query gradient");
    a.dz[1] = relx::heads_of(dk, uk, "norm and rotation: null key gradient");
    relx::writable(q_grad, a.rows, a.heads[0], a.dim);
    relx::writable(k_grad, a.rows, a.heads[1], a.dim);
    a.y[0] = relx::heads_of(q_grad, uq, "norm and rotation: null query gradient");
    a.y[1] = relx::heads_of(k_grad, uk, "norm and rotation: null key gradient");
    a.weight_grad[0] = q_weight_grad;
    a.weight_grad[1] = k_weight_grad;
    relx::need((!q_weight_grad || rot->q_weight) && (!k_weight_grad || rot->k_weight),
               "norm and rotation: a weight's gradient goes with the weight");
    if (q_weight_grad || k_weight_grad) {
      const size_t want = relx::rotate_partial(a);
      if (workspace_bytes < want || (want && !workspace))
        throw relx::Error("insufficient_capacity", "workspace holds " + std::to_string(workspace_bytes) +
                                                       " bytes, the call takes " + std::to_string(want));
      a.partial = static_cast<float *>(workspace);
    }
    relx::on_context(ctx, [&] {
      relx::launched(relx::rotate_launch(a, relx::kRotateBackward, type, relx::stream_of(stream)),
                     "norm and rotation, backward");
    });
  });
}

int relx_norm_rotate_append(relx_ctx *ctx, const relx_rotation *rot, const relx_heads *q,
                            const relx_heads *k, const relx_heads *v, const relx_heads *q_out,
                            const int64_t *slots, const relx_cache *cache, uint64_t stream,
                            relx_err *err) {
  return guarded(err, [&] {
    relx::need(rot && cache, "null arguments");
    int type;
    relx::RotateArgs a = relx::rotate_args(*rot, type);
    const relx::CacheBytes c = relx::cache_bytes(*cache);
    const bool i8 = c.type == relx::kI8;
    relx::layout(i8 || c.type == type, "append: a cache of the heads' type or int8");
    relx::need(cache->kv_heads == rot->kv_heads && cache->dim == rot->dim, "append: the cache has other heads");
    const bool uq = a.rows && a.heads[0], uk = a.rows && a.heads[1];
    a.x[0] = relx::heads_of(q, uq, "append: null queries");
    a.x[1] = relx::heads_of(k, uk, "append: null keys");
    a.x[2] = relx::heads_of(v, uk, "append: null values");
    relx::writable(q_out, a.rows, a.heads[0], a.dim);
    const auto apart = [&](int64_t page, int64_t slot, int64_t head) {
      return !relx::overlap(cache->pages, page, cache->page, slot, cache->dim) &&
             !relx::overlap(cache->pages, page, cache->kv_heads, head, cache->dim) &&
             !relx::overlap(cache->page, slot, cache->kv_heads, head, cache->dim);
    };
    relx::need(!uk || cache->pages == 0 || (apart(cache->key_page, cache->key_slot, cache->key_head) &&
                                            apart(cache->value_page, cache->value_slot, cache->value_head)),
               "append: the cache's elements overlap");
    a.y[0] = relx::heads_of(q_out, uq, "append: null query result");
    relx::need(!uk || slots, "append: null slots");
    a.chunks[2] = a.chunks[1];
    relx::fits_launch(a);
    a.slots = slots;
    a.page = relx::make_div(cache->page);
    a.pages_slots = cache->pages * cache->page;
    a.cache[0] = static_cast<char *>(cache->keys);
    a.cache[1] = static_cast<char *>(cache->values);
    const int64_t pages[2] = {cache->key_page, cache->value_page};
    const int64_t slot[2] = {cache->key_slot, cache->value_slot};
    const int64_t head[2] = {cache->key_head, cache->value_head};
    for (int i = 0; i < 2; ++i) {
      a.cache_page[i] = pages[i];
      a.cache_slot[i] = slot[i];
      a.cache_head[i] = head[i];
    }
    a.scale[0] = cache->key_scale;
    a.scale[1] = cache->value_scale;
    relx::on_context(ctx, [&] {
      if (uq || uk)
        relx::launched(relx::rotate_launch(a, i8 ? relx::kRotateAppendI8 : relx::kRotateAppend, type,
                                           relx::stream_of(stream)),
                       "append");
    });
  });
}

int relx_tree_attention_workspace(const relx_tree_attention_args *args, size_t *bytes,
                                  relx_err *err) {
  return guarded(err, [&] {
    relx::need(args && bytes, "null arguments");
    const relx_tree_attention_args &p = *args;
    relx::need(relx::fits32(p.rows) && relx::fits32(p.requests) && p.heads >= 1 && p.cache.kv_heads >= 1 &&
                   p.cache.page >= 1,
               "attention: sizes");
    *bytes = relx::attend_workspace(relx::attend_plan(p.rows, p.requests, p.heads / p.cache.kv_heads, p.cache.dim,
                                                      p.cache.page),
                                    p.requests);
  });
}

int relx_tree_attention(relx_ctx *ctx, const relx_tree_attention_args *args, uint64_t stream,
                        relx_err *err) {
  return guarded(err, [&] {
    relx::need(args != nullptr, "null arguments");
    relx::AttendPlan plan;
    int type;
    bool i8;
    relx::AttendArgs a = relx::attend_args(*args, plan, type, i8);
    if (a.rows > 0 && a.requests > 0) {
      const size_t want = relx::attend_workspace(plan, a.requests);
      if (args->workspace_bytes < 0 || static_cast<size_t>(args->workspace_bytes) < want || !args->workspace)
        throw relx::Error("insufficient_capacity", "workspace holds " + std::to_string(args->workspace_bytes) +
                                                       " bytes, the call takes " + std::to_string(want));
      const size_t rows = relx::attend_part_rows(plan);
      relx::need(reinterpret_cast<uintptr_t>(args->workspace) % 16 == 0, "attention: workspace alignment");
      a.partial = static_cast<float *>(args->workspace);
      a.stats = a.partial + rows * static_cast<size_t>(plan.width);
      a.schedule = reinterpret_cast<int64_t *>(a.stats + rows * 2);
    }
    relx::on_context(ctx, [&] {
      if (a.rows > 0)
        relx::launched(relx::attend_launch(a, plan, type, i8, relx::stream_of(stream)), "attention");
    });
  });
}

} // extern "C"
