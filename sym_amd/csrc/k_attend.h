// k_attend.h - attention of a step's query rows over a paged cache (device
// templates; instantiated in k_attend_f16.hip, k_attend_bf16.hip and, over int8
// caches, k_attend_f16_i8.hip and k_attend_bf16_i8.hip).
//
// One pass over the keys and values with the running maximum and sum of the
// softmax. The query rows of a request that share a key head (its new tokens
// times the heads of the group) are the columns of matrix products; a wave
// keeps 16 or 32 of them with their sums in registers:
//
//   S^T = K Q^T    16 tokens x 16 rows per product, dims contracted
//   O^T += V^T P^T 16 dims x 16 rows per product, 32 tokens contracted
//
// The layout of S^T in the registers (lane: row = lane % 16, tokens
// 4 (lane / 16) + 0..3 of each of two token tiles) is the layout of the
// second product's operand if its contracted tokens are numbered
// 8 (lane / 16) + 4 tile + 0..3, so the weights go from one product to the
// next without leaving their lane. Keys and values pass through shared memory, 32 tokens at a time:
// a lane reads its 16 bytes of a key row as they are, and values transposed
// (ds_read_b64_tr_b16: four tokens of one dim from four lanes' rows).
//
// How tokens get there (Source):
//   kAsync   pages of whole tiles of 16 tokens and rows at 16-byte addresses:
//            loads that write shared memory themselves, a ring of tiles ahead
//   kStaged  everything else: through registers, where what is no token
//            becomes zero
// and who works on them:
//   up to 4 query rows, int8 heads side by side (a view's): a wave has a head of its
//     own, so that four heads of a token are one piece of memory.
//   up to 16 query rows share a key head (decoding): bound by the cache's
//     bytes. The waves of a workgroup take turns at the tiles, each with a ring
//     of its own and no barrier, and add up at the end. int8 is widened in the
//     registers.
//   more (trees, chunks): the waves have rows of their own, 16 or 32 each, and
//     share the tiles. int8 is widened on its way there, once for all of them: with a
//     scale a block from a ring of int8 tiles that arrive by themselves (trees of 48 in
//     8 requests over up to 8192 tokens 107 us against 128 through registers, with 256
//     rows a workgroup).
//
// The work of a call is the list of its units of tokens over (request, key
// head, tile of query rows), cut into equal runs, one per workgroup; an item
// that lies in several runs leaves partial sums that k_attend_join adds up. So
// one long context fills the card as well as many short ones do, and uneven
// lengths cost nothing. A view's table of up to kWholeUnit tokens has units that hold
// an item: there nothing is cut, and nothing joined.
//
// Measured, with the join (8 key heads of 128 each, unless said):
//   64 requests of 1 row, 3000 int8 tokens on average, 32 key heads: 246 to 250
//     us, 6.3 TB/s of cache. Bound by the reads.
//   1 request of 13 rows x 4 heads, 131072 bf16 tokens: 100 to 101 us, 5.3 TB/s.
//     Bound by the reads, but for the join's 6.
//   64 requests of 1 row x 4 heads, 6100 int8 tokens with a scale a block on average, a
//     token's heads side by side: 136 us, 5.7 TB/s (a head at a time 153).
//   64 requests of 1 row x 4 heads, window of 2048 bf16 tokens: 98 us, 5.5 TB/s.
//   8 requests of 48 rows x 4 heads, up to 8192 int8 tokens, a scale a block: 88 us.
//   8 requests of 64 rows x 4 heads, up to 8192 tokens: 77 to 78 us, 455 TFLOP/s; up
//     to 32768: 274 to 315 us by the card's clock, 575 to 660 TFLOP/s. No unit is busy most of the time: the matrix
//     units for 0.27 of it, shared memory 0.21 (a third of that in bank conflicts),
//     the vector units a quarter by their count of instructions. The waves' steps
//     wait for one another (products, softmax, products) more than they overlap.
#pragma once

#include <algorithm>
#include <type_traits>
#include <utility>

#include "attend_share.h"
#include "attention.h"
#include "index.h"
#include "k_attend_wave.h"

namespace relx {
namespace {

constexpr int kScan = 128;    // runs of requests whose units a workgroup (of at least as many threads) adds up
constexpr int kTile = 32;     // tokens of a tile
constexpr int kSharedUnit = 64;
constexpr int turn_unit(int dp) { return turn_waves(dp) * kTile; }
// Unit of a call whose table holds no more tokens: no item is cut, so that no partial
// sums are left, and no launch that joins them.
constexpr int kWholeUnit = 512;
// Rows of an item of four heads at a time (k_attend_quads), which fit the places of
// sixteen, and its unit.
constexpr int kQuadRows = 4, kQuadUnit = 4 * kTile;
// Heads' items of a request.
template <int ROWS> __device__ __forceinline__ int head_items(const AttendArgs &a) {
  return ROWS == kQuadRows ? a.kv_heads >> 2 : a.kv_heads;
}

enum Source : int { kAsync, kStaged, kStagedEven };
// What a call's rows see, and how a cache's codes are scaled:
//   kWhole    all of the context; int8 by a scale a head
//   kWindow   the last `window` tokens and the first `sinks` ones; no int8
//   kBlocks   the same of an int8 cache with a scale a block of tokens and head
// With a window, an item's tiles of tokens are numbered without the ones that
// none of its rows sees: up to `edge`, the end of the tiles with first tokens,
// a place is the token's own, and from there on `jump` tokens before it.
enum Form : int { kWhole, kWindow, kBlocks };
// The kernel's arguments, read anew: what needs them now and then does not
// hold scalar registers through the loops.
__device__ __forceinline__ const AttendArgs &args_again() {
  uint64_t p = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(p));
  return *(const AttendArgs *)reinterpret_cast<const __attribute__((address_space(4))) AttendArgs *>(p);
}

// Two int8 values (byte K of x, byte M of y) as a pair of T, exactly.
template <int T, int K, int M> __device__ __forceinline__ uint32_t pair8(uint32_t x, uint32_t y) {
  if constexpr (T == kF16) {
    // 0x6400 | u is 1024 + u: with the sign bit flipped, 1152 more than the byte
    const uint32_t u = __builtin_amdgcn_perm(y, x, (0x0cu << 24) | ((4u + M) << 16) | (0x0cu << 8) | K) ^
                       0x64806480u;
    const f16x2 off = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, u) - off);
  } else {
    const int a = static_cast<int>(x << (24 - 8 * K)) >> 24, b = static_cast<int>(y << (24 - 8 * M)) >> 24;
    return pack16<T>(static_cast<float>(a), static_cast<float>(b));
  }
}

template <int T> __device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi) {
  return u32x4{pair8<T, 0, 1>(lo, lo), pair8<T, 2, 3>(lo, lo), pair8<T, 0, 1>(hi, hi),
               pair8<T, 2, 3>(hi, hi)};
}

__device__ __forceinline__ float max_over_groups(float x) {
  // the four lanes that hold a row's other tokens: 16 and 32 lanes away
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// n / d for n that hardly ever needs more than 32 bits: short code, since a
// kernel of a few microseconds waits for every line of it to be fetched.
__device__ __forceinline__ int64_t divide(int64_t n, int d) {
  if (__builtin_expect(n >> 32 == 0, 1))
    return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
  return n / d;
}

// Zeros for the rows of no request, where no join writes them.
__device__ __forceinline__ void zero_unowned(const AttendArgs &a) {
  const int r0 = min(max(a.starts[0], 0), a.rows), r1 = min(max(a.starts[a.requests], r0), a.rows);
  const int64_t none = static_cast<int64_t>(r0 + a.rows - r1) * a.heads;
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * waves + (threadIdx.x >> 6); i < none; i += static_cast<int64_t>(gridDim.x) * waves) {
    int64_t row = i / a.heads;
    const int64_t qh = i - row * a.heads;
    row += row < r0 ? 0 : r1 - r0;
    for (int d = lane; d < a.dim; d += 64)
      store(a.out + (row * a.out_row + qh * a.out_head + d) * 2, static_cast<uint16_t>(0));
    if (a.lse && lane == 0)
      a.lse[row * a.heads + qh] = -__builtin_inff();
  }
}

// ------------------------------------------------------------ the schedule

// The end of the tiles with first tokens.
__device__ __forceinline__ int edge_of(const AttendArgs &a, int length) {
  return (min(a.sinks, length) + kTile - 1) & ~(kTile - 1);
}

struct Request {
  int cached, length; // tokens in the cache before the step, and with it: at most 2^30
  int start, fresh;   // its rows
  int tiles;          // tiles of query rows
  int units;          // of one item
};

// ROWS: query rows of an item, UNIT: tokens of a unit.
template <int FORM, int ROWS, int UNIT>
__device__ __forceinline__ Request attend_request(const AttendArgs &a, int b) {
  Request r;
  const int s = min(max(a.starts[b], 0), a.rows), e = min(max(a.starts[b + 1], s), a.rows);
  r.start = s;
  r.fresh = e - s;
  const int room = a.pages > 0 ? a.columns * static_cast<int>(a.page.d) : 0;
  r.cached = min(max(a.cached[b], 0), room);
  r.length = r.fresh < room - r.cached ? r.cached + r.fresh : room;
  const int64_t q = static_cast<int64_t>(r.fresh) * a.group.d;
  r.tiles = static_cast<int>((q + ROWS - 1) / ROWS);
  int reach = r.length;
  if constexpr (FORM != kWhole) {
    // as many tokens as any of its items has: first ones, those that the windows
    // of an item's rows span, and the rest of the tile in which the span begins
    const uint32_t g = a.group.d;
    const uint32_t span = a.mask ? r.fresh : min(static_cast<uint32_t>(r.fresh), (ROWS - 1) / g + 2);
    const int64_t most = static_cast<int64_t>(edge_of(a, r.length)) + kTile - 1 + a.window + span;
    reach = static_cast<int>(min(static_cast<int64_t>(reach), most));
  }
  r.units = max((reach + UNIT - 1) / UNIT, 1);
  return r;
}

template <int FORM, int ROWS, int UNIT>
__device__ __forceinline__ int64_t request_units(const AttendArgs &a, int b) {
  const Request r = attend_request<FORM, ROWS, UNIT>(a, b);
  return static_cast<int64_t>(head_items<ROWS>(a)) * r.tiles * r.units;
}

// The units before each run of requests, which every workgroup adds up for
// itself.
struct Schedule {
  int64_t before[kScan + 1];
  int64_t waves[kScan / 64];
};

template <int FORM, int ROWS, int UNIT>
__device__ __forceinline__ void add_up(const AttendArgs &a, Schedule &sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int run = (a.requests + kScan - 1) / kScan;
  const int b0 = min(tid * run, a.requests), b1 = min(b0 + run, a.requests);
  const bool in = tid < kScan;
  int64_t mine = 0, upto = 0;
  if (in) {
    for (int b = b0; b < b1; ++b)
      mine += request_units<FORM, ROWS, UNIT>(a, b);
    upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t v = __shfl_up(upto, o);
      if (lane >= o)
        upto += v;
    }
    if (lane == 63)
      sh.waves[wave] = upto;
  }
  __syncthreads();
  if (in) {
    int64_t first = upto - mine;
    for (int w = 0; w < wave; ++w)
      first += sh.waves[w];
    sh.before[tid] = first;
    if (tid == kScan - 1)
      sh.before[kScan] = first + mine;
    if (blockIdx.x == 0) { // for the join
      int64_t at = first;
      for (int b = b0; b < b1; ++b) {
        a.schedule[b] = at;
        at += request_units<FORM, ROWS, UNIT>(a, b);
      }
      if (tid == kScan - 1)
        a.schedule[a.requests] = first + mine;
    }
  }
  __syncthreads();
}

// A workgroup's run of units. Workgroups go round the eight dies; neighbouring
// runs share a die, whose cache serves the tiles of query rows that read the
// same keys.
struct Run {
  int64_t wg, unit, end;
};
__device__ __forceinline__ int64_t units_of_run(int64_t total, int workgroups) {
  return (total + workgroups - 1) >> (31 - __builtin_clz(workgroups)); // a power of two
}
__device__ __forceinline__ Run my_run(const Schedule &sh) {
  const int64_t total = uniform64(sh.before[kScan]);
  const int64_t per = units_of_run(total, gridDim.x);
  Run r;
  r.wg = static_cast<int64_t>(blockIdx.x & 7u) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  r.wg = uniform64(r.wg);
  r.unit = uniform64(r.wg * per);
  r.end = uniform64(min(total, r.unit + per));
  return r;
}

// Partial sums of a part's rows: where dim d of row i lies. The shared kernel's
// lie as its lanes hold them, sixteen rows by sixteen dims, so that a store is
// one piece of memory.
template <int DP, int ROWS> __device__ __forceinline__ int part_at(int i, int d) {
  if constexpr (ROWS == 16)
    return i * DP + d;
  else
    return (i >> 4) * 16 * DP + (((d >> 4) * 4 + ((d >> 2) & 3)) * 16 + (i & 15)) * 4 + (d & 3);
}

// The part of an item that lies in a run: the units [s0, s1) of its `units`.
struct Item {
  int b, start, fresh, head, tile, cached, length, s0, s1, units;
  int reach;      // places of tokens: of the request, or those that its rows may see
  int edge, jump; // where places and tokens part, and by how much
  int position;   // of the first new token: the cached ones, of which the table may hold fewer
  int all_see;    // every row's window holds the tokens from here on
  template <int FORM> __device__ __forceinline__ int token(int place) const {
    return FORM == kWhole ? place : place < edge ? place : place + jump;
  }
  // Whether some rows' windows begin after the 32 tokens from x do.
  template <int FORM> __device__ __forceinline__ bool windowed(int x, int sinks) const {
    return FORM != kWhole && x < all_see && x + kTile > sinks;
  }
};
// Where the window of the j-th new token, at the d-th place after the cached ones, begins.
__device__ __forceinline__ int window_from(const AttendArgs &a, int position, int d) {
  const int64_t from = static_cast<int64_t>(position) + d - a.window + 1;
  return static_cast<int>(max(min(from, int64_t{1} << 30), int64_t{0}));
}
// The d of a row: the token's depth in its tree, or j. Of a mask's bits those of the
// request's `fresh` tokens count: the others are no tokens, and items are laid out
// for depths below fresh.
__device__ __forceinline__ int row_depth(const AttendArgs &a, int start, int fresh, int j) {
  if (!a.mask)
    return j;
  int n = 0;
  for (int w = 0, left = fresh; w < a.words && left > 0; ++w, left -= 64) {
    const uint64_t word = static_cast<uint64_t>(a.mask[(start + static_cast<int64_t>(j)) * a.words + w]);
    n += __builtin_popcountll(left >= 64 ? word : word & ((uint64_t{1} << left) - 1));
  }
  return max(n - 1, 0);
}
// Of the 32 tokens from x: the first ones, and those from `from` on.
__device__ __forceinline__ uint32_t window_sees(int x, int from, int sinks) {
  const int first = sinks - x, before = from - x;
  return (first >= 32 ? 0xffffffffu : first > 0 ? (1u << first) - 1u : 0u) |
         (before >= 32 ? 0u : before > 0 ? 0xffffffffu << before : 0xffffffffu);
}

template <int FORM, int ROWS, int UNIT>
__device__ __forceinline__ Item take(const AttendArgs &a, const Schedule &sh, Run &run) {
  int lo = 0, hi = kScan;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (uniform64(sh.before[mid]) <= run.unit)
      lo = mid;
    else
      hi = mid;
  }
  int b = lo * ((a.requests + kScan - 1) / kScan);
  int64_t at = uniform64(sh.before[lo]);
  Request r = attend_request<FORM, ROWS, UNIT>(a, b);
  for (;;) {
    const int64_t n = static_cast<int64_t>(head_items<ROWS>(a)) * r.tiles * r.units;
    if (run.unit < at + n)
      break;
    at += n;
    r = attend_request<FORM, ROWS, UNIT>(a, ++b);
  }
  Item i;
  i.b = uniform(b);
  at = uniform64(at);
  i.cached = uniform(r.cached);
  i.length = uniform(r.length);
  i.start = uniform(r.start);
  i.fresh = uniform(r.fresh);
  i.units = uniform(r.units);
  const int tiles = uniform(r.tiles);
  const int64_t item = uniform64(divide(run.unit - at, i.units));
  i.s0 = uniform(static_cast<int>(run.unit - at - item * i.units));
  i.s1 = uniform(static_cast<int>(min(static_cast<int64_t>(i.units), i.s0 + (run.end - run.unit))));
  i.head = uniform(static_cast<int>(divide(item, tiles)));
  i.tile = static_cast<int>(item - static_cast<int64_t>(i.head) * tiles);
  run.unit = uniform64(run.unit + i.s1 - i.s0);
  i.reach = i.length;
  i.edge = i.jump = i.all_see = i.position = 0;
  if constexpr (FORM != kWhole) {
    // the places of its first and last rows' tokens
    const int row0 = i.tile * ROWS;
    const int j0 = a.mask ? 0 : static_cast<int>(fdiv(static_cast<uint32_t>(row0), a.group));
    const int j1 = a.mask ? i.fresh - 1
                          : min(i.fresh - 1, static_cast<int>(fdiv(static_cast<uint32_t>(row0 + ROWS - 1), a.group)));
    if (j1 + 1 < i.length - i.cached)
      i.length = i.cached + j1 + 1;
    i.length = uniform(i.length);
    i.position = uniform(max(a.cached[b], 0));
    const int from = min(window_from(a, i.position, j0), i.length);
    i.all_see = uniform(min(window_from(a, i.position, j1), i.length));
    i.edge = uniform(edge_of(a, i.length));
    i.jump = uniform(max((from & ~(kTile - 1)) - i.edge, 0));
    i.reach = i.length - i.jump;
  }
  return i;
}

// What the j-th new token sees of the 32 tokens from `x`, as bits: all cached
// ones, and of the new ones those in its `mask` or, without one, up to itself.
__device__ __forceinline__ uint32_t sees(const Item &it, bool masked, int j, uint64_t mask, int x) {
  const int d = x - it.cached; // the first token's place among the new ones
  if (d + 32 <= 0)
    return 0xffffffffu;
  if (!masked) {
    const int n = j - d + 1;
    return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
  }
  const int old = d < 0 ? -d : 0; // cached tokens among the 32
  const uint64_t m = d <= 0 ? mask : d < 64 ? mask >> d : 0u;
  return static_cast<uint32_t>(m << old) | ((1u << old) - 1u);
}

// The same for the p-th query row of the item's request and key head, with a
// mask of any length.
__device__ __forceinline__ uint32_t row_sees(const AttendArgs &a, const Item &it, int p, int x) {
  const int j = static_cast<int>(fdiv(static_cast<uint32_t>(p), a.group));
  const int d = x - it.cached;
  if (!a.mask || d + 32 <= 0)
    return sees(it, false, j, 0u, x);
  if (j >= it.fresh)
    return 0u;
  const int64_t *mask = a.mask + (it.start + static_cast<int64_t>(j)) * a.words;
  const int from = d > 0 ? d : 0, word = from >> 6, sh = from & 63;
  uint64_t m = 0;
  if (word < a.words)
    m = static_cast<uint64_t>(mask[word]) >> sh;
  if (sh > 32 && word + 1 < a.words)
    m |= static_cast<uint64_t>(mask[word + 1]) << (64 - sh);
  const int old = d < 0 ? -d : 0;
  return static_cast<uint32_t>(m << old) | ((1u << old) - 1u);
}

// ------------------------------------------------------------ tiles

// Where the n-th 16-byte piece of a token's row lies in a tile of kTile rows of
// RB bytes: pieces are swapped by the token's number, so that sixteen lanes that
// read the same piece of sixteen tokens, or all pieces of one, meet no bank
// twice.
template <int RB> __device__ __forceinline__ int swap_of(int token) {
  constexpr int P = RB / 16;
  return P >= 16 ? token & 15 : (token / (16 / P)) & (P - 1);
}
template <int RB> __device__ __forceinline__ int piece(int token, int n) {
  return token * RB + (n ^ swap_of<RB>(token)) * 16;
}

// Eight tokens of one int8 dim: lane i of sixteen gives the address of eight
// dims of token i / 2, and gets dim i.
__device__ __forceinline__ u32x2 read_transposed8(uint32_t at) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) i32x2 *From;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(reinterpret_cast<From>(at)));
}

// Where a lane's reads of a tile begin: its first piece of a key, and of the
// values. Piece n + k of a token lies at the place of piece n with the bits of
// 16 k turned over (tiles lie at multiples of their tokens' bytes), and sixteen
// tokens on is the same piece: so all reads of a tile have one address each in
// registers outside the loop.
template <int DP, bool RAW> struct Reads {
  static constexpr int RB = DP * (RAW ? 1 : 2);
  uint32_t key, value;
  __device__ __forceinline__ explicit Reads(int lane) {
    const int c = lane & 15, g = lane >> 4;
    key = piece<RB>(c, g);
    if constexpr (RAW)
      value = piece<RB>(4 * g + ((c >> 1) & 3) + (c >> 3) * 16, 0) + (c & 1) * 8;
    else
      value = piece<RB>(4 * g + (c >> 2), (c & 3) >> 1) + (c & 1) * 8;
  }
};

// A tile's values as operands: at(e) has dim 16 e + lane % 16 of the lane's eight
// tokens. RAW: the tile holds int8. EARLY: all read at once, ahead of their use.
template <int T, int DP, bool RAW, bool EARLY> struct Values {
  static constexpr int E = DP / 16;
  uint32_t from;
  u32x2 lo[EARLY ? E : 1], hi[EARLY && !RAW ? E : 1];
  __device__ __forceinline__ u32x2 part(int e, int tile) const {
    if constexpr (RAW)
      return read_transposed8(from ^ (e * 16));
    else
      return read_transposed((from ^ (e * 32)) + tile * 16 * DP * 2);
  }
  __device__ __forceinline__ explicit Values(uint32_t from_) : from(from_) {
    if constexpr (EARLY) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        lo[e] = part(e, 0);
        if constexpr (!RAW)
          hi[e] = part(e, 1);
      }
      keep_order();
    }
  }
  __device__ __forceinline__ u32x4 at(int e) const {
    const u32x2 a = EARLY ? lo[e] : part(e, 0);
    if constexpr (RAW) {
      return widen8<T>(a.x, a.y);
    } else {
      const u32x2 b = EARLY ? hi[e] : part(e, 1);
      return u32x4{a.x, a.y, b.x, b.y};
    }
  }
};

template <int T> __device__ __forceinline__ bool finite16(uint32_t h) {
  constexpr uint32_t kExp = T == kF16 ? 0x7c00u : 0x7f80u;
  return (h & kExp) != kExp;
}

// Makes the values of a tile that no product may touch zero: of the tokens that
// are not `seen` everything, which may be anything, and, where the rows see
// different tokens (`mixed`), what is not finite: a product with a weight of
// zero would carry it over to rows that do not see it (Rows::add_odd puts it
// where it belongs). The NT tokens from `first`, by one wave; true if a token
// that is seen had such a value.
template <int T, int DP, int NT>
__device__ __forceinline__ bool clean(char *tv, int first, uint32_t seen, bool mixed, int lane) {
  constexpr int P = DP / 8;
  bool odd = false;
#pragma clang loop unroll(disable)
  for (int i = lane; i < NT * P; i += 64) {
    const int token = first + i / P;
    u32x4 *at = reinterpret_cast<u32x4 *>(tv + token * DP * 2 + (i % P) * 16);
    u32x4 v = *at;
    if (!(seen >> token & 1u)) {
      v = u32x4{0u, 0u, 0u, 0u};
    } else if (mixed) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const bool lo = finite16<T>(v[n]), hi = finite16<T>(v[n] >> 16);
        odd |= !lo || !hi;
        v[n] &= (lo ? 0xffffu : 0u) | (hi ? 0xffff0000u : 0u);
      }
    }
    *at = v;
  }
  return __any(odd);
}

// kBlocks: the scales of a tile's keys and values, of sixteen tokens each.
struct Scales {
  float key[2], value[2];
};

// A wave's query rows and their sums.
template <int FORM, int T, int DP, int RT, bool RAW, bool EARLY> struct Rows {
  static constexpr int E = DP / 16, QS = DP / 32;
  u32x4 q[RT][QS];
  float top[RT];     // reference maximum of a row's scaled scores
  float sum[RT];     // of its weights, over this lane's tokens; total(): over all
  f32x4 acc[RT][E];  // dims 16 e + 4 (lane / 16) + 0..3
  int place[RT];     // among the request's new tokens
  uint64_t mask[RT]; // of one word
  float scale;       // above zero: its sign is the queries'
  int words;         // of a mask; 0: none
  int from[FORM == kWhole ? 1 : RT]; // where a row's window begins
  int sinks;
  // kBlocks: the values' scales go into the weights of the second product. In f16
  // they go there over the largest that the row has seen so far, a power of two, of
  // which its sums are: else weights of up to 2^14 times a scale of four would be none.
  // For each row, since a page that it does not see may hold anything.
  static constexpr bool kOver = FORM == kBlocks && T == kF16;
  float back[kOver ? RT : 1]; // one over it: from 2^126, of the least normal number, to 2^-127
  __device__ __forceinline__ float whole(int t) const { return kOver ? 1.0f / back[kOver ? t : 0] : 1.0f; }

  __device__ __forceinline__ void start(const AttendArgs &a, const Item &it, int row0, int rows, float score_scale,
                                        int lane) {
    const int c = lane & 15, g = lane >> 4;
    // The maximum and the mask's -inf are those of unscaled scores, which goes for
    // a scale above zero alone: so a negative one turns the queries over, and zero
    // is the least normal number, by which no finite score reaches a bit of a weight.
    constexpr float kLeast = 1.17549435e-38f;
    const uint32_t sign = score_scale < 0.0f ? 0x80008000u : 0u;
    scale = fabsf(score_scale) < kLeast ? kLeast : fabsf(score_scale);
    words = a.mask ? a.words : 0;
    sinks = FORM == kWhole ? 0 : a.sinks;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if constexpr (kOver)
        back[t] = 0x1p126f;
      const uint32_t p = static_cast<uint32_t>(row0 + t * 16 + c);
      const uint32_t j = fdiv(p, a.group);
      place[t] = static_cast<int>(j);
      mask[t] = 0u;
      if (words == 1 && place[t] < it.fresh)
        mask[t] = static_cast<uint64_t>(a.mask[it.start + static_cast<int64_t>(j)]);
      if constexpr (FORM != kWhole)
        from[t] = place[t] < it.fresh ? window_from(a, it.position, row_depth(a, it.start, it.fresh, place[t])) : 0;
      const char *src = a.q + ((it.start + static_cast<int64_t>(j)) * a.q_row +
                               (static_cast<int64_t>(it.head) * a.group.d + (p - j * a.group.d)) * a.q_head) * 2;
#pragma unroll
      for (int s = 0; s < QS; ++s) {
        // the dims of contraction step s: those of a lane's piece of a key
        const int d = RAW ? (s >> 1) * 64 + g * 16 + (s & 1) * 8 : s * 32 + g * 8;
        q[t][s] = u32x4{0u, 0u, 0u, 0u};
        if (t * 16 + c < rows && d < a.dim)
          q[t][s] = load<u32x4>(src + d * 2);
        q[t][s] ^= sign;
      }
      top[t] = kNone;
      sum[t] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e)
        acc[t][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // Here, once: else the compiler, which cannot know in the loop whether the
    // queries have arrived, waits there for all loads in flight, every time.
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int s = 0; s < QS; ++s)
        asm volatile("" : "+v"(q[t][s]));
  }

  // Taking in a tile's 32 tokens from `x`, in three parts. `cut`: not every row
  // sees all of them, and the values are clean; `seen`: those inside the request
  // and on a page of the cache. One path, with little beside it that touches
  // the sums: where several meet, the compiler keeps the sums in several places.
  f32x4 s[RT][2];     // scores, unscaled
  u32x4 weights[RT];

  // from: the tile's place and the lane's first piece in it
  __device__ __forceinline__ void scores(uint32_t from) {
    constexpr int KR = RAW ? QS / 2 : QS; // reads of a token's key
    u32x4 k[2][KR];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < KR; ++i)
        k[n][i] = read16((from ^ (i * 64)) + n * 16 * DP * (RAW ? 1 : 2));
    keep_order(); // all reads on their way before the first is waited for
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
        s[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < QS; ++i) {
        u32x4 ki;
        if constexpr (RAW)
          ki = i & 1 ? widen8<T>(k[n][i >> 1].z, k[n][i >> 1].w) : widen8<T>(k[n][i >> 1].x, k[n][i >> 1].y);
        else
          ki = k[n][i];
#pragma unroll
        for (int t = 0; t < RT; ++t)
          s[t][n] = mfma<T>(ki, q[t][i], s[t][n]);
      }
    }
  }

  // The weights of a row, and their sum over the lane's tokens.
  __device__ __forceinline__ float weigh(int t, const float *value_scale) {
    float p[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[n][i] = __builtin_amdgcn_exp2f(s[t][n][i] * scale - top[t]);
      if constexpr (FORM == kBlocks) {
        const float f = value_scale[n];
        weights[t][n * 2] = pack16<T>(p[n][0] * f, p[n][1] * f);
        weights[t][n * 2 + 1] = pack16<T>(p[n][2] * f, p[n][3] * f);
      } else {
        weights[t][n * 2] = pack16<T>(p[n][0], p[n][1]);
        weights[t][n * 2 + 1] = pack16<T>(p[n][2], p[n][3]);
      }
    }
    return ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
  }

  // Weights go by the reference maximum, which moves only where some lane has
  // seen a score far above it: in a row's first tile and a few later ones. So
  // lanes compare theirs then and not at every tile.
  // kBlocks: the scales of the tile's keys and values, of sixteen tokens each.
  __device__ __forceinline__ void soften(const Item &it, int row0, int x, uint32_t seen, bool cut, int lane_,
                                         const Scales &tile) {
    constexpr float kBias = weight_bias<T>();
    float values[RT][2];
    if constexpr (FORM == kBlocks) {
      float v[2] = {tile.value[0], tile.value[1]};
#pragma unroll
      for (int n = 0; n < 2; ++n)
        if (!(seen >> (16 * n) & 0xffffu))
          v[n] = 0.0f; // of no token: may be anything
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        values[t][0] = v[0];
        values[t][1] = v[1];
#pragma unroll
        for (int n = 0; n < 2; ++n)
          s[t][n] *= tile.key[n];
      }
    }
    if (__builtin_expect(cut, 0)) {
      const int lane = anew(lane_), c = lane & 15, g = lane >> 4;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        uint32_t bits = seen & (words > 1 ? row_sees(args_again(), it, row0 + t * 16 + c, x)
                                          : sees(it, words == 1, place[t], mask[t], x));
        if constexpr (FORM != kWhole)
          bits &= window_sees(x, from[t], sinks);
        if constexpr (FORM == kBlocks)
#pragma unroll
          for (int n = 0; n < 2; ++n)
            values[t][n] = bits >> (16 * n) & 0xffffu ? values[t][n] : 0.0f;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(bits >> (n * 16 + 4 * g + i) & 1u))
              s[t][n][i] = -__builtin_inff();
      }
    }

    if constexpr (kOver) {
      bool larger = false;
#pragma unroll
      for (int t = 0; t < RT; ++t)
        larger |= fmaxf(fabsf(values[t][0]), fabsf(values[t][1])) * back[t] > 1.0f;
      if (__builtin_expect(__any(larger), 0)) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          // below 2^n, and at least half of it; 0: of no token that the row sees
          const float size = fmaxf(fabsf(values[t][0]), fabsf(values[t][1]));
          const int n = min(__builtin_amdgcn_frexp_expf(size), 127);
          const float next = size > 0.0f ? fminf(back[t], __builtin_amdgcn_ldexpf(1.0f, -n)) : back[t];
          const float shrink = next / back[t];
          back[t] = next;
#pragma unroll
          for (int e = 0; e < E; ++e)
            acc[t][e] *= shrink;
        }
      }
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int n = 0; n < 2; ++n)
          values[t][n] *= back[t];
    }

    float most[RT];
    bool above = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      most[t] = s[t][0][0];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          most[t] = fmaxf(most[t], s[t][n][i]);
      above |= most[t] * scale > top[t] + (kBias + kSlack);
    }
    if (__builtin_expect(__any(above), 0)) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const float next = fmaxf(top[t], max_over_groups(most[t]) * scale - kBias);
        const float shrink = __builtin_amdgcn_exp2f(top[t] - next);
        top[t] = next;
        sum[t] *= shrink;
#pragma unroll
        for (int e = 0; e < E; ++e)
          acc[t][e] *= shrink;
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
      sum[t] += weigh(t, values[t]);
  }

  __device__ __forceinline__ void add(const Values<T, DP, RAW, EARLY> &v) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const u32x4 ve = v.at(e);
#pragma unroll
      for (int t = 0; t < RT; ++t)
        acc[t][e] = mfma<T>(ve, weights[t], acc[t][e]);
    }
  }

  // tk, tv: the places of the tile's keys and values.
  __device__ __forceinline__ void step(const Item &it, int row0, int x, uint32_t seen, bool cut, uint32_t tk, uint32_t tv,
                                       const Reads<DP, RAW> &reads, int lane, const Scales &tile) {
    scores(tk + reads.key);
    const Values<T, DP, RAW, EARLY> v(tv + reads.value); // EARLY: they arrive during the softmax
    soften(it, row0, x, seen, cut, lane, tile);
    add(v);
  }

  __device__ __forceinline__ float total(int t) const {
    const float x = sum[t] + __shfl_xor(sum[t], 16);
    return x + __shfl_xor(x, 32);
  }

  // Gives `add` what clean() took out of the tiles at x0, x0 + pace, ... before
  // x_end: values that are not finite, of tokens that some rows see, times their
  // weights in those rows. Hardly ever; a dim at a time, from the cache, to
  // where the sums have been stored: they are not in registers here.
  template <class Add>
  __device__ __forceinline__ void add_odd(const Item &it, int row0, int rows, int x0, int x_end, int pace, int lane,
                                          Add add) const {
    const AttendArgs &a = args_again();
    const int c = lane & 15, g = lane >> 4;
    const int32_t *table = a.table + it.b * a.table_row;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int p = row0 + t * 16 + c;
      if (t * 16 + c >= rows)
        continue;
      const uint32_t j = fdiv(static_cast<uint32_t>(p), a.group);
      const char *q = a.q + ((it.start + static_cast<int64_t>(j)) * a.q_row +
                             (static_cast<int64_t>(it.head) * a.group.d + (p - j * a.group.d)) * a.q_head) * 2;
#pragma clang loop unroll(disable)
      for (int at0 = x0; at0 < x_end; at0 += pace) {
        const int x = it.token<FORM>(at0);
        if (x + kTile <= it.cached && !it.windowed<FORM>(x, sinks))
          continue;
        uint32_t sees = row_sees(a, it, p, x);
        if constexpr (FORM != kWhole)
          sees &= window_sees(x, from[t], sinks);
#pragma clang loop unroll(disable)
        for (int y = x; y < min(x + kTile, it.length); ++y) {
          const uint32_t at = fdiv(static_cast<uint32_t>(y), a.page), off = static_cast<uint32_t>(y) - at * a.page.d;
          const int id = table[at];
          if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.pages) || !(sees >> (y - x) & 1u))
            continue;
          const char *k = a.keys + it.head * a.key_head + id * a.key_page + off * a.key_slot;
          const char *v = a.values + it.head * a.value_head + id * a.value_page + off * a.value_slot;
          float score = 0.0f;
#pragma clang loop unroll(disable)
          for (int d = 0; d < a.dim; ++d)
            score += widen16<T>(load<uint16_t>(q + d * 2)) * widen16<T>(load<uint16_t>(k + d * 2));
          const float weight = __builtin_amdgcn_exp2f(score * a.scale - top[t]);
#pragma clang loop unroll(disable)
          for (int d = 4 * g; d < a.dim; d += (d & 3) == 3 ? 13 : 1) {
            const uint32_t h = load<uint16_t>(v + d * 2);
            if (!finite16<T>(h))
              add(t, d, weight * widen16<T>(h));
          }
        }
      }
    }
  }
};

// How a wave brings its tokens of a tile into shared memory: NT tokens from
// `first`, of every tile. Its tiles are PACE tokens apart.
template <int FORM, int T, bool I8, int DP, int SRC, int NT, bool RAW, int PACE> struct Loader {
  static constexpr int CELL = I8 ? 1 : 2;
  using Lanes = Share<DP, CELL, NT>;
  static constexpr int LB = Lanes::LB, TL = Lanes::TL, TPI = Lanes::TPI, LOADS = Lanes::LOADS;
  static constexpr bool EVEN = SRC != kStaged;             // pages of whole tiles of 16 tokens
  static constexpr int RB = DP * (RAW ? 1 : 2);            // bytes of a token in the tile

  const char *keys, *values;
  const int32_t *table;
  int64_t key_page, value_page;
  uint32_t key_slot, value_slot;
  int64_t key_slot64, value_slot64; // kStaged: of any size
  int edge, jump; // see Item
  const char *key_scale, *value_scale; // kBlocks: the head's
  uint32_t scale_page, scale_block;    // bytes
  FastDiv block;
  int length, pages, first, token, dim, cell_at, head_dims;
  uint32_t key_token, value_token; // kStagedEven: where the lane's token lies after the load's first
  bool full; // the head fills the tile's rows
  bool once; // one tile of query rows reads a key head
  FastDiv page;
  bool has;    // the lane's dims are the head's (all, or eight of an int8 load's)
  bool whole;  // all of them
  u32x4 stage[2][SRC == kAsync ? 1 : LOADS];
  uint32_t there; // loads that are a token's, by bit
  Scales fetched; // with them
  // kAsync: the lane's token of the first load in its group of sixteen, and its piece
  uint32_t key_lane, value_lane, place16;

  __device__ __forceinline__ Loader(const AttendArgs &a, int lane, int first_) {
    first = first_;
    token = lane / TL;
    dim = (lane % TL) * LB;
    key_page = a.key_page;
    key_slot = static_cast<uint32_t>(a.key_slot);
    value_page = a.value_page;
    value_slot = static_cast<uint32_t>(a.value_slot);
    key_slot64 = a.key_slot;
    value_slot64 = a.value_slot;
    head_dims = a.dim;
    full = a.dim == DP;
    once = a.once;
    pages = a.pages;
    page = a.page;
    if constexpr (FORM == kBlocks) {
      scale_page = a.scale_page;
      scale_block = a.scale_block;
      block = a.block;
    }
    has = dim < a.dim && Lanes::brings(lane);
    whole = dim + LB <= a.dim;
    cell_at = has ? dim * CELL : 0;
    there = 0u;
    key_token = static_cast<uint32_t>(Lanes::token(lane)) * key_slot;
    value_token = static_cast<uint32_t>(Lanes::token(lane)) * value_slot;
    key_lane = (token + (first & 15)) * key_slot;
    value_lane = (token + (first & 15)) * value_slot;
    place16 = ((dim / LB) ^ swap_of<RB>(first + token)) * 16;
  }
  __device__ __forceinline__ void item(const AttendArgs &a, const Item &it) {
    keys = a.keys + it.head * a.key_head;
    values = a.values + it.head * a.value_head;
    table = a.table + it.b * a.table_row;
    length = it.length;
    edge = it.edge;
    jump = it.jump;
    if constexpr (FORM == kBlocks) {
      key_scale = reinterpret_cast<const char *>(a.key_scale) + static_cast<uint64_t>(static_cast<uint32_t>(it.head)) * a.scale_head;
      value_scale = reinterpret_cast<const char *>(a.value_scale) + static_cast<uint64_t>(static_cast<uint32_t>(it.head)) * a.scale_head;
    }
  }
  __device__ __forceinline__ int token_of(int place) const {
    return FORM == kWhole ? place : place < edge ? place : place + jump;
  }

  __device__ __forceinline__ bool is_page(int id) const {
    return static_cast<uint32_t>(id) < static_cast<uint32_t>(pages);
  }
  // What the table says of the 16 tokens from x0 (past the length: -1); EVEN.
  // Nothing waits for it here.
  __device__ __forceinline__ int entry(int x0) const {
    return x0 < length ? scalar_load(table + fdiv(static_cast<uint32_t>(x0), page)) : -1;
  }
  // Where the 16-token groups of a wave's next kAhead tiles lie in the cache,
  // group g of them in lane g: one wave's worth of arithmetic, and two reads of a
  // lane a tile. The table's next entries come through shared memory like the
  // tiles: no wait, neither for them nor, as scalar loads would make it, for reads
  // of shared memory. kAsync, where there are tokens.
  static constexpr int kAhead = 32;
  static constexpr int GROUPS = NT > 16 ? 2 : 1; // that this wave brings of a tile
  struct Next {
    int64_t key[GROUPS], value[GROUPS];
    uint32_t on; // which of the tile's halves lie on a page
  };
  int64_t key_at, value_at;
  uint64_t paged; // the groups that lie on a page
  uint32_t room;  // [2][64] of this wave
  uint32_t scale_room; // kBlocks: [2][2][64], keys' and values' scales of the same groups
  __device__ __forceinline__ int group_at(int x, int lane) const {
    return token_of(x + (lane >> 1) * PACE) + (lane & 1) * 16;
  }
  __device__ __forceinline__ uint32_t entry_at(int x, int lane) const {
    return fdiv(static_cast<uint32_t>(min(group_at(x, lane), length - 1)), page);
  }
  // Past the length: the last page's first tokens; of no page: the first one's,
  // which nothing will see.
  // kBlocks: the groups' scales go on their way to shared memory, ahead of all of
  // the tiles that they are of, whose arrival is waited for: in this order.
  __device__ __forceinline__ void take_entries(int id, int x, int lane, uint32_t half) {
    const bool is = is_page(id);
    const int x0 = group_at(x, lane);
    const uint32_t off = is && x0 < length ? static_cast<uint32_t>(x0) - fdiv(static_cast<uint32_t>(x0), page) * page.d : 0u;
    const uint64_t at = is ? static_cast<uint32_t>(id) : 0u;
    key_at = static_cast<int64_t>(at * key_page + static_cast<uint64_t>(off) * key_slot);
    value_at = static_cast<int64_t>(at * value_page + static_cast<uint64_t>(off) * value_slot);
    paged = __ballot(is);
    if constexpr (FORM == kBlocks) {
      const uint32_t scale_at = static_cast<uint32_t>(at) * scale_page + fdiv(off, block) * scale_block;
      load_async4(key_scale, scale_at, scale_room + half * 2);
      load_async4(value_scale, scale_at, scale_room + half * 2 + 256);
    }
  }
  // kBlocks: the n-th tile's scales, once it has arrived.
  __device__ __forceinline__ Scales scales(int n) const {
    Scales t = {};
    if constexpr (FORM == kBlocks) {
      typedef const __attribute__((address_space(3))) f32x2 *Pair;
      const uint32_t from = scale_room + (n / kAhead % 2) * 512 + (n % kAhead) * 8;
      const f32x2 k = *reinterpret_cast<Pair>(from), v = *reinterpret_cast<Pair>(from + 256);
      t.key[0] = k.x, t.key[1] = k.y, t.value[0] = v.x, t.value[1] = v.y;
    }
    return t;
  }
  // The first entries, and the next on their way.
  __device__ __forceinline__ void first_entries(int x, int count, int lane) {
    const int id = table[entry_at(x, lane)];
    if (count > kAhead)
      load_async4(table, entry_at(x + kAhead * PACE, lane) * 4u, room + 256);
    take_entries(id, x, lane, 0);
  }
  // The n-th tile, at x; called for one after the other.
  __device__ __forceinline__ Next look(int n, int x, int lane) {
    if (n > 0 && n % kAhead == 0) {
      const uint32_t half = n / kAhead % 2 * 256;
      take_entries(*reinterpret_cast<const __attribute__((address_space(3))) int *>(room + half + lane * 4), x, lane, half);
      load_async4(table, entry_at(x + kAhead * PACE, lane) * 4u, room + (half ^ 256));
    }
    const int g = n % kAhead * 2;
    Next t;
#pragma unroll
    for (int h = 0; h < GROUPS; ++h) {
      const int from = g + (GROUPS == 2 ? h : first >> 4);
      t.key[h] = of_lane(key_at, from);
      t.value[h] = of_lane(value_at, from);
    }
    t.on = static_cast<uint32_t>(paged >> g) & 3u;
    return t;
  }
  // Which of the 32 tokens from x are there.
  __device__ __forceinline__ uint32_t seen(int x, uint32_t on) const {
    const int n = max(length - x, 0);
    const uint32_t in = n >= 32 ? 0xffffffffu : (1u << n) - 1u;
    return in & ((on & 1u ? 0xffffu : 0u) | (on & 2u ? 0xffff0000u : 0u));
  }

  // kAsync: the wave's tokens of a tile.
  template <bool ONCE> __device__ __forceinline__ void send(const Next &next, uint32_t to_k, uint32_t to_v) const {
#pragma unroll
    for (int h = 0; h < GROUPS; ++h) {
      const char *k = keys + next.key[h], *v = values + next.value[h];
#pragma unroll
      for (int i = 0; i < LOADS / GROUPS; ++i) {
        const int t = (GROUPS == 2 ? h * 16 : first) + i * TPI;
        // the piece that lies at this lane's place
        const uint32_t n16 = LOADS == 1 ? place16 : place16 ^ (swap_of<RB>((h * 16 + i * TPI) & 15) * 16);
        const char *ki = k + static_cast<uint64_t>(i * TPI) * key_slot, *vi = v + static_cast<uint64_t>(i * TPI) * value_slot;
        if ((NT >= TPI || token < NT) && (full || static_cast<int>(n16) < head_dims * CELL)) {
          load_async<ONCE>(ki, key_lane + n16, to_k + t * RB);
          load_async<ONCE>(vi, value_lane + n16, to_v + t * RB);
        }
      }
    }
  }

  // The wave's tokens of an int8 tile, keys and values; and as T in another tile.
  // Lanes that bring none read another place of the tile.
  struct Codes {
    u32x4 part[2][LOADS];
  };
  __device__ __forceinline__ Codes codes(uint32_t from, int lane) const {
    Codes c;
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        c.part[kv][i] = read16(from + kv * kTile * DP + piece<RB>((first + i * TPI + token) % kTile, lane % TL));
    return c;
  }
  __device__ __forceinline__ void widen(const Codes &c, uint32_t to, int lane) const {
    constexpr int WB = DP * 2;
    typedef __attribute__((address_space(3))) u32x4 *Place;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int t = first + i * TPI + token, n = lane % TL;
      if (NT >= TPI || token < NT)
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const u32x4 b = c.part[kv][i];
          const uint32_t at = to + kv * kTile * WB;
          *reinterpret_cast<Place>(at + piece<WB>(t, 2 * n)) = widen8<T>(b.x, b.y);
          *reinterpret_cast<Place>(at + piece<WB>(t, 2 * n + 1)) = widen8<T>(b.z, b.w);
        }
    }
  }

  // Through registers: the wave's tokens of the tile at x.
  __device__ __forceinline__ void fetch(int place) {
    const int x = token_of(place);
    there = 0u;
    if constexpr (FORM == kBlocks) { // pages are of whole blocks, and blocks of sixteen tokens
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int x0 = uniform(x + 16 * h), id = entry(x0);
        const uint32_t off = static_cast<uint32_t>(x0) - fdiv(static_cast<uint32_t>(x0), page) * page.d;
        const uint32_t at = is_page(id) ? static_cast<uint32_t>(id) * scale_page + fdiv(off, block) * scale_block : 0u;
        fetched.key[h] = scalar_load(reinterpret_cast<const float *>(key_scale + at));
        fetched.value[h] = scalar_load(reinterpret_cast<const float *>(value_scale + at));
      }
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int t0 = first + i * TPI;
      const int x0 = x + t0 + (EVEN ? 0 : token);
      int64_t id = -1;
      if constexpr (EVEN) {
        id = entry(x + (t0 & ~15));
      } else if (x0 < length && has) {
        id = table[fdiv(static_cast<uint32_t>(x0), page)];
      }
      id = is_page(static_cast<int>(id)) ? id : -1;
      if (id >= 0 && has && x + t0 + token < length)
        there |= 1u << i;
      const uint32_t off = id >= 0 ? static_cast<uint32_t>(x0) - fdiv(static_cast<uint32_t>(x0), page) * page.d : 0u;
      id = id >= 0 ? id : 0; // none: the first page, and zeros in its place
      const char *k = keys + id * key_page + off * key_slot64, *v = values + id * value_page + off * value_slot64;
      if constexpr (EVEN) {
        k += key_token + cell_at;
        v += value_token + cell_at;
      } else {
        k += cell_at;
        v += cell_at;
      }
      if (I8 && !whole) { // eight dims, or none
        const u32x2 hk = load<u32x2>(k), hv = load<u32x2>(v);
        stage[0][i] = u32x4{hk.x, hk.y, 0u, 0u};
        stage[1][i] = u32x4{hv.x, hv.y, 0u, 0u};
      } else {
        stage[0][i] = load<u32x4>(k);
        stage[1][i] = load<u32x4>(v);
      }
    }
  }
  __device__ __forceinline__ void put(char *tk, char *tv) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int t = first + i * TPI + token;
      const bool in = there >> i & 1u;
      if (NT >= TPI || token < NT)
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          char *to = kv ? tv : tk;
          const u32x4 b = in ? stage[kv][i] : u32x4{0u, 0u, 0u, 0u};
          if constexpr (I8 && !RAW) {
            *reinterpret_cast<u32x4 *>(to + piece<RB>(t, dim / 8)) = widen8<T>(b.x, b.y);
            *reinterpret_cast<u32x4 *>(to + piece<RB>(t, dim / 8 + 1)) = widen8<T>(b.z, b.w);
          } else {
            *reinterpret_cast<u32x4 *>(to + piece<RB>(t, dim / LB)) = b;
          }
        }
    }
  }
  // The wave's tokens that are there, by their place among its NT.
  __device__ __forceinline__ uint32_t tokens_there() const {
    uint32_t bits = 0u;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      uint64_t b = __ballot(dim == 0 && (there >> i & 1u)); // a lane of each token
#pragma unroll
      for (int t = 0; t < (TPI < NT ? TPI : NT); ++t)
        bits |= static_cast<uint32_t>(b >> (t * TL) & 1u) << (i * TPI + t);
    }
    return bits;
  }
};

// ---------------------------------------------------------- up to 16 rows

template <int FORM, int T, bool I8, int DP, int SRC, int UNIT>
__global__ __launch_bounds__(64 * turn_waves(DP), turn_workgroups(DP, I8, SRC == kAsync) == kMostWorkgroups ? 2 : 1)
void k_attend_turns(AttendArgs a) {
  constexpr int W = turn_waves(DP), STEP = turn_unit(DP), ROWS = 16, E = DP / 16;
  constexpr int TILE = kTile * DP * (I8 ? 1 : 2);
  constexpr int RING = SRC == kAsync ? 2 : 1; // tiles of a wave
  using Load = Loader<FORM, T, I8, DP, SRC, kTile, I8, STEP>;
  __shared__ int entries[SRC == kAsync ? W : 1][2][64];
  __shared__ float block_scales[FORM == kBlocks && SRC == kAsync ? W : 1][2][2][64];

  __shared__ Schedule schedule;
  constexpr int SUMS = W * 16 * (DP + 4) * sizeof(float); // the waves', at the end
  __shared__ __attribute__((aligned(16))) char room[W * RING * 2 * TILE > SUMS ? W * RING * 2 * TILE : SUMS];
  char(*tiles)[RING][2][TILE] = reinterpret_cast<char(*)[RING][2][TILE]>(room);
  __shared__ float row_max[W][ROWS], row_sum[W][ROWS];

  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  Load load(a, lane, 0);
  load.room = place(reinterpret_cast<const char *>(&entries[SRC == kAsync ? wave : 0][0][0]));
  if constexpr (FORM == kBlocks)
    load.scale_room = place(reinterpret_cast<const char *>(&block_scales[SRC == kAsync ? wave : 0][0][0][0]));
  Rows<FORM, T, DP, 1, I8, DP <= 128 && (I8 || SRC == kAsync)> r;
  const Reads<DP, I8> reads(lane);
  if (UNIT == kWholeUnit)
    zero_unowned(a);
  add_up<FORM, ROWS, UNIT>(a, schedule);
  Run run = my_run(schedule);

  while (run.unit < run.end) {
    const Item it = take<FORM, ROWS, UNIT>(args_again(), schedule, run);
    const int row0 = it.tile * ROWS;
    const int rows = it.fresh * static_cast<int>(args_again().group.d) - row0; // of this tile and later ones
    load.item(args_again(), it);
    const int x_end = min(it.s1 * UNIT, it.reach), x0 = it.s0 * UNIT + wave * kTile;
    const int count = x0 < x_end ? (x_end - x0 + STEP - 1) / STEP : 0; // this wave's tiles
    bool odd = false;
    auto start = [&] {
      const AttendArgs &b = args_again();
      r.start(b, it, row0, rows, I8 && FORM != kBlocks ? b.scale * b.key_scale[it.head] : b.scale, lane);
    };
    const uint32_t at = place(tiles[wave][0][0]);
    auto take_in = [&](int x, uint32_t seen, bool cut, int slot, const Scales &tile) {
      if (!I8 && __builtin_expect(cut, 0)) // what int8 holds is finite
        odd |= clean<T, DP, kTile>(tiles[wave][slot][1], 0, seen, x + kTile > it.cached || it.windowed<FORM>(x, r.sinks), lane);
      r.step(it, row0, x, seen, cut, at + slot * 2 * TILE, at + slot * 2 * TILE + TILE, reads, lane, tile);
    };

    if constexpr (SRC == kAsync) {
      if (!load.full) // places past the head's dims: no load writes them
        for (int i = lane * 16; i < RING * 2 * TILE; i += 64 * 16)
          *reinterpret_cast<u32x4 *>(&tiles[wave][0][0][0] + i) = u32x4{0u, 0u, 0u, 0u};
      shared_done();
      uint32_t on = 0u; // of the tiles on their way: their halves on a page
      auto send = [&](const typename Load::Next &next, int slot, int place) {
        load.template send<true>(next, at + slot * 2 * TILE, at + slot * 2 * TILE + TILE);
        on |= next.on << (2 * place);
      };
      if (count > 0)
        load.first_entries(x0, count, lane);
      start(); // the queries arrive while the table does
#pragma clang loop unroll(disable)
      for (int i = 0; i < min(count, RING); ++i)
        send(load.look(i, x0 + i * STEP, lane), i, i);
      typename Load::Next then = {}; // the next tile to send
      if (count > 0)
        then = load.look(RING, x0 + RING * STEP, lane);
      int x = x0;
      int slot = 0;
#pragma clang loop unroll(disable)
      for (int n = 0; n < count; ++n, x += STEP) {
        if (n + RING <= count)
          arrived<(RING - 1) * 2 * Load::LOADS>();
        else
          arrived<0>();
        const int xt = it.token<FORM>(x);
        const bool cut = (on & 3u) != 3u || xt + kTile > it.cached || it.windowed<FORM>(xt, r.sinks);
        take_in(xt, cut ? load.seen(xt, on) : 0xffffffffu, cut, slot, load.scales(n));
        shared_done(); // its place is free
        on >>= 2;
        if (n + RING < count)
          send(then, slot, RING - 1);
        then = load.look(n + RING + 1, x + (RING + 1) * STEP, lane);
        slot = slot + 1 == RING ? 0 : slot + 1;
      }
      arrived<0>(); // the last entries, wanted or not
    } else {
      start();
      char *tk = tiles[wave][0][0], *tv = tiles[wave][0][1];
      int x = x0;
      if (count > 0)
        load.fetch(x);
      for (int n = 0; n < count; ++n, x += STEP) {
        load.put(tk, tv);
        const uint32_t seen = load.tokens_there();
        const Scales tile = load.fetched;
        if (n + 1 < count)
          load.fetch(x + STEP);
        const int xt = it.token<FORM>(x);
        take_in(xt, seen, seen != 0xffffffffu || xt + kTile > it.cached || it.windowed<FORM>(xt, r.sinks), 0, tile);
      }
    }

    // ---- the waves' sums, where their tiles were
    float(*sums)[16][DP + 4] = reinterpret_cast<float(*)[16][DP + 4]>(room);
    const float sum = r.total(0);
    if (g == 0) {
      row_max[wave][c] = r.top[0];
      row_sum[wave][c] = sum;
    }
    __syncthreads();
    {
      float most = kNone;
#pragma unroll
      for (int w = 0; w < W; ++w)
        most = fmaxf(most, row_max[w][c]);
      const float f = __builtin_amdgcn_exp2f(r.top[0] - most) * r.whole(0);
      if (c < rows)
#pragma unroll
        for (int e = 0; e < E; ++e)
          *reinterpret_cast<f32x4 *>(&sums[wave][c][e * 16 + 4 * g]) = r.acc[0][e] * f;
      if (!I8 && __builtin_expect(odd, 0))
        r.add_odd(it, row0, rows, x0, x_end, STEP, lane, [&](int, int d, float v) { sums[wave][c][d] += v * f; });
    }
    __syncthreads();
    constexpr int DIMS = 16 * DP / (64 * W); // of a thread: sixteen rows over the workgroup
    const int i = tid / (DP / DIMS), d0 = (tid % (DP / DIMS)) * DIMS;
    if (i < rows) {
      const AttendArgs &a = args_again();
      float m = kNone, l = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w)
        m = fmaxf(m, row_max[w][i]);
#pragma unroll
      for (int w = 0; w < W; ++w)
        l += row_sum[w][i] * __builtin_amdgcn_exp2f(row_max[w][i] - m);
      const bool all = it.s0 == 0 && it.s1 == it.units;
      const uint32_t p = static_cast<uint32_t>(row0 + i);
      const uint32_t j = fdiv(p, a.group);
      const int64_t row = it.start + static_cast<int64_t>(j);
      const int64_t qh = static_cast<int64_t>(it.head) * a.group.d + (p - j * a.group.d);
      const int64_t part = (run.wg * 2 + (it.s0 == 0 ? 1 : 0)) * ROWS + i;
      const float f = finish(l, I8 && FORM != kBlocks ? a.value_scale[it.head] : 1.0f);
#pragma unroll
      for (int d = 0; d < DIMS; d += 4) {
        f32x4 o = *reinterpret_cast<const f32x4 *>(&sums[0][i][d0 + d]);
#pragma unroll
        for (int w = 1; w < W; ++w)
          o += *reinterpret_cast<const f32x4 *>(&sums[w][i][d0 + d]);
        if (!all) {
          *reinterpret_cast<f32x4 *>(a.partial + (part - i) * DP + part_at<DP, ROWS>(i, d0 + d)) = o;
        } else if (d0 + d < a.dim) {
          o *= f;
          store(a.out + (row * a.out_row + qh * a.out_head + d0 + d) * 2,
                u32x2{pack16<T>(o[0], o[1]), pack16<T>(o[2], o[3])});
        }
      }
      if (d0 == 0) {
        if (!all) {
          a.stats[part * 2] = m;
          a.stats[part * 2 + 1] = l;
        } else if (a.lse) {
          a.lse[row * a.heads + qh] = log_sum(m, l);
        }
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------- up to four rows, four heads at a time

// The same where a token's heads lie side by side: each wave has a head of its own,
// so that what the four read of a token is one piece of memory, 512 bytes for int8
// heads of 128. Nothing is added up between waves.
template <int T, int DP, int UNIT> __global__ __launch_bounds__(256, 2) void k_attend_quads(AttendArgs a) {
  constexpr int W = 4, ROWS = kQuadRows, E = DP / 16, TILE = kTile * DP, RING = 2;
  using Load = Loader<kBlocks, T, true, DP, kAsync, kTile, true, kTile>;
  __shared__ int entries[W][2][64];
  __shared__ float block_scales[W][2][2][64];
  __shared__ Schedule schedule;
  __shared__ __attribute__((aligned(16))) char tiles[W][RING][2][TILE];

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  Load load(a, lane, 0);
  load.room = place(reinterpret_cast<const char *>(&entries[wave][0][0]));
  load.scale_room = place(reinterpret_cast<const char *>(&block_scales[wave][0][0][0]));
  Rows<kBlocks, T, DP, 1, true, true> r;
  const Reads<DP, true> reads(lane);
  const uint32_t at = place(tiles[wave][0][0]);
  if (!load.full) // places past the head's dims: no load writes them
    for (int i = lane * 16; i < RING * 2 * TILE; i += 64 * 16)
      *reinterpret_cast<u32x4 *>(&tiles[wave][0][0][0] + i) = u32x4{0u, 0u, 0u, 0u};
  shared_done();
  if (UNIT == kWholeUnit)
    zero_unowned(a);
  add_up<kBlocks, ROWS, UNIT>(a, schedule);
  Run run = my_run(schedule);

  while (run.unit < run.end) {
    Item it = take<kBlocks, ROWS, UNIT>(args_again(), schedule, run);
    it.head = it.head * 4 + wave;
    const int row0 = it.tile * ROWS;
    const int rows = min(it.fresh * static_cast<int>(args_again().group.d) - row0, ROWS);
    load.item(args_again(), it);
    const int x0 = it.s0 * UNIT, x_end = min(it.s1 * UNIT, it.reach);
    const int count = x0 < x_end ? (x_end - x0 + kTile - 1) / kTile : 0;
    uint32_t on = 0u; // of the tiles on their way: their halves on a page
    auto send = [&](const typename Load::Next &next, int slot, int place) {
      load.template send<true>(next, at + slot * 2 * TILE, at + slot * 2 * TILE + TILE);
      on |= next.on << (2 * place);
    };
    if (count > 0)
      load.first_entries(x0, count, lane);
    r.start(args_again(), it, row0, rows, args_again().scale, lane); // the queries arrive while the table does
#pragma clang loop unroll(disable)
    for (int i = 0; i < min(count, RING); ++i)
      send(load.look(i, x0 + i * kTile, lane), i, i);
    typename Load::Next then = {}; // the next tile to send
    if (count > 0)
      then = load.look(RING, x0 + RING * kTile, lane);
    int x = x0, slot = 0;
#pragma clang loop unroll(disable)
    for (int n = 0; n < count; ++n, x += kTile) {
      if (n + RING <= count)
        arrived<(RING - 1) * 2 * Load::LOADS>();
      else
        arrived<0>();
      const int xt = it.token<kBlocks>(x);
      const bool cut = (on & 3u) != 3u || xt + kTile > it.cached || it.windowed<kBlocks>(xt, r.sinks);
      r.step(it, row0, xt, cut ? load.seen(xt, on) : 0xffffffffu, cut, at + slot * 2 * TILE, at + slot * 2 * TILE + TILE, reads,
             lane, load.scales(n));
      shared_done(); // its place is free
      on >>= 2;
      if (n + RING < count)
        send(then, slot, RING - 1);
      then = load.look(n + RING + 1, x + (RING + 1) * kTile, lane);
      slot = slot + 1 == RING ? 0 : slot + 1;
    }
    arrived<0>(); // the last entries, wanted or not

    const AttendArgs &b = args_again();
    const float sum = r.total(0), over = r.whole(0);
    if (c < rows) {
      if (it.s0 == 0 && it.s1 == it.units) {
        const uint32_t p = static_cast<uint32_t>(row0 + c);
        const uint32_t j = fdiv(p, b.group);
        const int64_t row = it.start + static_cast<int64_t>(j);
        const int64_t qh = static_cast<int64_t>(it.head) * b.group.d + (p - j * b.group.d);
        const float f = finish(sum, 1.0f) * over;
        char *dst = b.out + (row * b.out_row + qh * b.out_head + 4 * g) * 2;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e * 16 + 4 * g < b.dim) {
            const f32x4 o = r.acc[0][e] * f;
            store(dst + e * 32, u32x2{pack16<T>(o[0], o[1]), pack16<T>(o[2], o[3])});
          }
        if (b.lse && g == 0)
          b.lse[row * b.heads + qh] = log_sum(r.top[0], sum);
      } else {
        const int64_t part = (run.wg * 2 + (it.s0 == 0 ? 1 : 0)) * 16 + wave * ROWS + c;
#pragma unroll
        for (int e = 0; e < E; ++e)
          *reinterpret_cast<f32x4 *>(b.partial + part * DP + e * 16 + 4 * g) = r.acc[0][e] * over;
        if (g == 0) {
          b.stats[part * 2] = r.top[0];
          b.stats[part * 2 + 1] = sum;
        }
      }
    }
  }
}

// ---------------------------------------------------------- more rows

template <int FORM, int T, bool I8, int DP, int RT, int W, int SRC>
__global__ __launch_bounds__(64 * W, 2) void k_attend_shared(AttendArgs a) {
  constexpr int ROWS = 16 * RT * W, E = DP / 16, UNIT = kSharedUnit;
  constexpr int TILE = kTile * DP * 2;
  // int8 on its way by itself: a ring of tiles as they lie in the cache, of which a
  // wave widens the tokens that it has brought, into the other of two tiles
  constexpr bool WIDEN = I8 && SRC == kAsync;
  // tiles at a time: 64 KiB for each four waves
  constexpr int RING = SRC != kAsync || WIDEN ? 2 : 16 * 1024 * W / (2 * TILE) < 8 ? 16 * 1024 * W / (2 * TILE) : 8;
  constexpr int RAW = WIDEN ? (DP <= 128 ? 5 : 2) : 1; // tiles of int8
  using Load = Loader<FORM, T, I8, DP, SRC, kTile / W, WIDEN, kTile>;
  __shared__ int entries[SRC == kAsync ? W : 1][2][64];
  __shared__ float block_scales[FORM == kBlocks && SRC == kAsync ? W : 1][2][2][64];
  __shared__ __attribute__((aligned(16))) char raw[RAW][2][WIDEN ? kTile * DP : 16];

  __shared__ Schedule schedule;
  __shared__ __attribute__((aligned(16))) char tiles[RING][2][TILE];
  __shared__ uint8_t tokens[2][W]; // kStaged: each wave's tokens that are there
  __shared__ int odd_of[2];        // clean() found something, in every other item

  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  Load load(a, lane, wave * (kTile / W));
  load.room = place(reinterpret_cast<const char *>(&entries[SRC == kAsync ? wave : 0][0][0]));
  if constexpr (FORM == kBlocks)
    load.scale_room = place(reinterpret_cast<const char *>(&block_scales[SRC == kAsync ? wave : 0][0][0][0]));
  // A tile's values are read ahead of the softmax, where the registers hold them:
  // 77 us against 81 for 8 requests of 256 rows over up to 8192 tokens of 8 key
  // heads of 128, 280 against 287 up to 32768 (the fastest of 40). The same for the
  // next tile's keys was slower (81).
  constexpr bool EARLY = DP <= 128 && (I8 || SRC == kAsync);
  Rows<FORM, T, DP, RT, false, EARLY> r;
  if (tid < 2)
    odd_of[tid] = 0;
  add_up<FORM, ROWS, UNIT>(a, schedule);
  Run run = my_run(schedule);
  const Reads<DP, false> reads(lane);
  if (SRC == kAsync && a.dim < DP) // places past the head's dims: no load writes them
    for (int i = tid * 16; i < RING * 2 * TILE; i += 64 * W * 16)
      *reinterpret_cast<u32x4 *>(&tiles[0][0][0] + i) = u32x4{0u, 0u, 0u, 0u};
  if (WIDEN && a.dim < DP)
    for (int i = tid * 16; i < static_cast<int>(sizeof(raw)); i += 64 * W * 16)
      *reinterpret_cast<u32x4 *>(&raw[0][0][0] + i) = u32x4{0u, 0u, 0u, 0u};

  for (int turn = 0; run.unit < run.end; turn ^= 1) {
    const Item it = take<FORM, ROWS, UNIT>(args_again(), schedule, run);
    int &odd = odd_of[turn];
    const int row0 = (it.tile * W + wave) * 16 * RT;                // the wave's first
    const int rows = it.fresh * static_cast<int>(args_again().group.d) - row0; // and how many from there
    load.item(args_again(), it);
    const int x0 = it.s0 * UNIT, x_end = min(it.s1 * UNIT, it.reach);
    const int count = x0 < x_end ? (x_end - x0 + kTile - 1) / kTile : 0;
    // this wave's tokens of a tile that it has brought, before the others may read them
    auto clean_own = [&](int x, uint32_t seen, bool cut, int slot) {
      if (!I8 && __builtin_expect(cut, 0) &&
          clean<T, DP, kTile / W>(tiles[slot][1], wave * (kTile / W), seen,
                                  x + kTile > it.cached || it.windowed<FORM>(x, args_again().sinks), lane) &&
          lane == 0)
        odd = 1;
    };
    const uint32_t at = place(tiles[0][0]);
    __syncthreads(); // the tiles are free, and everybody has looked at the last item's `odd`
    if (tid == 0)
      odd_of[turn ^ 1] = 0;

    // A wave without rows brings its tokens all the same. Loops of their own, so
    // that in none the sums meet a way round them.
    auto work = [&](auto busy) {
      constexpr bool BUSY = decltype(busy)::value;
      auto take_in = [&](int x, uint32_t seen, bool cut, int slot, const Scales &tile) {
        if constexpr (BUSY)
          r.step(it, row0, x, seen, cut, at + slot * 2 * TILE, at + slot * 2 * TILE + TILE, reads, lane, tile);
      };
      auto start = [&] {
        const AttendArgs &b = args_again();
        r.start(b, it, row0, rows, I8 && FORM != kBlocks ? b.scale * b.key_scale[it.head] : b.scale, lane);
      };

      if constexpr (WIDEN) {
        uint32_t on = 0u; // of this tile and those on their way: their halves on a page
        const uint32_t raw_at = place(raw[0][0]);
        auto send = [&](const typename Load::Next &next, int slot, int place) {
          const uint32_t to = raw_at + slot * 2 * (kTile * DP);
          if (load.once)
            load.template send<true>(next, to, to + kTile * DP);
          else
            load.template send<false>(next, to, to + kTile * DP);
          on |= next.on << (2 * place);
        };
        if (count > 0)
          load.first_entries(x0, count, lane);
        if constexpr (BUSY)
          start();
#pragma clang loop unroll(disable)
        for (int i = 0; i < min(count, RAW); ++i)
          send(load.look(i, x0 + i * kTile, lane), i, i);
        typename Load::Next then = {}; // the next tile to send
        if (count > 0)
          then = load.look(RAW, x0 + RAW * kTile, lane);
        int slot = 0; // of the tile that is widened next, the n-th
        auto read = [&](int n) {
          if (n + RAW - 1 < count)
            arrived<(RAW - 1) * 2 * Load::LOADS>();
          else
            arrived<0>();
          return load.codes(raw_at + slot * 2 * (kTile * DP), lane);
        };
        auto widen = [&](const typename Load::Codes &codes, int n) {
          load.widen(codes, at + (n & 1) * 2 * TILE, lane); // which have been read: their place is free
          if (n + RAW < count)
            send(then, slot, RAW);
          then = load.look(n + RAW + 1, x0 + (n + RAW + 1) * kTile, lane);
          slot = slot + 1 == RAW ? 0 : slot + 1;
        };
        if (count > 0)
          widen(read(0), 0);
#pragma clang loop unroll(disable)
        for (int n = 0; n < count; ++n) {
          const int xt = it.token<FORM>(x0 + n * kTile);
          const bool cut = (on & 3u) != 3u || xt + kTile > it.cached || it.windowed<FORM>(xt, args_again().sinks);
          const uint32_t seen = cut ? load.seen(xt, on) : 0xffffffffu;
          on >>= 2;
          meet(); // the tile is whole, and everybody has read the one before
          typename Load::Codes codes;
          if (n + 1 < count)
            codes = read(n + 1); // on their way while this tile is worked on
          take_in(xt, seen, cut, n & 1, load.scales(n));
          if (n + 1 < count)
            widen(codes, n + 1);
        }
        arrived<0>(); // the last entries, wanted or not
      } else if constexpr (SRC == kAsync) {
        uint32_t on = 0u; // of the tiles on their way: their halves on a page
        auto send = [&](const typename Load::Next &next, int slot, int place) {
          const uint32_t to = at + slot * 2 * TILE;
          if (load.once)
            load.template send<true>(next, to, to + TILE);
          else
            load.template send<false>(next, to, to + TILE);
          on |= next.on << (2 * place);
        };
        if (count > 0)
          load.first_entries(x0, count, lane);
        if constexpr (BUSY)
          start(); // the queries arrive while the table does
#pragma clang loop unroll(disable)
        for (int i = 0; i < min(count, RING - 1); ++i)
          send(load.look(i, x0 + i * kTile, lane), i, i);
        typename Load::Next then = {}; // the next tile to send
        if (count > 0)
          then = load.look(RING - 1, x0 + (RING - 1) * kTile, lane);
        int x = x0, slot = 0;
        const int last = x0 + (count - 1) * kTile;
#pragma clang loop unroll(disable)
        for (int n = 0; x <= last; ++n, x += kTile) {
          // this wave's part of the tile is there, then everybody's, and everybody
          // has read the tile before, whose place the next takes
          if (x + (RING - 2) * kTile <= last)
            arrived<(RING - 2) * 2 * Load::LOADS>();
          else
            arrived<0>();
          const int xt = it.token<FORM>(x);
          const bool cut = (on & 3u) != 3u || xt + kTile > it.cached || (FORM != kWhole && it.windowed<FORM>(xt, args_again().sinks));
          const uint32_t seen = cut ? load.seen(xt, on) : 0xffffffffu;
          clean_own(xt, seen, cut, slot);
          meet();
          on >>= 2;
          if (x + (RING - 1) * kTile <= last)
            send(then, slot == 0 ? RING - 1 : slot - 1, RING - 2);
          take_in(xt, seen, cut, slot, Scales{});
          then = load.look(n + RING, x + RING * kTile, lane);
          slot = slot + 1 == RING ? 0 : slot + 1;
        }
        arrived<0>(); // the last entries, wanted or not
      } else {
        if constexpr (BUSY)
          start();
        int x = x0;
        auto put = [&](int slot) {
          load.put(tiles[slot][0], tiles[slot][1]);
          const uint32_t t = load.tokens_there();
          if (lane == 0)
            tokens[slot][wave] = static_cast<uint8_t>(t);
          // the tile put: this one or the next
          const int xp = it.token<FORM>(x + (slot == ((x - x0) / kTile & 1) ? 0 : kTile));
          const uint32_t seen = t << (wave * (kTile / W)) | ~(((1u << (kTile / W)) - 1u) << (wave * (kTile / W)));
          clean_own(xp, seen, seen != 0xffffffffu || xp + kTile > it.cached || it.windowed<FORM>(xp, args_again().sinks), slot);
        };
        Scales tile = {}, next_tile = {}; // of this tile and of the next, which has been put
        if (count > 0) {
          load.fetch(x);
          next_tile = load.fetched;
          put(0);
        }
        if (count > 1)
          load.fetch(x + kTile);
        for (int n = 0; n < count; ++n, x += kTile) {
          const int slot = n & 1;
          __syncthreads();
          uint32_t seen = 0u;
#pragma unroll
          for (int w = 0; w < W; ++w)
            seen |= static_cast<uint32_t>(tokens[slot][w]) << (w * (kTile / W));
          seen = static_cast<uint32_t>(uniform(static_cast<int>(seen)));
          tile = next_tile;
          if (n + 1 < count) {
            next_tile = load.fetched;
            put(slot ^ 1);
          }
          if (n + 2 < count)
            load.fetch(x + 2 * kTile);
          const int xt = it.token<FORM>(x);
          take_in(xt, seen, seen != 0xffffffffu || xt + kTile > it.cached || it.windowed<FORM>(xt, args_again().sinks), slot, tile);
        }
      }

      __syncthreads();
      if constexpr (!BUSY)
        return;
      const bool any_odd = !I8 && odd;
      // ---- every wave's rows are its own
      const AttendArgs &b = args_again();
      const bool whole = it.s0 == 0 && it.s1 == it.units;
      const int ln = anew(lane), c = ln & 15, g = ln >> 4;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const float sum = r.total(t);
        if (t * 16 + c >= rows)
          continue;
        if (whole) {
          const uint32_t p = static_cast<uint32_t>(row0 + t * 16 + c);
          const uint32_t j = fdiv(p, b.group);
          const int64_t row = it.start + static_cast<int64_t>(j);
          const int64_t qh = static_cast<int64_t>(it.head) * b.group.d + (p - j * b.group.d);
          const float f = finish(sum, I8 && FORM != kBlocks ? b.value_scale[it.head] : 1.0f) * r.whole(t);
          char *dst = b.out + (row * b.out_row + qh * b.out_head + 4 * g) * 2;
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (e * 16 + 4 * g < b.dim) {
              const f32x4 o = r.acc[t][e] * f;
              store(dst + e * 32, u32x2{pack16<T>(o[0], o[1]), pack16<T>(o[2], o[3])});
            }
          if (b.lse && g == 0)
            b.lse[row * b.heads + qh] = log_sum(r.top[t], sum);
        } else {
          const int64_t part = (run.wg * 2 + (it.s0 == 0 ? 1 : 0)) * ROWS + wave * 16 * RT + t * 16 + c;
          float *dst = b.partial + (part - c) * DP + part_at<DP, ROWS>(c, 4 * g);
#pragma unroll
          for (int e = 0; e < E; ++e)
            *reinterpret_cast<f32x4 *>(dst + e * 256) = r.kOver ? r.acc[t][e] * r.whole(t) : r.acc[t][e];
          if (g == 0) {
            b.stats[part * 2] = r.top[t];
            b.stats[part * 2 + 1] = sum;
          }
        }
      }
      if (__builtin_expect(any_odd, 0)) {
        r.add_odd(it, row0, rows, x0, x_end, kTile, lane, [&](int t, int d, float v) {
          const AttendArgs &b = args_again();
          const int i = wave * 16 * RT + t * 16 + c;
          if (!whole) {
            b.partial[(run.wg * 2 + (it.s0 == 0 ? 1 : 0)) * ROWS * DP + part_at<DP, ROWS>(i, d)] += v;
            return;
          }
          // what is rounded is finite, and what comes to it is not
          const uint32_t p = static_cast<uint32_t>(it.tile * ROWS + i);
          const uint32_t j = fdiv(p, b.group);
          char *o = b.out + ((it.start + static_cast<int64_t>(j)) * b.out_row +
                             (static_cast<int64_t>(it.head) * b.group.d + (p - j * b.group.d)) * b.out_head + d) * 2;
          store(o, static_cast<uint16_t>(pack16<T>(widen16<T>(relx::load<uint16_t>(o)) + v, 0.0f)));
        });
      }
    };
    if (rows > 0) // the same for the whole wave
      work(std::true_type());
    else
      work(std::false_type());
  }
}

// The rows of items that lie in several workgroups' runs: their partial sums,
// added up; and zeros for the rows of no request. A column of blocks takes the
// rows of a request, PHASES waves a piece of 64 times four dims at a time. It is
// bound by how long a read takes of what other dies have written: so all parts
// are on their way at once, where there are many by sharing them among waves.
template <int FORM, int T, bool I8, int DP, int ROWS, int UNIT, int PHASES>
__global__ __launch_bounds__(PHASES == 1 ? 256 : 64 * PHASES) void k_attend_join(AttendArgs a) {
  constexpr bool LANED = ROWS > 16;                   // see part_at
  constexpr int N = LANED ? 16 : 256 / DP;            // rows of a piece
  constexpr int E = LANED ? DP / 16 : 1;              // pieces of N rows
  constexpr int WAVES = PHASES == 1 ? 4 : PHASES;     // of a block
  constexpr int PIECES = WAVES / PHASES;              // of a block
  __shared__ f32x4 sums[PHASES][64];
  __shared__ float tops[PHASES][64], totals[PHASES][64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), phase = PHASES == 1 ? 0 : wave;
  const int c = LANED ? lane & 15 : lane / (DP / 4);
  const int b = blockIdx.x;
  if (b == a.requests) { // rows of no request: where there is none, all
    int r0 = 0, r1 = 0;
    if (a.requests > 0) {
      r0 = min(max(a.starts[0], 0), a.rows);
      r1 = min(max(a.starts[a.requests], r0), a.rows);
    }
    const int64_t none = static_cast<int64_t>(r0 + a.rows - r1) * a.heads;
    for (int64_t i = static_cast<int64_t>(blockIdx.y) * WAVES + wave; i < none; i += static_cast<int64_t>(gridDim.y) * WAVES) {
      int64_t row = i / a.heads;
      const int64_t qh = i - row * a.heads;
      row += row < r0 ? 0 : r1 - r0;
      for (int d = lane; d < a.dim; d += 64)
        store(a.out + (row * a.out_row + qh * a.out_head + d) * 2, static_cast<uint16_t>(0));
      if (a.lse && lane == 0)
        a.lse[row * a.heads + qh] = -__builtin_inff();
    }
    return;
  }
  const Request r = attend_request<FORM, ROWS, UNIT>(a, b);
  const int64_t total = a.schedule[a.requests], first = a.schedule[b];
  const int64_t per = units_of_run(total, a.workgroups);
  const int64_t rows = static_cast<int64_t>(r.fresh) * a.group.d;
  const int groups = static_cast<int>((rows + N - 1) / N); // of a key head's rows
  const int64_t count = static_cast<int64_t>(groups) * a.kv_heads * E;
  for (int64_t i = static_cast<int64_t>(blockIdx.y) * PIECES + (PHASES == 1 ? wave : 0); i < count;
       i += static_cast<int64_t>(gridDim.y) * PIECES) {
    const int e = static_cast<int>(i % E), head = static_cast<int>(divide(i / E, groups));
    const int row0 = static_cast<int>(i / E - static_cast<int64_t>(head) * groups) * N;
    const int d = LANED ? e * 16 + (lane >> 4) * 4 : lane % (DP / 4) * 4;
    const int64_t u0 = first + (static_cast<int64_t>(ROWS == kQuadRows ? head >> 2 : head) * r.tiles + row0 / ROWS) * r.units;
    const int64_t w0 = uniform64(divide(u0, static_cast<int>(per)));
    const int64_t w1 = uniform64(divide(u0 + r.units - 1, static_cast<int>(per)));
    if (w0 == w1)
      continue; // written whole
    const bool valid = row0 + c < rows;
    float top = kNone, sum = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    int64_t w = w0 + phase;
    auto take = [&](auto many) { // the next parts of this phase
      constexpr int MANY = decltype(many)::value;
      f32x4 o[MANY];
      f32x2 ml[MANY];
      float most = top;
#pragma unroll
      for (int k = 0; k < MANY; ++k) {
        // a run that begins inside the item left its part in its first place,
        // the run in which the item begins in its second
        const int64_t wk = min(w + k * PHASES, w1);
        const int64_t at = ROWS == kQuadRows ? (wk * 2 + (wk == w0 ? 1 : 0)) * 16 + head % 4 * ROWS + row0 % ROWS
                                             : (wk * 2 + (wk == w0 ? 1 : 0)) * ROWS + row0 % ROWS;
        ml[k] = *reinterpret_cast<const f32x2 *>(a.stats + (at + c) * 2);
        o[k] = *reinterpret_cast<const f32x4 *>(a.partial + at * DP + (e * 64 + lane) * 4);
      }
#pragma unroll
      for (int k = 0; k < MANY; ++k)
        most = fmaxf(most, ml[k].x);
      const float f = __builtin_amdgcn_exp2f(top - most);
      top = most;
      sum *= f;
      acc *= f;
#pragma unroll
      for (int k = 0; k < MANY; ++k)
        if (w + k * PHASES <= w1) {
          const float fk = __builtin_amdgcn_exp2f(ml[k].x - top);
          sum += ml[k].y * fk;
          acc += o[k] * fk;
        }
      w += MANY * PHASES;
    };
    if (valid) {
      while (w + 4 * PHASES <= w1)
        take(std::integral_constant<int, 8>());
      if (w <= w1)
        take(std::integral_constant<int, 4>());
    }
    if constexpr (PHASES > 1) {
      sums[phase][lane] = acc;
      tops[phase][lane] = top;
      totals[phase][lane] = sum;
      __syncthreads();
      if (phase == 0) {
#pragma unroll
        for (int k = 1; k < PHASES; ++k)
          top = fmaxf(top, tops[k][lane]);
        float f = __builtin_amdgcn_exp2f(tops[0][lane] - top);
        sum *= f;
        acc *= f;
#pragma unroll
        for (int k = 1; k < PHASES; ++k) {
          f = __builtin_amdgcn_exp2f(tops[k][lane] - top);
          sum += totals[k][lane] * f;
          acc += sums[k][lane] * f;
        }
      }
    }
    if (valid && phase == 0) {
      const uint32_t p = static_cast<uint32_t>(row0 + c);
      const uint32_t j = fdiv(p, a.group);
      const int64_t row = r.start + static_cast<int64_t>(j);
      const int64_t qh = static_cast<int64_t>(head) * a.group.d + (p - j * a.group.d);
      acc *= finish(sum, I8 && FORM != kBlocks ? a.value_scale[head] : 1.0f);
      if (d < a.dim)
        store(a.out + (row * a.out_row + qh * a.out_head + d) * 2,
              u32x2{pack16<T>(acc[0], acc[1]), pack16<T>(acc[2], acc[3])});
      if (a.lse && d == 0)
        a.lse[row * a.heads + qh] = log_sum(top, sum);
    }
    if constexpr (PHASES > 1)
      __syncthreads();
  }
}

template <int FORM, int T, bool I8, int DP, int ROWS, int UNIT>
hipError_t attend_start(const void *kernel, int threads, const AttendArgs &args, const AttendPlan &p,
                        hipStream_t s) {
  AttendArgs a = args;
  void *pa[] = {&a};
  hipError_t e = hipSuccess;
  if (a.requests > 0)
    e = hipLaunchKernel(kernel, dim3(static_cast<uint32_t>(p.workgroups)), dim3(static_cast<uint32_t>(threads)), pa, 0, s);
  if (e != hipSuccess || (UNIT == kWholeUnit && a.requests > 0))
    return e;
  // A wave for every piece of an even batch, within 2^16 blocks a request; eight
  // where an item lies in more than eight runs, on average: 6.7 us against 10.0
  // for 64 parts of 64 rows (14 MB), but 28 against 8.9 for five of 256 (31 MB).
  const int64_t requests = std::max(a.requests, 1);
  const int64_t rows = (a.rows + requests - 1) / requests * a.group.d;
  const int64_t n = ROWS > 16 ? 16 : 256 / DP;
  const int64_t pieces = (rows + n - 1) / n * a.kv_heads * (ROWS > 16 ? DP / 16 : 1);
  const int64_t items = (rows + ROWS - 1) / ROWS * a.kv_heads * requests;
  const bool many = p.workgroups > 8 * items;
  return hipLaunchKernel(many ? reinterpret_cast<const void *>(k_attend_join<FORM, T, I8, DP, ROWS, UNIT, 8>)
                              : reinterpret_cast<const void *>(k_attend_join<FORM, T, I8, DP, ROWS, UNIT, 1>),
                         dim3(static_cast<uint32_t>(a.requests) + 1,
                              static_cast<uint32_t>(std::min<int64_t>(many ? pieces : (pieces + 3) / 4, 65535))),
                         dim3(many ? 512 : 256), pa, 0, s);
}

template <int FORM, int T, bool I8, int DP, int RT, int W, int SRC>
hipError_t attend_start_shared(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  return attend_start<FORM, T, I8, DP, 16 * RT * W, kSharedUnit>(
      reinterpret_cast<const void *>(k_attend_shared<FORM, T, I8, DP, RT, W, SRC>), 64 * W, a, p, s);
}

template <int FORM, int T, bool I8, int DP, int SRC>
hipError_t attend_shared(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  if constexpr (DP < 256) { // 32 rows of a wave with a head of 256 would not fit its registers
    if (p.rows == 128)
      return attend_start_shared<FORM, T, I8, DP, 2, 4, SRC>(a, p, s);
    if (p.rows == 256)
      return attend_start_shared<FORM, T, I8, DP, 2, 8, SRC>(a, p, s);
  }
  return attend_start_shared<FORM, T, I8, DP, 1, 4, SRC>(a, p, s);
}

template <int FORM, int T, bool I8, int DP>
hipError_t attend_source(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  if constexpr (FORM == kBlocks && DP <= 128)
    if (p.quads)
      return p.whole ? attend_start<FORM, T, I8, DP, kQuadRows, kWholeUnit>(
                           reinterpret_cast<const void *>(k_attend_quads<T, DP, kWholeUnit>), 256, a, p, s)
                     : attend_start<FORM, T, I8, DP, kQuadRows, kQuadUnit>(
                           reinterpret_cast<const void *>(k_attend_quads<T, DP, kQuadUnit>), 256, a, p, s);
  if constexpr (FORM != kWhole)
    if (p.whole)
      return attend_start<FORM, T, I8, DP, 16, kWholeUnit>(
          reinterpret_cast<const void *>(k_attend_turns<FORM, T, I8, DP, kAsync, kWholeUnit>), 64 * turn_waves(DP), a, p, s);
  if (p.rows == 16)
    return attend_start<FORM, T, I8, DP, 16, turn_unit(DP)>(
        p.async ? reinterpret_cast<const void *>(k_attend_turns<FORM, T, I8, DP, kAsync, turn_unit(DP)>)
                : reinterpret_cast<const void *>(k_attend_turns<FORM, T, I8, DP, kStaged, turn_unit(DP)>),
        64 * turn_waves(DP), a, p, s);
  // int8 is widened once for all waves, on its way through registers
  if constexpr (FORM == kBlocks)
    if (p.async)
      return attend_shared<FORM, T, I8, DP, kAsync>(a, p, s);
  if constexpr (I8)
    return p.even ? attend_shared<FORM, T, I8, DP, kStagedEven>(a, p, s) : attend_shared<FORM, T, I8, DP, kStaged>(a, p, s);
  else
    return p.async ? attend_shared<FORM, T, I8, DP, kAsync>(a, p, s) : attend_shared<FORM, T, I8, DP, kStaged>(a, p, s);
}

template <int FORM, int T, bool I8>
hipError_t attend_width(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  switch (p.width) {
  case 64:
    return attend_source<FORM, T, I8, 64>(a, p, s);
  case 128:
    return attend_source<FORM, T, I8, 128>(a, p, s);
  default:
    return attend_source<FORM, T, I8, 256>(a, p, s);
  }
}

} // namespace
} // namespace relx
