// k_attend.h - attention of a step's query rows over a paged cache (device
// templates; instantiated in k_attend_f16.hip and k_attend_bf16.hip).
//
// One pass over the keys and values with the running maximum and sum of the
// softmax. The query rows of a request that share a key head (its new tokens
// times the heads of the group) are the columns of matrix products; a wave
// keeps 16, 32 or 64 of them with their sums in registers and takes 32 tokens
// at a time:
//
//   S^T = K Q^T    16 tokens x 16 rows per product, dims contracted
//   O^T += V^T P^T 16 dims x 16 rows per product, 32 tokens contracted
//
// The layout of S^T in the registers (lane: row = lane % 16, tokens
// 4 (lane / 16) + 0..3 of each of two token tiles) is the layout of the
// second product's operand if its contracted tokens are numbered
// 8 (lane / 16) + 4 tile + 0..3, so the weights go from one product to the
// next without leaving their lane. Keys and values come from the cache
// straight into registers: a lane's 16 bytes of a key row are its operand, and
// of values it loads 16 bytes (for a head of 128) from each of its eight
// tokens and transposes the 8 x 8 block in place with byte permutes; the
// dims that a product's rows stand for are numbered to suit. No shared memory
// is touched between the products.
//
// The tokens of a wave's tiles lie `kUnit` apart: four waves take 128 tokens
// in turn and add up at the end. The work of a call is the list of these
// units over (request, key head, tile of query rows), cut into equal runs, one
// per workgroup; an item that lies in several runs leaves partial sums that
// k_attend_join adds up. So one long context fills the card as well as many
// short ones do, and uneven lengths cost nothing.
#pragma once

#include <algorithm>
#include <type_traits>
#include <utility>

#include "attention.h"
#include "index.h"

namespace relx {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kAttendWaves = 4;
constexpr int kStep = 32;                       // tokens of a wave at a time
constexpr int kUnit = kStep * kAttendWaves;     // tokens of a workgroup at a time
constexpr int kScan = 64 * kAttendWaves;        // threads
// Where a row's running maximum starts: finite, so that a difference with a
// masked score's -inf stays -inf.
constexpr float kNone = -1e30f;
// A row's reference maximum moves only once a score exceeds it by this many
// powers of two; until then weights up to 2^8 are summed as they are.
constexpr float kSlack = 8.0f;

template <class T> struct __attribute__((packed)) Loose { T v; };
template <class T> __device__ __forceinline__ T load(const char *p) {
  return reinterpret_cast<const Loose<T> *>(p)->v;
}
template <class T> __device__ __forceinline__ void store(char *p, const T &v) {
  reinterpret_cast<Loose<T> *>(p)->v = v;
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

template <int T> __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (T == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two values rounded to nearest even. The weights of the second product are
// rounded so too: unbiased, and no coarser than the result's own type.
template <int T> __device__ __forceinline__ uint32_t pack16(float x, float y) {
  const f32x2 v = {x, y};
  if constexpr (T == kF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
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
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}

// acc += weights times values, dims e, e + 1, ... of each lane's.
template <int T, int E, class F, class V, int... I>
__device__ __forceinline__ void add_dims(f32x4 (&acc)[E], u32x4 weights, const F &operand, const V &v,
                                         std::integer_sequence<int, I...>) {
  ((acc[I] = mfma<T>(operand(v, std::integral_constant<int, I>{}), weights, acc[I])), ...);
}
template <int T, int E, class F, class V>
__device__ __forceinline__ void add_values(f32x4 (&acc)[E], u32x4 weights, const F &operand, const V &v) {
  add_dims<T, E>(acc, weights, operand, v, std::make_integer_sequence<int, E>{});
}

// The same for one row (the lanes that are `mine`), of the tokens that `sees`
// has: the others' values do not enter.
template <int T, int E, int I, class F, class V>
__device__ __forceinline__ void add_row_dim(f32x4 (&acc)[E], u32x4 weights, const F &operand, const V &v,
                                            u32x4 sees, bool mine) {
  const u32x4 o = operand(v, std::integral_constant<int, I>{}) & sees;
  const f32x4 one = mfma<T>(o, weights, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
  for (int i = 0; i < 4; ++i)
    acc[I][i] += mine ? one[i] : 0.0f;
}
template <int T, int E, class F, class V, int... I>
__device__ __forceinline__ void add_row_dims(f32x4 (&acc)[E], u32x4 weights, const F &operand, const V &v,
                                             u32x4 sees, bool mine, std::integer_sequence<int, I...>) {
  (add_row_dim<T, E, I>(acc, weights, operand, v, sees, mine), ...);
}
template <int T, int E, class F, class V>
__device__ __forceinline__ void add_row(f32x4 (&acc)[E], u32x4 weights, const F &operand, const V &v,
                                        u32x4 sees, bool mine) {
  add_row_dims<T, E>(acc, weights, operand, v, sees, mine, std::make_integer_sequence<int, E>{});
}

// ------------------------------------------------------------ the schedule

struct Request {
  int64_t cached, length; // tokens in the cache before the step, and with it
  int start, fresh;       // its rows
  int tiles;              // tiles of query rows
  int64_t units;          // of one item
};

template <int ROWS>
__device__ __forceinline__ Request attend_request(const AttendArgs &a, int b) {
  Request r;
  const int s = min(max(a.starts[b], 0), a.rows), e = min(max(a.starts[b + 1], s), a.rows);
  r.start = s;
  r.fresh = e - s;
  const int64_t room = a.pages > 0 ? static_cast<int64_t>(a.columns) * a.page.d : 0;
  const int64_t c = max(a.cached[b], 0);
  r.cached = min(c, room);
  r.length = min(c + r.fresh, room);
  const int64_t q = static_cast<int64_t>(r.fresh) * a.group.d;
  r.tiles = static_cast<int>((q + ROWS - 1) / ROWS);
  r.units = max((r.length + kUnit - 1) / kUnit, int64_t{1});
  return r;
}

template <int ROWS>
__device__ __forceinline__ int64_t request_units(const AttendArgs &a, int b) {
  const Request r = attend_request<ROWS>(a, b);
  return static_cast<int64_t>(a.kv_heads) * r.tiles * r.units;
}

// ------------------------------------------------------------ the kernel

template <int T, bool I8, int DP, int RT, bool FAST>
__global__ __launch_bounds__(kScan, RT <= 2 && DP <= 128 ? 2 : 1) void k_attend(AttendArgs a) {
  constexpr int ROWS = 16 * RT;
  constexpr int E = DP / 16;              // dims of a lane's values
  constexpr int CELL = I8 ? 1 : 2;        // bytes of a cache element
  constexpr int KB = 16 / CELL;           // dims of a key load
  constexpr int KS = DP / (4 * KB);       // key loads of a token
  constexpr int QS = DP / 32;             // contraction steps
  constexpr int VW = E * CELL / 4;        // words of a lane's values of a token
  constexpr float kBias = T == kF16 ? 6.0f : 0.0f; // weights up to 2^14 in f16: small ones keep their bits

  __shared__ int64_t before[kScan + 1];
  __shared__ int64_t wave_units[kAttendWaves];
  __shared__ float sums[kAttendWaves][16][DP + 4];
  __shared__ float row_max[kAttendWaves][ROWS], row_sum[kAttendWaves][ROWS];

  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int c = lane & 15, g = lane >> 4;

  // every workgroup adds up the requests' units for itself
  const int run = (a.requests + kScan - 1) / kScan;
  {
    const int b0 = min(tid * run, a.requests), b1 = min(b0 + run, a.requests);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b)
      mine += request_units<ROWS>(a, b);
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t v = __shfl_up(upto, o);
      if (lane >= o)
        upto += v;
    }
    if (lane == 63)
      wave_units[wave] = upto;
    __syncthreads();
    int64_t first = upto - mine;
    for (int w = 0; w < wave; ++w)
      first += wave_units[w];
    before[tid] = first;
    if (tid == kScan - 1)
      before[kScan] = first + mine;
    if (blockIdx.x == 0) { // for the join
      int64_t at = first;
      for (int b = b0; b < b1; ++b) {
        a.schedule[b] = at;
        at += request_units<ROWS>(a, b);
      }
      if (tid == kScan - 1)
        a.schedule[a.requests] = first + mine;
    }
    __syncthreads();
  }
  const int64_t total = uniform64(before[kScan]);
  const int64_t per = (total + gridDim.x - 1) / gridDim.x;
  // Workgroups go round the eight dies; neighbouring runs share a die, whose
  // cache serves the tiles of query rows that read the same keys.
  const uint32_t die = blockIdx.x & 7u;
  const int64_t wg = static_cast<int64_t>(die) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  int64_t unit = wg * per;
  const int64_t unit_end = min(total, unit + per);

  while (unit < unit_end) {
    // the item that holds `unit`
    int lo = 0, hi = kScan;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (uniform64(before[mid]) <= unit)
        lo = mid;
      else
        hi = mid;
    }
    int b = lo * run;
    int64_t at = uniform64(before[lo]);
    Request r = attend_request<ROWS>(a, b);
    for (;;) {
      const int64_t n = static_cast<int64_t>(a.kv_heads) * r.tiles * r.units;
      if (unit < at + n)
        break;
      at += n;
      r = attend_request<ROWS>(a, ++b);
    }
    b = uniform(b);
    at = uniform64(at);
    const int64_t cached = uniform64(r.cached), length = uniform64(r.length);
    const int start = uniform(r.start), fresh = uniform(r.fresh), tiles = uniform(r.tiles);
    const int64_t units = uniform64(r.units);
    const int64_t item = (unit - at) / units;
    const int64_t s0 = unit - at - item * units;
    const int64_t s1 = min(units, s0 + (unit_end - unit));
    const int head = static_cast<int>(item / tiles);
    const int tile = static_cast<int>(item - static_cast<int64_t>(head) * tiles);
    unit += s1 - s0;

    // ---- queries: this lane's row of each tile
    const int rows = fresh * static_cast<int>(a.group.d) - tile * ROWS; // of this tile and later ones
    u32x4 q[RT][QS];
    int row_j[RT]; // the row's token among the new ones
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int i = t * 16 + c;
      const uint32_t p = static_cast<uint32_t>(tile * ROWS + i);
      const uint32_t j = fdiv(p, a.group);
      row_j[t] = static_cast<int>(j);
      const char *src = a.q + ((start + static_cast<int64_t>(j)) * a.q_row +
                               (static_cast<int64_t>(head) * a.group.d + (p - j * a.group.d)) * a.q_head) * 2;
#pragma unroll
      for (int s = 0; s < QS; ++s) {
        // the dims of contraction step s: those of this lane's keys
        const int d = I8 ? (s >> 1) * 64 + g * 16 + (s & 1) * 8 : s * 32 + g * 8;
        q[t][s] = u32x4{0u, 0u, 0u, 0u};
        if (i < rows && d < a.dim)
          q[t][s] = load<u32x4>(src + d * 2);
      }
    }

    const float scale = I8 ? a.scale * a.key_scale[head] : a.scale;
    float top[RT], weight[RT];
    f32x4 acc[RT][E];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      top[t] = kNone;
      weight[t] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e)
        acc[t][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const char *keys = a.keys + head * a.key_head;
    const char *values = a.values + head * a.value_head;
    const int32_t *table = a.table + b * a.table_row;
    const int key_lane = FAST ? c * static_cast<int>(a.key_slot) + g * 16 : 0;
    int value_lane[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      value_lane[i] = FAST ? (4 * g + i) * static_cast<int>(a.value_slot) + c * E * CELL : 0;
    const int value_dim = c * E < a.dim ? c * E : 0; // dims past the head's: any of its bytes

    // Where the 32 tokens from `x` lie. FAST: pages hold whole tiles of 16
    // tokens, so a tile's page is the same for all lanes; else lane l knows
    // token l's. `seen`: tokens inside the request and on a page of the cache.
    struct Where {
      const char *k[2], *v[2];
      int64_t k_off, v_off;
      uint32_t seen;
    };
    auto find = [&](int64_t x) {
      Where w;
      w.seen = 0u;
      if constexpr (FAST) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int64_t x0 = x + t * 16;
          const int n = static_cast<int>(min(max(length - x0, int64_t{0}), int64_t{16}));
          int id = 0;
          uint32_t off = 0;
          if (n > 0) {
            const uint32_t p = fdiv(static_cast<uint32_t>(x0), a.page);
            off = static_cast<uint32_t>(x0) - p * a.page.d;
            id = uniform(table[p]);
            if (static_cast<uint32_t>(id) < static_cast<uint32_t>(a.pages))
              w.seen |= ((1u << n) - 1u) << (16 * t);
            else
              id = 0;
          }
          w.k[t] = keys + id * a.key_page + off * a.key_slot;
          w.v[t] = values + id * a.value_page + off * a.value_slot;
        }
      } else {
        const int64_t x0 = x + (lane & 31);
        w.k_off = w.v_off = 0;
        bool ok = x0 < length;
        if (ok) {
          const uint32_t p = fdiv(static_cast<uint32_t>(x0), a.page);
          const uint32_t off = static_cast<uint32_t>(x0) - p * a.page.d;
          const int id = table[p];
          ok = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.pages);
          if (ok) {
            w.k_off = id * a.key_page + off * a.key_slot;
            w.v_off = id * a.value_page + off * a.value_slot;
          }
        }
        w.seen = static_cast<uint32_t>(__ballot(ok));
      }
      return w;
    };
    auto load_keys = [&](const Where &w, u32x4 (&k)[2][KS]) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const char *p = FAST ? w.k[t] + key_lane : keys + __shfl(w.k_off, t * 16 + c);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          if constexpr (FAST) {
            k[t][s] = load<u32x4>(p + s * 64);
          } else {
            const int d = s * 4 * KB + g * KB;
            if (d + KB <= a.dim) {
              k[t][s] = load<u32x4>(p + d * CELL);
            } else { // past the head's end (an int8 head may end inside a load)
              k[t][s] = u32x4{0u, 0u, 0u, 0u};
              if (I8 && d < a.dim) {
                const u32x2 h = load<u32x2>(p + d);
                k[t][s].x = h.x;
                k[t][s].y = h.y;
              }
            }
          }
        }
      }
    };
    auto load_values = [&](const Where &w, uint32_t (&v)[8][VW]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const char *p = FAST ? w.v[i >> 2] + value_lane[i & 3]
                             : values + __shfl(w.v_off, (i >> 2) * 16 + 4 * g + (i & 3)) + value_dim * CELL;
        if constexpr (VW == 1) {
          v[i][0] = load<uint32_t>(p);
        } else if constexpr (VW == 2) {
          const u32x2 h = load<u32x2>(p);
          v[i][0] = h.x;
          v[i][1] = h.y;
        } else {
          // a head of fewer than DP dims may end inside a lane's sixteen
          const bool in = FAST || value_dim + 8 < a.dim;
          if (I8 && !in) {
            const u32x2 h = load<u32x2>(p);
            v[i][0] = h.x;
            v[i][1] = h.y;
            v[i][2] = v[i][3] = 0u;
            continue;
          }
#pragma unroll
          for (int n = 0; n < VW; n += 4) {
            const u32x4 h = load<u32x4>(p + (in ? n * 4 : 0));
            v[i][n] = h.x;
            v[i][n + 1] = h.y;
            v[i][n + 2] = h.z;
            v[i][n + 3] = h.w;
          }
        }
      }
    };
    // The values of the lane's eight tokens at its dim e, as an operand.
    auto operand = [&](const uint32_t (&v)[8][VW], auto ec) {
      constexpr int e = decltype(ec)::value;
      u32x4 o;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        if constexpr (I8)
          o[p] = pair8<T, e & 3, e & 3>(v[2 * p][e >> 2], v[2 * p + 1][e >> 2]);
        else
          o[p] = __builtin_amdgcn_perm(v[2 * p + 1][e >> 1], v[2 * p][e >> 1],
                                       e & 1 ? 0x07060302u : 0x05040100u);
      }
      return o;
    };

    auto step = [&](int64_t x, const Where &w, const u32x4 (&k)[2][KS], uint32_t (&v)[8][VW]) {
      f32x4 s[RT][2];
#pragma unroll
      for (int t = 0; t < RT; ++t)
        s[t][0] = s[t][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < QS; ++i) {
          u32x4 ka;
          if constexpr (I8)
            ka = widen8<T>(k[n][i >> 1][(i & 1) * 2], k[n][i >> 1][(i & 1) * 2 + 1]);
          else
            ka = k[n][i];
#pragma unroll
          for (int t = 0; t < RT; ++t)
            s[t][n] = mfma<T>(ka, q[t][i], s[t][n]);
        }

      // what a row sees of these tokens, as bits
      const bool cut = w.seen != 0xffffffffu || x + kStep > cached;
      uint32_t bits[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t)
        bits[t] = 0xffffffffu;
      bool odd = false; // a value that is not finite, in tokens that not every row sees
      if (cut) {
        const int64_t d = x - cached; // the first token's place among the new ones
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if (d + kStep > 0) {
            if (a.mask) {
              const int64_t from = d > 0 ? d : 0;
              const int word = static_cast<int>(from >> 6), sh = static_cast<int>(from & 63);
              uint64_t m = 0;
              if (t * 16 + c < rows) {
                const int64_t *mp = a.mask + (start + static_cast<int64_t>(row_j[t])) * a.words;
                if (word < a.words)
                  m = static_cast<uint64_t>(mp[word]) >> sh;
                if (sh > 32 && word + 1 < a.words)
                  m |= static_cast<uint64_t>(mp[word + 1]) << (64 - sh);
              }
              const int old = d < 0 ? static_cast<int>(-d) : 0; // cached tokens of the step
              bits[t] = static_cast<uint32_t>(m << old) | ((1u << old) - 1u);
            } else {
              const int64_t n = row_j[t] - d + 1;
              bits[t] = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
            }
          }
          bits[t] &= w.seen;
        }
        // tokens that no row may read hold anything: out of the products
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool in = w.seen >> ((i >> 2) * 16 + 4 * g + (i & 3)) & 1u;
#pragma unroll
          for (int n = 0; n < VW; ++n)
            v[i][n] = in ? v[i][n] : 0u;
        }
        if constexpr (!I8) {
          constexpr uint32_t kExp = T == kF16 ? 0x7c00u : 0x7f80u;
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int n = 0; n < VW; ++n)
              odd |= (v[i][n] & kExp) == kExp || (v[i][n] >> 16 & kExp) == kExp;
          odd = __any(odd);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!(bits[t] >> (n * 16 + 4 * g + i) & 1u))
                s[t][n][i] = -__builtin_inff();
      }

#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float most = fmaxf(fmaxf(fmaxf(s[t][0][0], s[t][0][1]), fmaxf(s[t][0][2], s[t][0][3])),
                           fmaxf(fmaxf(s[t][1][0], s[t][1][1]), fmaxf(s[t][1][2], s[t][1][3])));
        most = max_over_groups(most) * scale;
        if (__any(most > top[t] + (kBias + kSlack))) {
          const float next = fmaxf(top[t], most - kBias);
          const float shrink = __builtin_amdgcn_exp2f(top[t] - next);
          top[t] = next;
          weight[t] *= shrink;
#pragma unroll
          for (int e = 0; e < E; ++e)
            acc[t][e] *= shrink;
        }
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(s[t][i >> 2][i & 3] * scale - top[t]);
          weight[t] += p[i];
        }
        const u32x4 pb = {pack16<T>(p[0], p[1]), pack16<T>(p[2], p[3]), pack16<T>(p[4], p[5]),
                          pack16<T>(p[6], p[7])};
        if (!odd) {
          add_values<T, E>(acc[t], pb, operand, v);
        } else {
          // A product with a weight of zero would carry the value over: row by
          // row, without the tokens that the row does not see.
#pragma clang loop unroll(disable)
          for (int n = 0; n < 16; ++n) {
            // keeps the operands of all sixteen rounds from being made at once
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int m = 0; m < VW; ++m)
                asm volatile("" : "+v"(v[i][m]));
            const uint32_t mine = __shfl(bits[t], n);
            u32x4 sees;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t two = mine >> ((i >> 1) * 16 + 4 * g + (i & 1) * 2);
              sees[i] = (two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u);
            }
            add_row<T, E>(acc[t], pb, operand, v, sees, c == n);
          }
        }
      }
    };

    // ---- the tokens of this run: the next step's keys are on their way
    // while this one's are used
    const int64_t x_end = min(s1 * kUnit, length);
    int64_t x = s0 * kUnit + wave * kStep;
    if (x < x_end) {
      Where w = find(x);
      u32x4 k[2][KS];
      load_keys(w, k);
      for (;;) {
        uint32_t v[8][VW];
        load_values(w, v);
        const int64_t next = x + kUnit;
        Where wn = w;
        u32x4 kn[2][KS];
        if (next < x_end) {
          wn = find(next);
          load_keys(wn, kn);
        }
        step(x, w, k, v);
        if (next >= x_end)
          break;
        x = next;
        w = wn;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int s = 0; s < KS; ++s)
            k[n][s] = kn[n][s];
      }
    }

    // ---- the four waves' sums
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      weight[t] += __shfl_xor(weight[t], 16);
      weight[t] += __shfl_xor(weight[t], 32);
      if (g == 0) {
        row_max[wave][t * 16 + c] = top[t];
        row_sum[wave][t * 16 + c] = weight[t];
      }
    }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == units;
    const int64_t part = (wg * 2 + (s0 == 0 ? 1 : 0)) * ROWS;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float most = kNone;
      {
        const int i = t * 16 + c;
#pragma unroll
        for (int w = 0; w < kAttendWaves; ++w)
          most = fmaxf(most, row_max[w][i]);
        const float f = __builtin_amdgcn_exp2f(top[t] - most);
        if (i < rows)
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
            for (int e = 0; e < E; e += 4)
              *reinterpret_cast<f32x4 *>(&sums[wave][c][(4 * g + i4) * E + e]) =
                  f32x4{acc[t][e][i4] * f, acc[t][e + 1][i4] * f, acc[t][e + 2][i4] * f,
                        acc[t][e + 3][i4] * f};
      }
      __syncthreads();
      {
        const int r16 = tid >> 4, i = t * 16 + r16, d0 = (tid & 15) * E;
        if (i < rows) {
          float m = kNone, l = 0.0f;
#pragma unroll
          for (int w = 0; w < kAttendWaves; ++w)
            m = fmaxf(m, row_max[w][i]);
#pragma unroll
          for (int w = 0; w < kAttendWaves; ++w)
            l += row_sum[w][i] * __builtin_amdgcn_exp2f(row_max[w][i] - m);
          float o[E];
#pragma unroll
          for (int e = 0; e < E; ++e) {
            o[e] = sums[0][r16][d0 + e];
#pragma unroll
            for (int w = 1; w < kAttendWaves; ++w)
              o[e] += sums[w][r16][d0 + e];
          }
          if (whole) {
            const uint32_t p = static_cast<uint32_t>(tile * ROWS + i);
            const uint32_t j = fdiv(p, a.group);
            const int64_t row = start + static_cast<int64_t>(j);
            const int64_t qh = static_cast<int64_t>(head) * a.group.d + (p - j * a.group.d);
            const float f = l > 0.0f ? (I8 ? a.value_scale[head] : 1.0f) / l : l == 0.0f ? 0.0f : l;
            char *dst = a.out + (row * a.out_row + qh * a.out_head + d0) * 2;
#pragma unroll
            for (int e = 0; e < E; e += 4)
              if (d0 + e < a.dim)
                store(dst + e * 2, u32x2{pack16<T>(o[e] * f, o[e + 1] * f), pack16<T>(o[e + 2] * f, o[e + 3] * f)});
            if (a.lse && d0 == 0)
              a.lse[row * a.heads + qh] =
                  l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * 0.693147180559945309f;
          } else {
            float *dst = a.partial + (part + i) * DP + d0;
#pragma unroll
            for (int e = 0; e < E; e += 4)
              *reinterpret_cast<f32x4 *>(dst + e) = f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]};
            if (d0 == 0) {
              a.stats[(part + i) * 2] = m;
              a.stats[(part + i) * 2 + 1] = l;
            }
          }
        }
      }
      __syncthreads();
    }
  }
}

// The rows of items that lie in several workgroups' runs: their partial sums,
// added up; and zeros for the rows of no request. A wave takes an output row at
// a time, a column of blocks the rows of a request.
template <int T, bool I8, int DP, int RT>
__global__ __launch_bounds__(256) void k_attend_join(AttendArgs a) {
  constexpr int ROWS = 16 * RT;
  constexpr int N = DP / 64; // dims of a lane
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int b = blockIdx.x;
  if (b == a.requests) { // rows of no request
    const int r0 = min(max(a.starts[0], 0), a.rows), r1 = min(max(a.starts[a.requests], r0), a.rows);
    const int64_t none = static_cast<int64_t>(r0 + a.rows - r1) * a.heads;
    for (int64_t i = static_cast<int64_t>(blockIdx.y) * 4 + wave; i < none; i += static_cast<int64_t>(gridDim.y) * 4) {
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
  const Request r = attend_request<ROWS>(a, b);
  const int64_t total = a.schedule[a.requests], first = a.schedule[b];
  const int64_t per = (total + a.workgroups - 1) / a.workgroups;
  const int64_t count = static_cast<int64_t>(r.fresh) * a.heads;
  for (int64_t i = static_cast<int64_t>(blockIdx.y) * 4 + wave; i < count; i += static_cast<int64_t>(gridDim.y) * 4) {
    const int j = static_cast<int>(i / a.heads), qh = static_cast<int>(i - static_cast<int64_t>(j) * a.heads);
    const int head = static_cast<int>(fdiv(static_cast<uint32_t>(qh), a.group));
    const int p = j * static_cast<int>(a.group.d) + qh - head * static_cast<int>(a.group.d);
    const int tile = p / ROWS, row = p % ROWS;
    const int64_t u0 = first + (static_cast<int64_t>(head) * r.tiles + tile) * r.units;
    const int64_t w0 = u0 / per, w1 = (u0 + r.units - 1) / per;
    if (w0 == w1)
      continue; // written whole
    // a run that begins inside the item left its part in its first place, the
    // run in which the item begins in its second
    auto at = [&](int64_t w) { return (w * 2 + (w == w0 ? 1 : 0)) * ROWS + row; };
    float most = kNone;
    for (int64_t w = w0 + lane; w <= w1; w += 64)
      most = fmaxf(most, a.stats[at(w) * 2]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
      most = fmaxf(most, __shfl_xor(most, o));
    float sum = 0.0f, out[N];
#pragma unroll
    for (int n = 0; n < N; ++n)
      out[n] = 0.0f;
#pragma unroll 4
    for (int64_t w = w0; w <= w1; ++w) {
      const int64_t k = at(w);
      const float f = __builtin_amdgcn_exp2f(a.stats[k * 2] - most);
      sum += a.stats[k * 2 + 1] * f;
#pragma unroll
      for (int n = 0; n < N; ++n)
        out[n] += a.partial[k * DP + lane * N + n] * f;
    }
    const float f = sum > 0.0f ? (I8 ? a.value_scale[head] : 1.0f) / sum : sum == 0.0f ? 0.0f : sum;
    const int64_t orow = r.start + static_cast<int64_t>(j);
    char *dst = a.out + (orow * a.out_row + qh * a.out_head + lane * N) * 2;
    if (lane * N < a.dim) {
      if constexpr (N == 1) {
        store(dst, static_cast<uint16_t>(pack16<T>(out[0] * f, 0.0f)));
      } else {
#pragma unroll
        for (int n = 0; n < N; n += 2)
          store(dst + n * 2, pack16<T>(out[n] * f, out[n + 1] * f));
      }
    }
    if (a.lse && lane == 0)
      a.lse[orow * a.heads + qh] =
          sum == 0.0f ? -__builtin_inff() : (most + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f;
  }
}

template <int T, bool I8, int DP, int RT>
hipError_t attend_start(const AttendArgs &args, const AttendPlan &p, hipStream_t s) {
  AttendArgs a = args;
  void *pa[] = {&a};
  const void *k = p.fast ? reinterpret_cast<const void *>(k_attend<T, I8, DP, RT, true>)
                         : reinterpret_cast<const void *>(k_attend<T, I8, DP, RT, false>);
  hipError_t e = hipLaunchKernel(k, dim3(static_cast<uint32_t>(p.workgroups)), dim3(kScan), pa, 0, s);
  if (e != hipSuccess)
    return e;
  // a wave for every output row of an even batch, within 2^16 blocks a request
  const int64_t rows = (static_cast<int64_t>(a.rows) * a.heads + a.requests - 1) / a.requests;
  const int64_t y = std::min<int64_t>((rows + 3) / 4, 65535);
  return hipLaunchKernel(reinterpret_cast<const void *>(k_attend_join<T, I8, DP, RT>),
                         dim3(static_cast<uint32_t>(a.requests) + 1, static_cast<uint32_t>(y)), dim3(256), pa, 0, s);
}

template <int T, bool I8, int DP>
hipError_t attend_tiles(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  switch (p.row_tiles) {
  case 1:
    return attend_start<T, I8, DP, 1>(a, p, s);
  case 2:
    return attend_start<T, I8, DP, 2>(a, p, s);
  default:
    if constexpr (DP <= 128)
      return attend_start<T, I8, DP, 4>(a, p, s);
    return hipErrorInvalidValue;
  }
}

template <int T, bool I8>
hipError_t attend_width(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  switch (p.width) {
  case 64:
    return attend_tiles<T, I8, 64>(a, p, s);
  case 128:
    return attend_tiles<T, I8, 128>(a, p, s);
  default:
    return attend_tiles<T, I8, 256>(a, p, s);
  }
}

} // namespace
} // namespace relx
