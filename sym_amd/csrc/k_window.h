// k_window.h - attention over packed sequences with a window and first tokens
// that stay, and its gradients (device templates; instantiated in
// k_window_f16.hip and k_window_bf16.hip).
//
//   see(p, x)  x <= p and (x < sinks or p - x < window), p and x of one sequence
//   S = scale Q K^T, P = softmax(S), O = P V, lse = log sum exp S
//   dV = P^T dO, dP = dO V^T, D = rowsum(dO O), dS = P (dP - D) scale,
//   dQ = dS K, dK = dS^T Q, dK and dV summed over the heads of a group
//
// All products are 32 x 32 x 16 matrix instructions. What a wave owns, 32 query
// rows or 32 keys, are the columns of their results; what goes past it, keys or
// query rows, are the rows, in tiles that all waves of a workgroup share through
// shared memory. So a product's result lies in the lanes as the next product
// wants its operand (lane: column lane % 32, rows 8 i + 4 (lane / 32) + 0..3), if
// the rows that are summed over are taken in the order in which they lie:
// weights go from one product to the next in registers, and the other operand is
// read from shared memory transposed (ds_read_b64_tr_b16).
//
//   forward  S^T = K Q^T, O^T += V^T P^T             32 rows a wave, tiles of keys
//   dQ       S^T, dP^T = V dO^T, dQ^T += K^T dS^T    the same
//   dK, dV   S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
//                                                    32 keys a wave, tiles of rows
//
// Scores are computed twice in the backward pass rather than added up in memory:
// no atomics, the same bits every time. A key head's rows are (token, head of the
// group), so a tile of keys serves a whole group, and its gradients are summed
// over the group in registers.
//
// The first tokens' gradients come from all rows of their sequence: those within
// the window with the other keys, the rest in pieces of rows, by a launch of
// their own that leaves sums in 32 bits; they are added in order at the end.
//
// Measured, 24.6k rows of 32 + 8 heads of 128 in bf16, window 1024, 4 first tokens:
// forward 490 us (850 TFLOP/s), dQ 695, dK and dV 974, the first tokens' 95, D of rows
// that see few 11; 16384 rows of 16 heads of 64 in f16, window 4096: 307, 424, 632, 25
// and 7 (each at least, in traces; steps in a row take 2250 and 1369). Matrix units are
// busy for 0.47 to 0.49 of the cycles (at 1.7 to 1.8 GHz under this load), vector
// units for 0.56 (forward), 0.41 and 0.32, shared memory for 0.23, 0.24 and 0.37,
// without bank conflicts: products and softmax of one wave follow one another, and
// only the two or three waves of a SIMD overlap them. (Where 32 keys are a workgroup's,
// shared memory holds two with heads of 64, and one, of a wave a SIMD, with wider.)
#pragma once

#include <algorithm>
#include <type_traits>

#include "attention.h"
#include "index.h"
#include "k_attend_wave.h"
#include "window.h"

namespace relx {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;
constexpr int kAhead = 4; // reads of shared memory ahead of their product

template <int T> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (T == kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zero16() {
  return f32x16{0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
}

// ------------------------------------------------------------ sequences

// A piece of a sequence: `index` pieces of a size after its first row. Rows of no
// sequence, before the first and after the last, are two more, not `real`.
struct Piece {
  int begin, n, index, number;
  bool real;
};

// The number of a sequence's first piece: begin / size and one for each sequence
// before, since n rows are at most n / size + 1 pieces. LONG: of sequences of more
// rows than the window has, of which no two begin in the same span of so many rows;
// others have no pieces.
template <bool LONG> __device__ __forceinline__ int first_piece(const WindowArgs &a, FastDiv size, int begin, int sequence) {
  const int before = LONG ? min(sequence, static_cast<int>(fdiv(static_cast<uint32_t>(begin), a.longer))) : sequence;
  return static_cast<int>(fdiv(static_cast<uint32_t>(begin), size)) + before;
}

// Piece `number`, of all sequences, with the two. Lanes compare 64 of them at a time.
// n = 0: there is no such piece.
template <bool LONG> __device__ __forceinline__ Piece find(const WindowArgs &a, FastDiv size, int number) {
  const int lane = threadIdx.x & 63, many = a.sequences + 2;
  int lo = 0, hi = many, st = 0, en = 0;
  for (;;) {
    const int step = (hi - lo + 63) >> 6, b = lo + lane * step;
    bool upto = false;
    if (b < hi) {
      st = b == 0 ? 0 : min(max(a.starts[b - 1], 0), a.rows);
      if (step == 1)
        en = b == many - 1 ? a.rows : min(max(a.starts[b], 0), a.rows);
      upto = first_piece<LONG>(a, size, st, b) <= number;
    }
    const uint64_t not_yet = ~__ballot(upto);
    const int n = max(not_yet ? __builtin_ctzll(not_yet) : 64, 1) - 1;
    lo += n * step;
    if (step == 1) {
      st = __builtin_amdgcn_readlane(st, n);
      en = __builtin_amdgcn_readlane(en, n);
      break;
    }
    hi = min(hi, lo + step);
  }
  Piece p;
  p.begin = uniform(st);
  p.n = uniform(max(en - st, 0));
  p.number = uniform(lo);
  p.index = uniform(number - first_piece<LONG>(a, size, st, lo));
  p.real = lo > 0 && lo < many - 1;
  if (p.index < 0 || static_cast<int64_t>(p.index) * size.d >= p.n)
    p.n = 0;
  return p;
}

// The first pieces alone, `few_pieces` of each sequence.
__device__ __forceinline__ Piece first_of(const WindowArgs &a, FastDiv size, int number) {
  const int sequence = number / a.few_pieces;
  const int st = min(max(a.starts[sequence], 0), a.rows), en = min(max(a.starts[sequence + 1], 0), a.rows);
  Piece p;
  p.begin = uniform(st);
  p.number = sequence + 1;
  p.index = number - sequence * a.few_pieces;
  p.n = uniform(max(en - st, 0));
  p.real = true;
  if (p.index * static_cast<int>(size.d) >= p.n)
    p.n = 0;
  return p;
}

// A workgroup's piece and key head: neighbours share a die, whose cache serves the
// tiles that they both read. Later pieces, which in a sequence read more, first.
struct Work {
  int number, head;
  bool none;
};
__device__ __forceinline__ Work my_work(int numbers, int heads) {
  const int id = static_cast<int>(blockIdx.x), total = numbers * heads;
  const int item = (id & 7) * static_cast<int>(gridDim.x >> 3) + (id >> 3);
  Work w;
  w.none = item >= total;
  w.head = uniform(item / numbers);
  w.number = uniform(numbers - 1 - (item - w.head * numbers));
  return w;
}

// ------------------------------------------------------------ tiles

// Where the n-th 16-byte piece of a token's row lies in a tile of rows of RB
// bytes. Sixteen tokens' n-th pieces, and two neighbouring pairs of pieces of
// four tokens (what sixteen lanes of two transposed reads want), lie in banks of
// their own.
template <int RB> __device__ __forceinline__ int swap_of(int token) {
  return RB == 256 ? (token & 3) << 2 | (token >> 2 & 3) : (token >> 1 & 1) << 2 | (token >> 2 & 3);
}

// Brings NT tokens of a tile, from its `first` on, by one wave.
template <int DP, int NT> struct Bring {
  static constexpr int RB = DP * 2, LT = RB / 16, TPI = 64 / LT, LOADS = NT / TPI;
  int token, first, piece0, dims;
  __device__ __forceinline__ Bring(int lane, int first_, int dim) {
    token = lane / LT;
    first = first_;
    piece0 = lane % LT ^ swap_of<RB>(first + token);
    dims = dim;
  }
  // The tile's tokens begin at `base`, `row` bytes apart; those past the `left`
  // first are the last of them over again: nothing outside the sequence is read,
  // and what its rows do not see is at least its own.
  __device__ __forceinline__ void send(const char *base, uint32_t row, int left, uint32_t to) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      // TPI tokens on: of the swap's bits, those that the lane's token has stay
      const int n = piece0 ^ (swap_of<RB>(i * TPI));
      const int t = min(first + i * TPI + token, left - 1);
      if (n * 8 < dims)
        load_async<false>(base, static_cast<uint32_t>(t) * row + n * 16, to + (first + i * TPI) * RB);
    }
  }
};

// A lane's place in a tile for operands read as they lie: token lane % 32, and of
// contraction step s the dims 16 s + 8 (lane / 32) on. Step s: ^ 32 s.
template <int RB> __device__ __forceinline__ uint32_t direct_at(int lane) {
  const int c = lane & 31;
  return c * RB + ((lane >> 5) ^ swap_of<RB>(c)) * 16;
}
// And transposed: of 16 tokens from 16 s on, 4 (lane / 32) + 0..3 and 8 more (half 1),
// dim 32 m + lane % 32. m: ^ 64 m; s: + 16 s RB.
template <int RB> __device__ __forceinline__ uint32_t turned_at(int lane, int half) {
  const int i = lane & 15, g = lane >> 4, t = 8 * half + 4 * (g >> 1) + (i >> 2);
  return t * RB + ((((g & 1) * 2 + ((i & 3) >> 1)) ^ swap_of<RB>(t)) * 16) + (i & 1) * 8;
}
__device__ __forceinline__ u32x4 turned(uint32_t first, uint32_t second) {
  const u32x2 a = read_transposed(first), b = read_transposed(second);
  return u32x4{a.x, a.y, b.x, b.y};
}

// Sixteen values of a lane as two operands.
template <int T> __device__ __forceinline__ void pack_operands(const f32x16 &p, u32x4 (&w)[2]) {
#pragma unroll
  for (int s = 0; s < 2; ++s)
    w[s] = u32x4{pack16<T>(p[8 * s], p[8 * s + 1]), pack16<T>(p[8 * s + 2], p[8 * s + 3]),
                 pack16<T>(p[8 * s + 4], p[8 * s + 5]), pack16<T>(p[8 * s + 6], p[8 * s + 7])};
}

// Where element i of a result lies among the 32 rows.
__device__ __forceinline__ int row_of(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }

// Places of a head past its dims: no load writes them.
template <int THREADS> __device__ __forceinline__ void clear(char *tiles, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += THREADS * 16)
    *reinterpret_cast<u32x4 *>(tiles + i) = u32x4{0u, 0u, 0u, 0u};
}

// A lane's dims of its row or key, as an operand: zeros past the head.
template <int DP> __device__ __forceinline__ void take_row(u32x4 (&w)[DP / 16], const char *row, int dim, int lane) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = 16 * s + 8 * (lane >> 5);
    w[s] = u32x4{0u, 0u, 0u, 0u};
    if (d < dim)
      w[s] = *reinterpret_cast<const u32x4 *>(row + d * 2);
  }
}

// A result's columns, 32 dims of each `m`, to their rows.
template <int T, int DP>
__device__ __forceinline__ void put_row(char *row, const f32x16 (&acc)[DP / 32], float f, int dim, int lane) {
#pragma unroll
  for (int m = 0; m < DP / 32; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * m + 8 * i + 4 * (lane >> 5);
      if (d < dim)
        *reinterpret_cast<u32x2 *>(row + d * 2) =
            u32x2{pack16<T>(acc[m][4 * i] * f, acc[m][4 * i + 1] * f), pack16<T>(acc[m][4 * i + 2] * f, acc[m][4 * i + 3] * f)};
    }
}

// f16 has few bits for small numbers: P is taken 2^10 times as large (it is at
// most one), and dS over a power of two that holds the largest so far, of which
// the sums then are.
constexpr float kMore = 10.0f;
template <int T> __device__ __forceinline__ constexpr float less() { return T == kF16 ? 0.0009765625f : 1.0f; }
template <int T, int E> struct Over {
  int e = 1; // exponent of the power of two, as a float holds it
  __device__ __forceinline__ float up() const { return T == kF16 ? __uint_as_float(static_cast<uint32_t>(e) << 23) : 1.0f; }
  __device__ __forceinline__ float down() const { return T == kF16 ? __uint_as_float(static_cast<uint32_t>(254 - e) << 23) : 1.0f; }
  __device__ __forceinline__ void hold(const f32x16 &ds, f32x16 (&acc)[E]) {
    if constexpr (T == kF16) {
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        most = fmaxf(most, fabsf(ds[i]));
      if (__builtin_expect(__any(most * down() > 32768.0f), 0)) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
          most = fmaxf(most, __shfl_xor(most, o));
        // the largest becomes 2^11 to 2^12: a few times larger ones still fit
        const int next = uniform(max(static_cast<int>(__float_as_uint(most) >> 23) - 11, 1));
        const float shrink = up() * __uint_as_float(static_cast<uint32_t>(254 - next) << 23);
        e = next;
#pragma unroll
        for (int m = 0; m < E; ++m)
          acc[m] *= shrink;
      }
    }
  }
};

// A workgroup's query rows: (token, head of the group) in this order, 128 at most.
struct RowsOf {
  int first, tokens, head, heads;
  __device__ __forceinline__ RowsOf(const WindowArgs &a, const Piece &p, int which) {
    first = p.index * static_cast<int>(a.tile_tokens.d);
    tokens = min(static_cast<int>(a.tile_tokens.d), p.n - first);
    const int parts = a.parts, kv = which / parts, part = which - kv * parts;
    const int group = a.heads / a.kv_heads;
    head = kv * group + part * static_cast<int>(a.tile_heads.d);
    heads = min(static_cast<int>(a.tile_heads.d), group - part * static_cast<int>(a.tile_heads.d));
  }
};
// A lane's row: where none is, another of the tile's.
struct MyRow {
  int token, head; // of the sequence, of all heads
  bool there;
  __device__ __forceinline__ MyRow(const WindowArgs &a, const RowsOf &r, int row) {
    const int t = static_cast<int>(fdiv(static_cast<uint32_t>(row), a.tile_heads)), h = row - t * static_cast<int>(a.tile_heads.d);
    there = t < r.tokens && h < r.heads;
    token = r.first + min(t, r.tokens - 1);
    head = r.head + min(h, r.heads - 1);
  }
};

// The tiles of keys that a tile of rows reads: those with first tokens, then those
// of its rows' windows.
template <int KEYS> struct KeyTiles {
  int first, jump, count;
  __device__ __forceinline__ KeyTiles(const WindowArgs &a, int from_row, int to_row) {
    const int from = max(from_row - a.window + 1, 0) / KEYS;
    first = min((a.sinks + KEYS - 1) / KEYS, from);
    jump = from - first;
    count = to_row / KEYS - jump + 1;
  }
  __device__ __forceinline__ int token(int n) const { return (n < first ? n : n + jump) * KEYS; }
};
// Whether rows from p0 to p1 see none, or all, of the tokens from x0 to x1.
__device__ __forceinline__ bool see_none(const WindowArgs &a, int p0, int p1, int x0, int x1) {
  return x0 > p1 || (p0 - x1 >= a.window && x0 >= a.sinks);
}
__device__ __forceinline__ bool see_all(const WindowArgs &a, int p0, int p1, int x0, int x1) {
  return x1 <= p0 && (p1 - x0 < a.window || x1 < a.sinks);
}

// Puts `none` in the place of what a lane's row does not see of the 32 tokens from
// x. Compares and selects only: as branches, which the compiler makes of conditions
// that are read one after the other, a tile with an edge took three times as long.
__device__ __forceinline__ void hide(const WindowArgs &a, f32x16 &s, int row, int x, int first_row, int last_row, int lane, float none) {
  const int at = x + 4 * (lane >> 5);
  if (x + 31 > first_row) {
    const int most = row - at;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s[i] = row_of(i, 0) > most ? none : s[i];
  }
  if (x <= last_row - a.window) {
    const int upto = row - a.window - at, stay = a.sinks - at;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s[i] = (row_of(i, 0) <= upto) & (row_of(i, 0) >= stay) ? none : s[i];
  }
}

// Rows of no sequence: zeros.
__device__ __forceinline__ void zero_rows(const WindowArgs &a, const Heads &h, int begin, int from, int tokens, int head, int heads) {
  const int pieces = a.dim / 8;
  for (int i = threadIdx.x; i < tokens * heads * pieces; i += 64 * kWaves) {
    const int row = i / pieces, t = row / heads;
    *reinterpret_cast<u32x4 *>(h.data + ((static_cast<int64_t>(begin) + from + t) * h.row + (head + row - t * heads) * h.head) * 2 +
                               (i - row * pieces) * 16) = u32x4{0u, 0u, 0u, 0u};
  }
}

// ------------------------------------------------------------ forward

// Three waves a SIMD, for which a head of 128 takes 32 tokens at a time: 497 us
// against 536 with 64 and two waves (24.6k rows of 32 + 8 heads, window 1024).
template <int T, int DP> __global__ __launch_bounds__(64 * kWaves, 3) void k_window_forward(WindowArgs a) {
  constexpr int KEYS = DP == 128 ? 32 : 64, B = KEYS / 32; // tokens of a tile
  constexpr int RB = DP * 2, TILE = KEYS * RB, E = DP / 32, KS = DP / 16, RING = DP == 128 ? 3 : 2;
  using Loads = Bring<DP, KEYS / kWaves>;
  __shared__ __attribute__((aligned(256))) char tiles[RING][2][TILE];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const Work w = my_work(a.row_pieces, a.kv_heads * a.parts);
  if (w.none)
    return;
  const Piece piece = find<false>(a, a.tile_tokens, w.number);
  if (piece.n == 0)
    return;
  const RowsOf rows(a, piece, w.head);
  if (!piece.real) {
    zero_rows(a, a.o, piece.begin, rows.first, rows.tokens, rows.head, rows.heads);
    if (a.lse)
      for (int i = threadIdx.x; i < rows.tokens * rows.heads; i += 64 * kWaves)
        a.lse[static_cast<int64_t>(rows.head + i / rows.tokens) * a.rows + piece.begin + rows.first + i % rows.tokens] =
            -__builtin_inff();
    return;
  }
  if (a.dim < DP) {
    clear<64 * kWaves>(&tiles[0][0][0], sizeof(tiles));
    __syncthreads();
  }
  const int last = rows.first + rows.tokens - 1;
  const KeyTiles<KEYS> keys(a, rows.first, last);
  const int kv = w.head / a.parts;
  const char *k0 = a.k.data + (static_cast<int64_t>(piece.begin) * a.k.row + kv * a.k.head) * 2;
  const char *v0 = a.v.data + (static_cast<int64_t>(piece.begin) * a.v.row + kv * a.v.head) * 2;
  const uint32_t krow = static_cast<uint32_t>(a.k.row) * 2, vrow = static_cast<uint32_t>(a.v.row) * 2;
  const Loads bring(lane, wave * (KEYS / kWaves), a.dim);
  const uint32_t at = place(&tiles[0][0][0]);
  auto send = [&](int n, int slot) {
    const int x = keys.token(n);
    bring.send(k0 + static_cast<int64_t>(x) * krow, krow, piece.n - x, at + slot * 2 * TILE);
    bring.send(v0 + static_cast<int64_t>(x) * vrow, vrow, piece.n - x, at + slot * 2 * TILE + TILE);
  };
  for (int n = 0; n < min(keys.count, RING - 1); ++n)
    send(n, n);

  const MyRow row(a, rows, wave * 32 + (lane & 31));
  const int first_row = uniform(MyRow(a, rows, wave * 32).token), last_row = uniform(MyRow(a, rows, wave * 32 + 31).token);
  const bool busy = wave * 32 < rows.tokens * static_cast<int>(a.tile_heads.d);
  u32x4 q[KS];
  take_row<DP>(q, a.q.data + ((static_cast<int64_t>(piece.begin) + row.token) * a.q.row + row.head * a.q.head) * 2, a.dim, lane);
  // masks and maxima are those of unscaled scores, which goes for a scale above
  // zero: a negative one turns the queries over, zero is the least normal number
  const float scale = fmaxf(fabsf(a.scale), 1.17549435e-38f);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    q[s] ^= a.scale < 0.0f ? 0x80008000u : 0u;
    asm volatile("" : "+v"(q[s])); // arrived, once: not waited for in the loop
  }
  constexpr float kBias = weight_bias<T>();
  float top = kNone, sum = 0.0f;
  f32x16 acc[E];
#pragma unroll
  for (int m = 0; m < E; ++m)
    acc[m] = zero16();
  const uint32_t direct = direct_at<RB>(lane), turn0 = turned_at<RB>(lane, 0), turn1 = turned_at<RB>(lane, 1);

#pragma clang loop unroll(disable)
  for (int n = 0, next = 0; n < keys.count; ++n) {
    const int slot = next, x = keys.token(n);
    next = slot + 1 == RING ? 0 : slot + 1;
    if (n + RING - 2 < keys.count)
      arrived<(RING - 2) * 2 * Loads::LOADS>();
    else
      arrived<0>();
    meet(); // the tile is there, and everybody has read the one before
    if (n + RING - 1 < keys.count)
      send(n + RING - 1, slot == 0 ? RING - 1 : slot - 1);
    if (!busy || see_none(a, first_row, last_row, x, x + KEYS - 1))
      continue;
    const uint32_t tk = at + slot * 2 * TILE + direct, tv = at + slot * 2 * TILE + TILE;
    f32x16 s[B];
    // reads go out ahead of their products, in this order: see dK and dV
    auto operand = [&](int n) {
      const int b = n / KS % B, i = n % KS, m = i / 2 * 64, tokens = (b * 32 + i % 2 * 16) * RB;
      return n < B * KS ? read16((tk ^ (i * 32)) + b * 32 * RB)
                        : turned((tv + turn0 ^ m) + tokens, (tv + turn1 ^ m) + tokens);
    };
    u32x4 ahead[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n)
      ahead[n] = operand(n);
    keep_order();
#pragma unroll
    for (int b = 0; b < B; ++b) {
      s[b] = zero16();
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        s[b] = mfma32<T>(ahead[i % kAhead], q[i], s[b]);
        ahead[i % kAhead] = operand(b * KS + i + kAhead);
        keep_order();
      }
    }
    if (!see_all(a, first_row, last_row, x, x + KEYS - 1)) {
#pragma unroll
      for (int b = 0; b < B; ++b)
        hide(a, s[b], row.token, x + 32 * b, first_row, last_row, lane, -__builtin_inff());
    }
    float most = s[0][0];
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        most = fmaxf(most, s[b][i]);
    if (__builtin_expect(__any(most * scale > top + (kBias + kSlack)), 0)) {
      const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
      most = fmaxf(__uint_as_float(other[0]), __uint_as_float(other[1]));
      const float next = fmaxf(top, most * scale - kBias);
      const float shrink = __builtin_amdgcn_exp2f(top - next);
      top = next;
      sum *= shrink;
#pragma unroll
      for (int m = 0; m < E; ++m)
        acc[m] *= shrink;
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = __builtin_amdgcn_exp2f(s[b][i] * scale - top);
        part[i & 3] += s[b][i];
      }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
      u32x4 p[2];
      pack_operands<T>(s[b], p);
#pragma unroll
      for (int i = 0; i < 2 * E; ++i) {
        acc[i / 2] = mfma32<T>(ahead[i % kAhead], p[i % 2], acc[i / 2]);
        if (b * KS + i + kAhead < B * KS)
          ahead[i % kAhead] = operand((B + b) * KS + i + kAhead);
      }
    }
  }
  arrived<0>();
  sum += __shfl_xor(sum, 32);
  if (row.there) {
    const int64_t at_row = static_cast<int64_t>(piece.begin) + row.token;
    put_row<T, DP>(a.o.data + (at_row * a.o.row + row.head * a.o.head) * 2, acc, finish(sum, 1.0f), a.dim, lane);
    if (a.lse && lane < 32)
      a.lse[static_cast<int64_t>(row.head) * a.rows + at_row] = log_sum(top, sum);
  }
}

// ------------------------------------------------------------ dQ

// SUMS: D alone, as the sum of P dP. D of the rounded result is off by as much as a
// rounded weight is, over the root of the number of tokens that a row sees, and in
// all of them alike: with a few tokens gradients are 1.7 times as far off as their own
// rounding is, and 1.4 times with this D (with 128 tokens 1.5 and 1.4). So it is for
// tiles of rows that see up to kFew, in long sequences too: their first tokens'
// gradients are the largest, and mostly of rows that see few.
template <int T, int DP, bool SUMS> __global__ __launch_bounds__(64 * kWaves, 2) void k_window_dq(WindowArgs a) {
  constexpr int kKeys = 64; // tokens of a tile
  constexpr int RB = DP * 2, TILE = kKeys * RB, E = DP / 32, KS = DP / 16, RING = 2;
  __shared__ __attribute__((aligned(256))) char tiles[RING][2][TILE];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const bool of_few = SUMS && a.few_pieces > 0;
  const Work w = my_work(of_few ? a.sequences * a.few_pieces : a.row_pieces, a.kv_heads * a.parts);
  if (w.none)
    return;
  const Piece piece = of_few ? first_of(a, a.tile_tokens, w.number) : find<false>(a, a.tile_tokens, w.number);
  if (piece.n == 0)
    return;
  const RowsOf rows(a, piece, w.head);
  if (!piece.real) {
    if constexpr (!SUMS)
      zero_rows(a, a.dq, piece.begin, rows.first, rows.tokens, rows.head, rows.heads);
    return;
  }
  if (a.dim < DP) {
    clear<64 * kWaves>(&tiles[0][0][0], sizeof(tiles));
    __syncthreads();
  }
  const int last = rows.first + rows.tokens - 1;
  const bool few = min(last + 1, a.window + a.sinks) <= kFew;
  if (SUMS && !few)
    return;
  const KeyTiles<kKeys> keys(a, rows.first, last);
  const int kv = w.head / a.parts;
  const char *k0 = a.k.data + (static_cast<int64_t>(piece.begin) * a.k.row + kv * a.k.head) * 2;
  const char *v0 = a.v.data + (static_cast<int64_t>(piece.begin) * a.v.row + kv * a.v.head) * 2;
  const uint32_t krow = static_cast<uint32_t>(a.k.row) * 2, vrow = static_cast<uint32_t>(a.v.row) * 2;
  const Bring<DP, kKeys / kWaves> bring(lane, wave * (kKeys / kWaves), a.dim);
  const uint32_t at = place(&tiles[0][0][0]);
  auto send = [&](int n, int slot) {
    const int x = keys.token(n);
    bring.send(k0 + static_cast<int64_t>(x) * krow, krow, piece.n - x, at + slot * 2 * TILE);
    bring.send(v0 + static_cast<int64_t>(x) * vrow, vrow, piece.n - x, at + slot * 2 * TILE + TILE);
  };
  send(0, 0);

  const MyRow row(a, rows, wave * 32 + (lane & 31));
  const int first_row = uniform(MyRow(a, rows, wave * 32).token), last_row = uniform(MyRow(a, rows, wave * 32 + 31).token);
  const bool busy = wave * 32 < rows.tokens * static_cast<int>(a.tile_heads.d);
  const int64_t at_row = static_cast<int64_t>(piece.begin) + row.token;
  u32x4 q[KS], g[KS];
  take_row<DP>(q, a.q.data + (at_row * a.q.row + row.head * a.q.head) * 2, a.dim, lane);
  take_row<DP>(g, a.dout.data + (at_row * a.dout.row + row.head * a.dout.head) * 2, a.dim, lane);
  float *stats = a.stats + static_cast<int64_t>(row.head) * 2 * a.rows + at_row; // of the row: -lse / scale
  float *stats_d = stats + a.rows;                                               // and -D
  float d = 0.0f;
  if (!SUMS && few) {
    d = -*stats_d;
  } else if constexpr (!SUMS) {
    u32x4 o[KS];
    take_row<DP>(o, a.o.data + (at_row * a.o.row + row.head * a.o.head) * 2, a.dim, lane);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        d += widen16<T>(o[s][i] & 0xffffu) * widen16<T>(g[s][i] & 0xffffu) + widen16<T>(o[s][i] >> 16) * widen16<T>(g[s][i] >> 16);
  }
  if (!SUMS && !few)
    d += __shfl_xor(d, 32);
  const float lse = a.lse[static_cast<int64_t>(row.head) * a.rows + at_row] * 1.44269504088896341f;
  if (!SUMS && row.there && lane < 32) {
    *stats = -lse / a.scale;
    *stats_d = -d;
  }
#pragma unroll
  for (int s = 0; s < KS; ++s)
    asm volatile("" : "+v"(q[s]), "+v"(g[s]));
  Over<T, E> over;
  f32x16 acc[E];
#pragma unroll
  for (int m = 0; m < E; ++m)
    acc[m] = zero16();
  const uint32_t direct = direct_at<RB>(lane), turn0 = turned_at<RB>(lane, 0), turn1 = turned_at<RB>(lane, 1);

#pragma clang loop unroll(disable)
  for (int n = 0; n < keys.count; ++n) {
    const int slot = n & 1, x = keys.token(n);
    arrived<0>();
    meet();
    if (n + 1 < keys.count)
      send(n + 1, slot ^ 1);
    if (!busy || see_none(a, first_row, last_row, x, x + kKeys - 1))
      continue;
    const uint32_t tk = at + slot * 2 * TILE, tv = tk + TILE;
    const bool cut = !see_all(a, first_row, last_row, x, x + kKeys - 1);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (DP == 128 && see_none(a, first_row, last_row, x + 32 * b, x + 32 * b + 31))
        continue; // heads of 64 have too little to gain
      f32x16 s = zero16(), dp = zero16();
      auto operand = [&](int n) {
        const int i = n % KS, m = i / 2 * 64, tokens = (b * 32 + i % 2 * 16) * RB;
        return n < KS       ? read16((tk + direct ^ (i * 32)) + b * 32 * RB)
               : n < 2 * KS ? read16((tv + direct ^ (i * 32)) + b * 32 * RB)
                            : turned((tk + turn0 ^ m) + tokens, (tk + turn1 ^ m) + tokens);
      };
      u32x4 ahead[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n)
        ahead[n] = operand(n);
      keep_order();
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        s = mfma32<T>(ahead[i % kAhead], q[i], s);
        ahead[i % kAhead] = operand(i + kAhead);
        keep_order();
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        dp = mfma32<T>(ahead[i % kAhead], g[i], dp);
        if (!SUMS || i + kAhead < KS)
          ahead[i % kAhead] = operand(KS + i + kAhead);
#pragma unroll
        for (int n = 16 / KS * i; n < 16 / KS * (i + 1); ++n)
          s[n] = __builtin_amdgcn_exp2f(s[n] * a.scale - lse);
        keep_order();
      }
      if constexpr (SUMS) {
        if (cut)
          hide(a, s, row.token, x + 32 * b, first_row, last_row, lane, 0.0f);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          d += s[i] > 0.0f ? s[i] * dp[i] : 0.0f;
        continue;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] *= dp[i] - d;
      if (cut)
        hide(a, s, row.token, x + 32 * b, first_row, last_row, lane, 0.0f);
      over.hold(s, acc);
      if constexpr (T == kF16)
        s *= over.down();
      u32x4 p[2];
      pack_operands<T>(s, p);
#pragma unroll
      for (int i = 0; i < 2 * E; ++i) {
        acc[i / 2] = mfma32<T>(ahead[i % kAhead], p[i % 2], acc[i / 2]);
        if (i + kAhead < KS)
          ahead[i % kAhead] = operand(2 * KS + i + kAhead);
      }
    }
  }
  arrived<0>();
  if constexpr (SUMS) {
    d += __shfl_xor(d, 32);
    if (row.there && lane < 32)
      *stats_d = -d;
    return;
  }
  if (row.there)
    put_row<T, DP>(a.dq.data + (at_row * a.dq.row + row.head * a.dq.head) * 2, acc, a.plain_scale * over.up(), a.dim, lane);
}

// ------------------------------------------------------------ dK and dV

// A wave's keys stay in registers with their gradients' sums, its values in shared
// memory: both in registers left too few (1842 us against 1396 with heads of 128;
// 1422 against 1378 for a step with heads of 64, which three waves a SIMD fit so).
//   kWide    128 keys a workgroup, 32 a wave, over the rows in whose windows they are
//   kNarrow  32 keys a workgroup, whose waves take turns at the tiles of rows and add
//            up at the end: where there are few keys, four times the workgroups
//   kFirst   the same, of first tokens over the rows whose window has left them
// The last two take 70 KiB of shared memory with heads of 64 and 138 KiB with wider
// ones: that, and not their 126 and 164 registers, says how many run on a compute unit.
enum KeyMode : int { kWide, kNarrow, kFirst };
template <int T, int DP, int MODE>
__global__ __launch_bounds__(64 * kWaves, DP == 64 ? 3 : 2) void k_window_dkv(WindowArgs a) {
  constexpr bool FIRST = MODE == kFirst, TURNS = MODE != kWide;
  constexpr int RB = DP * 2, TILE = 32 * RB, E = DP / 32, KS = DP / 16, KEYS = TURNS ? 32 : 32 * kWaves;
  constexpr int RING = TURNS || DP == 128 ? 2 : 3; // tiles at a time; TURNS: of each wave
  constexpr int SLOTS = TURNS ? kWaves * RING : RING;
  constexpr int NT = TURNS ? 32 : 32 / kWaves; // tokens that a wave brings
  using Loads = Bring<DP, NT>;
  constexpr int ROOM = SLOTS * 2 * TILE;
  __shared__ __attribute__((aligned(256))) char tiles[ROOM];
  __shared__ __attribute__((aligned(16))) float stats[SLOTS][2][32];
  __shared__ __attribute__((aligned(256))) char values[KEYS * RB];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int group = a.heads / a.kv_heads;
  const Work w = my_work(FIRST ? a.first_pieces : a.key_pieces, FIRST ? a.kv_heads * a.first_blocks : a.kv_heads);
  if (w.none)
    return;
  const Piece piece = find<FIRST>(a, FIRST ? a.first_tokens : a.key_tokens, w.number);
  if (piece.n == 0)
    return;
  const int kv = FIRST ? w.head / a.first_blocks : w.head;
  // the keys, and the rows' tokens [p0, p1)
  const int x0 = FIRST ? (w.head - kv * a.first_blocks) * 32 : piece.index * KEYS;
  int p0, p1;
  if constexpr (FIRST) {
    p0 = max(piece.index * static_cast<int>(a.first_tokens.d), a.window + x0);
    p1 = min(piece.index * static_cast<int>(a.first_tokens.d) + static_cast<int>(a.first_tokens.d), piece.n);
    if (!piece.real || p0 >= p1)
      return;
  } else {
    if (!piece.real) {
      const int tokens = min(KEYS, piece.n - x0);
      zero_rows(a, a.dk, piece.begin, x0, tokens, kv, 1);
      zero_rows(a, a.dv, piece.begin, x0, tokens, kv, 1);
      return;
    }
    p0 = x0;
    p1 = static_cast<int>(min(static_cast<int64_t>(piece.n), static_cast<int64_t>(x0) + KEYS - 1 + a.window));
  }
  if (a.dim < DP) {
    clear<64 * kWaves>(tiles, ROOM);
    __syncthreads();
  }
  const int per = (p1 - p0 + 31) >> 5; // tiles of a head
  const int count = per * group;
  const Loads bring(lane, TURNS ? 0 : wave * NT, a.dim);
  const uint32_t at = place(tiles), stats_at = place(reinterpret_cast<const char *>(&stats[0][0][0]));
  const uint32_t qrow = static_cast<uint32_t>(a.q.row) * 2, grow = static_cast<uint32_t>(a.dout.row) * 2;
  auto send = [&](int h, int i, int slot) { // the i-th tile of a head of the group
    const int p = p0 + i * 32, head = kv * group + h;
    const int64_t row = static_cast<int64_t>(piece.begin) + p;
    bring.send(a.q.data + (row * a.q.row + head * a.q.head) * 2, qrow, piece.n - p, at + slot * 2 * TILE);
    bring.send(a.dout.data + (row * a.dout.row + head * a.dout.head) * 2, grow, piece.n - p, at + slot * 2 * TILE + TILE);
    // 64 numbers of the tile's rows: each wave a quarter, TURNS: all
    const int number = TURNS ? lane : wave * 16 + lane;
    if (TURNS || lane < 16)
      load_async4(a.stats + static_cast<int64_t>(head) * 2 * a.rows + row, // rows: 2^29 at most
                  static_cast<uint32_t>(min(number & 31, piece.n - p - 1) + (number < 32 ? 0 : a.rows)) * 4,
                  stats_at + slot * 256 + (TURNS ? 0 : wave * 64));
  };
  constexpr int SENT = 2 * Loads::LOADS + 1;

  const int x_first = x0 + (TURNS ? 0 : wave * 32), x_last = x_first + 31, key = x_first + (lane & 31);
  const int64_t key_row = static_cast<int64_t>(piece.begin) + min(key, piece.n - 1);
  u32x4 k[KS], v[KS];
  take_row<DP>(k, a.k.data + (key_row * a.k.row + kv * a.k.head) * 2, a.dim, lane);
  take_row<DP>(v, a.v.data + (key_row * a.v.row + kv * a.v.head) * 2, a.dim, lane);
  const uint32_t direct = direct_at<RB>(lane), turn0 = turned_at<RB>(lane, 0), turn1 = turned_at<RB>(lane, 1);
  const uint32_t values_at = place(values) + (TURNS ? 0 : wave * 32 * RB) + direct;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    // TURNS: the same by all waves
    *reinterpret_cast<__attribute__((address_space(3))) u32x4 *>(values_at ^ (s * 32)) = v[s];
    asm volatile("" : "+v"(k[s]));
  }
  Over<T, E> over;
  f32x16 dk[E], dv[E];
#pragma unroll
  for (int m = 0; m < E; ++m)
    dk[m] = dv[m] = zero16();

  // Reads of shared memory go out a product or more ahead of their use, each where
  // the product before has freed its registers, and the order is kept: left to
  // itself the compiler, short of registers, waits for each read where it uses it.
  auto take_in = [&](int p, int slot) {
    const uint32_t tq = at + slot * 2 * TILE, tg = tq + TILE, st = stats_at + slot * 256 + (lane >> 5) * 16;
    // S and dP begin with -lse / scale and -D of their rows
    f32x16 s, dp;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 x = read16(st + i * 32);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        s[4 * i + r] = __uint_as_float(x[r]);
    }
    auto operand = [&](int n) {
      const int i = n % KS, m = i / 2 * 64, tokens = i % 2 * 16 * RB;
      return n < KS       ? read16(tq + direct ^ (i * 32))
             : n < 2 * KS ? read16(tg + direct ^ (i * 32))
             : n < 3 * KS ? turned((tg + turn0 ^ m) + tokens, (tg + turn1 ^ m) + tokens)
                          : turned((tq + turn0 ^ m) + tokens, (tq + turn1 ^ m) + tokens);
    };
    u32x4 ahead[kAhead], w[2];
#pragma unroll
    for (int n = 0; n < kAhead; ++n)
      ahead[n] = operand(n);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 x = read16(st + 128 + i * 32);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        dp[4 * i + r] = __uint_as_float(x[r]);
    }
    keep_order();
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      s = mfma32<T>(ahead[i % kAhead], k[i], s);
      ahead[i % kAhead] = operand(i + kAhead);
      if (i >= KS - 2)
        w[i - KS + 2] = read16(values_at ^ ((i - KS + 2) * 32));
      keep_order();
    }
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      dp = mfma32<T>(ahead[i % kAhead], w[i % 2], dp);
      ahead[i % kAhead] = operand(KS + i + kAhead);
      if (i + 2 < KS)
        w[i % 2] = read16(values_at ^ ((i + 2) * 32));
#pragma unroll
      for (int n = 16 / KS * i; n < 16 / KS * (i + 1); ++n)
        s[n] = __builtin_amdgcn_exp2f(T == kF16 ? s[n] * a.scale + kMore : s[n] * a.scale);
      keep_order();
    }
    const bool whole = p + 31 < p1 && (FIRST ? x_last < a.sinks && p - x_last >= a.window
                                             : x_last <= p && p + 31 - x_first < a.window);
    if (!whole) {
      // the rows from `low` on and before `high` see the lane's key
      const int at_row = p + 4 * (lane >> 5);
      const int low = (FIRST ? key < a.sinks ? key + a.window : p1 : key) - at_row;
      const int high = (FIRST ? p1 : static_cast<int>(min(static_cast<int64_t>(p1), static_cast<int64_t>(key) + a.window))) - at_row;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool sees = (row_of(i, 0) >= low) & (row_of(i, 0) < high);
        s[i] = sees ? s[i] : 0.0f;
        dp[i] = sees ? dp[i] : 0.0f;
      }
    }
    u32x4 p2[2];
    pack_operands<T>(s, p2);
    keep_order();
#pragma unroll
    for (int i = 0; i < 2 * E; ++i) {
      dv[i / 2] = mfma32<T>(ahead[i % kAhead], p2[i % 2], dv[i / 2]);
      ahead[i % kAhead] = operand(2 * KS + i + kAhead);
#pragma unroll
      for (int n = 16 / KS * i; n < 16 / KS * (i + 1); ++n)
        s[n] *= dp[n];
      keep_order();
    }
    over.hold(s, dk);
    if constexpr (T == kF16)
      s *= over.down();
    pack_operands<T>(s, p2);
#pragma unroll
    for (int i = 0; i < 2 * E; ++i) {
      dk[i / 2] = mfma32<T>(ahead[i % kAhead], p2[i % 2], dk[i / 2]);
      if (i + kAhead < KS)
        ahead[i % kAhead] = operand(3 * KS + i + kAhead);
      keep_order();
    }
  };

  if constexpr (TURNS) {
    int slot = wave * RING;
    if (wave < count)
      send(wave / per, wave % per, slot);
#pragma clang loop unroll(disable)
    for (int n = wave; n < count; n += kWaves, slot ^= 1) { // tiles of its own
      if (n + kWaves < count) {
        send((n + kWaves) / per, (n + kWaves) % per, slot ^ 1);
        arrived<SENT>();
      } else {
        arrived<0>();
      }
      take_in(p0 + n % per * 32, slot);
      shared_done(); // its place is free
    }
  } else {
    int slot = 0, in_head = 0, next_head = 0, next_in = 0; // of this tile, and the next to send
    auto send_next = [&](int to) {
      send(next_head, next_in, to);
      const bool end = next_in + 1 == per;
      next_head += end;
      next_in = end ? 0 : next_in + 1;
    };
    for (int n = 0; n < min(count, RING - 1); ++n)
      send_next(n);
#pragma clang loop unroll(disable)
    for (int n = 0; n < count; ++n) {
      if (n + RING - 2 < count)
        arrived<(RING - 2) * SENT>();
      else
        arrived<0>();
      meet();
      if (n + RING - 1 < count)
        send_next(slot == 0 ? RING - 1 : slot - 1);
      const int p = p0 + in_head * 32;
      if (p + 31 >= x_first && p - x_last < a.window)
        take_in(p, slot);
      slot = slot + 1 == RING ? 0 : slot + 1;
      in_head = in_head + 1 == per ? 0 : in_head + 1;
    }
    arrived<0>();
  }

  const float fk = a.plain_scale * over.up() * less<T>(), fv = less<T>();
  const int sinks = min(a.sinks, piece.n);
  // what the later rows, whose windows have left them, add to first tokens from
  // x_first on: `add` takes the place of each sum
  const int size = static_cast<int>(a.first_tokens.d);
  const bool more = !FIRST && x_first < sinks && a.window + x_first < piece.n;
  auto add_first = [&](auto add) {
    const int64_t base = first_piece<true>(a, a.first_tokens, piece.begin, piece.number);
    for (int c = (a.window + x_first) / size; static_cast<int64_t>(c) * size < piece.n; ++c)
      add(a.first_sums + ((base + c) * a.kv_heads + kv) * a.sinks * 2 * DP);
  };
  if constexpr (TURNS) {
    // the waves' sums, in order, keys' then values'
    float *room = reinterpret_cast<float *>(tiles);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int m = 0; m < E; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x16 &x = which ? dv[m] : dk[m];
          const float f = which ? fv : fk;
          *reinterpret_cast<f32x4 *>(room + (wave * 32 + (lane & 31)) * DP + 32 * m + 8 * i + 4 * (lane >> 5)) =
              f32x4{x[4 * i] * f, x[4 * i + 1] * f, x[4 * i + 2] * f, x[4 * i + 3] * f};
        }
      __syncthreads();
      for (int i = threadIdx.x * 4; i < min(32, (FIRST ? a.sinks : piece.n) - x0) * DP; i += 64 * kWaves * 4) {
        f32x4 sum = *reinterpret_cast<const f32x4 *>(room + i);
#pragma unroll
        for (int o = 1; o < kWaves; ++o)
          sum += *reinterpret_cast<const f32x4 *>(room + o * 32 * DP + i);
        const int x = x0 + i / DP, d = i % DP;
        const int64_t at_sum = (static_cast<int64_t>(x) * 2 + which) * DP + d;
        if constexpr (FIRST) {
          *reinterpret_cast<f32x4 *>(a.first_sums + (static_cast<int64_t>(w.number) * a.kv_heads + kv) * a.sinks * 2 * DP + at_sum) = sum;
        } else {
          if (more && x < sinks)
            add_first([&](const float *from) { sum += *reinterpret_cast<const f32x4 *>(from + at_sum); });
          const Heads &to = which ? a.dv : a.dk;
          if (d < a.dim)
            *reinterpret_cast<u32x2 *>(to.data + ((static_cast<int64_t>(piece.begin) + x) * to.row + kv * to.head + d) * 2) =
                u32x2{pack16<T>(sum[0], sum[1]), pack16<T>(sum[2], sum[3])};
        }
      }
    }
  } else {
#pragma unroll
    for (int m = 0; m < E; ++m) {
      dk[m] *= fk;
      dv[m] *= fv;
    }
    if (more && key < sinks)
      add_first([&](const float *from) {
        from += key * 2 * DP + 4 * (lane >> 5);
#pragma unroll
        for (int m = 0; m < E; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(from + 32 * m + 8 * i);
            const f32x4 y = *reinterpret_cast<const f32x4 *>(from + DP + 32 * m + 8 * i);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              dk[m][4 * i + r] += x[r];
              dv[m][4 * i + r] += y[r];
            }
          }
      });
    if (key < piece.n) {
      put_row<T, DP>(a.dk.data + (key_row * a.dk.row + kv * a.dk.head) * 2, dk, 1.0f, a.dim, lane);
      put_row<T, DP>(a.dv.data + (key_row * a.dv.row + kv * a.dv.head) * 2, dv, 1.0f, a.dim, lane);
    }
  }
}

// ------------------------------------------------------------ launches

inline hipError_t window_start(const void *kernel, WindowArgs a, int64_t items, hipStream_t s) {
  void *pa[] = {&a};
  return hipLaunchKernel(kernel, dim3(static_cast<uint32_t>((items + 7) / 8 * 8)), dim3(64 * kWaves), pa, 0, s);
}

template <int T, int DP> hipError_t window_forward(const WindowArgs &a, hipStream_t s) {
  return window_start(reinterpret_cast<const void *>(k_window_forward<T, DP>), a,
                      static_cast<int64_t>(a.row_pieces) * a.kv_heads * a.parts, s);
}

template <int T, int DP> hipError_t window_backward(const WindowArgs &a, hipStream_t s) {
  const int64_t tiles = static_cast<int64_t>(a.row_pieces) * a.kv_heads * a.parts;
  hipError_t e = hipSuccess;
  const int64_t few = a.few_pieces ? static_cast<int64_t>(a.sequences) * a.few_pieces * a.kv_heads * a.parts : tiles;
  if (few > 0)
    e = window_start(reinterpret_cast<const void *>(k_window_dq<T, DP, true>), a, few, s);
  if (e == hipSuccess)
    e = window_start(reinterpret_cast<const void *>(k_window_dq<T, DP, false>), a, tiles, s);
  if (e == hipSuccess && a.sinks > 0)
    e = window_start(reinterpret_cast<const void *>(k_window_dkv<T, DP, kFirst>), a,
                     static_cast<int64_t>(a.first_pieces) * a.kv_heads * a.first_blocks, s);
  if (e == hipSuccess)
    e = window_start(a.key_tokens.d == 32 ? reinterpret_cast<const void *>(k_window_dkv<T, DP, kNarrow>)
                                            : reinterpret_cast<const void *>(k_window_dkv<T, DP, kWide>),
                     a,
                     static_cast<int64_t>(a.key_pieces) * a.kv_heads, s);
  return e;
}

template <int T> hipError_t window_by_width(const WindowArgs &a, bool back, hipStream_t s) {
  if (back)
    return a.dim <= 64 ? window_backward<T, 64>(a, s) : window_backward<T, 128>(a, s);
  return a.dim <= 64 ? window_forward<T, 64>(a, s) : window_forward<T, 128>(a, s);
}

} // namespace
} // namespace relx
