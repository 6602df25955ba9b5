// k_blocks.hip - a step's keys and values into an int8 cache whose blocks of
// tokens have a scale each for every head.
//
//   scale' = max(amax of the block's new tokens / 127, 2^-126, the scale so far
//            where the block holds tokens of the request already)
//   codes  round(x / scale') of the new tokens; of those already there
//          round(q scale / scale'), where the scale has grown
//
// A wave takes one block of one head, keys or values: no two waves write to one
// scale, and nothing needs an order among them. Which block is worked out from
// the wave's number: request b's blocks are the numbers from starts[b] / block +
// 2 b on, since n tokens in a row touch at most n / block + 2 blocks; numbers
// that are left over have nothing to do. Lanes compare 64 requests at a time
// with the number, so a batch of up to 64 costs one read.
//
// A block's tokens stay in the registers between the pass that finds their
// largest magnitude and the one that rounds, up to `kHold` reads of a lane;
// those past them are read again, from the cache that the first pass filled.
//
// Measured, 8 key heads of 128 in bf16: 12.9k rows of four requests 18.7 us (79 MB,
// 4.2 TB/s; bound by how long its few waves' reads take), 48k rows of sixteen 52 (5.6
// TB/s), 64 rows of one token each 4.9, where the chain of reads that find a block is
// all of it.
#include "attention.h"
#include "index.h"

namespace relx {
namespace {

constexpr int kWaves = 4;
constexpr float kLeast = 1.17549435e-38f; // 2^-126: its inverse is finite

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <class T> struct __attribute__((packed)) Loose { T v; };
template <class T> __device__ __forceinline__ T load(const void *p) {
  return static_cast<const Loose<T> *>(p)->v;
}
template <class T> __device__ __forceinline__ T load_past(const void *p) {
  return __builtin_nontemporal_load(&static_cast<const Loose<T> *>(p)->v);
}
template <class T> __device__ __forceinline__ void store(void *p, const T &v) {
  static_cast<Loose<T> *>(p)->v = v;
}

template <int T> constexpr int width() { return T == kF32 ? 4 : 2; }

// Eight elements of a row, the first `n` of them there, as they lie in memory.
template <int T> struct Raw {
  u32x4 w[T == kF32 ? 2 : 1];
  __device__ __forceinline__ void take(const char *p, int n) {
    if (n >= 8) {
      w[0] = load<u32x4>(p);
      if constexpr (T == kF32)
        w[1] = load<u32x4>(p + 16);
      return;
    }
    w[0] = u32x4{0u, 0u, 0u, 0u};
    if constexpr (T == kF32)
      w[1] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) {
        if constexpr (T == kF32)
          w[i >> 2][i & 3] = load<uint32_t>(p + i * 4);
        else
          w[0][i >> 1] |= static_cast<uint32_t>(load<uint16_t>(p + i * 2)) << (16 * (i & 1));
      }
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (T == kF32)
      return __uint_as_float(w[i >> 2][i & 3]);
    const uint32_t h = w[0][i >> 1] >> (16 * (i & 1)) & 0xffffu;
    if constexpr (T == kF16)
      return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
    else
      return __uint_as_float(h << 16);
  }
  // The largest finite magnitude.
  __device__ __forceinline__ float most() const {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = fabsf(at(i));
      m = fmaxf(m, x < __builtin_inff() ? x : 0.0f);
    }
    return m;
  }
};

// clamp(round half even(x * inv)) to a byte, as the quantize stage rounds:
// adding 1.5 * 2^23 leaves the integer in the low bits.
__device__ __forceinline__ uint32_t quantize(float x, float inv) {
  float y = x * inv;
  y = __builtin_fmaxf(y, -128.0f);
  y = __builtin_fminf(y, 127.0f);
  return __float_as_uint(y + 12582912.0f) & 0xffu;
}

__device__ __forceinline__ void put_codes(char *p, u32x2 b, int n) {
  if (n >= 8) {
    store(p, b);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n)
      p[i] = static_cast<char>(b[i >> 2] >> (8 * (i & 3)));
}

// L lanes hold a token's head, eight elements each.
template <int T, int L> __global__ __launch_bounds__(64 * kWaves) void k_block_append(BlockArgs a) {
  constexpr int kTokens = 64 / L;               // of a read
  constexpr int kHold = T == kF32 ? 8 : 16;     // reads that stay in registers
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int which = static_cast<int>(blockIdx.y) * kWaves + wave;
  if (which >= 2 * a.kv_heads)
    return;
  const int kind = which >= a.kv_heads, head = which - kind * a.kv_heads;
  const int64_t number = blockIdx.x;
  const int block = static_cast<int>(a.block.d), page = static_cast<int>(a.page.d);

  // the last request whose first number is at most this one
  int lo = 0, hi = a.requests, st = 0, en = 0, have = 0;
  for (;;) {
    const int step = (hi - lo + 63) >> 6, b = lo + lane * step;
    bool upto = false;
    if (b < hi) {
      st = min(max(a.starts[b], 0), a.rows);
      if (step == 1) {
        en = a.starts[b + 1];
        have = a.cached[b];
      }
      upto = static_cast<int64_t>(fdiv(static_cast<uint32_t>(st), a.block)) + 2 * static_cast<int64_t>(b) <= number;
    }
    const uint64_t not_yet = ~__ballot(upto);
    const int n = max(not_yet ? __builtin_ctzll(not_yet) : 64, 1) - 1;
    lo += n * step;
    if (step == 1) {
      st = __builtin_amdgcn_readlane(st, n);
      en = __builtin_amdgcn_readlane(en, n);
      have = __builtin_amdgcn_readlane(have, n);
      break;
    }
    hi = min(hi, lo + step);
  }
  const int room = a.columns * page; // at most 2^30
  have = min(max(have, 0), room);
  const int fresh = min(min(max(en, st), a.rows) - st, room - have);
  const int64_t i = number - fdiv(static_cast<uint32_t>(st), a.block) - 2 * static_cast<int64_t>(lo);
  const int64_t first64 = (static_cast<int64_t>(fdiv(static_cast<uint32_t>(have), a.block)) + i) * block;
  if (i < 0 || first64 >= static_cast<int64_t>(have) + fresh)
    return;
  const int first = static_cast<int>(first64); // the block's first place
  const int from = max(first, have), upto = min(first + block, have + fresh);
  const int column = static_cast<int>(fdiv(static_cast<uint32_t>(first), a.page)), off = first - column * page;
  const int id = a.table[lo * a.table_row + column];

  const int dim = (lane % L) * 8, n = a.dim - dim; // the lane's first element, and how many from there
  const int mine = from + lane / L;                // the lane's token of the first read
  const char *src = a.x[kind].data +
                    ((st + static_cast<int64_t>(mine - have)) * a.x[kind].row + head * a.x[kind].head + dim) * width<T>();
  const int64_t pace = kTokens * a.x[kind].row * width<T>();

  Raw<T> held[kHold];
  float most = 0.0f;
#pragma unroll
  for (int k = 0; k < kHold; ++k)
    if (mine + k * kTokens < upto && n > 0)
      held[k].take(src + k * pace, n);
#pragma unroll
  for (int k = 0; k < kHold; ++k)
    if (mine + k * kTokens < upto && n > 0)
      most = fmaxf(most, held[k].most());
  for (int x = mine + kHold * kTokens, k = kHold; x < upto; x += kTokens, ++k)
    if (n > 0) {
      Raw<T> r;
      r.take(src + k * pace, n);
      most = fmaxf(most, r.most());
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    most = fmaxf(most, __shfl_xor(most, o));
  if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.pages))
    return;

  float *scale_at = a.scale[kind] + id * a.scale_page + fdiv(static_cast<uint32_t>(off), a.block) * a.scale_block +
                    head * a.scale_head;
  const float old = from > first ? *scale_at : 0.0f;
  const float scale = fmaxf(fmaxf(most * static_cast<float>(1.0 / 127.0), old), kLeast);
  const float inv = 1.0f / scale;
  char *cells = a.cache[kind] + id * a.page_stride[kind] + head * a.head_stride[kind] + dim;
  const int64_t slot = a.slot_stride[kind];

  if (from > first && scale != old) {
    const float shrink = old * inv;
    for (int x = first + lane / L; x < from; x += kTokens)
      if (n > 0) {
        char *at = cells + (off + x - first) * slot;
        u32x2 b = {0u, 0u};
        if (n >= 8) {
          b = load<u32x2>(at);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < n)
              b[e >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(at[e])) << (8 * (e & 3));
        }
        u32x2 out = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int q = static_cast<int>(b[e >> 2] << (24 - 8 * (e & 3))) >> 24;
          out[e >> 2] |= quantize(static_cast<float>(q), shrink) << (8 * (e & 3));
        }
        put_codes(at, out, n);
      }
  }
  auto round_to = [&](const Raw<T> &r, int x) {
    u32x2 b = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      b[e >> 2] |= quantize(r.at(e), inv) << (8 * (e & 3));
    put_codes(cells + (off + x - first) * slot, b, n);
  };
#pragma unroll
  for (int k = 0; k < kHold; ++k)
    if (mine + k * kTokens < upto && n > 0)
      round_to(held[k], mine + k * kTokens);
  for (int x = mine + kHold * kTokens, k = kHold; x < upto; x += kTokens, ++k)
    if (n > 0) {
      Raw<T> r;
      r.take(src + k * pace, n);
      round_to(r, x);
    }
  if (lane == 0)
    *scale_at = scale;
}

template <int T, int L> hipError_t start(const BlockArgs &args, hipStream_t s) {
  BlockArgs a = args;
  void *pa[] = {&a};
  const uint32_t numbers = static_cast<uint32_t>(a.rows) / a.block.d + 2u * static_cast<uint32_t>(a.requests) + 1u;
  return hipLaunchKernel(reinterpret_cast<const void *>(k_block_append<T, L>),
                         dim3(numbers, static_cast<uint32_t>((2 * a.kv_heads + kWaves - 1) / kWaves)), dim3(64 * kWaves), pa, 0, s);
}

template <int T> hipError_t by_width(const BlockArgs &a, hipStream_t s) {
  return a.dim <= 64 ? start<T, 8>(a, s) : a.dim <= 128 ? start<T, 16>(a, s) : a.dim <= 256 ? start<T, 32>(a, s) : start<T, 64>(a, s);
}

} // namespace

hipError_t blocks_launch(const BlockArgs &a, int type, hipStream_t s) {
  return type == kF32 ? by_width<kF32>(a, s) : type == kF16 ? by_width<kF16>(a, s) : by_width<kBF16>(a, s);
}

} // namespace relx
