// k_rotate.hip - per-head norms of queries and keys with the position
// rotation in the same pass: forward, backward, and the serving form that
// puts keys and values into a paged cache.
//
// A head lies over L = 8..64 lanes, eight elements each, so a wave holds
// 64 / L heads per row of its block of heads; sums over a head stay in
// registers (DPP), and a rotated element's partner comes from another lane
// (or, where halves do not begin on a lane, through shared memory). A block
// of heads belongs to one kind (queries, keys, values), so a wave keeps its
// weights, and walks the rows of the batch: a row's angles are loaded once
// for all heads of the block.
//
//   forward   n = x / sqrt(mean(x^2) + eps), y = n w, z = R(position) y
//   backward  g = R^T dz, u = g w, dx = (u - n mean(u n)) / sqrt(..),
//             dw = sum over rows and heads of g n
//
// Bound by bytes: everything is read once and written once, past the caches.
// What decides is how much is on its way, so a wave loads its next row before
// it works on this one. 32768 rows of 32 + 8 heads of 128 in bf16, from views
// of a fused projection: forward 125 us (5.4 TB/s; 119 now and then; 177 without
// the next row ahead, 155 with stores through the caches), backward with the
// weights' gradients 185 to 188 us (5.4 TB/s; 310 before). 8192 rows into a cache
// 78 us (5.2 TB/s; 113 before). The sums of the weights' gradients are added block
// by block in a fixed order by a second launch (4 us): no atomics.
#include "attention.h"
#include "index.h"

namespace relx {
namespace {

constexpr int kWaves = 4;
constexpr int kV = 8; // elements of a lane

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// A vector that may lie at any element's address.
template <class T> struct __attribute__((packed)) Loose { T v; };
template <class T> __device__ __forceinline__ T load(const void *p) {
  return static_cast<const Loose<T> *>(p)->v;
}
template <class T> __device__ __forceinline__ void store(void *p, const T &v) {
  static_cast<Loose<T> *>(p)->v = v;
}

template <class T> __device__ __forceinline__ void store_past(void *p, const T &v) {
  __builtin_nontemporal_store(v, &static_cast<Loose<T> *>(p)->v);
}

// The same for the whole wave: through the scalar cache, which does not queue
// behind the vector loads in flight.
template <class T> __device__ __forceinline__ T scalar_load(const T *p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) T *>(reinterpret_cast<uint64_t>(p));
}

template <int T> constexpr int width() { return T == kF32 ? 4 : 2; }

template <int T> __device__ __forceinline__ float widen16(uint32_t h) {
  if constexpr (T == kF16)
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
  else
    return __uint_as_float(h << 16);
}

// Two values rounded to nearest even.
template <int T> __device__ __forceinline__ uint32_t pack16(float x, float y) {
  const f32x2 v = {x, y};
  if constexpr (T == kF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// Eight elements as they lie in memory, of which the first `n` are the head's
// (the others zero). Loads are nothing but loads, so they can be on their way
// while the row before is worked on. Everything is read once: past the caches.
template <int T> struct Raw {
  u32x4 v[T == kF32 ? 2 : 1];
};
template <int T> __device__ __forceinline__ Raw<T> load_raw(const char *p, int n) {
  Raw<T> r;
  if (n >= kV) {
#pragma unroll
    for (int i = 0; i < (T == kF32 ? 2 : 1); ++i)
      r.v[i] = __builtin_nontemporal_load(&reinterpret_cast<const Loose<u32x4> *>(p + i * 16)->v);
    return r;
  }
  uint32_t b[T == kF32 ? kV : kV / 2] = {};
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    if constexpr (T == kF32)
      b[e] = e < n ? load<uint32_t>(p + e * 4) : 0u;
    else
      b[e >> 1] |= (e < n ? load<uint16_t>(p + e * 2) : 0u) << ((e & 1) * 16);
  }
#pragma unroll
  for (int i = 0; i < (T == kF32 ? 2 : 1); ++i)
    r.v[i] = u32x4{b[i * 4], b[i * 4 + 1], b[i * 4 + 2], b[i * 4 + 3]};
  return r;
}
template <int T> __device__ __forceinline__ void widen(const Raw<T> &r, float *v) {
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    if constexpr (T == kF32)
      v[e] = __uint_as_float(r.v[e >> 2][e & 3]);
    else
      v[e] = widen16<T>((r.v[0][e >> 1] >> ((e & 1) * 16)) & 0xffffu);
  }
}

template <int T> __device__ __forceinline__ void store8(char *p, int n, const float *v) {
  if (n >= kV) {
    if constexpr (T == kF32) {
      store_past(p, f32x4{v[0], v[1], v[2], v[3]});
      store_past(p + 16, f32x4{v[4], v[5], v[6], v[7]});
    } else {
      store_past(p, u32x4{pack16<T>(v[0], v[1]), pack16<T>(v[2], v[3]), pack16<T>(v[4], v[5]),
                          pack16<T>(v[6], v[7])});
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < kV; ++e)
    if (e < n) {
      if constexpr (T == kF32)
        store(p + e * 4, v[e]);
      else
        store(p + e * 2, static_cast<uint16_t>(pack16<T>(v[e], 0.0f)));
    }
}

__device__ __forceinline__ void load_weight(const void *w, int type, int at, int n, float *v) {
#pragma unroll
  for (int e = 0; e < kV; ++e)
    v[e] = e < n ? 1.0f : 0.0f;
  if (!w || n <= 0)
    return;
  const char *p = static_cast<const char *>(w) + static_cast<int64_t>(at) * (type == kF32 ? 4 : 2);
  if (type == kF32)
    widen(load_raw<kF32>(p, n), v);
  else if (type == kF16)
    widen(load_raw<kF16>(p, n), v);
  else
    widen(load_raw<kBF16>(p, n), v);
}

template <int CTRL> __device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// The sum over a head's L lanes, in each of them.
template <int L> __device__ __forceinline__ float head_sum(float x) {
  x += dpp<0xb1>(x);  // quad_perm 1 0 3 2
  x += dpp<0x4e>(x);  // quad_perm 2 3 0 1
  x += dpp<0x141>(x); // row_half_mirror: the other four of eight
  if constexpr (L >= 16)
    x += dpp<0x140>(x); // row_mirror: the other eight of sixteen
  if constexpr (L >= 32)
    x += __shfl_xor(x, 16);
  if constexpr (L >= 64)
    x += __shfl_xor(x, 32);
  return x;
}

// Where a lane's rotation takes its partners from.
enum Partner : int { kPairs, kLanes, kShared };

struct Turn {
  Partner how;
  int first; // the lane's first element
  int half, rotary;
  int from; // kLanes: the partner's lane
};

template <int L>
__device__ __forceinline__ Turn make_turn(const RotateArgs &a, int lane, int first) {
  Turn t;
  t.first = first;
  t.rotary = a.rotary;
  t.half = a.rotary >> 1;
  t.how = a.pairs ? kPairs : t.half % kV == 0 ? kLanes : kShared;
  t.from = lane;
  if (t.how == kLanes && first < t.rotary)
    t.from = first < t.half ? lane + t.half / kV : lane - t.half / kV;
  return t;
}

// The angles of the lane's elements at a row's position (kPairs: four, of two
// elements each).
struct Angles {
  f32x4 c[2], s[2];
};
__device__ __forceinline__ Angles load_angles(const RotateArgs &a, const Turn &t, int64_t position) {
  Angles r = {};
  if (position < 0 || position >= a.angles) { // loud, and nothing read
    const float nan = __builtin_nanf("");
    r.c[0] = r.c[1] = f32x4{nan, nan, nan, nan};
    return r;
  }
  if (t.first >= t.rotary)
    return r;
  const float *c = a.cos + position * t.half, *s = a.sin + position * t.half;
  if (t.how == kPairs && t.first + kV <= t.rotary) {
    r.c[0] = load<f32x4>(c + (t.first >> 1));
    r.s[0] = load<f32x4>(s + (t.first >> 1));
  } else if (t.how == kLanes) {
    const int at = t.first < t.half ? t.first : t.first - t.half;
    r.c[0] = load<f32x4>(c + at);
    r.c[1] = load<f32x4>(c + at + 4);
    r.s[0] = load<f32x4>(s + at);
    r.s[1] = load<f32x4>(s + at + 4);
  } else {
    // some of the lane's elements do not turn, or turn in the other half:
    // what they load is not used
    float vc[kV], vs[kV];
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      const int i = t.first + e;
      const int at = min(t.how == kPairs ? (t.first >> 1) + e : i < t.half ? i : i - t.half, t.half - 1);
      vc[e] = c[at];
      vs[e] = s[at];
    }
    r.c[0] = f32x4{vc[0], vc[1], vc[2], vc[3]};
    r.c[1] = f32x4{vc[4], vc[5], vc[6], vc[7]};
    r.s[0] = f32x4{vs[0], vs[1], vs[2], vs[3]};
    r.s[1] = f32x4{vs[4], vs[5], vs[6], vs[7]};
  }
  return r;
}

// cos and sin of each of the lane's elements, sin with the sign that its
// partner's product takes: z = y * cos + partner * sin.
__device__ __forceinline__ void angles(const Turn &t, const Angles &r, float *co, float *si) {
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    if (t.how == kPairs) {
      co[e] = r.c[0][e >> 1];
      si[e] = e & 1 ? r.s[0][e >> 1] : -r.s[0][e >> 1];
    } else {
      co[e] = r.c[e >> 2][e & 3];
      si[e] = t.first + e < t.half ? -r.s[e >> 2][e & 3] : r.s[e >> 2][e & 3];
    }
  }
}

// Each element's partner (itself where it does not turn). `room`: this wave's
// shared memory, [64 / L heads][L * 8 + 4].
template <int L>
__device__ __forceinline__ void partners(const Turn &t, int lane, const float *y, float *p,
                                         float *room) {
  if (t.how == kPairs) {
#pragma unroll
    for (int e = 0; e < kV; ++e)
      p[e] = y[e ^ 1];
  } else if (t.how == kLanes) {
#pragma unroll
    for (int e = 0; e < kV; ++e)
      p[e] = __shfl(y[e], t.from);
  } else {
    float *head = room + (lane / L) * (L * kV + 4);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int v = 0; v < kV; v += 4)
      *reinterpret_cast<f32x4 *>(head + t.first + v) = f32x4{y[v], y[v + 1], y[v + 2], y[v + 3]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      const int i = t.first + e;
      p[e] = head[i < t.half ? i + t.half : i < t.rotary ? i - t.half : i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// clamp(round half even(x * inv)) to a byte, as the quantize stage rounds:
// NaN to -128.
__device__ __forceinline__ uint32_t quantize(float x, float inv) {
  float y = x * inv;
  y = __builtin_fmaxf(y, -128.0f);
  y = __builtin_fminf(y, 127.0f);
  return __float_as_uint(y + 12582912.0f) & 0xffu;
}

template <int T, int L, int U, int FORM>
__global__ __launch_bounds__(64 * kWaves) void k_rotate(RotateArgs a) {
  constexpr int W = width<T>();
  constexpr int H = 64 / L; // heads of a wave at a time
  constexpr bool kBack = FORM == kRotateBackward;
  constexpr bool kServe = FORM == kRotateAppend || FORM == kRotateAppendI8;
  __shared__ float room[kWaves][H * (L * kV + 4)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int chunk = blockIdx.y, kind = 0;
  while (chunk >= a.chunks[kind])
    chunk -= a.chunks[kind++];
  const int first = (lane & (L - 1)) * kV;
  const int n = min(a.dim - first, kV); // the lane's elements (none: <= 0)
  const bool turns = kind < 2;
  float w[kV], dw[kV];
#pragma unroll
  for (int e = 0; e < kV; ++e)
    dw[e] = 0.0f;
  if (turns)
    load_weight(a.weight[kind], a.weight_type, first, n, w);
  const Turn t = make_turn<L>(a, lane, first);

  const int heads = a.heads[kind < 2 ? kind : 1];
  const int head0 = chunk * a.chunk_heads + lane / L;
  bool live[U];
  float inv[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    live[u] = u * H < a.chunk_heads && head0 + u * H < heads && n > 0;
    inv[u] = 0.0f;
    if constexpr (FORM == kRotateAppendI8)
      if (live[u] && kind > 0)
        inv[u] = 1.0f / a.scale[kind - 1][head0 + u * H];
  }
  const Heads xs = a.x[kind];

  // The next row's elements and angles are on their way while a row is worked
  // on, and the position of the one after it.
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWaves;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(wave);
  int64_t position = turns && row < a.rows ? scalar_load(a.positions + row) : 0;
  Raw<T> next_x[U] = {}, next_dz[kBack ? U : 1] = {};
  Angles next_angles = {};
  int64_t next_slot = -1;
  auto fetch = [&](int64_t r) {
    if (r >= a.rows)
      return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t head = head0 + u * H;
      if (live[u]) {
        next_x[u] = load_raw<T>(xs.data + (r * xs.row + head * xs.head + first) * W, n);
        if constexpr (kBack)
          next_dz[u] = load_raw<T>(a.dz[kind].data + (r * a.dz[kind].row + head * a.dz[kind].head + first) * W, n);
      }
    }
    if (turns) {
      next_angles = load_angles(a, t, position);
      if (r + step < a.rows)
        position = scalar_load(a.positions + r + step);
    }
    if (kServe && kind > 0)
      next_slot = scalar_load(a.slots + r);
  };
  fetch(row);
  for (; row < a.rows; row += step) {
    Raw<T> now_x[U], now_dz[kBack ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      now_x[u] = next_x[u];
      if constexpr (kBack)
        now_dz[u] = next_dz[u];
    }
    const Angles now_angles = next_angles;
    const int64_t slot = next_slot;
    fetch(row + step);
    int64_t cache_at = 0;
    if constexpr (kServe) {
      if (kind > 0) {
        if (slot < 0 || slot >= a.pages_slots)
          continue;
        const uint32_t page = fdiv(static_cast<uint32_t>(slot), a.page);
        cache_at = page * a.cache_page[kind - 1] +
                   (static_cast<uint32_t>(slot) - page * a.page.d) * a.cache_slot[kind - 1];
      }
    }
    float co[kV], si[kV];
    if (turns)
      angles(t, now_angles, co, si);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (chunk * a.chunk_heads + u * H >= heads || u * H >= a.chunk_heads)
        break; // no heads left: the same for the whole wave
      const int64_t head = head0 + u * H;
      float x[kV], dz[kV];
      widen(now_x[u], x);
      if constexpr (kBack)
        widen(now_dz[u], dz);
      float z[kV];
      if (kServe && !turns) {
#pragma unroll
        for (int e = 0; e < kV; ++e)
          z[e] = x[e];
      } else if constexpr (!kBack) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < kV; ++e)
          ss += x[e] * x[e];
        const float r = rsqrtf(head_sum<L>(ss) * a.inv_dim + a.eps);
        float y[kV], p[kV];
#pragma unroll
        for (int e = 0; e < kV; ++e)
          y[e] = x[e] * r * w[e];
        partners<L>(t, lane, y, p, room[wave]);
#pragma unroll
        for (int e = 0; e < kV; ++e)
          z[e] = first + e < a.rotary ? y[e] * co[e] + p[e] * si[e] : y[e];
      } else {
        // the transposed rotation: the partner's product with the other sign
        float g[kV], p[kV], ss = 0.0f, ux = 0.0f;
        partners<L>(t, lane, dz, p, room[wave]);
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          g[e] = first + e < a.rotary ? dz[e] * co[e] - p[e] * si[e] : dz[e];
          ss += x[e] * x[e];
          ux += g[e] * w[e] * x[e];
        }
        // lanes without a head add nothing to the weight's gradient, also where
        // eps = 0 makes their root infinite
        const float mean = head_sum<L>(ss) * a.inv_dim;
        const float r = live[u] ? rsqrtf(mean + a.eps) : 0.0f;
        const float m = head_sum<L>(ux) * r * a.inv_dim; // mean(u n)
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          const float nx = x[e] * r;
          dw[e] += g[e] * nx;
          z[e] = r * (g[e] * w[e] - nx * m);
        }
      }
      if (!live[u])
        continue;
      if (kServe && kind > 0) {
        const int64_t at = cache_at + head * a.cache_head[kind - 1] + first;
        if constexpr (FORM == kRotateAppendI8) {
          uint32_t b[2] = {0u, 0u};
#pragma unroll
          for (int e = 0; e < kV; ++e)
            b[e >> 2] |= quantize(z[e], inv[u]) << ((e & 3) * 8);
          char *o = a.cache[kind - 1] + at;
          if (n >= kV) {
            store(o, static_cast<uint64_t>(b[1]) << 32 | b[0]);
          } else {
#pragma unroll
            for (int e = 0; e < kV; ++e)
              if (e < n)
                o[e] = static_cast<char>(b[e >> 2] >> ((e & 3) * 8));
          }
        } else {
          store8<T>(a.cache[kind - 1] + at * W, n, z);
        }
      } else {
        store8<T>(a.y[kind].data + (row * a.y[kind].row + head * a.y[kind].head + first) * W, n, z);
      }
    }
  }

  if constexpr (kBack) {
    if (!a.weight_grad[kind])
      return;
    // the block's part of the weight's gradient, its heads and waves added in
    // a fixed order
#pragma unroll
    for (int o = L; o < 64; o <<= 1)
#pragma unroll
      for (int e = 0; e < kV; ++e)
        dw[e] += __shfl_xor(dw[e], o);
    float *sum = &room[0][0]; // [kWaves][L * kV]
    __syncthreads();
    if (lane < L)
#pragma unroll
      for (int e = 0; e < kV; ++e)
        sum[wave * L * kV + lane * kV + e] = dw[e];
    __syncthreads();
    const int64_t part = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
    for (int i = threadIdx.x; i < a.dim; i += 64 * kWaves) {
      float v = sum[i];
#pragma unroll
      for (int k = 1; k < kWaves; ++k)
        v += sum[k * L * kV + i];
      a.partial[part * a.dim + i] = v;
    }
  }
}

// The weights' gradients from the blocks' parts: a block sums 64 elements,
// its sixteen waves a sixteenth of the parts each.
__global__ __launch_bounds__(1024) void k_weight_grad(const float *partial, int parts_q, int parts_k,
                                                      int dim, float *q, float *k) {
  __shared__ float sum[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = blockIdx.x * 64 + lane;
  const bool keys = blockIdx.y != 0;
  float *out = keys ? k : q;
  if (!out)
    return;
  const float *p = partial + (keys ? static_cast<int64_t>(parts_q) * dim : 0);
  const int parts = keys ? parts_k : parts_q;
  float v = 0.0f;
  if (i < dim)
#pragma unroll 8
    for (int j = wave; j < parts; j += 16)
      v += p[static_cast<int64_t>(j) * dim + i];
  sum[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && i < dim) {
    for (int w = 1; w < 16; ++w)
      v += sum[w][lane];
    out[i] = v;
  }
}

template <int T, int L, int U> const void *kernel_of(int form) {
  switch (form) {
  case kRotateForward:
    return reinterpret_cast<const void *>(k_rotate<T, L, U, kRotateForward>);
  case kRotateBackward:
    return reinterpret_cast<const void *>(k_rotate<T, L, U, kRotateBackward>);
  case kRotateAppend:
    return reinterpret_cast<const void *>(k_rotate<T, L, U, kRotateAppend>);
  default:
    return reinterpret_cast<const void *>(k_rotate<T, L, U, kRotateAppendI8>);
  }
}

template <int T> const void *kernel_for(int lanes, int form) {
  switch (lanes) {
  case 8:
    return kernel_of<T, 8, 2>(form);
  case 16:
    return kernel_of<T, 16, 2>(form);
  case 32:
    return kernel_of<T, 32, 2>(form);
  default:
    return kernel_of<T, 64, 2>(form);
  }
}

} // namespace

int rotate_lanes(int dim) {
  int l = 8;
  while (l * kV < dim)
    l <<= 1;
  return l;
}

int rotate_blocks(int form, int64_t rows, int64_t chunks) {
  const int64_t blocks = (rows + kWaves - 1) / kWaves;
  // As many waves as the card holds at once (three on a SIMD), or twice that
  // where no block leaves a part of a sum. 32768 rows of 40 heads of 128, bf16,
  // in a kernel trace: forward 135 us with 1024 or 2048 blocks, 141 with 4096, 158 with 8192;
  // backward 188 with 768, 190 with 1536, 195 with 2048.
  const int64_t most = 256 * (form == kRotateBackward ? 3 : 8);
  const int64_t cap = most / chunks > 0 ? most / chunks : 1;
  return static_cast<int>(blocks < cap ? blocks : cap);
}

hipError_t rotate_launch(const RotateArgs &a, int form, int type, hipStream_t s) {
  RotateArgs args = a;
  const int lanes = rotate_lanes(a.dim);
  const int chunks = a.chunks[0] + a.chunks[1] + a.chunks[2];
  const int blocks = chunks ? rotate_blocks(form, a.rows, chunks) : 0;
  const void *k = type == kF32   ? kernel_for<kF32>(lanes, form)
                  : type == kF16 ? kernel_for<kF16>(lanes, form)
                                 : kernel_for<kBF16>(lanes, form);
  void *p[] = {&args};
  hipError_t e = hipSuccess;
  if (blocks)
    e = hipLaunchKernel(k, dim3(static_cast<uint32_t>(blocks), static_cast<uint32_t>(chunks)),
                        dim3(64 * kWaves), p, 0, s);
  if (e != hipSuccess || form != kRotateBackward || (!a.weight_grad[0] && !a.weight_grad[1]))
    return e;
  const float *partial = a.partial;
  int parts_q = blocks * a.chunks[0], parts_k = blocks * a.chunks[1], dim = a.dim;
  float *q = a.weight_grad[0], *kw = a.weight_grad[1];
  void *p2[] = {&partial, &parts_q, &parts_k, &dim, &q, &kw};
  return hipLaunchKernel(reinterpret_cast<const void *>(k_weight_grad),
                         dim3(static_cast<uint32_t>((dim + 63) / 64), 2), dim3(1024), p2, 0, s);
}

} // namespace relx
