// k_attend_wave.h - what the attention kernels share: vectors, a wave's scalars, matrix
// instructions, reads of shared memory and loads into it.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention.h"

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

template <class T> struct __attribute__((packed)) Loose { T v; };
template <class T> __device__ __forceinline__ T load(const char *p) {
  return reinterpret_cast<const Loose<T> *>(p)->v;
}
template <class T> __device__ __forceinline__ void store(char *p, const T &v) {
  reinterpret_cast<Loose<T> *>(p)->v = v;
}

// Reads that are the same for the whole wave, through the scalar cache: they
// do not queue behind the vector loads in flight.
__device__ __forceinline__ int32_t scalar_load(const int32_t *p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int32_t *>(reinterpret_cast<uint64_t>(p));
}

__device__ __forceinline__ float scalar_load(const float *p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) float *>(reinterpret_cast<uint64_t>(p));
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t of_lane(int64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(x), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(static_cast<uint64_t>(x) >> 32), lane);
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}
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

// Keeps the scheduler from moving anything across.
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }

// The same number, of which the compiler no longer knows what it is: what is
// worked out from it in a loop stays there instead of filling registers outside.
__device__ __forceinline__ int anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <int T> __device__ __forceinline__ float widen16(uint32_t h) {
  if constexpr (T == kF16)
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
  else
    return __uint_as_float(h << 16);
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

typedef __attribute__((address_space(3))) char lds_char;
typedef short i16x4 __attribute__((ext_vector_type(4)));

// A shared array's place.
__device__ __forceinline__ uint32_t place(const char *p) {
  return uniform(static_cast<int>(reinterpret_cast<uintptr_t>((lds_char *)const_cast<char *>(p))));
}
__device__ __forceinline__ u32x4 read16(uint32_t at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4 *>(at);
}

// Four tokens of one dim, a pair of words: lane i of sixteen gives the address
// of four dims of token i / 4, and gets dim i.
__device__ __forceinline__ u32x2 read_transposed(uint32_t at) {
  typedef __attribute__((address_space(3))) i16x4 *From;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<From>(at)));
}

// 16 bytes per lane from base + at into shared memory, lane after lane from
// `to`. The compiler does not count it: arrived<N>() waits until at most the N
// latest are on their way. ONCE: past the caches, for what no other workgroup
// reads.
template <bool ONCE> __device__ __forceinline__ void load_async(const char *base, uint32_t at, uint32_t to) {
  const int m0 = uniform(static_cast<int>(to));
  const int64_t from = uniform64(reinterpret_cast<int64_t>(base));
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 :
                 : "s"(m0), "v"(at), "s"(from)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(m0), "v"(at), "s"(from)
                 : "memory", "m0");
}
// The same for four bytes a lane.
__device__ __forceinline__ void load_async4(const void *base, uint32_t at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               :
               : "s"(uniform(static_cast<int>(to))), "v"(at), "s"(uniform64(reinterpret_cast<int64_t>(base)))
               : "memory", "m0");
}
template <int N> __device__ __forceinline__ void arrived() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// Waits for the wave's own reads and writes of shared memory.
__device__ __forceinline__ void shared_done() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// Waits for the workgroup's other waves, and for the wave's own reads of shared
// memory, whose place another wave's load may take next; for no other memory.
__device__ __forceinline__ void meet() {
  shared_done();
  __builtin_amdgcn_s_barrier();
  asm volatile("" : : : "memory");
}

// ------------------------------------------------------------ softmax

// Where a row's reference maximum starts: finite, so that a difference with a
// masked score's -inf stays -inf.
constexpr float kNone = -3.402823466e38f;
// A row's reference maximum moves only once a score exceeds it by this many
// powers of two; until then weights up to 2^8 are summed as they are.
constexpr float kSlack = 8.0f;

template <int T> constexpr float weight_bias() {
  return T == kF16 ? 6.0f : 0.0f; // weights up to 2^14 in f16: small ones keep their bits
}

// One over a row's sum of weights, with the values' scale; 0 for a row that
// saw nothing.
__device__ __forceinline__ float finish(float sum, float scale) {
  return sum > 0.0f ? scale / sum : sum == 0.0f ? 0.0f : sum;
}
__device__ __forceinline__ float log_sum(float top, float sum) {
  return sum == 0.0f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f;
}

} // namespace
} // namespace relx
