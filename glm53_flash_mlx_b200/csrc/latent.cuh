// Shared device helpers of the latent-attention operators: 16-bit element
// types, fail-closed status reports and shape limits.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace glm53 {
namespace latent {

constexpr uint32_t kStatusBadPage = 1u << 3;  // a page id or slot outside the cache
constexpr uint32_t kStatusNoPages = 1u << 4;  // a page plan that does not fit its pages, table or token capacity

// OR a bit into the device status word and, where given, store the word in
// the pinned host mirror: the success path needs no mirror launch.
__device__ __forceinline__ void report(uint32_t* status, uint32_t* host, uint32_t bit) {
  if (!status) return;
  const uint32_t word = atomicOr(status, bit) | bit;
  if (host) {
    *reinterpret_cast<volatile uint32_t*>(host) = word;
    __threadfence_system();
  }
}

template <typename E>
struct Elem;

template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  static __device__ __forceinline__ float to_float(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t from_float(float f) {
    const __nv_bfloat16 h = __float2bfloat16_rn(f);
    return *reinterpret_cast<const uint16_t*>(&h);
  }
};

template <>
struct Elem<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  static __device__ __forceinline__ float to_float(uint16_t v) {
    return __half2float(*reinterpret_cast<const __half*>(&v));
  }
  static __device__ __forceinline__ uint16_t from_float(float f) {
    const __half h = __float2half_rn(f);
    return *reinterpret_cast<const uint16_t*>(&h);
  }
};

template <typename E>
__device__ __forceinline__ void unpack8(uint4 w, float (&f)[8]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Elem<E>::unpack(v[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}

template <typename E>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(Elem<E>::pack(f[0], f[1]), Elem<E>::pack(f[2], f[3]), Elem<E>::pack(f[4], f[5]),
                    Elem<E>::pack(f[6], f[7]));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// True in every thread of `threads` when `p` holds in any of them (named barrier `id`).
__device__ __forceinline__ bool any_of(bool p, int id, int threads) {
  uint32_t r;
  asm volatile(
      "{ .reg .pred a, b; setp.ne.u32 a, %1, 0; barrier.cta.red.or.pred b, %2, %3, a; selp.u32 %0, 1, 0, b; }"
      : "=r"(r)
      : "r"((uint32_t)p), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Running maxima are replaced (and results rescaled) only when a score passes
// the one in use by this much, in powers of two: weights stay below 2^8, which
// every type here holds, and most tiles rescale nothing.
constexpr float kMaxSlack = 8.0f;
// FP16 weights are held times 2^7, that is relative to the maximum less 7: 2^15
// at most, which FP16 holds, and what is below 2^-32 of the largest is lost, not
// what is below 2^-25 (keys 17.5 nats under one of their tile all vanished from
// the result, but not from its divisor).  BF16 has the exponents of FP32.
template <typename E>
constexpr float kWeightShift = std::is_same<E, __half>::value ? 7.0f : 0.0f;
// A row whose scores are all -inf has no weight anywhere: 0, as one that sees no key.
__device__ __forceinline__ float inverse_sum(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

}  // namespace latent
}  // namespace glm53
