// Two elements of a row as one thread reads, holds and writes them, for bf16, fp16 and fp32 rows.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace fla {

template <typename T>
struct PairOf {  // 16-bit types
  using Raw = uint32_t;
  using Element = uint16_t;
};
template <>
struct PairOf<float> {
  using Raw = float2;
  using Element = float;
};

__device__ __forceinline__ uint32_t join_pair(uint16_t a, uint16_t b) { return a | static_cast<uint32_t>(b) << 16; }
__device__ __forceinline__ float2 join_pair(float a, float b) { return make_float2(a, b); }
__device__ __forceinline__ void zero_pair(uint32_t& r) { r = 0u; }
__device__ __forceinline__ void zero_pair(float2& r) { r = make_float2(0.f, 0.f); }

template <typename T>
__device__ __forceinline__ float2 unpack_pair(const typename PairOf<T>::Raw& r);
template <>
__device__ __forceinline__ float2 unpack_pair<float>(const float2& r) {
  return r;
}
template <>
__device__ __forceinline__ float2 unpack_pair<__nv_bfloat16>(const uint32_t& r) {
  return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack_pair<__half>(const uint32_t& r) {
  return __half22float2(*reinterpret_cast<const __half2*>(&r));
}

// Rounded to nearest, once.
template <typename T>
__device__ __forceinline__ typename PairOf<T>::Raw pack_pair(float2 v);
template <>
__device__ __forceinline__ float2 pack_pair<float>(float2 v) {
  return v;
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float2 v) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float2 v) {
  const __half2 r = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// sm_100 multiplies and adds pairs of floats in one instruction.
__device__ __forceinline__ uint64_t bits(float2 v) { return *reinterpret_cast<const uint64_t*>(&v); }
__device__ __forceinline__ float2 floats(uint64_t v) { return *reinterpret_cast<const float2*>(&v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return floats(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
  return floats(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
  return floats(d);
}

// Where a thread's two columns are: next to each other in an aligned pair (one access), or `gap` columns apart (two
// accesses, each of which a warp makes to neighbouring elements).
template <typename T, bool PAIR>
__device__ __forceinline__ typename PairOf<T>::Raw load_pair(const T* p, int gap, bool ok0, bool ok1) {
  using Raw = typename PairOf<T>::Raw;
  using Element = typename PairOf<T>::Element;
  Raw r;
  zero_pair(r);
  if (PAIR) {
    if (ok0) r = __ldg(reinterpret_cast<const Raw*>(p));
    return r;
  }
  Element a = 0, b = 0;
  if (ok0) a = __ldg(reinterpret_cast<const Element*>(p));
  if (ok1) b = __ldg(reinterpret_cast<const Element*>(p) + gap);
  return join_pair(a, b);
}

template <typename T, bool PAIR>
__device__ __forceinline__ void store_pair(T* p, int gap, bool ok0, bool ok1, float2 v) {
  using Raw = typename PairOf<T>::Raw;
  using Element = typename PairOf<T>::Element;
  const Raw r = pack_pair<T>(v);
  if (PAIR) {
    if (ok0) *reinterpret_cast<Raw*>(p) = r;
    return;
  }
  const Element* e = reinterpret_cast<const Element*>(&r);
  if (ok0) reinterpret_cast<Element*>(p)[0] = e[0];
  if (ok1) reinterpret_cast<Element*>(p)[gap] = e[1];
}

}  // namespace fla
