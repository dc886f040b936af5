// Pairs of values: two fp32 of one packed instruction (fma.rn.f32x2 and its like), or two fp64; and
// the same operations on single values, for code that takes either.
#pragma once

#include "common.cuh"

namespace fdwt {
namespace {

// Two values that every operation is done to: packed instructions for 32 bits.
template <typename A> struct Two;
template <> struct Two<float> {
  unsigned long long v;
};
template <> struct Two<double> {
  double x, y;
};
__device__ __forceinline__ Two<float> two(float x, float y) {
  Two<float> r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ Two<double> two(double x, double y) { return {x, y}; }
__device__ __forceinline__ float first(Two<float> a) {
  return __uint_as_float(static_cast<uint32_t>(a.v));
}
__device__ __forceinline__ float second(Two<float> a) {
  return __uint_as_float(static_cast<uint32_t>(a.v >> 32));
}
__device__ __forceinline__ double first(Two<double> a) { return a.x; }
__device__ __forceinline__ double second(Two<double> a) { return a.y; }
__device__ __forceinline__ Two<float> mul(Two<float> a, Two<float> b) {
  Two<float> r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two<double> mul(Two<double> a, Two<double> b) {
  return {a.x * b.x, a.y * b.y};
}
__device__ __forceinline__ Two<float> add(Two<float> a, Two<float> b) {
  Two<float> r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two<double> add(Two<double> a, Two<double> b) {
  return {a.x + b.x, a.y + b.y};
}
__device__ __forceinline__ Two<float> fma(Two<float> a, Two<float> b, Two<float> c) {
  Two<float> r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two<double> fma(Two<double> a, Two<double> b, Two<double> c) {
  return {::fma(a.x, b.x, c.x), ::fma(a.y, b.y, c.y)};
}
// single values
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ double mul(double a, double b) { return a * b; }
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ double add(double a, double b) { return a + b; }
__device__ __forceinline__ float fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma(double a, double b, double c) { return ::fma(a, b, c); }

}  // namespace
}  // namespace fdwt
