// Pairs of values: two fp32 of one packed instruction (fma.rn.f32x2 and its like), or two fp64; and
// the same operations on single values, for code that takes either.
#pragma once

#include <type_traits>

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
__device__ __forceinline__ Two<float> both(float x) { return two(x, x); }
// 2^x
__device__ __forceinline__ float exp_2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ double exp_2(double x) { return exp2(x); }
template <typename A> __device__ __forceinline__ Two<A> exp_2(Two<A> x) {
  return two(exp_2(first(x)), exp_2(second(x)));
}
constexpr double kLog2e = 1.4426950408889634074, kLn2 = 0.69314718055994530942;
// 1 / x to a rounding; 0 for the largest
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ Two<float> reciprocal(Two<float> x) {
  return two(reciprocal(first(x)), reciprocal(second(x)));
}
// single values
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ double mul(double a, double b) { return a * b; }
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ double add(double a, double b) { return a + b; }
__device__ __forceinline__ float fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma(double a, double b, double c) { return ::fma(a, b, c); }

template <typename E> __device__ __forceinline__ E splat(float x) {
  if constexpr (std::is_same_v<E, Two<float>>) return both(x);
  else return static_cast<E>(x);
}

}  // namespace
}  // namespace fdwt
