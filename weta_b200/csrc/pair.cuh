// Two values at a time: sm_100 has packed f32 arithmetic, two IEEE operations per instruction and lane; f64 stays scalar
// behind the same names.
#pragma once

#include <cstdint>

template <class T>
struct Pair;
template <>
struct Pair<float> {
    uint64_t v;
};
template <>
struct Pair<double> {
    double a, b;
};
__device__ __forceinline__ Pair<float> pair(float a, float b) {
    Pair<float> r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ Pair<double> pair(double a, double b) { return {a, b}; }
__device__ __forceinline__ void unpair(const Pair<float>& p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ void unpair(const Pair<double>& p, double& a, double& b) {
    a = p.a;
    b = p.b;
}
__device__ __forceinline__ Pair<float> operator+(const Pair<float>& x, const Pair<float>& y) {
    Pair<float> r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(x.v), "l"(y.v));
    return r;
}
__device__ __forceinline__ Pair<float> operator*(const Pair<float>& x, const Pair<float>& y) {
    Pair<float> r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(x.v), "l"(y.v));
    return r;
}
// A product that is rounded by itself whatever is added to it.  The assembler contracts a packed multiplication and a packed
// addition into one fused operation, -fmad=false or not, and does so with x * y + (-0), too, where it knows the constant:
// `minus_zero` is a value that it cannot know (a kernel's argument).
__device__ __forceinline__ Pair<float> rounded_product(const Pair<float>& x, const Pair<float>& y, const Pair<float>& minus_zero) {
    Pair<float> r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(x.v), "l"(y.v), "l"(minus_zero.v));
    return r;
}
__device__ __forceinline__ Pair<float> muladd(const Pair<float>& x, const Pair<float>& y, const Pair<float>& z) {
    Pair<float> r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(x.v), "l"(y.v), "l"(z.v));
    return r;
}
// f64: two separate operations
__device__ __forceinline__ Pair<double> operator+(const Pair<double>& x, const Pair<double>& y) { return {x.a + y.a, x.b + y.b}; }
__device__ __forceinline__ Pair<double> operator*(const Pair<double>& x, const Pair<double>& y) { return {x.a * y.a, x.b * y.b}; }
__device__ __forceinline__ Pair<double> muladd(const Pair<double>& x, const Pair<double>& y, const Pair<double>& z) {
    return {fma(x.a, y.a, z.a), fma(x.b, y.b, z.b)};
}
