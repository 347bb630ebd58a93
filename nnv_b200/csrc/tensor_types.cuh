// Element types of the device-tensor entry points (layer normalisation, attention): conversions to and from the
// type sums are held in (float for the 16- and 32-bit types, double for double) and 16-byte vector access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace nnvb {

template <typename T> struct AccOf { using type = float; };
template <> struct AccOf<double> { using type = double; };

__device__ __forceinline__ float to_acc(float x) { return x; }
__device__ __forceinline__ double to_acc(double x) { return x; }
__device__ __forceinline__ float to_acc(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_acc(__half x) { return __half2float(x); }

// one rounding to nearest even, where a result leaves for memory
template <typename T, typename A> __device__ __forceinline__ T from_acc(A x);
template <> __device__ __forceinline__ float from_acc<float, float>(float x) { return x; }
template <> __device__ __forceinline__ double from_acc<double, double>(double x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16, float>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_acc<__half, float>(float x) { return __float2half_rn(x); }

// N elements that are loaded and stored as one access
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// Pairs of sums: two float operations are one instruction (f32x2), two doubles are two.
template <typename A> struct Pair { A x, y; };
__device__ __forceinline__ uint64_t pair_bits(Pair<float> a) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ Pair<float> pair_of(uint64_t b) {
    Pair<float> a;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(b));
    return a;
}
__device__ __forceinline__ Pair<float> add2(Pair<float> a, Pair<float> b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
    return pair_of(r);
}
__device__ __forceinline__ Pair<float> mul2(Pair<float> a, Pair<float> b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
    return pair_of(r);
}
__device__ __forceinline__ Pair<float> fma2(Pair<float> a, Pair<float> b, Pair<float> c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
    return pair_of(r);
}
__device__ __forceinline__ Pair<double> add2(Pair<double> a, Pair<double> b) { return {a.x + b.x, a.y + b.y}; }
__device__ __forceinline__ Pair<double> mul2(Pair<double> a, Pair<double> b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ Pair<double> fma2(Pair<double> a, Pair<double> b, Pair<double> c) {
    return {fma(a.x, b.x, c.x), fma(a.y, b.y, c.y)};
}
template <typename A> __device__ __forceinline__ Pair<A> both(A x) { return {x, x}; }
// a single sum, for elements that do not come in pairs
__device__ __forceinline__ float add2(float a, float b) { return a + b; }
__device__ __forceinline__ float mul2(float a, float b) { return a * b; }
__device__ __forceinline__ float fma2(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double add2(double a, double b) { return a + b; }
__device__ __forceinline__ double mul2(double a, double b) { return a * b; }
__device__ __forceinline__ double fma2(double a, double b, double c) { return fma(a, b, c); }
template <typename A> __device__ __forceinline__ A across(Pair<A> a) { return a.x + a.y; }
__device__ __forceinline__ float across(float a) { return a; }
__device__ __forceinline__ double across(double a) { return a; }

__device__ __forceinline__ float rsqrt_acc(float x) { return rsqrtf(x); }
__device__ __forceinline__ double rsqrt_acc(double x) { return rsqrt(x); }

}  // namespace nnvb
