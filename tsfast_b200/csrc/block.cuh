// What the block operators (gated recurrence, block norms, quantised product) share: conversions between the sequence
// types and float32, and the gates' function.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200 {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rsq(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 1 / (1 + e^-x): the two approximations are within a few units of 2^-23 each, the sum of one and a positive number loses
// nothing, and rounding the argument of the exponential adds 1.5 |x| 2^-24 where x is negative (1e-6 at -20, 7e-6 at -80:
// relative to a gate that is as good as shut, and less than 16-bit gates lose by being rounded themselves)
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-1.4426950408889634f * x)); }


// Two float32 operations per instruction (sm_100): the two halves of a 64-bit register pair
__device__ __forceinline__ unsigned long long bits2(float2 v) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ float2 pair2(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
typedef unsigned long long Pair;
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return pair2(fma2(bits2(a), bits2(b), bits2(c))); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return pair2(mul2(bits2(a), bits2(b))); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return pair2(add2(bits2(a), bits2(b))); }
// A constant in both halves that stays in its registers: a packed instruction takes no immediate, and the compiler would
// rather make the pair anew with two moves at every use
__device__ __forceinline__ Pair resident(float v) {
    Pair r;
    asm volatile("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(v));
    return r;
}

// an error word in device memory: read after the work on the stream, and cleared if it was set
inline int take_error_word(unsigned int& word, cudaStream_t st) {
    unsigned int error = 0, zero = 0;
    if (cudaMemcpyFromSymbolAsync(&error, word, sizeof(error), 0, cudaMemcpyDeviceToHost, st) != cudaSuccess) return B200_ERR_LAUNCH;
    if (cudaStreamSynchronize(st) != cudaSuccess) return B200_ERR_LAUNCH;
    if (error && cudaMemcpyToSymbolAsync(word, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, st) != cudaSuccess) return B200_ERR_LAUNCH;
    if (error && cudaStreamSynchronize(st) != cudaSuccess) return B200_ERR_LAUNCH;
    return (int)error;
}

// whether every pointer is on a boundary of so many bytes (null ones are)
template <typename... P>
inline bool on_boundary(size_t bytes, P... p) {
    return ((reinterpret_cast<uintptr_t>(p) % bytes == 0) && ...);
}
inline int block_elem_size(int dtype) { return dtype == B200_F32 ? 4 : dtype == B200_BF16 || dtype == B200_F16 ? 2 : 0; }

}  // namespace b200
