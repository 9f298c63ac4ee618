// Element types of the tensor operators (recurrence, distillation, verification): what is stored, and what sums are held in.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mz {

// Sums, states and softmax statistics of 16- and 32-bit tensors are held in float32, those of float64 tensors in float64.
template <typename T> struct AccOf { using type = float; };
template <> struct AccOf<double> { using type = double; };
template <typename T> using acc_t = typename AccOf<T>::type;

template <typename T> __device__ __forceinline__ acc_t<T> widen(T v) { return (acc_t<T>)v; }
// One rounding to nearest even, at the store (v_cvt_pk_bf16_f32 / v_cvt_f16_f32 on gfx950).
template <typename T> __device__ __forceinline__ T narrow(acc_t<T> v) { return (T)v; }

__device__ __forceinline__ float fma_acc(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_acc(double a, double b, double c) { return __builtin_fma(a, b, c); }

// Workgroup barrier that orders LDS traffic only: global loads and stores in flight stay in flight across it.
__device__ __forceinline__ void lds_fence_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// N elements that travel as one load or store; aligned to its size.
template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };
// ... aligned to one element only (one wide access all the same: gfx950 takes any element-aligned address).
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Loose { T v[N]; };

}  // namespace mz
