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

// What a rounding to 16 bits lost, in 8 more bits: the distance of the float32 pattern from that of the rounded value (patterns
// of one sign are ordered like their values, across exponents too) in steps of 2^FINE_SHIFT, held in byte 1 of what
// fine_of() returns.  refined() is then within one such step of the float32 value, 2^-15 of it (bfloat16) or 2^-18 (float16).
// A bfloat16 has float32's exponents: half a step of its own is 2^15 everywhere, what rounds to infinity comes back finite, and
// adding up to 2^15 to a quiet NaN leaves one.  A float16 among its subnormal numbers is off by more than fits and is never
// further off than the rounded value; its infinities and NaN are left as they are.
template <typename T> constexpr int FINE_SHIFT = 8;
template <> constexpr int FINE_SHIFT<_Float16> = 5;
__device__ __forceinline__ int pattern(float v) { return __builtin_bit_cast(int, v); }
__device__ __forceinline__ unsigned fine_of(float v, __bf16 rounded)   // in byte 1
{
    return (unsigned)(min(pattern(v) - pattern((float)rounded), 0x7f7f) + 0x80);
}
__device__ __forceinline__ unsigned fine_of(float v, _Float16 rounded)
{
    const int w = pattern((float)rounded), d = min(max(pattern(v) - w, -0x1000), 0xfef) + 0x10;
    return (w & 0x7f800000) == 0x7f800000 ? 0u : (unsigned)d << 3;
}
template <typename A, typename T> __device__ __forceinline__ unsigned fine_of(A, T) { return 0; }
template <typename T> __device__ __forceinline__ float refined(T rounded, signed char fine)
{
    return __builtin_bit_cast(float, pattern((float)rounded) + (int)fine * (1 << FINE_SHIFT<T>));
}

__device__ __forceinline__ float fma_acc(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_acc(double a, double b, double c) { return __builtin_fma(a, b, c); }

// Workgroup barrier that orders LDS traffic only: global loads and stores in flight stay in flight across it.
__device__ __forceinline__ void lds_fence_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Value of another lane of the same 16 by a register move (0 where there is none): a few cycles, against about a hundred for a
// shuffle through LDS.
template <int CTRL> __device__ __forceinline__ float lane_move(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
template <int CTRL> __device__ __forceinline__ double lane_move(double v)
{
    const long long b = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_mov_dpp((int)b, CTRL, 0xF, 0xF, true), hi = __builtin_amdgcn_mov_dpp((int)(b >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (long long)hi << 32 | (unsigned)lo);
}
__device__ __forceinline__ float lane_read(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
__device__ __forceinline__ double lane_read(double v, int lane)
{
    const long long b = __builtin_bit_cast(long long, v);
    return __builtin_bit_cast(double, (long long)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)b, lane));
}
// f over G neighbouring lanes (4, 16 or 64, all of them at work), in every one of them, always in the same order.
template <int G, typename V, typename F> __device__ __forceinline__ V group_fold(V v, F f)
{
    static_assert(G == 4 || G == 16 || G == 64, "groups of 4, 16 or 64 lanes");
    v = f(v, lane_move<0xB1>(v));    // lanes 1, 0, 3, 2 of every four
    v = f(v, lane_move<0x4E>(v));    // lanes 2, 3, 0, 1
    if constexpr (G > 4) {
        v = f(v, lane_move<0x141>(v));   // mirrored in every eight
        v = f(v, lane_move<0x140>(v));   // mirrored in every sixteen
    }
    if constexpr (G == 64) v = f(f(lane_read(v, 0), lane_read(v, 16)), f(lane_read(v, 32), lane_read(v, 48)));
    return v;
}
template <int G, typename V> __device__ __forceinline__ V group_sum(V v)
{
    return group_fold<G>(v, [](V a, V b) { return a + b; });
}
template <int G> __device__ __forceinline__ float group_max(float v)
{
    return group_fold<G>(v, [](float a, float b) { return fmaxf(a, b); });
}

// N elements that travel as one load or store; aligned to its size.
template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };
// ... aligned to one element only (one wide access all the same: gfx950 takes any element-aligned address).
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Loose { T v[N]; };

}  // namespace mz
