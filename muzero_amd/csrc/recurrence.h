// Gated linear recurrence y[s] = a[s] * y[s-1] + x[s] along one axis of a [B][T][D] tensor, and its gradients: the shape of
// discounted returns and traces over long records, and of recurrent state.
//
// A run of steps is the map y -> A y + X with A = a[s1] ... a[s0], X = what the run makes of y = 0, and two runs compose as
// (A1, X1), (A2, X2) -> (A1 A2, A2 X1 + X2).  Every kernel below cuts the axis into short runs held in registers, composes
// the runs' maps to get each run's first state, and then walks the run once more in registers: inputs are read once,
// outputs written once.
//
// Gradients: g[s] = dy[s] + a[s+1] g[s+1] is the same recurrence in the opposite order with the gate taken one position
// earlier in that order; dx = g, da[s] = g[s] y[s-1], dstate = a[0] g[0].
#pragma once
#include "element_types.h"

namespace mz {

struct RecurrenceArgs {
    // Scan order: position s lies at pointer + b * sb + s * st + d * sd (in elements; st is negative where the pass runs
    // from the last position to the first, the pointer then stands on the last).
    struct View { const void *p; long long sb, st, sd; };
    int B, D;
    long long T;
    View a, x;           // gates and inputs (backward: dy)
    View y;              // backward: the forward pass's outputs, or p = NULL where no gate gradient is wanted
    View out, da;        // y (backward: dx), gate gradients
    const void *first;   // acc[B][D] what goes into position 0 (backward: gradient of the last state), NULL = 0
    const void *state0;  // backward: acc[B][D] the forward pass's first state, NULL = 0
    void *last;          // acc[B][D] the state behind the last position (backward: gradient of the first state), may be NULL
};

template <typename T> __device__ __forceinline__ const T *at(const RecurrenceArgs::View &v, int b, long long s, int d)
{
    return (const T *)v.p + (long long)b * v.sb + s * v.st + (long long)d * v.sd;
}

// Channels contiguous: CL neighbouring lanes hold CL * VEC neighbouring channels, and each such group of lanes ("strand")
// walks L consecutive positions in registers; the block's NV strands follow each other in time and exchange their maps
// through LDS, one barrier per NV * L positions.
template <typename T, int VEC, int CL, int THREADS, int L, bool BWD>
__global__ __launch_bounds__(THREADS) void k_recurrence_channels(RecurrenceArgs q)
{
    using A = acc_t<T>;
    using P = Pack<T, VEC>;
    constexpr int NV = THREADS / CL;
    __shared__ A run_a[2][NV][CL * VEC], run_x[2][NV][CL * VEC];
    const int tiles = (q.D + CL * VEC - 1) / (CL * VEC);
    const int b = blockIdx.x / tiles, c = (threadIdx.x % CL) * VEC, d = (blockIdx.x % tiles) * CL * VEC + c;
    const int v = threadIdx.x / CL;
    const bool live = d < q.D;
    A carry[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) carry[j] = live && q.first ? ((const A *)q.first)[(long long)b * q.D + d + j] : A(0);
    const bool want_da = BWD && q.da.p;
    int buf = 0;
    for (long long base = 0; base < q.T; base += NV * L, buf ^= 1) {
        const long long s0 = base + v * L;
        P a[L], x[L], y[L];
#pragma unroll
        for (int i = 0; i < L; i++) {
            const long long s = s0 + i;
            if (live && s < q.T) {
                x[i] = *(const P *)at<T>(q.x, b, s, d);
                if (!BWD || s > 0) a[i] = *(const P *)at<T>(q.a, b, BWD ? s - 1 : s, d);
                else
#pragma unroll
                    for (int j = 0; j < VEC; j++) a[i].v[j] = T(1.0f);
                if (want_da && s + 1 < q.T) y[i] = *(const P *)at<T>(q.y, b, s + 1, d);
            } else
#pragma unroll
                for (int j = 0; j < VEC; j++) a[i].v[j] = T(1.0f), x[i].v[j] = T(0.0f);
        }
        A ra[VEC], rx[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            ra[j] = A(1), rx[j] = A(0);
#pragma unroll
            for (int i = 0; i < L; i++) {
                rx[j] = fma_acc(widen(a[i].v[j]), rx[j], widen(x[i].v[j]));
                ra[j] *= widen(a[i].v[j]);
            }
            run_a[buf][v][c + j] = ra[j], run_x[buf][v][c + j] = rx[j];
        }
        __syncthreads();
        A h[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++)
#pragma unroll 8
            for (int i = 0; i < NV; i++) {
                if (i == v) h[j] = carry[j];
                carry[j] = fma_acc(run_a[buf][i][c + j], carry[j], run_x[buf][i][c + j]);
            }
#pragma unroll
        for (int i = 0; i < L; i++) {
            const long long s = s0 + i;
            if (!live || s >= q.T) continue;
            P o, da;
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                h[j] = fma_acc(widen(a[i].v[j]), h[j], widen(x[i].v[j]));
                o.v[j] = narrow<T>(h[j]);
                if (want_da) {
                    const A before = s + 1 < q.T ? widen(y[i].v[j]) : q.state0 ? ((const A *)q.state0)[(long long)b * q.D + d + j] : A(0);
                    da.v[j] = narrow<T>(h[j] * before);
                }
            }
            *(P *)at<T>(q.out, b, s, d) = o;
            if (want_da) *(P *)at<T>(q.da, b, s, d) = da;
        }
    }
    if (q.last && live && v == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            A z = carry[j];
            if (BWD) z *= widen(at<T>(q.a, b, q.T - 1, d)[j]);
            ((A *)q.last)[(long long)b * q.D + d + j] = z;
        }
    }
}

// Any strides, one row (b, d) per block: every thread walks E consecutive positions, the maps are composed across the wave
// by shuffles and across the waves through LDS.
template <typename T, int E, bool BWD>
__global__ __launch_bounds__(1024) void k_recurrence_rows(RecurrenceArgs q)
{
    using A = acc_t<T>;
    __shared__ A run_a[2][16], run_x[2][16];
    const int b = blockIdx.x / q.D, d = blockIdx.x % q.D, lane = threadIdx.x % 64, w = threadIdx.x / 64, nw = blockDim.x / 64;
    A carry = q.first ? ((const A *)q.first)[blockIdx.x] : A(0);
    const A state0 = BWD && q.state0 ? ((const A *)q.state0)[blockIdx.x] : A(0);
    const bool want_da = BWD && q.da.p;
    int buf = 0;
    for (long long base = 0; base < q.T; base += (long long)blockDim.x * E, buf ^= 1) {
        const long long s0 = base + (long long)threadIdx.x * E;
        A a[E], x[E], y[E];
        A ra = A(1), rx = A(0);
#pragma unroll
        for (int i = 0; i < E; i++) {
            const long long s = s0 + i;
            a[i] = A(1), x[i] = A(0), y[i] = state0;
            if (s < q.T) {
                x[i] = widen(*at<T>(q.x, b, s, d));
                if (!BWD || s > 0) a[i] = widen(*at<T>(q.a, b, BWD ? s - 1 : s, d));
                if (want_da && s + 1 < q.T) y[i] = widen(*at<T>(q.y, b, s + 1, d));
            }
        }
#pragma unroll
        for (int i = 0; i < E; i++) rx = fma_acc(a[i], rx, x[i]), ra *= a[i];
#pragma unroll
        for (int k = 1; k < 64; k *= 2) {
            const A pa = __shfl_up(ra, k), px = __shfl_up(rx, k);
            if (lane >= k) rx = fma_acc(ra, px, rx), ra *= pa;
        }
        if (lane == 63) run_a[buf][w] = ra, run_x[buf][w] = rx;
        A ea = __shfl_up(ra, 1), ex = __shfl_up(rx, 1);
        if (lane == 0) ea = A(1), ex = A(0);
        __syncthreads();
        A h = carry;
        for (int i = 0; i < nw; i++) {
            if (i == w) h = carry;
            carry = fma_acc(run_a[buf][i], carry, run_x[buf][i]);
        }
        h = fma_acc(ea, h, ex);
#pragma unroll
        for (int i = 0; i < E; i++) {
            const long long s = s0 + i;
            if (s >= q.T) break;
            h = fma_acc(a[i], h, x[i]);
            *(T *)at<T>(q.out, b, s, d) = narrow<T>(h);
            if (want_da) *(T *)at<T>(q.da, b, s, d) = narrow<T>(h * y[i]);
        }
    }
    if (q.last && threadIdx.x == 0) {
        if (BWD) carry *= widen(*at<T>(q.a, b, q.T - 1, d));
        ((A *)q.last)[blockIdx.x] = carry;
    }
}

}  // namespace mz
