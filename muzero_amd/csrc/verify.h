// Verification of drafted moves against the target policy: per sequence, drafted token x_k is kept while
// u_k q_k(x_k) < p_k(x_k); at the first that is not, a token is drawn from max(p - q, 0), and where all are kept, one more
// from the target's next row.  What comes out is distributed as the target's own moves.  The draw is the inverse of the
// running sum at u (first index whose sum exceeds u times the whole), in float64 as numpy.random.choice takes it.
#pragma once
#include "element_types.h"

namespace mz {

struct VerifyArgs {
    const void *tokens;          // [B][K] int32 or int64
    const void *draft;           // [B][K][V], or NULL: each draft was its policy's only choice
    const void *target;          // [B][K + 1][V]
    long long draft_b, draft_k, target_b, target_k;   // strides in elements; V is contiguous
    const double *u_accept;      // [B][K]
    const double *u_sample;      // [B]
    const int *lengths;          // [B] drafted tokens of each sequence, or NULL: K
    int *accepted;               // [B]
    void *out;                   // [B][K + 1], type of tokens; -1 behind the last token
    int B, K, V, token64;
};

// Entries that are no probability (negative, NaN, infinite) count as zero.
template <typename T> __device__ __forceinline__ double mass_of(T v)
{
    const double d = (double)v;
    return d > 0 && d < HUGE_VAL ? d : 0.0;
}

__device__ __forceinline__ long long drafted(const VerifyArgs &q, long long i)
{
    return q.token64 ? ((const long long *)q.tokens)[i] : (long long)((const int *)q.tokens)[i];
}

// How many drafts of sequence b are kept; every thread of the block gets the answer.
template <typename T> __device__ __forceinline__ int kept(const VerifyArgs &q, int b, int length, int *first)
{
    if (threadIdx.x == 0) *first = length;
    __syncthreads();
    for (int k = threadIdx.x; k < length; k += blockDim.x) {
        const long long x = drafted(q, (long long)b * q.K + k);
        bool ok = false;
        if (x >= 0 && x < q.V) {
            const double p = mass_of(((const T *)q.target)[(long long)b * q.target_b + (long long)k * q.target_k + x]);
            const double d = q.draft ? mass_of(((const T *)q.draft)[(long long)b * q.draft_b + (long long)k * q.draft_k + x]) : 1.0;
            ok = q.u_accept[(long long)b * q.K + k] * d < p;
        }
        if (!ok) atomicMin(first, k);
    }
    __syncthreads();
    return *first;
}

// The row to draw from: p, or what p has more than q.
template <typename T> struct Left {
    const T *p, *d;
    int only;        // a draft without probabilities: the action that is taken out, else -1
    __device__ __forceinline__ double at(int j) const
    {
        double v = mass_of(p[j]);
        if (d) v = fmax(v - mass_of(d[j]), 0.0);
        return j == only ? 0.0 : v;
    }
};

__device__ __forceinline__ double block_sum_d(double v, double *red)
{
    for (int k = 32; k; k /= 2) v += __shfl_xor(v, k);
    __syncthreads();
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < (int)blockDim.x / 64; i++) v += red[i];
    return v;
}

// One block per sequence.
template <typename T> __global__ __launch_bounds__(1024) void k_verify(VerifyArgs q)
{
    __shared__ int first;
    __shared__ double red[16], part[16];
    __shared__ int found;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid % 64, w = tid / 64, nw = blockDim.x / 64;
    int length = q.lengths ? q.lengths[b] : q.K;
    length = length < 0 ? 0 : length > q.K ? q.K : length;
    const int n = kept<T>(q, b, length, &first);
    Left<T> left{(const T *)q.target + (long long)b * q.target_b + (long long)n * q.target_k, nullptr, -1};
    if (n < length) {
        if (q.draft) left.d = (const T *)q.draft + (long long)b * q.draft_b + (long long)n * q.draft_k;
        else left.only = (int)drafted(q, (long long)b * q.K + n);
    }
    int token = -1;
    for (int again = 0; again < 2; again++) {
        // the range that holds the answer shrinks to the part of one wave until a wave covers it by one element a lane
        int lo = 0, hi = q.V;
        double below = 0, goal = 0;
        bool any = true;
        while (true) {
            const int step = (hi - lo + nw - 1) / nw;
            const int a = min(lo + w * step, hi), z = min(a + step, hi);
            double s = 0;
            for (int j = a + lane; j < z; j += 64) s += left.at(j);
            for (int k = 32; k; k /= 2) s += __shfl_xor(s, k);
            __syncthreads();
            if (lane == 0) part[w] = s;
            __syncthreads();
            if (lo == 0 && hi == q.V) {
                double all = 0;
                for (int i = 0; i < nw; i++) all += part[i];
                any = all > 0;
                goal = q.u_sample[b] * all;
            }
            if (!any) break;
            int pick = -1, last = -1;
            double at = below, last_at = below;
            for (int i = 0; i < nw; i++) {
                if (part[i] > 0) last = i, last_at = at;
                if (part[i] > 0 && at + part[i] > goal) { pick = i; break; }
                at += part[i];
            }
            if (pick < 0) pick = last, at = last_at;   // rounding put the goal behind the last element
            below = at;
            const int na = min(lo + pick * step, hi), nz = min(na + step, hi);
            lo = na, hi = nz;
            if (hi - lo <= 64) break;
        }
        if (any) {
            if (w == 0) {
                const double v = lo + lane < hi ? left.at(lo + lane) : 0.0;
                double c = v;
                for (int k = 1; k < 64; k *= 2) {
                    const double o = __shfl_up(c, k);
                    if (lane >= k) c += o;
                }
                const unsigned long long over = __ballot(v > 0 && below + c > goal), some = __ballot(v > 0);
                if (lane == 0) found = lo + (over ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)some));
            }
            __syncthreads();
            token = found;
            break;
        }
        if (!left.d && left.only < 0) break;   // the target itself has nothing: no token
        left.d = nullptr, left.only = -1;      // p nowhere above q: the target's own row
    }
    for (int k = tid; k <= q.K; k += blockDim.x) {
        const long long x = k < n ? drafted(q, (long long)b * q.K + k) : k == n ? token : -1;
        if (q.token64) ((long long *)q.out)[(long long)b * (q.K + 1) + k] = x;
        else ((int *)q.out)[(long long)b * (q.K + 1) + k] = (int)x;
    }
    if (tid == 0) q.accepted[b] = n;
}

}  // namespace mz
