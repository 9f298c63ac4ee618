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

// Entries that are no probability (negative, NaN, infinite) count as zero; looked at in the type's own precision, which costs a
// third of the same in float64.
template <typename T> __device__ __forceinline__ double mass_of(T v)
{
    const float f = (float)v;
    return (double)fmaxf(f < HUGE_VALF ? f : 0.0f, 0.0f);
}
template <> __device__ __forceinline__ double mass_of(double d) { return d > 0 && d < HUGE_VAL ? d : 0.0; }

__device__ __forceinline__ long long drafted(const VerifyArgs &q, long long i)
{
    return q.token64 ? ((const long long *)q.tokens)[i] : (long long)((const int *)q.tokens)[i];
}

__device__ __forceinline__ int length_of(const VerifyArgs &q, long long b)
{
    const int n = q.lengths ? q.lengths[b] : q.K;
    return n < 0 ? 0 : n > q.K ? q.K : n;
}

// Whether draft k of sequence b is kept.
template <typename T> __device__ __forceinline__ bool passes(const VerifyArgs &q, long long b, int k)
{
    const long long x = drafted(q, b * q.K + k);
    const double u = q.u_accept[b * q.K + k];
    if (x < 0 || x >= q.V) return false;
    const double p = mass_of(((const T *)q.target)[b * q.target_b + k * q.target_k + x]);
    const double d = q.draft ? mass_of(((const T *)q.draft)[b * q.draft_b + k * q.draft_k + x]) : 1.0;
    return u * d < p;
}

// The row to draw from once n of `length` drafts are kept: p, or what p has more than the draft's policy.
template <typename T> struct Left {
    const T *p, *d;
    int only;        // a draft without probabilities: the action that is taken out, else -1
    __device__ __forceinline__ Left(const VerifyArgs &q, long long b, int n, int length)
        : p((const T *)q.target + b * q.target_b + n * q.target_k), d(nullptr), only(-1)
    {
        if (n >= length) return;
        if (q.draft) d = (const T *)q.draft + b * q.draft_b + n * q.draft_k;
        else {
            const long long x = drafted(q, b * q.K + n);
            only = x >= 0 && x < q.V ? (int)x : -1;
        }
    }
    __device__ __forceinline__ bool whole() const { return !d && only < 0; }
    __device__ __forceinline__ double of(T pj, T dj, int j) const
    {
        if (d) return fmax(mass_of(pj) - mass_of(dj), 0.0);
        return j == only ? 0.0 : mass_of(pj);
    }
};

__device__ __forceinline__ void put_token(const VerifyArgs &q, long long b, int n, int k, int token)
{
    const long long x = k < n ? drafted(q, b * q.K + k) : k == n ? token : -1;
    if (q.token64) ((long long *)q.out)[b * (q.K + 1) + k] = x;
    else ((int *)q.out)[b * (q.K + 1) + k] = (int)x;
}

template <int G> __device__ __forceinline__ double running_sum(double v, int lane)
{
#pragma unroll
    for (int k = 1; k < G; k *= 2) {
        const double o = __shfl_up(v, k, G);
        if (lane >= k) v += o;
    }
    return v;
}

// The lowest lane of the G (a power of two) whose flag is set, or G; and the highest, or -1.
template <int G> __device__ __forceinline__ int lowest_lane(bool flag)
{
    unsigned long long m = __ballot(flag);
    if (G < 64) m = m >> (threadIdx.x % 64 / G * G) & ((1ull << (G & 63)) - 1);
    return m ? __ffsll((long long)m) - 1 : G;
}
template <int G> __device__ __forceinline__ int highest_lane(bool flag)
{
    unsigned long long m = __ballot(flag);
    if (G < 64) m = m >> (threadIdx.x % 64 / G * G) & ((1ull << (G & 63)) - 1);
    return m ? 63 - __clzll((long long)m) : -1;
}

// Small action sets: G lanes of a wave serve a sequence, 4 neighbouring actions a lane, all in registers.
// 16384 sequences of 5 drafts over 9 actions in float64: 5.0 us, three dependent loads behind the launch.
template <typename T, int G> __global__ __launch_bounds__(256) void k_verify_group(VerifyArgs q)
{
    constexpr int E = 4;
    const int lane = threadIdx.x % G;
    const long long seq = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
    const bool live = seq < q.B;
    const long long b = live ? seq : q.B - 1;   // the last block's idle groups follow its last sequence and write nothing
    const int length = length_of(q, b);
    int n = length;
    for (int k = lane; k < q.K; k += G)   // past its length too: the loads do not wait for the length
        if (!passes<T>(q, b, k)) { n = min(n, k); break; }
#pragma unroll
    for (int k = G / 2; k; k /= 2) n = min(n, __shfl_xor(n, k));
    Left<T> left(q, b, n, length);
    int token = -1;
    const double u = q.u_sample[b];
    T p[E], d[E];
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int j = lane * E + i;
        p[i] = j < q.V ? left.p[j] : T(0.0f);
        d[i] = left.d && j < q.V ? left.d[j] : T(0.0f);
    }
    for (int again = 0; again < 2; again++) {
        double c[E], own = 0;
        bool some = false;
#pragma unroll
        for (int i = 0; i < E; i++) {
            const double v = left.of(p[i], d[i], lane * E + i);
            own += v;
            c[i] = v > 0 ? own : -1.0;   // the running sum where an action can be drawn
            some |= v > 0;
        }
        const double to = running_sum<G>(own, lane);
        double before = __shfl_up(to, 1, G);
        if (lane == 0) before = 0;
        const double goal = u * __shfl(to, G - 1, G);
        int pick = -1, last = -1;
#pragma unroll
        for (int i = E - 1; i >= 0; i--) {
            if (c[i] >= 0 && before + c[i] > goal) pick = lane * E + i;
            if (c[i] >= 0 && last < 0) last = lane * E + i;
        }
        const int lo = lowest_lane<G>(pick >= 0), hi = highest_lane<G>(some);
        const int picked = __shfl(pick, lo % G, G), end = __shfl(last, hi < 0 ? 0 : hi, G);
        const int found = lo < G ? picked : hi >= 0 ? end : -1;   // rounding can put the goal behind the last element
        if (token < 0) token = found;
        const bool retry = token < 0 && !left.whole();   // p nowhere above q: the target's own row
        if (!__any(retry)) break;
        if (retry) left.d = nullptr, left.only = -1;
    }
    if (!live) return;
    for (int k = lane; k <= q.K; k += G) put_token(q, b, n, k, token);
    if (lane == 0) q.accepted[b] = n;
}

// Wide action sets: one block per sequence.  The row is cut into stretches of two wide loads of a wave; a wave sums whole
// stretches, the first wave finds the stretch in which the running sum passes the goal and walks that one again.
// 256 x 100003 float32: 34 us (205 MB, 6 TB/s with part of the rows in cache); 2000 x 32000 bfloat16 100 us (256 MB; waves wait for
// three quarters of their cycles and the vector units issue in a tenth of theirs: a stretch's sixteen dependent float64 additions
// and its fold stand between a wave's loads); one sequence of 32000 float32: 10 us, of which the launch is 3 and four dependent trips
// to memory most of the rest; one of 130000: 25 us, what one compute unit can read.
constexpr int STRETCH_LOADS = 2;
template <typename T> constexpr int STRETCH = STRETCH_LOADS * 64 * (16 / (int)sizeof(T));

template <typename T> struct StretchOf {
    static constexpr int E = 16 / sizeof(T), N = STRETCH_LOADS;
    Loose<T, E> p[N], d[N];

    __device__ __forceinline__ void load(const Left<T> &left, int j0, int V)
    {
        const int lane = threadIdx.x % 64;
        if (j0 + STRETCH<T> <= V) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int j = j0 + (i * 64 + lane) * E;
                p[i] = *(const Loose<T, E> *)(left.p + j);
                if (left.d) d[i] = *(const Loose<T, E> *)(left.d + j);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int j = j0 + (i * 64 + lane) * E + e;
                    p[i].v[e] = j < V ? left.p[j] : T(0.0f);
                    d[i].v[e] = left.d && j < V ? left.d[j] : T(0.0f);
                }
        }
    }
    __device__ __forceinline__ double at(const Left<T> &left, int j0, int i, int e) const
    {
        return left.of(p[i].v[e], left.d ? d[i].v[e] : T(0.0f), j0 + (i * 64 + (int)(threadIdx.x % 64)) * E + e);
    }
    __device__ __forceinline__ double sum(const Left<T> &left, int j0) const
    {
        double s = 0;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int e = 0; e < E; e++) s += at(left, j0, i, e);
        return group_sum<64>(s);
    }
};

template <typename T> __global__ __launch_bounds__(1024) void k_verify(VerifyArgs q)
{
    constexpr int E = 16 / sizeof(T);
    extern __shared__ double part[];   // [stretches]
    __shared__ int first, found;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid % 64, w = tid / 64, nw = blockDim.x / 64;
    const int length = length_of(q, b), stretches = (q.V + STRETCH<T> - 1) / STRETCH<T>;
    if (tid == 0) first = q.K;
    __syncthreads();
    for (int k = tid; k < q.K; k += blockDim.x)   // past its length too: the loads do not wait for the length
        if (!passes<T>(q, b, k)) atomicMin(&first, k);
    __syncthreads();
    const int n = min(first, length);
    Left<T> left(q, b, n, length);
    int token = -1;
    while (true) {
        constexpr int AHEAD = 2;   // stretches of a wave on their way at a time (four: 1 x 130000 float32 26 instead of 24 us)
        for (int i = w; i < stretches; i += AHEAD * nw) {
            StretchOf<T> some[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; u++) some[u].load(left, min(i + u * nw, stretches - 1) * STRETCH<T>, q.V);
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const double s = some[u].sum(left, min(i + u * nw, stretches - 1) * STRETCH<T>);
                if (lane == 0 && i + u * nw < stretches) part[i + u * nw] = s;
            }
        }
        __syncthreads();
        if (w == 0) {
            const int run = (stretches + 63) / 64;
            double own = 0;
            for (int i = lane * run; i < min(lane * run + run, stretches); i++) own += part[i];
            const double to = running_sum<64>(own, lane), goal = q.u_sample[b] * __shfl(to, 63);
            int pick = -1, last = -1;
            double at = __shfl_up(to, 1), pick_at = 0, last_at = 0;
            if (lane == 0) at = 0;
            for (int i = lane * run; i < min(lane * run + run, stretches); i++) {
                if (part[i] > 0) {
                    if (pick < 0 && at + part[i] > goal) pick = i, pick_at = at;
                    last = i, last_at = at;
                }
                at += part[i];
            }
            const int lo = lowest_lane<64>(pick >= 0), hi = highest_lane<64>(last >= 0);
            int ans = -1;
            if (hi >= 0) {   // the row has mass
                const int s = lo < 64 ? __shfl(pick, lo) : __shfl(last, hi);
                double below = lo < 64 ? __shfl(pick_at, lo) : __shfl(last_at, hi);
                StretchOf<T> walk;
                walk.load(left, s * STRETCH<T>, q.V);
                int end = -1;
#pragma unroll
                for (int a = 0; a < STRETCH_LOADS; a++) {
                    double mine = 0, c[E], v[E];
#pragma unroll
                    for (int e = 0; e < E; e++) v[e] = walk.at(left, s * STRETCH<T>, a, e), mine += v[e], c[e] = mine;
                    const double incl = running_sum<64>(mine, lane);
                    double before = __shfl_up(incl, 1);
                    if (lane == 0) before = 0;
                    int hit = -1, some = -1;
#pragma unroll
                    for (int e = E - 1; e >= 0; e--) {
                        if (v[e] > 0 && below + (before + c[e]) > goal) hit = e;
                        if (v[e] > 0 && some < 0) some = e;
                    }
                    const int l = lowest_lane<64>(hit >= 0), h = highest_lane<64>(some >= 0);
                    const int base = s * STRETCH<T> + a * 64 * E;
                    const int at_hit = base + (l % 64) * E + __shfl(hit, l % 64), at_end = base + max(h, 0) * E + __shfl(some, max(h, 0));
                    if (ans < 0 && l < 64) ans = at_hit;
                    if (h >= 0) end = at_end;
                    below += __shfl(incl, 63);
                }
                if (ans < 0) ans = end;   // rounding put the goal behind the last element
            }
            if (lane == 0) found = ans;
        }
        __syncthreads();
        token = found;
        if (token >= 0 || left.whole()) break;
        left.d = nullptr, left.only = -1;   // p nowhere above q: the target's own row
        __syncthreads();
    }
    for (int k = tid; k <= q.K; k += blockDim.x) put_token(q, b, n, k, token);
    if (tid == 0) q.accepted[b] = n;
}

}  // namespace mz
