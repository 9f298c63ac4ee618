// Distillation of a policy from a teacher's top logits: per row, the Kullback-Leibler divergence between the teacher's
// distribution over its entries and the student's softmax over all V actions, and its gradient with respect to the logits.
//
//   p_k = softmax(t / tau) over the entries, or exp(t_k / tau - lse) where the teacher's log-sum-exp over all actions is
//         given; rest = 1 - sum p is then one more class: everything outside the entries
//   q   = softmax(z / tau)
//   loss = w tau^2 [ sum_k p_k (log p_k - log q_k) + rest (log rest - log qrest) ],  k over the entries: those of one action have
//         a term each, which is the divergence of their sum less the entropy of the choice between them, no matter of q
//   dz_j = w tau [ q_j (sum p + rest) - p_j ]  inside the entries,  w tau q_j [ sum p + rest - rest / qrest ]  outside
//
// Sums of exponentials run in float32 per thread and are joined in float64; what concerns the few entries is float64
// throughout, since the loss is a small difference of large logarithms.
#pragma once
#include "element_types.h"

namespace mz {

struct DistillArgs {
    const void *logits;      // [R][V], rows ld elements apart
    long long ld;
    const void *index;       // [R][K] int32 or int64, entries outside [0, V) are absent
    const void *teacher;     // [R][K]
    const float *lse;        // [R] or NULL
    const float *weight;     // [R] or NULL: 1
    const float *up;         // [R] gradient of the loss, or NULL: 1
    float *loss;             // [R] or NULL
    void *grad;              // [R][V] contiguous, or NULL
    // [R][4] maximum, sum (0: nothing of the row counts), sum outside the entries and what that one is relative to: written by
    // the loss pass, read by a later gradient pass
    float *stats;
    int R, V, K;
    int index64, teacher_type;
    float tau;
    double inv_tau;
};

__device__ __forceinline__ float teacher_at(const DistillArgs &q, long long i)
{
    return q.teacher_type == 0 ? ((const float *)q.teacher)[i]
         : q.teacher_type == 1 ? (float)((const __bf16 *)q.teacher)[i] : (float)((const _Float16 *)q.teacher)[i];
}

__device__ __forceinline__ int entry_at(const DistillArgs &q, long long i)
{
    const long long j = q.index64 ? ((const long long *)q.index)[i] : (long long)((const int *)q.index)[i];
    return j >= 0 && j < q.V ? (int)j : -1;
}



// What a row's entries come to: sum p, sum p u with p = exp(u) / norm, the norm, and what the teacher has left.
struct Mass { double mass, ent, norm, rest; bool some; };

// From the sums over unnormalised p.
__device__ __forceinline__ void settle(const DistillArgs &q, Mass &e)
{
    const double sum = e.norm;
    if (q.lse) {
        e.mass = sum, e.norm = 1.0;
        e.rest = sum != sum ? sum : fmax(1.0 - sum, 0.0);
    } else {
        e.mass = sum == 0 ? 0.0 : sum != sum ? sum : 1.0;
        e.ent = sum == 0 ? 0.0 : e.ent / sum;
        e.rest = 0.0;
    }
}

// G lanes, C entries each: action, teacher's logit -> probability p.  An absent entry has action -1 and p = 0.
template <int G, int C>
__device__ __forceinline__ Mass weigh(const DistillArgs &q, long long row, const int (&index)[C], const float (&t)[C], double (&p)[C])
{
    float top = -HUGE_VALF;
    bool any = false;
#pragma unroll
    for (int i = 0; i < C; i++) {
        top = fmaxf(top, t[i]);
        any |= index[i] >= 0;
    }
    Mass e;
    e.some = group_max<G>(any ? 1.0f : 0.0f) != 0.0f;
    const double from = q.lse ? (double)q.lse[row] : (double)group_max<G>(top) * q.inv_tau;
    double sum = 0, ent = 0;
#pragma unroll
    for (int i = 0; i < C; i++) {
        const double u = (double)t[i] * q.inv_tau - from;
        p[i] = t[i] == -HUGE_VALF ? 0.0 : exp(u);
        sum += p[i];
        if (!(p[i] == 0)) ent += p[i] * u;
    }
    e.norm = group_sum<G>(sum), e.ent = group_sum<G>(ent);
    settle(q, e);
    if (!q.lse) {
        const double scale = 1.0 / e.norm;
#pragma unroll
        for (int i = 0; i < C; i++) p[i] = p[i] == 0 ? 0.0 : p[i] * scale;
    }
    return e;
}

// exp(d / tau) as exp2 of the product with c = log2(e) / tau.  d = z - m is at most 0, so c's rounding is a change of the
// temperature by 2^-25 of itself, and a -inf logit stays at 0.
__device__ __forceinline__ float expo(float d, float c) { return __builtin_amdgcn_exp2f(d * c); }

// Exponentials of the actions outside the entries are summed relative to the row's maximum m, as all others, where that leaves
// TAIL_LEAST or more.  Below, float32 runs out of exponents (nothing is left of an action 87 tau under the maximum) and the
// gradient's factor rest / sum grows towards overflow: the sum is then taken again relative to the largest logit outside, mt.
// Logits of -inf and of the type's lowest value are masked: where nothing else is outside, the class is left out.
constexpr float TAIL_LEAST = 0x1p-24f;
template <typename T> constexpr float LOWEST = -0x1.fffffep127f;
template <> constexpr float LOWEST<__bf16> = -0x1.fep127f;
template <> constexpr float LOWEST<_Float16> = -65504.0f;

// What q_j, relative to mt, is multiplied with outside the entries.
__device__ __forceinline__ float outside_factor(const DistillArgs &q, const Mass &e, double dsum, double dtail, float m, float mt, float scale)
{
    const double of_row = (e.mass + e.rest) * (mt == m ? 1.0 : exp(((double)mt - (double)m) * q.inv_tau)) / dsum;
    return (float)((of_row - (e.rest == 0 ? 0.0 : e.rest / dtail)) * (double)scale);
}

// The divergence, in lane 0 of G: cross = sum p (z - m) / tau; dsum, dtail: sums of the student's exponentials over all
// actions and over those outside the entries, the latter relative to mt.  Three logarithms, taken by three lanes at once.
template <int G>
__device__ __forceinline__ double divergence(const DistillArgs &q, const Mass &e, double cross, double dsum, double dtail, float m, float mt, int lane)
{
    const double ratio = e.rest == 0 ? 1.0 : e.rest * dsum / dtail;
    const double l = log(lane == 1 ? dsum : lane == 2 && !(e.rest == 0) ? ratio : lane == 0 && e.norm > 0 ? e.norm : 1.0);
    const double of_sum = __shfl(l, 1, G), of_ratio = __shfl(l, 2, G);
    const double below = mt == m ? 0.0 : ((double)m - (double)mt) * q.inv_tau;
    return e.ent - e.mass * l - (cross - e.mass * of_sum) + (e.rest == 0 ? 0.0 : e.rest * (of_ratio + below));
}

// Small action sets: G lanes of a wave hold a row, E actions and 4 entries a lane, all of it in registers.  MODE 0: loss and
// statistics, 1: loss and gradient, 2: gradient from the statistics of an earlier loss pass.  98304 rows of 9 float32, 4
// entries: 8.4 us for the loss, 7.8 for the gradient - two to three times their bytes.  A wave runs 470 (350) vector instructions,
// most of them for the entries in float64, the vector units issue in a sixth of their cycles and waves wait for half of theirs:
// index, logit, exponential, sums over lanes and logarithm each need the one before.  40000 rows of 64, 20 entries: 21 us.
template <typename T, int G, int E, int MODE>
__global__ __launch_bounds__(256) void k_distill_group(DistillArgs q, float c)
{
    constexpr int C = 4;
    const int lane = threadIdx.x % G;
    const long long row = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (row >= q.R) return;
    const T *zr = (const T *)q.logits + row * q.ld;
    T *gr = (T *)q.grad + row * q.V;
    const float weight = q.weight ? q.weight[row] : 1.0f;
    const float scale = MODE == 0 ? 0.0f : weight * q.tau * (q.up ? q.up[row] : 1.0f);
    float z[E], ze[C], t[C];
    int index[C];
#pragma unroll
    for (int i = 0; i < C; i++) {
        const int k = lane + i * G;
        index[i] = k < q.K ? entry_at(q, row * q.K + k) : -1;
        t[i] = index[i] >= 0 ? teacher_at(q, row * q.K + k) : -HUGE_VALF;
        ze[i] = index[i] >= 0 ? widen(zr[index[i]]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int j = lane + i * G;
        z[i] = j < q.V ? widen(zr[j]) : -HUGE_VALF;
    }
    double p[C];
    Mass e = weigh<G, C>(q, row, index, t, p);
    if (!e.some || (MODE == 2 ? scale == 0.0f || q.stats[row * 4 + 1] == 0.0f : weight == 0.0f)) {   // nothing of the row counts
        if (MODE != 0)
#pragma unroll
            for (int i = 0; i < E; i++) if (lane + i * G < q.V) gr[lane + i * G] = T(0.0f);
        if (MODE != 2 && lane == 0) {
            q.loss[row] = 0.0f;
            if (MODE == 0) q.stats[row * 4 + 1] = 0.0f;
        }
        return;
    }
    // which of the lane's actions are entries; an action that several entries name gets their sum, at the first of them
    unsigned inside = 0;
    double total[C];
    bool first[C];
#pragma unroll
    for (int i = 0; i < C; i++) total[i] = p[i], first[i] = index[i] >= 0;
    if (MODE != 0 || q.lse) {
        bool again = false;
#pragma unroll
        for (int i = 0; i < C; i++)
            for (int l = 0; l < G; l++) {
                if (l + i * G >= q.K) break;
                const int j = __shfl(index[i], l, G);
                if (j >= 0 && j % G == lane) inside |= 1u << (j / G);
#pragma unroll
                for (int c = 0; c < C; c++) again |= index[c] == j && j >= 0 && l + i * G < lane + c * G;
            }
        if (MODE != 0 && __any(again)) {
#pragma unroll
            for (int c = 0; c < C; c++) total[c] = 0;
#pragma unroll
            for (int i = 0; i < C; i++)
                for (int l = 0; l < G; l++) {
                    if (l + i * G >= q.K) break;
                    const int j = __shfl(index[i], l, G);
                    const double pj = __shfl(p[i], l, G);
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        total[c] += index[c] == j ? pj : 0.0;
                        if (index[c] == j && l + i * G < lane + c * G) first[c] = false;
                    }
                }
        }
    }
    float m, mt;
    double dsum, dtail;
    if (MODE != 2) {
        m = -HUGE_VALF;
#pragma unroll
        for (int i = 0; i < E; i++) m = fmaxf(m, z[i]);
        m = group_max<G>(m);
        float sum = 0, tail = 0;
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float x = expo(z[i] - m, c);
            sum += x;
            if (q.lse && !(inside >> i & 1)) tail += x;
        }
        dsum = group_sum<G>((double)sum), dtail = group_sum<G>((double)tail), mt = m;
        if (q.lse && dtail < TAIL_LEAST) {
            mt = -HUGE_VALF, tail = 0;
#pragma unroll
            for (int i = 0; i < E; i++) mt = fmaxf(mt, !(inside >> i & 1) && z[i] > LOWEST<T> ? z[i] : -HUGE_VALF);
            mt = group_max<G>(mt);
#pragma unroll
            for (int i = 0; i < E; i++) tail += !(inside >> i & 1) && z[i] > LOWEST<T> ? expo(z[i] - mt, c) : 0.0f;
            dtail = group_sum<G>((double)tail);   // 0 where all is masked
            mt = dtail == 0 ? m : mt;
        }
        double cross = 0;
#pragma unroll
        for (int i = 0; i < C; i++)
            if (!(p[i] == 0)) cross += p[i] * (((double)ze[i] - (double)m) * q.inv_tau);
        cross = group_sum<G>(cross);
        if (dtail == 0) e.rest = 0;   // no action outside the entries has anything left
        const double kl = divergence<G>(q, e, cross, dsum, dtail, m, mt, lane);
        if (lane == 0) {
            q.loss[row] = (float)((double)weight * q.tau * q.tau * kl);
            if (MODE == 0) *(float4 *)(q.stats + row * 4) = make_float4(m, (float)dsum, (float)dtail, mt);
        }
    } else {
        const float4 st = *(const float4 *)(q.stats + row * 4);
        m = st.x, dsum = st.y, dtail = st.z, mt = st.w;
        if (dtail == 0) e.rest = 0;
    }
    if (MODE == 0) return;
    const float f = outside_factor(q, e, dsum, dtail, m, mt, scale), fi = (float)((e.mass + e.rest) * ((double)scale / dsum));
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int j = lane + i * G;
        if (j < q.V && !(inside >> i & 1)) gr[j] = narrow<T>(expo(z[i] - mt, c) * f);
    }
#pragma unroll
    for (int i = 0; i < C; i++)
        if (first[i]) gr[index[i]] = narrow<T>(__builtin_fmaf(expo(ze[i] - m, c), fi, -(float)(total[i] * scale)));
}

// A pack of 16 bytes as it lies in memory.
struct alignas(16) Raw {
    unsigned w[4];
    template <typename P> __device__ __forceinline__ P as() const
    {
        P v;
        __builtin_memcpy(&v, w, 16);
        return v;
    }
    // ... held as four plain registers: the compiler is kept from carrying unpacked values from one step to the next
    template <typename P> __device__ __forceinline__ P again()
    {
        asm("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));
        return as<P>();
    }
    __device__ __forceinline__ void fill(unsigned u) { w[0] = w[1] = w[2] = w[3] = u; }
};
template <typename T> __device__ __forceinline__ unsigned lowest_bits();   // a register of -inf
template <> __device__ __forceinline__ unsigned lowest_bits<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ unsigned lowest_bits<__bf16>() { return 0xff80ff80u; }
template <> __device__ __forceinline__ unsigned lowest_bits<_Float16>() { return 0xfc00fc00u; }

// Wide action sets: one block per row.  A row is a run of whole packs, aligned in memory, between two edges of less than a
// pack, which the block's last two threads take element by element.  The sums take one pass over the row with a running
// maximum per thread, the gradient another; the loss and gradient pass keeps rows of up to NP packs a thread in registers
// between the two (NP > 0) and reads wider ones again.
// 4096 x 32000 bfloat16, 32 entries, loss and gradient: 116 us (524 MB, 4.5 TB/s; a copy 5.1).  1023 x 131071, 64 entries and the
// remaining mass: loss 76 us (268 MB, 3.5 TB/s: 4 rows a compute unit, whose first and last steps overlap little), gradient 106 us
// (536 MB, 5.1 TB/s).  Short rows are bound by the same chain as above, one row at a time: 40000 x 200 float32, 20 entries in 57 us,
// 790 vector instructions a wave and units that issue in a quarter of their cycles.
template <typename T, int THREADS, int NP, int MODE>
__global__ __launch_bounds__(THREADS, NP == 16 ? 4 : NP ? 6 : 8) void k_distill_row(DistillArgs q, float c)
{
    constexpr int E = 16 / sizeof(T), NW = THREADS / 64, U = NP ? NP : 2;   // packs of a thread on their way at a time
    using P = Pack<T, E>;
    extern __shared__ double lds[];
    __shared__ double red[2][NW];
    __shared__ float red_m[NW];
    __shared__ double share[4];
    __shared__ int share_some, repeated;
    double *ep = lds;                                     // [K] probability of an entry
    float *ez = (float *)(lds + q.K);                     // [K] the student's logit of its action
    int *ei = (int *)(ez + q.K);                          // [K] its action, -1: absent
    unsigned *bits = q.lse && MODE != 2 ? (unsigned *)(ei + q.K) : nullptr;   // the entries' actions, E bits a pack
    const long long row = blockIdx.x;
    const T *z = (const T *)q.logits + row * q.ld;
    T *g = MODE ? (T *)q.grad + row * q.V : nullptr;
    const int tid = threadIdx.x, w = tid / 64, lane = tid % 64;
    // pack i covers actions i * E - shift ..; whole packs are [first, last)
    const int shift = (int)(((uintptr_t)z / sizeof(T)) % E);
    const bool same = MODE && (int)(((uintptr_t)g / sizeof(T)) % E) == shift;
    const int first = shift ? 1 : 0, last = max((q.V + shift) / E, first), n_packs = (q.V + shift + E - 1) / E;
    // the edges: pack 0 if it is cut, pack `last` if there is one
    const int edge = tid == THREADS - 1 && shift ? 0 : tid == THREADS - 2 && n_packs > last ? last : -1;
    const float weight = q.weight ? q.weight[row] : 1.0f;
    const float scale = MODE == 0 ? 0.0f : weight * q.tau * (q.up ? q.up[row] : 1.0f);

    auto load_edge = [&]() {
        P v;
#pragma unroll
        for (int k = 0; k < E; k++) {
            const int j = edge * E - shift + k;
            v.v[k] = edge >= 0 && j >= 0 && j < q.V ? z[j] : T(-HUGE_VALF);
        }
        return v;
    };
    auto store_edge = [&](const P &v) {
#pragma unroll
        for (int k = 0; k < E; k++) {
            const int j = edge * E - shift + k;
            if (edge >= 0 && j >= 0 && j < q.V) g[j] = v.v[k];
        }
    };
    // whole pack i; -inf from `last` on (read where the last one is: nothing is read behind the row)
    auto load = [&](int i) {
        Raw r = *(const Raw *)(z + (long long)min(i, last - 1) * E - shift);
        if (i >= last) r.fill(lowest_bits<T>());
        return r;
    };
    auto store = [&](int i, const P &v) {
        T *to = g + (long long)i * E - shift;
        if (same) *(P *)to = v;
        else *(Loose<T, E> *)to = *(const Loose<T, E> *)&v;
    };
    auto nothing = [&]() {   // of the row counts
        if (MODE != 0) {
            P v;
#pragma unroll
            for (int k = 0; k < E; k++) v.v[k] = T(0.0f);
            for (int i = first + tid; i < last; i += THREADS) store(i, v);
            store_edge(v);
        }
        if (MODE != 2 && tid == 0) {
            q.loss[row] = 0.0f;
            if (MODE == 0) q.stats[row * 4 + 1] = 0.0f;
        }
    };

    const int start = first + tid;
    const bool inner = last > first;
    Raw r[U];
    auto begin = [&]() {
        if (inner)
#pragma unroll
            for (int u = 0; u < U; u++) r[u] = load(start + u * THREADS);
    };
    if (MODE == 2 ? (scale == 0.0f || q.stats[row * 4 + 1] == 0.0f) : weight == 0.0f) {
        nothing();
        return;
    }
    if (bits) {
        for (int i = tid; i < (n_packs * E + 31) / 32; i += THREADS) bits[i] = 0;
        __syncthreads();
    }
    if (w == 0) {   // the first wave weighs the entries
        if (lane == 0) repeated = 0;
        auto put = [&](int k, int j) {
            ei[k] = j, ez[k] = j >= 0 ? widen(z[j]) : 0.0f;
            if (bits && j >= 0) atomicOr(&bits[(j + shift) / 32], 1u << ((j + shift) % 32));
        };
        if (q.K <= 64) {
            int index[1] = {lane < q.K ? entry_at(q, row * q.K + lane) : -1};
            float t[1] = {index[0] >= 0 ? teacher_at(q, row * q.K + lane) : -HUGE_VALF};
            double p[1];
            if (lane < q.K) put(lane, index[0]);
            const Mass e = weigh<64, 1>(q, row, index, t, p);
            if (lane < q.K) ep[lane] = p[0];
            if (lane == 0) share[0] = e.mass, share[1] = e.ent, share[2] = e.norm, share[3] = e.rest, share_some = e.some;
        } else {   // in rounds of 64, over lists in LDS
            float top = -HUGE_VALF;
            bool some = false;
            for (int k = lane; k < q.K; k += 64) {
                const int j = entry_at(q, row * q.K + k);
                const float t = j >= 0 ? teacher_at(q, row * q.K + k) : -HUGE_VALF;
                put(k, j);
                ep[k] = t;
                some |= j >= 0;
                top = fmaxf(top, t);
            }
            const double from = q.lse ? (double)q.lse[row] : (double)group_max<64>(top) * q.inv_tau;
            double total = 0, ent = 0;
            for (int k = lane; k < q.K; k += 64) {
                const double u = ep[k] * q.inv_tau - from, x = ep[k] == -HUGE_VAL ? 0.0 : exp(u);
                ep[k] = x;
                total += x;
                if (!(x == 0)) ent += x * u;
            }
            Mass e;
            e.norm = group_sum<64>(total), e.ent = group_sum<64>(ent), e.some = __any(some);
            settle(q, e);
            if (!q.lse) {
                const double scale_p = 1.0 / e.norm;
                for (int k = lane; k < q.K; k += 64) ep[k] = ep[k] == 0 ? 0.0 : ep[k] * scale_p;
            }
            if (lane == 0) share[0] = e.mass, share[1] = e.ent, share[2] = e.norm, share[3] = e.rest, share_some = e.some;
        }
        begin();
    } else begin();   // the other waves' first packs are on their way meanwhile
    float m = -HUGE_VALF, mt, sum = 0, tail = 0;
    // adds a pack's exponentials to the sums
    auto add = [&](int i, const P &v) {
        float x[E], s = 0;
#pragma unroll
        for (int k = 0; k < E; k++) x[k] = expo(widen(v.v[k]) - m, c), s += x[k];
        sum += s;
        if (bits && i < n_packs) {
            const unsigned in = E == 8 ? ((const uint8_t *)bits)[i] : ((const uint8_t *)bits)[i / 2] >> (i % 2 * 4) & 15;
            if (in) {
                s = 0;
#pragma unroll
                for (int k = 0; k < E; k++) s += in >> k & 1 ? 0.0f : x[k];
            }
            tail += s;
        }
    };
    auto top_of = [&](const P &v) {
        float t = widen(v.v[0]);
#pragma unroll
        for (int k = 1; k < E; k++) t = fmaxf(t, widen(v.v[k]));
        return t;
    };
    __syncthreads();
    Mass e{share[0], share[1], share[2], share[3], share_some != 0};
    if (!e.some) {
        nothing();
        return;
    }
    double dsum, dtail;
    if (MODE != 2) {
        // one pass: whenever the thread's maximum rises, what it has summed so far is scaled down to the new one
        auto rise = [&](float top) {
            if (top > m) {
                const float down = m == -HUGE_VALF ? 0.0f : expo(m - top, c);
                sum *= down, tail *= down, m = top;
            }
        };
        auto take = [&](int i, const P &v) {
            if (m != -HUGE_VALF) add(i, v);
            else
#pragma unroll
                for (int k = 0; k < E; k++) if (v.v[k] != v.v[k]) sum = tail = widen(v.v[k]);   // not a number among nothing but -inf
        };
        auto take_all = [&](int i) {
            float top = top_of(r[0].template again<P>());
#pragma unroll
            for (int u = 1; u < U; u++) top = fmaxf(top, top_of(r[u].template again<P>()));
            rise(top);
#pragma unroll
            for (int u = 0; u < U; u++) take(i + u * THREADS, r[u].template again<P>());
        };
        if (inner) {
            if constexpr (NP > 0) take_all(start);
            else
                for (int i = start;;) {
                    const int next = i + U * THREADS;
                    Raw ahead[U];
                    if (next < last)
#pragma unroll
                        for (int u = 0; u < U; u++) ahead[u] = load(next + u * THREADS);
                    take_all(i);
                    if (next >= last) break;
                    i = next;
#pragma unroll
                    for (int u = 0; u < U; u++) r[u] = ahead[u];
                }
        }
        if (edge >= 0) {
            const P cut = load_edge();
            rise(top_of(cut));
            take(edge, cut);
        }
        const float own = m;
        m = group_max<64>(m);
        if (lane == 0) red_m[w] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; i++) m = fmaxf(m, red_m[i]);
        const float down = own == -HUGE_VALF ? 1.0f : expo(own - m, c);
        sum *= down, tail *= down;
        if (m == -HUGE_VALF) sum = tail = m - m;   // no logit above -inf: not a number
        dsum = group_sum<64>((double)sum), dtail = group_sum<64>((double)tail);
        if (lane == 0) red[0][w] = dsum, red[1][w] = dtail;
        __syncthreads();
        dsum = dtail = 0;
#pragma unroll
        for (int i = 0; i < NW; i++) dsum += red[0][i], dtail += red[1][i];
        mt = m;
        if (bits && !(e.rest == 0) && dtail < TAIL_LEAST) {   // seldom: one more pass, action by action
            float top = -HUGE_VALF, low = 0;
            for (int j = tid; j < q.V; j += THREADS) {
                const float v = widen(z[j]);
                if (bits[(j + shift) / 32] >> ((j + shift) % 32) & 1 || !(v > LOWEST<T>)) continue;
                if (v > top) low = top == -HUGE_VALF ? 0.0f : low * expo(top - v, c), top = v;
                low += expo(v - top, c);
            }
            mt = group_max<64>(top);
            if (lane == 0) red_m[w] = mt;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NW; i++) mt = fmaxf(mt, red_m[i]);
            dtail = group_sum<64>(top == -HUGE_VALF ? 0.0 : (double)(low * expo(top - mt, c)));
            if (lane == 0) red[1][w] = dtail;
            __syncthreads();
            dtail = 0;   // and stays so where all is masked
#pragma unroll
            for (int i = 0; i < NW; i++) dtail += red[1][i];
            mt = dtail == 0 ? m : mt;
        }
        if (dtail == 0) e.rest = 0;   // no action outside the entries has anything left
        if (w == NW - 1) {
            double cross = 0;
            for (int k = lane; k < q.K; k += 64)
                if (!(ep[k] == 0)) cross += ep[k] * (((double)ez[k] - (double)m) * q.inv_tau);
            cross = group_sum<64>(cross);
            const double kl = divergence<64>(q, e, cross, dsum, dtail, m, mt, lane);
            if (lane == 0) {
                q.loss[row] = (float)((double)weight * q.tau * q.tau * kl);
                if (MODE == 0) *(float4 *)(q.stats + row * 4) = make_float4(m, (float)dsum, (float)dtail, mt);
            }
        }
    } else {
        const float4 st = *(const float4 *)(q.stats + row * 4);
        m = st.x, dsum = st.y, dtail = st.z, mt = st.w;
        if (dtail == 0) e.rest = 0;
    }
    if (MODE == 0) return;
    // q_j times what stands outside the entries; the entries themselves are put right behind the barrier
    const float f = outside_factor(q, e, dsum, dtail, m, mt, scale), fi = (float)((e.mass + e.rest) * ((double)scale / dsum));
    for (int k = tid; k < q.K; k += THREADS) {
        bool other = false;
        for (int i = 0; i < q.K; i++) other |= i != k && ei[i] == ei[k];
        if (other && ei[k] >= 0) repeated = 1;
    }
    auto emit = [&](const P &v) {
        P o;
#pragma unroll
        for (int k = 0; k < E; k++) o.v[k] = narrow<T>(expo(widen(v.v[k]) - mt, c) * f);
        return o;
    };
    if (inner)
        for (int i = start; i < last; i += U * THREADS) {
            if (NP == 0 && (MODE == 1 || i != start))
#pragma unroll
                for (int u = 0; u < U; u++) r[u] = load(i + u * THREADS);
#pragma unroll
            for (int u = 0; u < U; u++) if (i + u * THREADS < last) store(i + u * THREADS, emit(r[u].template again<P>()));
        }
    if (edge >= 0) store_edge(emit(load_edge()));
    __syncthreads();
    for (int k = tid; k < q.K; k += THREADS) {
        const int j = ei[k];
        if (j < 0) continue;
        double total = ep[k];
        bool lead = true;
        if (repeated) {   // an action that several entries name gets the sum, in the order of the entries
            total = 0;
            for (int i = 0; i < q.K; i++)
                if (ei[i] == j) {
                    total += ep[i];
                    lead &= i >= k;
                }
        }
        if (lead) g[j] = narrow<T>(__builtin_fmaf(expo(ez[k] - m, c), fi, -(float)(total * scale)));
    }
}

}  // namespace mz
