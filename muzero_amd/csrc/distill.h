// Distillation of a policy from a teacher's top logits: per row, the Kullback-Leibler divergence between the teacher's
// distribution over its entries and the student's softmax over all V actions, and its gradient with respect to the logits.
//
//   p_k = softmax(t / tau) over the entries, or exp(t_k / tau - lse) where the teacher's log-sum-exp over all actions is
//         given; rest = 1 - sum p is then one more class: everything outside the entries
//   q   = softmax(z / tau)
//   loss = w tau^2 [ sum_k p_k (log p_k - log q_k) + rest (log rest - log qrest) ]
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
    float *stats;            // [R][4] maximum, sum, tail sum: written by the loss pass, read by a later gradient pass
    int R, V, K;
    int index64, teacher_type;
    float tau;
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


// The teacher's side of a row, in LDS: what one wave makes of the K entries.
struct Entries {
    int *index;      // [K] action of the entry, -1: absent
    double *p;       // [K] the entry's probability
    double *total;   // [K] probability of its action over all entries that name it; < 0: not the first of them
    double mass, ent, rest;   // sum p, sum p log p, 1 - mass (>= 0; 0 without lse)
    bool some;
};

__device__ __forceinline__ double wave_sum(double v)
{
    for (int k = 32; k; k /= 2) v += __shfl_xor(v, k);
    return v;
}
__device__ __forceinline__ float wave_max(float v)
{
    for (int k = 32; k; k /= 2) v = fmaxf(v, __shfl_xor(v, k));
    return v;
}

// One wave; the lists are complete for the whole block after its next barrier.
__device__ __forceinline__ void read_entries(const DistillArgs &q, long long row, Entries &e, unsigned *bits)
{
    const int lane = threadIdx.x % 64;
    const double inv_tau = 1.0 / (double)q.tau;
    bool some = false;
    double top = -HUGE_VAL;
    for (int k = lane; k < q.K; k += 64) {
        const int j = entry_at(q, row * q.K + k);
        const double t = j >= 0 ? (double)teacher_at(q, row * q.K + k) * inv_tau : -HUGE_VAL;
        e.index[k] = j, e.p[k] = t;
        some |= j >= 0;
        top = t > top || t != t ? t : top;
        if (bits && j >= 0) atomicOr(&bits[j / 32], 1u << (j % 32));
    }
    for (int k = 32; k; k /= 2) {
        const double o = __shfl_xor(top, k);
        top = o > top || o != o ? o : top;
    }
    e.some = __any(some);
    if (q.lse) top = (double)q.lse[row];
    double z = 0, sum = 0;
    if (!q.lse) {
        for (int k = lane; k < q.K; k += 64) z += e.p[k] == -HUGE_VAL ? 0.0 : exp(e.p[k] - top);
        z = wave_sum(z);
    }
    const double logz = q.lse ? 0.0 : log(z), inv_z = q.lse ? 1.0 : 1.0 / z;
    double ent = 0;
    for (int k = lane; k < q.K; k += 64) {
        const bool none = e.p[k] == -HUGE_VAL;
        const double u = e.p[k] - top, p = none ? 0.0 : exp(u) * inv_z;
        e.p[k] = p;
        sum += p;
        if (!(p == 0)) ent += p * (u - logz);
    }
    e.mass = wave_sum(sum);
    e.ent = wave_sum(ent);
    e.rest = q.lse ? fmax(1.0 - e.mass, 0.0) : 0.0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int k = lane; k < q.K; k += 64) {   // an action that several entries name gets the sum, in the order of the entries
        const int j = e.index[k];
        double tot = 0;
        bool first = j >= 0;
        for (int i = 0; i < q.K; i++)
            if (e.index[i] == j) {
                tot += e.p[i];
                if (i < k) first = false;
            }
        e.total[k] = first ? tot : -1.0;
    }
}

// One block per row.  The row's packs of 16 bytes stay in registers between the passes where NP of them per thread hold it
// (KEEP); otherwise each pass reads it again.  MODE 0: loss and statistics, 1: loss and gradient, 2: gradient from the
// statistics of an earlier loss pass.
template <typename T, int THREADS, int NP, bool KEEP, int MODE>
__global__ __launch_bounds__(THREADS) void k_distill_row(DistillArgs q, float c_hi, float c_lo)
{
    constexpr int E = 16 / sizeof(T), NW = THREADS / 64;
    using P = Pack<T, E>;
    extern __shared__ double lds[];
    __shared__ double red[3][NW];
    __shared__ double share[4];
    Entries e;
    e.p = lds, e.total = lds + q.K, e.index = (int *)(lds + 2 * q.K);
    unsigned *bits = q.lse && MODE != 2 ? (unsigned *)(e.index + q.K) : nullptr;
    const long long row = blockIdx.x;
    const T *z = (const T *)q.logits + row * q.ld;
    T *g = q.grad ? (T *)q.grad + row * q.V : nullptr;
    const int tid = threadIdx.x, w = tid / 64;
    // packs are aligned in memory: the first one begins up to E - 1 elements in front of the row
    const int shift = (int)(((uintptr_t)z / sizeof(T)) % E);
    const bool same = g && (int)(((uintptr_t)g / sizeof(T)) % E) == shift;
    const int n_packs = (q.V + shift + E - 1) / E;
    const float weight = q.weight ? q.weight[row] : 1.0f;
    const float scale = MODE == 0 ? 0.0f : weight * q.tau * (q.up ? q.up[row] : 1.0f);

    auto load = [&](int i, P &v) {
        const int j = i * E - shift;
        if (j >= 0 && j + E <= q.V) v = *(const P *)(z + j);
        else
#pragma unroll
            for (int k = 0; k < E; k++) v.v[k] = j + k >= 0 && j + k < q.V ? z[j + k] : T(-HUGE_VALF);
    };
    auto store = [&](int i, const P &v) {
        const int j = i * E - shift;
        if (same && j >= 0 && j + E <= q.V) *(P *)(g + j) = v;
        else
#pragma unroll
            for (int k = 0; k < E; k++) if (j + k >= 0 && j + k < q.V) g[j + k] = v.v[k];
    };
    auto zeros = [&]() {
        P v;
#pragma unroll
        for (int k = 0; k < E; k++) v.v[k] = T(0.0f);
        for (int i = tid; i < n_packs; i += THREADS) store(i, v);
    };

    if (MODE == 2 ? (scale == 0.0f || q.stats[row * 4 + 3] == 0.0f) : weight == 0.0f) {   // nothing of the row counts
        if (MODE != 0) zeros();
        if (MODE != 2 && tid == 0) {
            q.loss[row] = 0.0f;
            if (MODE == 0) q.stats[row * 4 + 3] = 0.0f;
        }
        return;
    }
    P keep[KEEP ? NP : 1];
    float m = -HUGE_VALF;
    if (KEEP)
#pragma unroll
        for (int n = 0; n < NP; n++) load(tid + n * THREADS, keep[n]);   // -inf behind the row
    if (bits) {
        for (int i = tid; i < (q.V + 31) / 32; i += THREADS) bits[i] = 0;
        __syncthreads();
    }
    if (w == 0) {
        read_entries(q, row, e, bits);
        if (tid == 0) share[0] = e.mass, share[1] = e.ent, share[2] = e.rest, share[3] = e.some ? 1.0 : 0.0;
    }
    double dsum = 0, dtail = 0;
    if (MODE != 2) {
        if (KEEP)
#pragma unroll
            for (int n = 0; n < NP; n++)
#pragma unroll
                for (int k = 0; k < E; k++) m = fmaxf(m, widen(keep[n].v[k]));
        else
            for (int i = tid; i < n_packs; i += THREADS) {
                P v;
                load(i, v);
#pragma unroll
                for (int k = 0; k < E; k++) m = fmaxf(m, widen(v.v[k]));
            }
        m = wave_max(m);
        if (tid % 64 == 0) red[0][w] = m;
    }
    __syncthreads();
    if (MODE != 2) {
#pragma unroll
        for (int i = 0; i < NW; i++) m = fmaxf(m, (float)red[0][i]);
    } else m = q.stats[row * 4];
    e.mass = share[0], e.ent = share[1], e.rest = share[2], e.some = share[3] != 0.0;
    if (!e.some) {
        if (MODE != 0) zeros();
        if (MODE != 2 && tid == 0) {
            q.loss[row] = 0.0f;
            if (MODE == 0) q.stats[row * 4 + 3] = 0.0f;
        }
        return;
    }
    // exp((z - m) / tau) as exp2 of the product with log2(e) / tau in two parts (c_lo > 0 keeps a -inf logit at -inf)
    auto expo = [&](T v) {
        const float d = widen(v) - m;
        return __builtin_amdgcn_exp2f(__builtin_fmaf(d, c_lo, d * c_hi));
    };
    if (MODE != 2) {
        float sum = 0, tail = 0;
        auto add = [&](int i, const P &v) {
            const int j = i * E - shift;
#pragma unroll
            for (int k = 0; k < E; k++) {
                const float x = expo(v.v[k]);
                sum += x;
                if (bits && j + k >= 0 && j + k < q.V && !(bits[(j + k) / 32] >> ((j + k) % 32) & 1)) tail += x;
            }
        };
        if (KEEP)
#pragma unroll
            for (int n = 0; n < NP; n++) add(tid + n * THREADS, keep[n]);
        else
            for (int i = tid; i < n_packs; i += THREADS) {
                P v;
                load(i, v);
                add(i, v);
            }
        dsum = wave_sum(sum), dtail = wave_sum(tail);
        if (tid % 64 == 0) red[1][w] = dsum, red[2][w] = dtail;
        __syncthreads();
        dsum = dtail = 0;
#pragma unroll
        for (int i = 0; i < NW; i++) dsum += red[1][i], dtail += red[2][i];
        if (!(dtail != 0)) e.rest = 0;   // no action outside the entries has anything left
        if (w == 0) {
            double cross = 0;
            const double lsum = log(dsum), inv_tau = 1.0 / (double)q.tau;
            for (int k = tid; k < q.K; k += 64)
                if (e.index[k] >= 0 && !(e.p[k] == 0))
                    cross += e.p[k] * (((double)widen(z[e.index[k]]) - (double)m) * inv_tau - lsum);
            cross = wave_sum(cross);
            if (tid == 0) {
                double kl = e.ent - cross;
                if (!(e.rest == 0)) kl += e.rest * (log(e.rest) - log(dtail) + lsum);
                q.loss[row] = (float)((double)weight * q.tau * q.tau * kl);
                if (MODE == 0) {
                    float *st = q.stats + row * 4;
                    st[0] = m, st[1] = (float)dsum, st[2] = (float)dtail, st[3] = 1.0f;
                }
            }
        }
    } else {
        dsum = q.stats[row * 4 + 1], dtail = q.stats[row * 4 + 2];
        if (!(dtail != 0)) e.rest = 0;
    }
    if (MODE == 0) return;
    // q_j times what stands outside the entries; the entries themselves are put right behind the barrier
    const double whole = e.mass + e.rest;
    const double outside = e.rest == 0 ? whole : whole - e.rest * dsum / dtail;
    const float f = (float)(outside / dsum * scale);
    auto emit = [&](int i, const P &v) {
        P o;
#pragma unroll
        for (int k = 0; k < E; k++) o.v[k] = narrow<T>(expo(v.v[k]) * f);
        store(i, o);
    };
    if (KEEP)
#pragma unroll
        for (int n = 0; n < NP; n++) {
            if (tid + n * THREADS < n_packs) emit(tid + n * THREADS, keep[n]);
        }
    else
        for (int i = tid; i < n_packs; i += THREADS) {
            P v;
            load(i, v);
            emit(i, v);
        }
    __syncthreads();
    for (int k = tid; k < q.K; k += THREADS) {
        const double tot = e.total[k];
        const int j = e.index[k];
        if (j >= 0 && !(tot < 0)) g[j] = narrow<T>((float)(((double)expo(z[j]) / dsum * whole - tot) * scale));
    }
}

}  // namespace mz
