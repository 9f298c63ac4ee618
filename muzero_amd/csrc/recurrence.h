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
    // What y's rounding to 16 bits lost (fine_of), a byte a position of the FORWARD pass's scan order: position s lies at
    // p + b * sb + s / 4 * st + d * sd + s % 4.  p = NULL: not kept.
    View fine;
    const void *first;   // acc[B][D] what goes into position 0 (backward: gradient of the last state), NULL = 0
    const void *state0;  // backward: acc[B][D] the forward pass's first state, NULL = 0
    void *last;          // acc[B][D] the state behind the last position (backward: gradient of the first state), may be NULL
    unsigned long long *granules;   // k_recurrence_chain: a counter of 64 bytes, then what its links hand on, zero before the call
    int links;
};

template <typename T> __device__ __forceinline__ const T *at(const RecurrenceArgs::View &v, int b, long long s, int d)
{
    return (const T *)v.p + (long long)b * v.sb + s * v.st + (long long)d * v.sd;
}

template <typename A> __device__ __forceinline__ A state_at(const void *p, long long i) { return p ? ((const A *)p)[i] : A(0); }

// The bytes of `fine` that L positions need, in words of four positions each: 4 x 8192 x 4096 bfloat16 in 243 us forward and 315
// backward (199 and 294 without them); a load or store of two bytes a lane for every position took 248 and 398.
template <int VEC, int L> struct Fine {
    using W = Pack<unsigned, VEC>;
    W w[L / 4 + 1];
    static __device__ __forceinline__ W *word(const RecurrenceArgs &q, int b, long long k, int d)
    {
        return (W *)((char *)q.fine.p + (long long)b * q.fine.sb + k * q.fine.st + (long long)d * q.fine.sd);
    }
    // Backward: those of what precedes the L positions from s0 on, the forward pass's T - 2 - s0 and the ones in front of it.
    __device__ __forceinline__ void load(const RecurrenceArgs &q, int b, long long s0, int d)
    {
        const long long k = (q.T - 1 - s0 - L) >> 2, last = (q.T - 1) >> 2;   // a word outside 0 .. last holds no position that is used
        if (!q.fine.p) {
#pragma unroll
            for (int j = 0; j <= L / 4; j++) w[j] = W{};
            return;
        }
        const char *at = (const char *)word(q, b, min(max(k, 0ll), last), d);
#pragma unroll
        for (int j = 0; j <= L / 4; j++) {
            w[j] = *(const W *)at;
            if (k + j >= 0 && k + j < last) at += q.fine.st;
        }
    }
    __device__ __forceinline__ void line_up(const RecurrenceArgs &q)   // lets the last of the L positions begin a word
    {
        const unsigned shift = (unsigned)(q.T - 1 - L) & 3;   // s0 is a multiple of 4
#pragma unroll
        for (int j = 0; j < L / 4; j++)
#pragma unroll
            for (int v = 0; v < VEC; v++) w[j].v[v] = __builtin_amdgcn_alignbyte(w[j + 1].v[v], w[j].v[v], shift);
    }
    __device__ __forceinline__ signed char at(int i, int v) const { return (signed char)(w[(L - 1 - i) / 4].v[v] >> (L - 1 - i) % 4 * 8); }
    // Forward: byte 1 of `fine` for position s0 + i, in order, and all of them together.
    __device__ __forceinline__ void put(int i, int v, unsigned fine)
    {
        // v_perm: bytes 0 .. 3 are those of the second operand, 4 .. 7 those of the first, 12 is zero
        constexpr unsigned at[4] = {0x0c0c0c05u, 0x0c0c0500u, 0x0c050100u, 0x05020100u};
        w[i / 4].v[v] = __builtin_amdgcn_perm(fine, i % 4 ? w[i / 4].v[v] : 0u, at[i % 4]);
    }
    __device__ __forceinline__ void store(const RecurrenceArgs &q, int b, long long s0, int d, int left) const
    {
#pragma unroll
        for (int j = 0; j < L / 4; j++) if (4 * j < left) *word(q, b, (s0 >> 2) + j, d) = w[j];
    }
};
// ... of fewer than four positions: byte by byte.
template <int VEC> struct Fine<VEC, 2> {
    signed char f[2];
    static __device__ __forceinline__ signed char *byte(const RecurrenceArgs &q, int b, long long s, int d)
    {
        return (signed char *)q.fine.p + (long long)b * q.fine.sb + (s >> 2) * q.fine.st + (long long)d * q.fine.sd + (s & 3);
    }
    __device__ __forceinline__ void load(const RecurrenceArgs &q, int b, long long s0, int d)
    {
#pragma unroll
        for (int i = 0; i < 2; i++) f[i] = q.fine.p ? *byte(q, b, max(q.T - 2 - s0 - i, 0ll), d) : 0;
    }
    __device__ __forceinline__ void line_up(const RecurrenceArgs &) {}
    __device__ __forceinline__ signed char at(int i, int) const { return f[i]; }
    __device__ __forceinline__ void put(int i, int, unsigned fine) { f[i] = (signed char)(fine >> 8); }
    __device__ __forceinline__ void store(const RecurrenceArgs &q, int b, long long s0, int d, int left) const
    {
#pragma unroll
        for (int i = 0; i < 2; i++) if (i < left) *byte(q, b, s0 + i, d) = f[i];
    }
};
// 32- and 64-bit tensors keep nothing of the kind.
struct NoFine {
    __device__ __forceinline__ void load(const RecurrenceArgs &, int, long long, int) {}
    __device__ __forceinline__ void line_up(const RecurrenceArgs &) {}
    __device__ __forceinline__ signed char at(int, int) const { return 0; }
    __device__ __forceinline__ void put(int, int, unsigned) {}
    __device__ __forceinline__ void store(const RecurrenceArgs &, int, long long, int, int) const {}
};
template <typename T, int VEC, int L> struct FineOf { using type = Fine<VEC, L>; };
template <int VEC, int L> struct FineOf<float, VEC, L> { using type = NoFine; };
template <int VEC, int L> struct FineOf<double, VEC, L> { using type = NoFine; };

// What precedes a position, for its gate's gradient: the forward pass's state there as y and fine hold it.
template <typename T> __device__ __forceinline__ acc_t<T> before_of(T y, signed char fine)
{
    if constexpr (sizeof(T) == 2) return refined(y, fine);
    else return widen(y);
}

// L positions of one strand in registers, all loads asked for at once.
template <typename T, int VEC, int L, bool BWD> struct Strand {
    using P = Pack<T, VEC>;
    using F = typename FineOf<T, VEC, L>::type;
    P a[L], x[L], y[BWD ? L : 1];
    F f;   // forward: empty until the walk

    // FULL: every position is below the end (and, backward, so is the one behind it); otherwise addresses are clamped and
    // positions from `end` on become the identity map.
    template <bool FULL>
    __device__ __forceinline__ void load(const RecurrenceArgs &q, int b, long long s0, long long end, int d, bool want_da)
    {
#pragma unroll
        for (int i = 0; i < L; i++) {
            const long long s = FULL ? s0 + i : min(s0 + i, q.T - 1);
            x[i] = *(const P *)at<T>(q.x, b, s, d);
            a[i] = *(const P *)at<T>(q.a, b, !BWD ? s : FULL && i ? s - 1 : max(s - 1, 0ll), d);
        }
        if constexpr (BWD) {
            if (want_da)
#pragma unroll
                for (int i = 0; i < L; i++) y[i] = *(const P *)at<T>(q.y, b, FULL ? s0 + i + 1 : min(s0 + i + 1, q.T - 1), d);
            if (s0 == 0)
#pragma unroll
                for (int j = 0; j < VEC; j++) a[0].v[j] = T(1.0f);   // nothing precedes the first position: its carry enters as it is
        }
        if (!FULL)
#pragma unroll
            for (int i = 0; i < L; i++)
                if (s0 + i >= end)
#pragma unroll
                    for (int j = 0; j < VEC; j++) a[i].v[j] = T(1.0f), x[i].v[j] = T(0.0f);
    }
    __device__ __forceinline__ void load_fine(const RecurrenceArgs &q, int b, long long s0, int d, bool want_da)
    {
        if (BWD && want_da) f.load(q, b, s0, d);
    }
    // The strand's outputs from the state h in front of it, each rounded once from the 32- or 64-bit state.  A gate's gradient
    // multiplies two states: of 16-bit tensors the forward pass keeps 8 bits of what y's rounding lost beside it (one more byte
    // an element each way), since the stored y alone made that gradient's error 1.4 times a rounding.
    __device__ __forceinline__ void walk(const RecurrenceArgs &q, int b, long long s0, long long end, int d, bool want_da, acc_t<T> (&h)[VEC])
    {
        using A = acc_t<T>;
        if (BWD && want_da) f.line_up(q);
        const int left = (int)min((long long)L, max(end - s0, 0ll));
#pragma unroll
        for (int i = 0; i < L; i++) {
            if (i >= left) continue;
            P o, da;
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                h[j] = fma_acc(widen(a[i].v[j]), h[j], widen(x[i].v[j]));
                o.v[j] = narrow<T>(h[j]);
            }
            *(P *)at<T>(q.out, b, s0 + i, d) = o;
            if constexpr (!BWD && sizeof(T) == 2) {
                if (q.fine.p)
#pragma unroll
                    for (int j = 0; j < VEC; j++) f.put(i, j, fine_of(h[j], o.v[j]));
            }
            if constexpr (BWD) {
                if (want_da) {
                    const bool first = s0 + i + 1 == q.T;   // of the forward pass: what precedes it is the first state
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const A before = first ? state_at<A>(q.state0, (long long)b * q.D + d + j) : before_of<T>(y[i].v[j], f.at(i, j));
                        da.v[j] = narrow<T>(h[j] * before);
                    }
                    *(P *)at<T>(q.da, b, s0 + i, d) = da;
                }
            }
        }
        if constexpr (!BWD) {
            if (q.fine.p) f.store(q, b, s0, d, left);
        }
    }
    // The strand's map behind the map (ra, rx).
    __device__ __forceinline__ void compose(acc_t<T> (&ra)[VEC], acc_t<T> (&rx)[VEC]) const
    {
#pragma unroll
        for (int i = 0; i < L; i++)
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                rx[j] = fma_acc(widen(a[i].v[j]), rx[j], widen(x[i].v[j]));
                ra[j] *= widen(a[i].v[j]);
            }
    }
};

// Neighbouring tiles go to the same compute die (workgroups are dealt to the 8 dies in turn), whose cache then holds the lines
// that tiles share where rows are no multiple of them.
__device__ __forceinline__ unsigned tile_index()
{
    return gridDim.x % 8 ? blockIdx.x : blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
}

constexpr int REC_THREADS = 512;   // of a block: strands of 32 or 64 lanes along the channels

// Channels contiguous: LANES neighbouring lanes hold LANES * VEC neighbouring channels (a "strand") and walk L consecutive
// positions in registers; the block's strands follow each other in time and exchange their maps through LDS,
// one barrier per round of strands, while the next round's loads are on their way.
// Bound by HBM: 8 x 4096 x 2048 bfloat16 in 102 us (403 MB, 3.95 TB/s where a copy reaches 5.1), 4 x 8192 x 4096 in 195 us
// (4.1 TB/s), 32 x 2048 x 4096 in 330 us (4.9 TB/s).  256 tiles are one block of eight waves a compute unit; twice the waves,
// or twice the positions ahead, change nothing.
template <typename T, int VEC, int LANES, int L, bool BWD>
__global__ __launch_bounds__(REC_THREADS) void k_recurrence_channels(RecurrenceArgs q)
{
    constexpr int STRANDS = REC_THREADS / LANES;
    using A = acc_t<T>;
    using P = Pack<T, VEC>;
    struct Map { A a[VEC], x[VEC]; };
    __shared__ Map run[2][STRANDS][LANES];
    const int nv = blockDim.x / LANES;
    const int tiles = (q.D + LANES * VEC - 1) / (LANES * VEC);
    const int tile = tile_index();
    const int b = tile / tiles, c = threadIdx.x % LANES, v = threadIdx.x / LANES;
    const int d0 = (tile % tiles) * LANES * VEC + c * VEC;
    const bool live = d0 < q.D;
    const int d = live ? d0 : q.D - VEC;   // idle lanes read what the last live one reads
    const long long row = (long long)b * q.D + d;
    const long long end = q.T;
    const bool want_da = BWD && q.da.p;
    A carry[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) carry[j] = state_at<A>(q.first, row + j);
    const int round = nv * L;
    int buf = 0;
    Strand<T, VEC, L, BWD> now, next;
    const long long inside = BWD ? end - 1 : end;   // a round that ends here or earlier needs no clamping
    auto load = [&](Strand<T, VEC, L, BWD> &w, long long base) {
        if (base + round <= inside) w.template load<true>(q, b, base + v * L, end, d, want_da);
        else w.template load<false>(q, b, base + v * L, end, d, want_da);
        w.load_fine(q, b, base + v * L, d, want_da);
    };
    load(now, 0);
    for (long long base = 0; base < end; base += round, buf ^= 1) {
        const bool more = base + round < end;
        if (more) load(next, base + round);
        Map m;
#pragma unroll
        for (int j = 0; j < VEC; j++) m.a[j] = A(1), m.x[j] = A(0);
        now.compose(m.a, m.x);
        run[buf][v][c] = m;
        lds_fence_barrier();
        A h[VEC];
        for (int i = 0; i < nv; i++) {
            const Map o = run[buf][i][c];
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                h[j] = i == v ? carry[j] : h[j];
                carry[j] = fma_acc(o.a[j], carry[j], o.x[j]);
            }
        }
        const long long s0 = base + v * L;
        now.walk(q, b, s0, live ? end : s0, d, want_da, h);
        if (more) now = next;
    }
    if (q.last && live && v == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            A z = carry[j];
            if (BWD) z *= widen(at<T>(q.a, b, q.T - 1, d)[j]);
            ((A *)q.last)[row + j] = z;
        }
    }
}

// Long records of few channels: a block for every tile would leave compute units idle, so the axis is cut into links of
// 256 positions (128 backward or in float64) and every link of a tile is a block of its own, with its inputs
// in registers from the first read to the output.  A link hands two things on through memory: its map, as soon as it has it, and the state behind it, once it
// knows the state in front.  To learn that, it looks back over its predecessors: past those that have only a map yet, to one
// whose state is known, and folds the maps in between from there on - the same operations in the same order however far it
// had to look, so results do not depend on timing.
// A value travels as an 8-byte granule of its 32 bits and a tag, written and read as one access at the scope of the device;
// granules are zero before the call.  Links are dealt by a counter, so a block waits for blocks only that are already running
// and that wait for earlier ones in turn: every wait ends.
// 50000 x 1000 float32 in 140 us (600 MB, 4.3 TB/s) and 5 us for the granules; reading the inputs once for the maps and once for
// the outputs instead took 211 us, links of half the positions 150, asking four predecessors at once 142 (registers spill).
// The gradients of 4 x 8192 x 4096 bfloat16 in 315 us (five tensors and a byte an element, 4.7 TB/s) and 7 for the granules.
constexpr int CHAIN_BACK = 16;
constexpr int CHAIN_LENGTH(int size) { return size == 8 ? 8 : 16; }   // positions of a wave; float64 takes twice the registers
constexpr int CHAIN_WAVES(int size, bool backward) { return backward && size != 8 ? 8 : 16; }   // backward: a third tensor in registers
constexpr int CHAIN_ROWS(int size, bool backward) { return CHAIN_LENGTH(size) * CHAIN_WAVES(size, backward); }

template <typename A> __device__ __forceinline__ void granule_put(unsigned long long *to, A v)
{
    unsigned w[sizeof(A) / 4];
    __builtin_memcpy(w, &v, sizeof(A));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(A) / 4); i++)
        __hip_atomic_store(to + i, (unsigned long long)w[i] << 32 | 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename A> __device__ __forceinline__ bool granule_get(const unsigned long long *from, A &v)
{
    unsigned w[sizeof(A) / 4];
    bool there = true;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(A) / 4); i++) {
        const unsigned long long g = __hip_atomic_load(from + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        w[i] = (unsigned)(g >> 32);
        there &= (unsigned)g == 1u;
    }
    __builtin_memcpy(&v, w, sizeof(A));
    return there;
}

__global__ void k_zero_granules(unsigned long long *p, long long n)
{
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) p[i] = 0;
}

template <typename T, int VEC, bool BWD>
__global__ __launch_bounds__(64 * CHAIN_WAVES(sizeof(T), BWD)) void k_recurrence_chain(RecurrenceArgs q)
{
    using A = acc_t<T>;
    using P = Pack<T, VEC>;
    constexpr int L = CHAIN_LENGTH(sizeof(T)), WAVES = CHAIN_WAVES(sizeof(T), BWD), ROWS = CHAIN_ROWS(sizeof(T), BWD), W = sizeof(A) / 4;
    struct Map { A a[VEC], x[VEC]; };
    struct State { A h[VEC]; };
    __shared__ Map run[WAVES][64], back[CHAIN_BACK][64];
    __shared__ State front[64];
    __shared__ unsigned ticket;
    if (threadIdx.x == 0) ticket = atomicAdd((unsigned *)q.granules, 1u);
    __syncthreads();
    const int tiles = (q.D + 64 * VEC - 1) / (64 * VEC), all = tiles * q.B;
    const int link = (int)(ticket / (unsigned)all), tile = (int)(ticket % (unsigned)all);
    const int b = tile / tiles, c = threadIdx.x % 64, v = threadIdx.x / 64;
    const int d0 = (tile % tiles) * 64 * VEC + c * VEC;
    const bool live = d0 < q.D;
    const int d = live ? d0 : q.D - VEC;
    const long long row = (long long)b * q.D + d, s0 = (long long)link * ROWS + v * L;
    const long long end = min((link + 1ll) * ROWS, q.T);
    const bool want_da = BWD && q.da.p;
    Strand<T, VEC, L, BWD> w;
    if (end + (BWD ? 1 : 0) <= q.T && end == (link + 1ll) * ROWS) w.template load<true>(q, b, s0, end, d, want_da);
    else w.template load<false>(q, b, s0, end, d, want_da);
    Map m;
#pragma unroll
    for (int j = 0; j < VEC; j++) m.a[j] = A(1), m.x[j] = A(0);
    w.compose(m.a, m.x);
    run[v][c] = m;
    lds_fence_barrier();
    if (v == 0) {
        // granules of a channel and link: map (a, x), then the state behind it
        auto place = [&](int l, int j) { return q.granules + 8 + (((long long)l * q.B * q.D + row + j) * 3) * W; };
        for (int i = 1; i < WAVES; i++) {
            const Map o = run[i][c];
#pragma unroll
            for (int j = 0; j < VEC; j++) m.x[j] = fma_acc(o.a[j], m.x[j], o.x[j]), m.a[j] *= o.a[j];
        }
        A h[VEC];
        if (link == 0) {
#pragma unroll
            for (int j = 0; j < VEC; j++) h[j] = state_at<A>(q.first, row + j);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; j++) granule_put(place(link, j), m.a[j]), granule_put(place(link, j) + W, m.x[j]);
            int n = 0;   // maps looked past
            while (true) {
                const int l = link - 1 - n;   // >= 0: link 0 hands on its state alone, the look back ends there at the latest
                bool known = true, mapped = true;
                Map o;
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    known &= granule_get(place(l, j) + 2 * W, h[j]);
                    mapped &= granule_get(place(l, j), o.a[j]);
                    mapped &= granule_get(place(l, j) + W, o.x[j]);
                }
                if (__all(known)) break;
                if (n < CHAIN_BACK && __all(mapped)) back[n++][c] = o;
                else __builtin_amdgcn_s_sleep(1);
            }
            for (int i = n - 1; i >= 0; i--) {
                const Map o = back[i][c];
#pragma unroll
                for (int j = 0; j < VEC; j++) h[j] = fma_acc(o.a[j], h[j], o.x[j]);
            }
        }
        State behind, before;
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            before.h[j] = h[j];
            behind.h[j] = fma_acc(m.a[j], h[j], m.x[j]);
            if (link + 1 < q.links) granule_put(place(link, j) + 2 * W, behind.h[j]);
        }
        front[c] = before;
        if (q.last && live && link + 1 == q.links) {
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                A z = behind.h[j];
                if (BWD) z *= widen(at<T>(q.a, b, q.T - 1, d)[j]);
                ((A *)q.last)[row + j] = z;
            }
        }
    }
    // Not before the look back: held across it, they take the registers past 128 and with that half of the waves of a unit.
    w.load_fine(q, b, s0, d, want_da);
    lds_fence_barrier();
    const State before = front[c];
    A h[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) h[j] = before.h[j];
    for (int i = 0; i < v; i++) {
        const Map o = run[i][c];
#pragma unroll
        for (int j = 0; j < VEC; j++) h[j] = fma_acc(o.a[j], h[j], o.x[j]);
    }
    w.walk(q, b, s0, live ? end : s0, d, want_da, h);
}

// Few positions (a step of serving, short records): a thread walks VEC channels of one sequence through all of them.
// 64 x 1 x 2560 bfloat16 in 3.4 us, which is what an empty launch takes.
template <typename T, int VEC, bool BWD>
__global__ __launch_bounds__(256) void k_recurrence_short(RecurrenceArgs q)
{
    using A = acc_t<T>;
    using P = Pack<T, VEC>;
    constexpr int L = 4;
    const int per = q.D / VEC;
    const long long id = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= (long long)per * q.B) return;
    const int b = (int)(id / per), d = (int)(id % per) * VEC;
    const long long row = (long long)b * q.D + d;
    const bool want_da = BWD && q.da.p;
    A h[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) h[j] = state_at<A>(q.first, row + j);
    for (long long s0 = 0; s0 < q.T; s0 += L) {
        Strand<T, VEC, L, BWD> w;
        w.template load<false>(q, b, s0, q.T, d, want_da);
        w.load_fine(q, b, s0, d, want_da);
        w.walk(q, b, s0, q.T, d, want_da, h);
    }
    if (q.last)
#pragma unroll
        for (int j = 0; j < VEC; j++)
            ((A *)q.last)[row + j] = BWD ? h[j] * widen(at<T>(q.a, b, q.T - 1, d)[j]) : h[j];
}

// E consecutive positions of one row; one wide access where they are neighbours in memory (st = 1 or -1).
template <typename T, int E> struct Stretch {
    T v[E];
    __device__ __forceinline__ void load(const RecurrenceArgs::View &w, const T *row, long long s, long long T_, T fill)
    {
        if (s >= 0 && s + E <= T_ && (w.st == 1 || w.st == -1)) {
            const Loose<T, E> p = *(const Loose<T, E> *)(row + (w.st == 1 ? s : -(s + E - 1)));
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = w.st == 1 ? p.v[i] : p.v[E - 1 - i];
        } else
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = s + i >= 0 && s + i < T_ ? row[(s + i) * w.st] : fill;
    }
    __device__ __forceinline__ void store(const RecurrenceArgs::View &w, T *row, long long s, long long T_) const
    {
        if (s + E <= T_ && (w.st == 1 || w.st == -1)) {
            Loose<T, E> p;
#pragma unroll
            for (int i = 0; i < E; i++) p.v[i] = w.st == 1 ? v[i] : v[E - 1 - i];
            *(Loose<T, E> *)(row + (w.st == 1 ? s : -(s + E - 1))) = p;
        } else
#pragma unroll
            for (int i = 0; i < E; i++) if (s + i < T_) row[(s + i) * w.st] = v[i];
    }
};

// Any strides, one row (b, d) per block: every thread walks E consecutive positions, the maps are composed across the wave
// by shuffles and across the waves through LDS.  1000 rows of 4097 float32 in 11.7 us forward and 20.6 backward (49 and 82 MB,
// 4.2 and 4.0 TB/s); a block walks 8192 float32 positions of a long row in about 2.3 us.
template <typename T, int E, bool BWD>
__global__ __launch_bounds__(1024) void k_recurrence_rows(RecurrenceArgs q)
{
    using A = acc_t<T>;
    __shared__ A run_a[2][16], run_x[2][16];
    const int b = blockIdx.x / q.D, d = blockIdx.x % q.D, lane = threadIdx.x % 64, w = threadIdx.x / 64, nw = blockDim.x / 64;
    A carry = state_at<A>(q.first, blockIdx.x);
    const bool want_da = BWD && q.da.p;
    int buf = 0;
    for (long long base = 0; base < q.T; base += (long long)blockDim.x * E, buf ^= 1) {
        const long long s0 = base + (long long)threadIdx.x * E;
        Stretch<T, E> a, x, y;
        typename FineOf<T, 1, E>::type f;
        x.load(q.x, at<T>(q.x, b, 0, d), s0, q.T, T(0.0f));
        // a position behind the end is the identity map; backward, the one in front of the first as well
        if (!BWD) a.load(q.a, at<T>(q.a, b, 0, d), s0, q.T, T(1.0f));
        else {
            a.load(q.a, at<T>(q.a, b, 0, d), s0 - 1, q.T, T(1.0f));
            if (want_da) y.load(q.y, at<T>(q.y, b, 0, d), s0 + 1, q.T, T(0.0f)), f.load(q, b, s0, d), f.line_up(q);
            if (s0 + E > q.T)
#pragma unroll
                for (int i = 0; i < E; i++) if (s0 + i >= q.T) a.v[i] = T(1.0f);
        }
        A ra = A(1), rx = A(0);
#pragma unroll
        for (int i = 0; i < E; i++) rx = fma_acc(widen(a.v[i]), rx, widen(x.v[i])), ra *= widen(a.v[i]);
#pragma unroll
        for (int k = 1; k < 64; k *= 2) {
            const A pa = __shfl_up(ra, k), px = __shfl_up(rx, k);
            if (lane >= k) rx = fma_acc(ra, px, rx), ra *= pa;
        }
        if (lane == 63) run_a[buf][w] = ra, run_x[buf][w] = rx;
        A ea = __shfl_up(ra, 1), ex = __shfl_up(rx, 1);
        if (lane == 0) ea = A(1), ex = A(0);
        lds_fence_barrier();
        A h = carry;
        for (int i = 0; i < nw; i++) {
            if (i == w) h = carry;
            carry = fma_acc(run_a[buf][i], carry, run_x[buf][i]);
        }
        h = fma_acc(ea, h, ex);
        if (s0 >= q.T) continue;
        Stretch<T, E> o, da;
#pragma unroll
        for (int i = 0; i < E; i++) {
            h = fma_acc(widen(a.v[i]), h, widen(x.v[i]));
            o.v[i] = narrow<T>(h);
            if constexpr (BWD) {
                if (want_da) da.v[i] = narrow<T>(h * (s0 + i + 1 == q.T ? state_at<A>(q.state0, blockIdx.x) : before_of<T>(y.v[i], f.at(i, 0))));
            } else if (sizeof(T) == 2) f.put(i, 0, fine_of(h, o.v[i]));
        }
        o.store(q.out, (T *)at<T>(q.out, b, 0, d), s0, q.T);
        if (!BWD && q.fine.p) f.store(q, b, s0, d, (int)min((long long)E, q.T - s0));
        if constexpr (BWD) {
            if (want_da) da.store(q.da, (T *)at<T>(q.da, b, 0, d), s0, q.T);
        }
    }
    if (q.last && threadIdx.x == 0) {
        if (BWD) carry *= widen(*at<T>(q.a, b, q.T - 1, d));
        ((A *)q.last)[blockIdx.x] = carry;
    }
}

// A few long rows: links of ROW_LINK positions of one row, a block each, handed on as in k_recurrence_chain; a wave looks back
// over 64 predecessors at once, a lane each.  One row of 4 000 000 float32 in 32 us (48 MB; 1118 us walked by one block).
constexpr int ROW_STRETCH = 8, ROW_LINK = 1024 * ROW_STRETCH;

template <typename T, bool BWD>
__global__ __launch_bounds__(1024) void k_recurrence_row_chain(RecurrenceArgs q)
{
    using A = acc_t<T>;
    constexpr int E = ROW_STRETCH, W = sizeof(A) / 4, WAVES = 16;
    __shared__ A run_a[WAVES], run_x[WAVES], front;
    __shared__ unsigned ticket;
    if (threadIdx.x == 0) ticket = atomicAdd((unsigned *)q.granules, 1u);
    __syncthreads();
    const int rows = q.B * q.D, link = (int)(ticket / (unsigned)rows), row = (int)(ticket % (unsigned)rows);
    const int b = row / q.D, d = row % q.D, lane = threadIdx.x % 64, w = threadIdx.x / 64;
    const bool want_da = BWD && q.da.p;
    const long long s0 = (long long)link * ROW_LINK + threadIdx.x * E;
    Stretch<T, E> a, x, y;
    typename FineOf<T, 1, E>::type f;
    x.load(q.x, at<T>(q.x, b, 0, d), s0, q.T, T(0.0f));
    if (!BWD) a.load(q.a, at<T>(q.a, b, 0, d), s0, q.T, T(1.0f));
    else {
        a.load(q.a, at<T>(q.a, b, 0, d), s0 - 1, q.T, T(1.0f));
        if (want_da) y.load(q.y, at<T>(q.y, b, 0, d), s0 + 1, q.T, T(0.0f)), f.load(q, b, s0, d), f.line_up(q);
        if (s0 + E > q.T)
#pragma unroll
            for (int i = 0; i < E; i++) if (s0 + i >= q.T) a.v[i] = T(1.0f);
    }
    A ra = A(1), rx = A(0);
#pragma unroll
    for (int i = 0; i < E; i++) rx = fma_acc(widen(a.v[i]), rx, widen(x.v[i])), ra *= widen(a.v[i]);
#pragma unroll
    for (int k = 1; k < 64; k *= 2) {
        const A pa = __shfl_up(ra, k), px = __shfl_up(rx, k);
        if (lane >= k) rx = fma_acc(ra, px, rx), ra *= pa;
    }
    if (lane == 63) run_a[w] = ra, run_x[w] = rx;
    A ea = __shfl_up(ra, 1), ex = __shfl_up(rx, 1);
    if (lane == 0) ea = A(1), ex = A(0);
    lds_fence_barrier();
    if (w == 0) {
        auto place = [&](int l) { return q.granules + 8 + (((long long)l * rows + row) * 3) * W; };
        A ma = run_a[0], mx = run_x[0];
        for (int i = 1; i < WAVES; i++) mx = fma_acc(run_a[i], mx, run_x[i]), ma *= run_a[i];
        A h;
        if (link == 0) h = state_at<A>(q.first, row);
        else {
            if (lane == 0) granule_put(place(link), ma), granule_put(place(link) + W, mx);
            A oa, ox, oh;
            int known_at;
            while (true) {
                const bool there = lane < link;   // predecessor link - 1 - lane; link 0 hands on its state alone
                const unsigned long long *p = place(there ? link - 1 - lane : 0);
                const bool known = granule_get(p + 2 * W, oh), has_a = granule_get(p, oa), has_x = granule_get(p + W, ox);
                const unsigned long long states = __ballot(there && known), maps = __ballot(there && has_a && has_x);
                if (states) {
                    known_at = __ffsll((long long)states) - 1;
                    const unsigned long long nearer = (1ull << known_at) - 1;
                    if ((maps & nearer) == nearer) break;
                }
                __builtin_amdgcn_s_sleep(1);
            }
            known_at = __builtin_amdgcn_readfirstlane(known_at);
            h = lane_read(oh, known_at);
            for (int i = known_at - 1; i >= 0; i--) h = fma_acc(lane_read(oa, i), h, lane_read(ox, i));
        }
        const A behind = fma_acc(ma, h, mx);
        if (lane == 0) {
            if (link + 1 < q.links) granule_put(place(link) + 2 * W, behind);
            front = h;
            if (q.last && link + 1 == q.links) ((A *)q.last)[row] = BWD ? behind * widen(*at<T>(q.a, b, q.T - 1, d)) : behind;
        }
    }
    lds_fence_barrier();
    if (s0 >= q.T) return;
    A h = front;
    for (int i = 0; i < w; i++) h = fma_acc(run_a[i], h, run_x[i]);
    h = fma_acc(ea, h, ex);
    Stretch<T, E> o, da;
#pragma unroll
    for (int i = 0; i < E; i++) {
        h = fma_acc(widen(a.v[i]), h, widen(x.v[i]));
        o.v[i] = narrow<T>(h);
        if constexpr (BWD) {
            if (want_da) da.v[i] = narrow<T>(h * (s0 + i + 1 == q.T ? state_at<A>(q.state0, row) : before_of<T>(y.v[i], f.at(i, 0))));
        } else if (sizeof(T) == 2) f.put(i, 0, fine_of(h, o.v[i]));
    }
    o.store(q.out, (T *)at<T>(q.out, b, 0, d), s0, q.T);
    if (!BWD && q.fine.p) f.store(q, b, s0, d, (int)min((long long)E, q.T - s0));
    if constexpr (BWD) {
        if (want_da) da.store(q.da, (T *)at<T>(q.da, b, 0, d), s0, q.T);
    }
}

}  // namespace mz
