// C entry points of the tensor operators around a policy: gated linear recurrence, distillation, verification of drafts.
// Argument checks and launches; the kernels live in the headers included below.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/muzero_amd.h"
#include "api.h"
#include "distill.h"
#include "recurrence.h"
#include "verify.h"

using namespace mz;

// A launch takes fewer than 2^32 threads: larger calls are launched in slices of at most so many blocks (of 1024 threads at most).
constexpr long long SLICE = 1 << 20;
constexpr long long MOST_THREADS = (1ll << 32) - 1;

static const char *ahead(const void *p, long long bytes) { return p ? (const char *)p + bytes : nullptr; }
static char *ahead(void *p, long long bytes) { return p ? (char *)p + bytes : nullptr; }

static size_t size_of(int type) { return type == MZ_F64 ? 8 : type == MZ_F32 ? 4 : 2; }

// ------------------------------------------------------------------------------------------------ recurrence

// Which kernel serves a recurrence, as measured (one MI355X, kernel times):
// - REC_LENGTH, positions a strand of k_recurrence_channels holds in registers: 8 x 4096 x 2048 bfloat16 in 102 us with 8, 126
//   with 4, 195 with 16 (146 registers: one block a compute unit, its loads no longer ahead of its arithmetic).
// - From REC_MANY_TILES tiles on a strand is 64 lanes wide, 256 bytes of a position: 32 x 2048 x 4096 bfloat16 330 against 367 us.
// - Below REC_FEW_TILES tiles of 32 lanes, records of REC_LEAST_LINKS links or more are cut into chains (the zeroing of their granules
//   counted): 1 x 4096 x 512 bfloat16 13 against 49 us, 4 x 2048 x 1024 18 against 32, 6 x 2048 x 2048 (192 tiles) 40 against 46, at
//   256 tiles 109 against 102;
//   three links (1 x 600 x 512) 11.2 against 10.5, their gradients 15.3 against 17.6.  Gradients, with five tensors on their
//   way, gain up to REC_FEW_TILES_BACKWARD tiles: 4 x 8192 x 4096 (256 tiles) 301 against 334, 8 x 2048 x 2500 (320) 114
//   against 159, both without the byte an element that `fine` adds (321 and 125 with it).
// - Fewer than REC_FEW_ROWS rows of REC_LEAST_ROW_LINKS links or more are cut into links: 1 x 65536 float32 7.3 against 18.1 us (the
//   granules' 1.4 us included), 64 x 32768 12.7 against 13.3, its gradients 15.4 against 18.5; 200 x 32768 23.7 against 17.
constexpr int REC_LENGTH = 8;
constexpr long long REC_MANY_TILES = 512, REC_FEW_TILES = 256, REC_FEW_TILES_BACKWARD = 512, REC_LEAST_LINKS = 3;
constexpr long long REC_FEW_ROWS = 128, REC_LEAST_ROW_LINKS = 3;

// How a recurrence is run: chosen by sizes, strides and alignment alone, for the workspace query and the call alike.
struct RecurrencePlan {
    bool channels, brief;    // channels contiguous; so few positions that a thread walks them all
    int vec, lanes;          // channels a thread holds, lanes of a strand
    int strands, links;      // of a block; of a tile's chain, or 0: one block walks the tile
};

// VEC = 2 is a 4-byte access of a 16-bit type
static RecurrencePlan plan_recurrence(const mz_recurrence *a, bool backward)
{
    RecurrencePlan p{true, false, 1, 32, 1, 0};
    uint64_t low = 0;   // low bits of every address and step along the axis and the sequences
    const int size = (int)size_of(a->type);
    for (const mz_strided *t : {&a->gate, &a->x, &a->out, &a->y, &a->out_gate}) {
        if (!t->p) continue;
        if (t->stride_d != 1) p.channels = false;
        low |= (uint64_t)(uintptr_t)t->p | (uint64_t)t->stride_b * size | (uint64_t)t->stride_t * size;
    }
    if (size == 2 && a->fine.p)   // four bytes a channel where the others have two; only neighbouring ones travel together
        low |= (((uint64_t)(uintptr_t)a->fine.p | (uint64_t)a->fine.stride_b | (uint64_t)a->fine.stride_t) >> 1) | (a->fine.stride_d != 4 ? 2 : 0);
    if (a->D == 1) p.channels = false;
    if (!p.channels) {
        const long long links = (a->T + ROW_LINK - 1) / ROW_LINK;
        const long long rows = (long long)a->B * a->D;
        if (rows < REC_FEW_ROWS && links >= REC_LEAST_ROW_LINKS && links <= MOST_THREADS / 1024 / rows) p.links = (int)links;
        return p;
    }
    auto fits = [&](int n) { return a->D % n == 0 && low % (uint64_t)(n * size) == 0; };
    // a step, or a few: the block of strands would stand idle (64 x 4 x 4096 bfloat16 4.1 against 5.8 us, 8 positions 4.8 against
    // 6.4, 16 positions 7.2 against 6.6)
    const long long wide = 16 / size;
    p.brief = a->T <= 8;
    if (p.brief) {
        p.vec = fits((int)wide) ? (int)wide : 1;
        return p;
    }
    p.vec = size == 2 && fits(2) ? 2 : 1;
    auto tiles_of = [&](int lanes) { return (long long)a->B * ((a->D + lanes * p.vec - 1) / (lanes * p.vec)); };
    p.lanes = tiles_of(64) >= REC_MANY_TILES ? 64 : 32;
    p.strands = (int)std::min<long long>(REC_THREADS / p.lanes, std::max<long long>(2, (a->T + REC_LENGTH - 1) / REC_LENGTH));
    const long long links = (a->T + CHAIN_ROWS(size, backward) - 1) / CHAIN_ROWS(size, backward);
    if (a->T > 256 && tiles_of(32) < (backward ? REC_FEW_TILES_BACKWARD : REC_FEW_TILES) && links >= REC_LEAST_LINKS &&
        links <= MOST_THREADS / (64 * CHAIN_WAVES(size, backward)) / tiles_of(64)) p.links = (int)links;
    return p;
}

template <typename T, int VEC, int LANES, bool BWD> static void launch_channels(const RecurrencePlan &p, const RecurrenceArgs &q, hipStream_t st)
{
    const unsigned tiles = (unsigned)((long long)q.B * ((q.D + LANES * VEC - 1) / (LANES * VEC)));
    hipLaunchKernelGGL((k_recurrence_channels<T, VEC, LANES, REC_LENGTH, BWD>), dim3(tiles), dim3(LANES * p.strands), 0, st, q);
}

static size_t granule_count(const mz_recurrence *a, const RecurrencePlan &p)
{
    return p.links ? 8 + (size_t)p.links * a->B * a->D * 3 * (a->type == MZ_F64 ? 2 : 1) : 0;
}

template <typename T> static void zero_granules(const RecurrenceArgs &q, hipStream_t st)
{
    const long long granules = 8 + (long long)q.links * q.B * q.D * 3 * (long long)(sizeof(acc_t<T>) / 4);
    const unsigned blocks = (unsigned)std::min<long long>((granules + 255) / 256, 2048);
    hipLaunchKernelGGL(k_zero_granules, dim3(blocks), dim3(256), 0, st, q.granules, granules);
}

template <typename T, int VEC, bool BWD> static void launch_chain(const RecurrenceArgs &q, hipStream_t st)
{
    zero_granules<T>(q, st);
    const long long tiles = (long long)q.B * ((q.D + 64 * VEC - 1) / (64 * VEC));
    hipLaunchKernelGGL((k_recurrence_chain<T, VEC, BWD>), dim3((unsigned)(tiles * q.links)), dim3(64 * CHAIN_WAVES(sizeof(T), BWD)), 0, st, q);
}

template <typename T, int VEC, bool BWD> static void launch_channels(const RecurrencePlan &p, const RecurrenceArgs &q, hipStream_t st)
{
    if (p.links) launch_chain<T, VEC, BWD>(q, st);
    else if (p.lanes == 64) launch_channels<T, VEC, 64, BWD>(p, q, st);
    else launch_channels<T, VEC, 32, BWD>(p, q, st);
}

template <typename T, int VEC, bool BWD> static void launch_short(const RecurrenceArgs &q, hipStream_t st)
{
    const long long n = (long long)q.B * (q.D / VEC);
    const unsigned threads = n >= 65536 ? 256 : 64;   // small calls: spread over the compute units
    hipLaunchKernelGGL((k_recurrence_short<T, VEC, BWD>), dim3((unsigned)((n + threads - 1) / threads)), dim3(threads), 0, st, q);
}

template <typename T, int E, bool BWD> static void launch_rows(const RecurrenceArgs &q, hipStream_t st)
{
    const long long need = (q.T + E - 1) / E;
    const unsigned threads = need >= 1024 ? 1024 : (unsigned)((need + 63) / 64 * 64);
    hipLaunchKernelGGL((k_recurrence_rows<T, E, BWD>), dim3((unsigned)((long long)q.B * q.D)), dim3(threads), 0, st, q);
}

template <typename T, bool BWD> static void launch_recurrence(const RecurrencePlan &p, const RecurrenceArgs &q, hipStream_t st)
{
    constexpr int W = 16 / (int)sizeof(T);
    if (!p.channels && p.links) {
        zero_granules<T>(q, st);
        hipLaunchKernelGGL((k_recurrence_row_chain<T, BWD>), dim3((unsigned)((long long)q.B * q.D * q.links)), dim3(1024), 0, st, q);
    } else if (!p.channels) {
        // positions a thread: 4000 rows of 500 float32 in 7.5 us with 8, 9.9 with 2; of 250 in 6.3 and 6.5, of 60 in 6.0 and 4.8
        if (q.T > 256) launch_rows<T, 8, BWD>(q, st);
        else launch_rows<T, 2, BWD>(q, st);
    } else if (p.brief) {
        if (p.vec == W) launch_short<T, W, BWD>(q, st);
        else launch_short<T, 1, BWD>(q, st);
    } else if (sizeof(T) == 2 && p.vec == 2) launch_channels<T, sizeof(T) == 2 ? 2 : 1, BWD>(p, q, st);
    else launch_channels<T, 1, BWD>(p, q, st);
}

// q in slices of sequences, and one sequence in slices of channels, where it is more than one launch can take.
template <typename T, bool BWD> static void launch_slices(const RecurrencePlan &p, const RecurrenceArgs &q, hipStream_t st)
{
    // channels of a block; a chain is one launch by its plan, a thread of k_recurrence_short serves a channel at least
    const long long wide = p.channels ? (long long)p.lanes * p.vec : 1, blocks = (q.D + wide - 1) / wide;
    if (p.links || p.brief || blocks * q.B <= SLICE) return launch_recurrence<T, BWD>(p, q, st);
    const int sequences = (int)std::max(1ll, SLICE / blocks), channels = (int)std::min<long long>(q.D, SLICE * wide);
    for (int b = 0; b < q.B; b += sequences)
        for (int d = 0; d < q.D; d += channels) {
            RecurrenceArgs s = q;
            s.B = std::min(sequences, q.B - b), s.D = std::min(channels, q.D - d);
            for (RecurrenceArgs::View *v : {&s.a, &s.x, &s.y, &s.out, &s.da}) v->p = ahead(v->p, (b * v->sb + d * v->sd) * (long long)sizeof(T));
            s.fine.p = ahead(s.fine.p, b * s.fine.sb + d * s.fine.sd);
            const long long state = ((long long)b * q.D + d) * (long long)sizeof(acc_t<T>);
            s.first = ahead(s.first, state), s.state0 = ahead(s.state0, state), s.last = ahead(s.last, state);
            launch_recurrence<T, BWD>(p, s, st);
        }
}

static int check_recurrence(const mz_recurrence *a, bool backward, const char *fn)
{
    if (!a) return api_fail(MZ_ERR_ARG, std::string(fn) + ": null argument");
    if (a->type < MZ_F32 || a->type > MZ_F64) return api_fail(MZ_ERR_ARG, std::string(fn) + ": unknown element type");
    if (a->B < 1 || a->D < 1 || a->T < 1 || (int64_t)a->B * a->D > (1 << 30))
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": sizes must be positive, and B * D at most 2^30");
    if (!a->gate.p || !a->x.p || !a->out.p) return api_fail(MZ_ERR_ARG, std::string(fn) + ": null tensor");
    if (backward && (a->out_gate.p != nullptr) != (a->y.p != nullptr))
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": the gates' gradient needs the outputs, and nothing else does");
    const mz_strided &f = a->fine;
    if (size_of(a->type) == 2 && f.p && ((uintptr_t)f.p | (uint64_t)f.stride_b | (uint64_t)f.stride_t | (uint64_t)f.stride_d) % 4 != 0)
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": fine and its strides must be multiples of 4 bytes");
    return MZ_OK;
}

template <bool BWD> static int run_recurrence(const mz_recurrence *a, void *stream, const char *fn)
{
    (void)hipGetLastError();
    if (int rc = check_recurrence(a, BWD, fn)) return rc;
    const RecurrencePlan p = plan_recurrence(a, BWD);
    if (p.links && (a->workspace_bytes < (int64_t)(8 * granule_count(a, p)) || !a->workspace || (uintptr_t)a->workspace % 64))
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": the workspace is smaller than mz_linear_recurrence_workspace says, or not aligned to 64 bytes");
    RecurrenceArgs q{};
    q.B = a->B, q.D = a->D, q.T = a->T, q.granules = (unsigned long long *)a->workspace, q.links = p.links;
    // the pass runs along the axis, or against it: reversed recurrence and gradient each turn it round
    const bool turned = (a->reverse != 0) != BWD;
    auto view = [&](const mz_strided &t) {
        RecurrenceArgs::View v{t.p, t.stride_b, t.stride_t, t.stride_d};
        if (t.p && turned) v.p = (const char *)t.p + (q.T - 1) * t.stride_t * (int64_t)size_of(a->type), v.st = -t.stride_t;
        return v;
    };
    q.a = view(a->gate), q.x = view(a->x), q.out = view(a->out);
    if (BWD) q.y = view(a->y), q.da = view(a->out_gate), q.state0 = a->y.p ? a->state : nullptr;
    if (size_of(a->type) == 2 && (!BWD || a->y.p)) q.fine = {a->fine.p, a->fine.stride_b, a->fine.stride_t, a->fine.stride_d};
    q.first = BWD ? a->grad_last : a->state, q.last = BWD ? a->out_state : a->last;
    hipStream_t st = (hipStream_t)stream;
    switch (a->type) {
    case MZ_F32: launch_slices<float, BWD>(p, q, st); break;
    case MZ_BF16: launch_slices<__bf16, BWD>(p, q, st); break;
    case MZ_F16: launch_slices<_Float16, BWD>(p, q, st); break;
    default: launch_slices<double, BWD>(p, q, st);
    }
    return api_launch_status(fn);
}

extern "C" int mz_linear_recurrence(const mz_recurrence *args_h, void *stream)
{
    return run_recurrence<false>(args_h, stream, "mz_linear_recurrence");
}

extern "C" int mz_linear_recurrence_backward(const mz_recurrence *args_h, void *stream)
{
    return run_recurrence<true>(args_h, stream, "mz_linear_recurrence_backward");
}

extern "C" int mz_linear_recurrence_workspace(const mz_recurrence *args_h, int32_t backward, int64_t *out_bytes)
{
    if (int rc = check_recurrence(args_h, backward != 0, "mz_linear_recurrence_workspace")) return rc;
    if (!out_bytes) return api_fail(MZ_ERR_ARG, "mz_linear_recurrence_workspace: null argument");
    *out_bytes = (int64_t)(8 * granule_count(args_h, plan_recurrence(args_h, backward != 0)));
    return MZ_OK;
}

// ------------------------------------------------------------------------------------------------ distillation

template <typename T, int G, int E, int MODE> static void launch_group(const DistillArgs &q, float c, hipStream_t st)
{
    constexpr int rows = 256 / G;
    hipLaunchKernelGGL((k_distill_group<T, G, E, MODE>), dim3((unsigned)(((long long)q.R + rows - 1) / rows)), dim3(256), 0, st, q, c);
}

template <typename T, int THREADS, int NP, int MODE> static void launch_row(const DistillArgs &q, float c, hipStream_t st)
{
    // entries, and with lse a bit for every action of whole packs (up to 14 more than there are actions)
    const size_t lds = (size_t)q.K * (8 + 4 + 4) + (q.lse && MODE != 2 ? 4 * (((size_t)q.V + 16 + 31) / 32) : 0);
    hipLaunchKernelGGL((k_distill_row<T, THREADS, MODE == 1 ? NP : 0, MODE>), dim3((unsigned)q.R), dim3(THREADS), lds, st, q, c);
}

template <typename T, int MODE> static void launch_distill(const DistillArgs &q, float c, hipStream_t st)
{
    // Groups of lanes up to 64 actions (40000 x 64 float32, 20 entries, loss and gradient: 21 us, a block a row 82; at 200 actions
    // groups of a whole wave took 125, the block 57).  Then as few waves a row as keep its packs in registers: 12000 x 6000 bfloat16
    // in 79 us with 128 threads of 8 packs, 89 with 64 of 16; 4096 x 32000 in 118 with 256 of 16, 131 with 512 of 8, 165 with 1024 of
    // 4, 141 read twice; 20000 x 1000 float32 in 37 with 4 packs a thread, 45 with 8 (idle packs cost exponentials).  Wider rows are
    // read twice: 1023 x 131071 in 165, 183 where 1024 threads hold 17 packs each; their loss alone in 76 with 512 threads, 88 with 1024, their gradient
    // alone in 106 with 1024, 117 with 512.
    constexpr int W = 16 / (int)sizeof(T);   // actions of a pack
    const int packs = (q.V + W - 1) / W + 1;   // one more where a row begins inside a pack
    if (q.V <= 16 && q.K <= 16) launch_group<T, 4, 4, MODE>(q, c, st);
    else if (q.V <= 64 && q.K <= 64) launch_group<T, 16, 4, MODE>(q, c, st);
    else if (packs <= 64 * 2) launch_row<T, 64, 2, MODE>(q, c, st);
    else if (packs <= 64 * 4) launch_row<T, 64, 4, MODE>(q, c, st);
    else if (packs <= 64 * 8) launch_row<T, 64, 8, MODE>(q, c, st);
    else if (packs <= 128 * 8) launch_row<T, 128, 8, MODE>(q, c, st);
    else if (packs <= 256 * 8) launch_row<T, 256, 8, MODE>(q, c, st);
    else if (packs <= 512 * 8) launch_row<T, 256, 16, MODE>(q, c, st);
    else if (packs <= 8192) launch_row<T, 512, 0, MODE>(q, c, st);
    else launch_row<T, MODE == 0 ? 512 : 1024, 0, MODE>(q, c, st);
}

template <typename T, int MODE> static void launch_distill_slices(const DistillArgs &q, float c, hipStream_t st)
{
    for (long long r = 0; r < q.R; r += SLICE) {
        DistillArgs s = q;
        const long long k = r * q.K;
        s.R = (int)std::min(SLICE, q.R - r);
        s.logits = ahead(q.logits, r * q.ld * (long long)sizeof(T)), s.grad = ahead(q.grad, r * q.V * (long long)sizeof(T));
        s.index = ahead(q.index, k * (q.index64 ? 8 : 4)), s.teacher = ahead(q.teacher, k * (long long)size_of(q.teacher_type));
        s.lse = (const float *)ahead(q.lse, r * 4), s.weight = (const float *)ahead(q.weight, r * 4), s.up = (const float *)ahead(q.up, r * 4);
        s.loss = (float *)ahead(q.loss, r * 4), s.stats = (float *)ahead(q.stats, r * 16);
        launch_distill<T, MODE>(s, c, st);
    }
}

template <int MODE> static int run_distill(const mz_distill *a, void *stream, const char *fn)
{
    (void)hipGetLastError();
    if (!a) return api_fail(MZ_ERR_ARG, std::string(fn) + ": null argument");
    if (a->type < MZ_F32 || a->type >= MZ_F64 || a->teacher_type < MZ_F32 || a->teacher_type >= MZ_F64)
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": logits are float32, bfloat16 or float16");
    if (a->R < 1 || a->V < 1 || a->V > (1 << 30) || a->K < 1 || a->K > MZ_DISTILL_MAX_ENTRIES || (a->lse && a->V > MZ_DISTILL_MAX_TAIL_ACTIONS))
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": sizes outside the limits (entries 1.." + std::to_string(MZ_DISTILL_MAX_ENTRIES) +
                                        ", actions up to " + std::to_string(MZ_DISTILL_MAX_TAIL_ACTIONS) + " with lse)");
    if (!(a->temperature >= 1e-30f && a->temperature <= 1e30f)) return api_fail(MZ_ERR_ARG, std::string(fn) + ": temperature must lie in 1e-30 .. 1e30");
    if (!a->logits || !a->index || !a->teacher || (MODE != 2 && !a->loss) || (MODE != 0 && !a->grad) || (MODE != 1 && !a->stats))
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": null tensor");
    if ((uintptr_t)a->stats % 16) return api_fail(MZ_ERR_ARG, std::string(fn) + ": stats must be aligned to 16 bytes");
    DistillArgs q{};
    q.logits = a->logits, q.ld = a->logits_stride, q.index = a->index, q.teacher = a->teacher, q.lse = a->lse, q.weight = a->weight;
    q.up = MODE == 2 ? a->grad_loss : nullptr, q.loss = a->loss, q.grad = MODE ? a->grad : nullptr, q.stats = a->stats;
    q.R = a->R, q.V = a->V, q.K = a->K, q.index64 = a->index64, q.teacher_type = a->teacher_type, q.tau = a->temperature, q.inv_tau = 1.0 / (double)a->temperature;
    const float c = (float)(1.4426950408889634074 / (double)a->temperature);   // log2(e) / temperature
    hipStream_t st = (hipStream_t)stream;
    switch (a->type) {
    case MZ_F32: launch_distill_slices<float, MODE>(q, c, st); break;
    case MZ_BF16: launch_distill_slices<__bf16, MODE>(q, c, st); break;
    default: launch_distill_slices<_Float16, MODE>(q, c, st);
    }
    return api_launch_status(fn);
}

extern "C" int mz_distill_loss(const mz_distill *args_h, void *stream) { return run_distill<0>(args_h, stream, "mz_distill_loss"); }
extern "C" int mz_distill_loss_grad(const mz_distill *args_h, void *stream) { return run_distill<1>(args_h, stream, "mz_distill_loss_grad"); }
extern "C" int mz_distill_grad(const mz_distill *args_h, void *stream) { return run_distill<2>(args_h, stream, "mz_distill_grad"); }

// ------------------------------------------------------------------------------------------------ verification

template <typename T, int G> static void launch_verify_group(const VerifyArgs &q, hipStream_t st)
{
    constexpr int n = 256 / G;
    hipLaunchKernelGGL((k_verify_group<T, G>), dim3((unsigned)((q.B + (n - 1ll)) / n)), dim3(256), 0, st, q);
}

template <typename T> static void launch_verify(const VerifyArgs &q, hipStream_t st)
{
    // a wave's registers hold up to 256 actions: 4096 sequences in 6.3 us, 14.0 with a block each
    if (q.V <= 16) return launch_verify_group<T, 4>(q, st);
    if (q.V <= 64) return launch_verify_group<T, 16>(q, st);
    if (q.V <= 256) return launch_verify_group<T, 64>(q, st);
    const int stretches = (q.V + STRETCH<T> - 1) / STRETCH<T>;
    hipLaunchKernelGGL((k_verify<T>), dim3((unsigned)q.B), dim3(64 * std::min(stretches, 16)), 8 * (size_t)stretches, st, q);
}

template <typename T> static void launch_verify_slices(const VerifyArgs &q, hipStream_t st)
{
    const long long token = q.token64 ? 8 : 4, size = (long long)sizeof(T);
    for (long long b = 0; b < q.B; b += SLICE) {
        VerifyArgs s = q;
        s.B = (int)std::min(SLICE, q.B - b);
        s.tokens = ahead(q.tokens, b * q.K * token), s.draft = ahead(q.draft, b * q.draft_b * size), s.target = ahead(q.target, b * q.target_b * size);
        s.u_accept = (const double *)ahead(q.u_accept, b * q.K * 8), s.u_sample = q.u_sample + b, s.lengths = (const int *)ahead(q.lengths, b * 4);
        s.accepted = q.accepted + b, s.out = ahead(q.out, b * (q.K + 1ll) * token);
        launch_verify<T>(s, st);
    }
}

extern "C" int mz_verify_drafts(const mz_verify *a, void *stream)
{
    const char *fn = "mz_verify_drafts";
    (void)hipGetLastError();
    if (!a) return api_fail(MZ_ERR_ARG, std::string(fn) + ": null argument");
    if (a->type < MZ_F32 || a->type > MZ_F64) return api_fail(MZ_ERR_ARG, std::string(fn) + ": unknown element type");
    if (a->B < 1 || a->K < 0 || a->K >= INT32_MAX || a->V < 1 || a->V > MZ_VERIFY_MAX_ACTIONS)
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": sizes must be positive, and at most " + std::to_string(MZ_VERIFY_MAX_ACTIONS) + " actions");
    if (!a->target || !a->u_sample || !a->accepted || !a->out || (a->K && (!a->tokens || !a->u_accept)))
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": null tensor");
    VerifyArgs q{};
    q.tokens = a->tokens, q.draft = a->draft, q.target = a->target;
    q.draft_b = a->draft_stride_b, q.draft_k = a->draft_stride_k, q.target_b = a->target_stride_b, q.target_k = a->target_stride_k;
    q.u_accept = a->u_accept, q.u_sample = a->u_sample, q.lengths = a->lengths, q.accepted = a->accepted, q.out = a->out;
    q.B = a->B, q.K = a->K, q.V = a->V, q.token64 = a->token64;
    hipStream_t st = (hipStream_t)stream;
    switch (a->type) {
    case MZ_F32: launch_verify_slices<float>(q, st); break;
    case MZ_BF16: launch_verify_slices<__bf16>(q, st); break;
    case MZ_F16: launch_verify_slices<_Float16>(q, st); break;
    default: launch_verify_slices<double>(q, st);
    }
    return api_launch_status(fn);
}
