// C entry points of the tensor operators around a policy: gated linear recurrence, distillation, verification of drafts.
// Argument checks and launches; the kernels live in the headers included below.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>

#include "../../include/muzero_amd.h"
#include "api.h"
#include "distill.h"
#include "recurrence.h"
#include "verify.h"

using namespace mz;

static size_t size_of(int type) { return type == MZ_F64 ? 8 : type == MZ_F32 ? 4 : 2; }

// ------------------------------------------------------------------------------------------------ recurrence

template <typename T, int VEC, bool BWD> static void launch_channels(const RecurrenceArgs &q, hipStream_t st)
{
    constexpr int CL = 32, THREADS = 512, L = 8;
    const long long tiles = (q.D + CL * VEC - 1) / (CL * VEC);
    hipLaunchKernelGGL((k_recurrence_channels<T, VEC, CL, THREADS, L, BWD>), dim3((unsigned)(tiles * q.B)), dim3(THREADS), 0, st, q);
}

template <typename T, bool BWD> static void launch_recurrence(const RecurrenceArgs &q, bool channels, bool pairs, hipStream_t st)
{
    if (channels) {
        if (sizeof(T) == 2 && pairs) launch_channels<T, 2, BWD>(q, st);
        else launch_channels<T, 1, BWD>(q, st);
        return;
    }
    constexpr int E = 4;
    const long long need = (q.T + E - 1) / E;
    const unsigned threads = need >= 1024 ? 1024 : (unsigned)((need + 63) / 64 * 64);
    hipLaunchKernelGGL((k_recurrence_rows<T, E, BWD>), dim3((unsigned)((long long)q.B * q.D)), dim3(threads), 0, st, q);
}

template <bool BWD> static int run_recurrence(const mz_recurrence *a, void *stream, const char *fn)
{
    (void)hipGetLastError();
    if (!a) return api_fail(MZ_ERR_ARG, std::string(fn) + ": null argument");
    if (a->type < MZ_F32 || a->type > MZ_F64) return api_fail(MZ_ERR_ARG, std::string(fn) + ": unknown element type");
    if (a->B < 1 || a->D < 1 || a->T < 1 || (int64_t)a->B * a->D > INT32_MAX)
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": sizes must be positive, and B * D below 2^31");
    if (!a->gate.p || !a->x.p || !a->out.p) return api_fail(MZ_ERR_ARG, std::string(fn) + ": null tensor");
    if (BWD && (a->out_gate.p != nullptr) != (a->y.p != nullptr))
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": the gates' gradient needs the outputs, and nothing else does");
    RecurrenceArgs q{};
    q.B = a->B, q.D = a->D, q.T = a->T;
    // the pass runs along the axis, or against it: reversed recurrence and gradient each turn it round
    const bool turned = (a->reverse != 0) != BWD;
    bool channels = true, pairs = q.D % 2 == 0;
    auto view = [&](const mz_strided &t) {
        RecurrenceArgs::View v{t.p, t.stride_b, t.stride_t, t.stride_d};
        if (!t.p) return v;
        if (q.D > 1 && t.stride_d != 1) channels = false;
        if (((uintptr_t)t.p | (uintptr_t)(t.stride_b * 2) | (uintptr_t)(t.stride_t * 2)) % 4) pairs = false;
        if (turned) v.p = (const char *)t.p + (q.T - 1) * t.stride_t * (int64_t)size_of(a->type), v.st = -t.stride_t;
        return v;
    };
    q.a = view(a->gate), q.x = view(a->x), q.out = view(a->out);
    if (BWD) q.y = view(a->y), q.da = view(a->out_gate), q.state0 = a->y.p ? a->state : nullptr;
    q.first = BWD ? a->grad_last : a->state, q.last = BWD ? a->out_state : a->last;
    if (q.D == 1) channels = false;
    hipStream_t st = (hipStream_t)stream;
    switch (a->type) {
    case MZ_F32: launch_recurrence<float, BWD>(q, channels, pairs, st); break;
    case MZ_BF16: launch_recurrence<__bf16, BWD>(q, channels, pairs, st); break;
    case MZ_F16: launch_recurrence<_Float16, BWD>(q, channels, pairs, st); break;
    default: launch_recurrence<double, BWD>(q, channels, pairs, st);
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

// ------------------------------------------------------------------------------------------------ distillation

template <typename T, int THREADS, int NP, bool KEEP, int MODE>
static void launch_distill(const DistillArgs &q, float c_hi, float c_lo, hipStream_t st)
{
    const size_t lds = (size_t)q.K * (8 + 8 + 4) + (q.lse && MODE != 2 ? 4 * (((size_t)q.V + 31) / 32) : 0);
    hipLaunchKernelGGL((k_distill_row<T, THREADS, NP, KEEP, MODE>), dim3((unsigned)q.R), dim3(THREADS), lds, st, q, c_hi, c_lo);
}

template <typename T, int MODE> static void launch_distill(const DistillArgs &q, float c_hi, float c_lo, hipStream_t st)
{
    if (q.V <= 2048) launch_distill<T, 64, 1, false, MODE>(q, c_hi, c_lo, st);
    else if (q.V <= 16384) launch_distill<T, 256, 1, false, MODE>(q, c_hi, c_lo, st);
    else launch_distill<T, 1024, 1, false, MODE>(q, c_hi, c_lo, st);
}

template <int MODE> static int run_distill(const mz_distill *a, void *stream, const char *fn)
{
    (void)hipGetLastError();
    if (!a) return api_fail(MZ_ERR_ARG, std::string(fn) + ": null argument");
    if (a->type < MZ_F32 || a->type >= MZ_F64 || a->teacher_type < MZ_F32 || a->teacher_type >= MZ_F64)
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": logits are float32, bfloat16 or float16");
    if (a->R < 1 || a->V < 1 || a->K < 1 || a->K > MZ_DISTILL_MAX_ENTRIES || (a->lse && a->V > MZ_DISTILL_MAX_TAIL_ACTIONS))
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": sizes outside the limits (entries 1.." + std::to_string(MZ_DISTILL_MAX_ENTRIES) +
                                        ", actions up to " + std::to_string(MZ_DISTILL_MAX_TAIL_ACTIONS) + " with lse)");
    if (!(a->temperature > 0) || !std::isfinite(a->temperature)) return api_fail(MZ_ERR_ARG, std::string(fn) + ": temperature must be positive and finite");
    if (!a->logits || !a->index || !a->teacher || (MODE != 2 && !a->loss) || (MODE != 0 && !a->grad) || (MODE != 1 && !a->stats))
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": null tensor");
    DistillArgs q{};
    q.logits = a->logits, q.ld = a->logits_stride, q.index = a->index, q.teacher = a->teacher, q.lse = a->lse, q.weight = a->weight;
    q.up = MODE == 2 ? a->grad_loss : nullptr, q.loss = a->loss, q.grad = MODE ? a->grad : nullptr, q.stats = a->stats;
    q.R = a->R, q.V = a->V, q.K = a->K, q.index64 = a->index64, q.teacher_type = a->teacher_type, q.tau = a->temperature;
    // log2(e) / tau = c_hi + c_lo, c_hi rounded towards zero and c_lo kept above zero
    const double c = 1.4426950408889634074 / (double)a->temperature;
    float c_hi = (float)c;
    if ((double)c_hi > c) c_hi = std::nextafter(c_hi, 0.0f);
    const float c_lo = std::fmax((float)(c - (double)c_hi), 1e-30f);
    hipStream_t st = (hipStream_t)stream;
    switch (a->type) {
    case MZ_F32: launch_distill<float, MODE>(q, c_hi, c_lo, st); break;
    case MZ_BF16: launch_distill<__bf16, MODE>(q, c_hi, c_lo, st); break;
    default: launch_distill<_Float16, MODE>(q, c_hi, c_lo, st);
    }
    return api_launch_status(fn);
}

extern "C" int mz_distill_loss(const mz_distill *args_h, void *stream) { return run_distill<0>(args_h, stream, "mz_distill_loss"); }
extern "C" int mz_distill_loss_grad(const mz_distill *args_h, void *stream) { return run_distill<1>(args_h, stream, "mz_distill_loss_grad"); }
extern "C" int mz_distill_grad(const mz_distill *args_h, void *stream) { return run_distill<2>(args_h, stream, "mz_distill_grad"); }

// ------------------------------------------------------------------------------------------------ verification

template <typename T> static void launch_verify(const VerifyArgs &q, hipStream_t st)
{
    const unsigned threads = q.V <= 64 ? 64 : q.V <= 1024 ? 128 : q.V <= 8192 ? 256 : 1024;   // more than one wave above 64 actions
    hipLaunchKernelGGL((k_verify<T>), dim3((unsigned)q.B), dim3(threads), 0, st, q);
}

extern "C" int mz_verify_drafts(const mz_verify *a, void *stream)
{
    const char *fn = "mz_verify_drafts";
    (void)hipGetLastError();
    if (!a) return api_fail(MZ_ERR_ARG, std::string(fn) + ": null argument");
    if (a->type < MZ_F32 || a->type > MZ_F64) return api_fail(MZ_ERR_ARG, std::string(fn) + ": unknown element type");
    if (a->B < 1 || a->K < 0 || a->V < 1) return api_fail(MZ_ERR_ARG, std::string(fn) + ": sizes must be positive");
    if (!a->target || !a->u_sample || !a->accepted || !a->out || (a->K && (!a->tokens || !a->u_accept)))
        return api_fail(MZ_ERR_ARG, std::string(fn) + ": null tensor");
    VerifyArgs q{};
    q.tokens = a->tokens, q.draft = a->draft, q.target = a->target;
    q.draft_b = a->draft_stride_b, q.draft_k = a->draft_stride_k, q.target_b = a->target_stride_b, q.target_k = a->target_stride_k;
    q.u_accept = a->u_accept, q.u_sample = a->u_sample, q.lengths = a->lengths, q.accepted = a->accepted, q.out = a->out;
    q.B = a->B, q.K = a->K, q.V = a->V, q.token64 = a->token64;
    hipStream_t st = (hipStream_t)stream;
    switch (a->type) {
    case MZ_F32: launch_verify<float>(q, st); break;
    case MZ_BF16: launch_verify<__bf16>(q, st); break;
    case MZ_F16: launch_verify<_Float16>(q, st); break;
    default: launch_verify<double>(q, st);
    }
    return api_launch_status(fn);
}
