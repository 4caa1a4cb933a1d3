// distill.cu -- the loss against a teacher's top logits behind the C ABI: checks of arguments, rows by size, launches.
#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "distill.cuh"
#include "op_checks.h"

static int distill_check(const nncu_distill_shape *s)
{
    if (!s || s->n_rows < 1 || s->n_symbols < 1 || s->n_top < 0 || !(s->temperature > 0.0f) || !isfinite(s->temperature) ||
        !(s->teacher_share >= 0.0f && s->teacher_share <= 1.0f) || (s->ld_logits && s->ld_logits < s->n_symbols) ||
        (s->ld_dlogits && s->ld_dlogits < s->n_symbols))
        return nncu_fail(NNCU_ERR_INVALID, "distillation: bad shape");
    // what the loss and the logits are multiplied by
    if (s->teacher_share != 0.0f && !(isfinite(s->temperature * s->temperature) && isfinite(2.0f / s->temperature)))
        return nncu_fail(NNCU_ERR_INVALID, "distillation: the temperature's square or inverse is no fp32 number");
    if (s->n_top > NNCU_DISTILL_TOP_MAX || s->n_symbols > INT_MAX / 2)
        return nncu_fail(NNCU_ERR_RANGE, "distillation: more than %d entries of the teacher, or too many symbols", NNCU_DISTILL_TOP_MAX);
    return NNCU_OK;
}

// An SM takes as many CTAs as rows fit its shared memory, each with a place or, where eight fit twice, more: one loads
// while others compute (rows of 16384 fp32 logits, 2048 of them, loss and gradient: three CTAs of one place 46 us, two 58, one
// of three places 83).  Some 1024 threads an SM share them.
template <typename TZ, typename TG, int WHAT, int HARD> static int distill_launch(distill::Args &a, cudaStream_t st)
{
    const int entries = 2 * 3 * 4 * a.K4, fixed = entries + 4 * distill::PLACES + 2560; // static arrays and what a CTA costs
    const long long row = (((long long)a.V * sizeof(TZ)) + 31) & ~15ll;
    if (row + fixed > SMEM_MOST) {
        a.slots = a.slot_bytes = 0;
        CUDA_TRY(launch_k(distill::kernel<TZ, TG, WHAT, HARD, false, false>, dim3(a.N), dim3(distill::THREADS_MAX), (size_t)entries, st, a));
        KERNEL_CHECK();
        return NNCU_OK;
    }
    a.slot_bytes = (int)row;
    const int ctas = std::min(a.V <= 2048 ? 16 : 8, SMEM_MOST / (a.slot_bytes + fixed));
    int threads = 64;
    while (threads < distill::THREADS_MAX && 2 * threads * ctas <= 1024)
        threads *= 2;
    a.slots = std::max(1, std::min(distill::SLOTS_MAX, (SMEM_MOST / ctas - fixed) / a.slot_bytes));
    const int grid = std::min(a.N, ctas * SMS);
    auto launch = [&](auto late) {
        constexpr bool LATE = decltype(late)::value;
        static DeviceOnce once;
        NNCU_TRY(smem_limit(once, distill::kernel<TZ, TG, WHAT, HARD, true, LATE>, SMEM_MOST - 4 * distill::PLACES - 1536));
        CUDA_TRY(launch_k(distill::kernel<TZ, TG, WHAT, HARD, true, LATE>, dim3(grid), dim3(threads), (size_t)a.slots * a.slot_bytes + entries, st, a));
        KERNEL_CHECK();
        return (int)NNCU_OK;
    };
    return (WHAT & distill::GRAD) && a.N > grid ? launch(std::bool_constant<(WHAT & distill::GRAD) != 0>()) : launch(std::false_type());
}

template <typename TZ, typename TG, int WHAT> static int distill_run(distill::Args &a, cudaStream_t st)
{
    if (a.tau == 1.0f || a.share == 1.0f) // p is p_tau, or not there
        return distill_launch<TZ, TG, WHAT, distill::SAME>(a, st);
    return a.tau == 2.0f ? distill_launch<TZ, TG, WHAT, distill::SQUARE>(a, st) : distill_launch<TZ, TG, WHAT, distill::APART>(a, st);
}

template <int WHAT>
static int distill_any(const nncu_distill_shape *s, const void *logits, const int32_t *top_ids, const float *top_logits, const int32_t *targets,
                       const float *row_weight, float *loss_rows, float *lse, void *dlogits, void *cuda_stream)
{
    NNCU_TRY(distill_check(s));
    if (!logits || (s->n_top && (!top_ids || !top_logits)) || ((WHAT & distill::LOSS) && !loss_rows) ||
        (WHAT != (distill::LOSS | distill::GRAD) && !lse) || ((WHAT & distill::GRAD) && !dlogits))
        return nncu_fail(NNCU_ERR_INVALID, "null tensor");
    if (logits == dlogits)
        return nncu_fail(NNCU_ERR_INVALID, "distillation: the gradient cannot go over the logits");
    NNCU_TRY(elements_aligned({logits}, s->logits_bf16 ? 2 : 4));
    NNCU_TRY(elements_aligned({dlogits}, s->grad_bf16 ? 2 : 4));
    NNCU_TRY(elements_aligned({top_ids, top_logits, targets, row_weight, loss_rows, lse}, 4));
    NNCU_TRY(on_device({logits, top_ids, top_logits, targets, row_weight, loss_rows, lse, dlogits}));
    distill::Args a;
    memset(&a, 0, sizeof(a));
    a.z = logits; a.ids = top_ids; a.top = top_logits; a.targets = targets; a.weight = row_weight;
    a.loss = loss_rows; a.lse = lse; a.dz = dlogits;
    a.ldz = s->ld_logits ? s->ld_logits : s->n_symbols;
    a.lddz = s->ld_dlogits ? s->ld_dlogits : s->n_symbols;
    a.N = s->n_rows; a.V = s->n_symbols; a.K = s->n_top;
    a.K4 = (s->n_top + 1 + 3) & ~3;
    a.share = s->teacher_share;
    a.tau = a.share == 0.0f ? 1.0f : s->temperature; // of a term that is not there
    a.inv_tau = 1.0f / a.tau;
    ChainScope chain;
    cudaStream_t st = (cudaStream_t)cuda_stream;
    if (!(WHAT & distill::GRAD))
        return s->logits_bf16 ? distill_run<bf16, float, WHAT>(a, st) : distill_run<float, float, WHAT>(a, st);
    if (s->logits_bf16)
        return s->grad_bf16 ? distill_run<bf16, bf16, WHAT>(a, st) : distill_run<bf16, float, WHAT>(a, st);
    return s->grad_bf16 ? distill_run<float, bf16, WHAT>(a, st) : distill_run<float, float, WHAT>(a, st);
}

extern "C" {

int nncu_distill_forward(const nncu_distill_shape *s, const void *logits, const int32_t *top_ids, const float *top_logits,
                         const int32_t *targets, const float *row_weight, float *loss_rows, float *lse, void *cuda_stream)
{
    return distill_any<distill::LOSS>(s, logits, top_ids, top_logits, targets, row_weight, loss_rows, lse, nullptr, cuda_stream);
}

int nncu_distill_backward(const nncu_distill_shape *s, const void *logits, const int32_t *top_ids, const float *top_logits,
                          const int32_t *targets, const float *row_weight, const float *lse, void *dlogits, void *cuda_stream)
{
    return distill_any<distill::GRAD>(s, logits, top_ids, top_logits, targets, row_weight, nullptr, const_cast<float *>(lse), dlogits, cuda_stream);
}

int nncu_distill_gradient(const nncu_distill_shape *s, const void *logits, const int32_t *top_ids, const float *top_logits,
                          const int32_t *targets, const float *row_weight, float *loss_rows, void *dlogits, void *cuda_stream)
{
    return distill_any<distill::LOSS | distill::GRAD>(s, logits, top_ids, top_logits, targets, row_weight, loss_rows, nullptr, dlogits, cuda_stream);
}

} // extern "C"
