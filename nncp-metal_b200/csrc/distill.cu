// distill.cu -- the loss against a teacher's top logits behind the C ABI: checks of arguments, rows by size, launches.
#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>

#include "distill.cuh"
#include "op_checks.h"

static int distill_check(const nncu_distill_shape *s)
{
    if (!s || s->n_rows < 1 || s->n_symbols < 1 || s->n_top < 0 || !(s->temperature > 0.0f) || !isfinite(s->temperature) ||
        !(s->teacher_share >= 0.0f && s->teacher_share <= 1.0f) || (s->ld_logits && s->ld_logits < s->n_symbols) ||
        (s->ld_dlogits && s->ld_dlogits < s->n_symbols))
        return nncu_fail(NNCU_ERR_INVALID, "distillation: bad shape");
    if (s->n_top > NNCU_DISTILL_TOP_MAX || s->n_symbols > INT_MAX / 2)
        return nncu_fail(NNCU_ERR_RANGE, "distillation: more than %d entries of the teacher, or too many symbols", NNCU_DISTILL_TOP_MAX);
    return NNCU_OK;
}

template <typename TZ, typename TG, int WHAT, int THR, int PER, bool TWO> static int distill_launch(const distill::Args &a, cudaStream_t st)
{
    CUDA_TRY(launch_k(distill::kernel<TZ, TG, WHAT, THR, PER, TWO>, dim3(a.N), dim3(THR), sizeof(float) * 3 * (size_t)a.K4, st, a));
    KERNEL_CHECK();
    return NNCU_OK;
}

// Rows of up to 1024 logits take a CTA of four warps, up to 4096 one of eight, longer ones sixteen; a thread holds 32
// logits at most.  The gradient from sums that stand needs a logit only once.
template <typename TZ, typename TG, int WHAT, bool TWO> static int distill_sized(const distill::Args &a, cudaStream_t st)
{
    const bool begins = a.ldz % 4 == 0 && aligned(a.z, 4 * sizeof(TZ)); // every row with a group
    const int groups = begins ? ceil_div(a.V, 4) : (a.V + 6) / 4;
    if constexpr (WHAT == distill::GRAD) {
        return groups <= 512 ? distill_launch<TZ, TG, WHAT, 128, 0, TWO>(a, st) : distill_launch<TZ, TG, WHAT, 256, 0, TWO>(a, st);
    } else {
        if (groups <= 128)
            return distill_launch<TZ, TG, WHAT, 128, 1, TWO>(a, st);
        if (groups <= 256)
            return distill_launch<TZ, TG, WHAT, 128, 2, TWO>(a, st);
        if (groups <= 512)
            return distill_launch<TZ, TG, WHAT, 256, 2, TWO>(a, st);
        if (groups <= 1024)
            return distill_launch<TZ, TG, WHAT, 256, 4, TWO>(a, st);
        switch (ceil_div(groups, 512)) {
        case 3: return distill_launch<TZ, TG, WHAT, 512, 3, TWO>(a, st);
        case 4: return distill_launch<TZ, TG, WHAT, 512, 4, TWO>(a, st);
        case 5: return distill_launch<TZ, TG, WHAT, 512, 5, TWO>(a, st);
        case 6: return distill_launch<TZ, TG, WHAT, 512, 6, TWO>(a, st);
        case 7: return distill_launch<TZ, TG, WHAT, 512, 7, TWO>(a, st);
        case 8: return distill_launch<TZ, TG, WHAT, 512, 8, TWO>(a, st);
        default: return distill_launch<TZ, TG, WHAT, 512, 0, TWO>(a, st);
        }
    }
}

template <typename TZ, typename TG, int WHAT> static int distill_run(const distill::Args &a, cudaStream_t st)
{
    if constexpr (WHAT != distill::GRAD)
        if (!a.power)
            return distill_sized<TZ, TG, WHAT, true>(a, st);
    return distill_sized<TZ, TG, WHAT, false>(a, st);
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
    a.K4 = (s->n_top + 3) & ~3;
    a.share = s->teacher_share;
    a.tau = a.share == 0.0f ? 1.0f : s->temperature; // of a term that is not there
    a.inv_tau = 1.0f / a.tau;
    a.power = a.share == 1.0f ? 1 : a.tau <= 4.0f && a.tau == floorf(a.tau) ? (int)a.tau : 0; // of p too
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
