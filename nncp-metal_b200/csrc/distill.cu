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

template <typename TZ, typename TG, int WHAT, int THR, int VEC, int PER> static int distill_launch(const distill::Args &a, cudaStream_t st)
{
    CUDA_TRY(launch_k(distill::kernel<TZ, TG, WHAT, THR, VEC, PER>, dim3(a.N), dim3(THR), sizeof(float) * 2 * (size_t)a.K, st, a));
    KERNEL_CHECK();
    return NNCU_OK;
}

// Short rows take a CTA of four warps, long ones of sixteen; a thread holds 32 logits at most.
template <typename TZ, typename TG, int WHAT, int VEC> static int distill_sized(const distill::Args &a, cudaStream_t st)
{
    const int groups = ceil_div(a.V, VEC), most = 32 / VEC;
    if (groups <= 128 * most) {
        const int per = ceil_div(groups, 128);
        if (per <= most / 4)
            return distill_launch<TZ, TG, WHAT, 128, VEC, most / 4>(a, st);
        return per <= most / 2 ? distill_launch<TZ, TG, WHAT, 128, VEC, most / 2>(a, st) : distill_launch<TZ, TG, WHAT, 128, VEC, most>(a, st);
    }
    if (groups <= 512 * most) {
        const int per = ceil_div(groups, 512);
        if (per <= most / 2)
            return distill_launch<TZ, TG, WHAT, 512, VEC, most / 2>(a, st);
        return distill_launch<TZ, TG, WHAT, 512, VEC, most>(a, st);
    }
    return distill_launch<TZ, TG, WHAT, 512, VEC, 0>(a, st);
}

template <typename TZ, typename TG, int WHAT> static int distill_run(const distill::Args &a, cudaStream_t st)
{
    const bool wide = a.ldz % 4 == 0 && aligned(a.z, 4 * sizeof(TZ)) && (!(WHAT & distill::GRAD) || (a.lddz % 4 == 0 && aligned(a.dz, 4 * sizeof(TG))));
    return wide ? distill_sized<TZ, TG, WHAT, 4>(a, st) : distill_sized<TZ, TG, WHAT, 1>(a, st);
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
    a.share = s->teacher_share; a.tau = s->temperature; a.inv_tau = 1.0f / s->temperature;
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
