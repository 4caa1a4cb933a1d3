// linear_attention.cu -- attention with a decaying state behind the C ABI: checks of arguments, the choice of a
// kernel and of its launch shape.
#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "linear_attention.cuh"
#include "op_checks.h"

static int lin_check(const nncu_linear_attn_shape *s)
{
    if (!s || s->n_streams < 1 || s->n_head < 1 || s->d_key < 1 || s->d_value < 1 || s->seg_len < 1 || !isfinite(s->scale))
        return nncu_fail(NNCU_ERR_INVALID, "linear attention: bad shape");
    if (s->d_key > NNCU_LINEAR_ATTN_DIM_MAX || s->d_value > NNCU_LINEAR_ATTN_DIM_MAX || s->n_head > NNCU_LINEAR_ATTN_HEADS_MAX)
        return nncu_fail(NNCU_ERR_RANGE, "linear attention: more than %d heads or head sizes over %d", NNCU_LINEAR_ATTN_HEADS_MAX, NNCU_LINEAR_ATTN_DIM_MAX);
    if ((long long)s->n_streams * s->n_head > INT_MAX || s->seg_len > 1 << 30)
        return nncu_fail(NNCU_ERR_RANGE, "linear attention: too many streams or tokens");
    const int wk = s->n_head * s->d_key, wv = s->n_head * s->d_value;
    if ((s->ld_q && s->ld_q < wk) || (s->ld_k && s->ld_k < wk) || (s->ld_v && s->ld_v < wv) || (s->ld_out && s->ld_out < wv))
        return nncu_fail(NNCU_ERR_INVALID, "linear attention: a row pitch is less than the row");
    return NNCU_OK;
}

// In how many parts a stream's tokens are cut.  One part is one pass over the tokens; more parts read b and c
// twice, and pay where one CTA for each (stream, head) would leave most SMs without work.
static void lin_parts(const nncu_linear_attn_shape *s, int *n_seg, int *seg)
{
    const long long pairs = (long long)s->n_streams * s->n_head;
    const int chunk = s->dtype_bf16 ? lin::TC : lin::FC, chunks = ceil_div(s->seg_len, chunk);
    int n = (int)std::min<long long>(std::max<long long>(SMS / pairs, 1), std::max(chunks / 4, 1));
    const int each = ceil_div(chunks, n);
    *seg = each * chunk;
    *n_seg = ceil_div(chunks, each);
}

static size_t lin_need(const nncu_linear_attn_shape *s)
{
    if (s->seg_len <= lin::STEP_TOKENS)
        return 0;
    int n_seg, seg;
    lin_parts(s, &n_seg, &seg);
    return n_seg > 1 ? sizeof(float) * (size_t)s->n_streams * s->n_head * n_seg * s->d_key * s->d_value : 0;
}

static int lin_common(const nncu_linear_attn_shape *s, const float *decay_host, const void *workspace, size_t workspace_bytes)
{
    if (!decay_host)
        return nncu_fail(NNCU_ERR_INVALID, "null tensor");
    for (int h = 0; h < s->n_head; h++)
        if (!(decay_host[h] > 0.0f && decay_host[h] <= 1.0f))
            return nncu_fail(NNCU_ERR_INVALID, "linear attention: the decay of head %d is not in (0, 1]", h);
    if (lin_need(s) > workspace_bytes || (lin_need(s) && (!workspace || !aligned(workspace, 16))))
        return nncu_fail(NNCU_ERR_INVALID, "linear attention: a workspace of %zu bytes that begins at a multiple of 16 is needed", lin_need(s));
    return NNCU_OK;
}

static lin::Args lin_args(const nncu_linear_attn_shape *s, const float *decay_host, const int32_t *len, void *workspace)
{
    lin::Args a;
    memset(&a, 0, sizeof(a));
    a.len = len;
    a.parts = (float *)workspace;
    a.B = s->n_streams; a.H = s->n_head; a.T = s->seg_len;
    lin_parts(s, &a.n_seg, &a.seg);
    for (int h = 0; h < s->n_head; h++)
        a.rate[h] = (float)log2((double)decay_host[h]);
    return a;
}

template <typename T, int VEC> static int lin_step(const lin::Args &a, cudaStream_t st)
{
    CUDA_TRY(launch_k(lin::step_kernel<T, VEC>, dim3(a.B * a.H, ceil_div(a.dc, 8 * VEC)), dim3(128), 0, st, a));
    KERNEL_CHECK();
    return NNCU_OK;
}

template <typename T, bool STATES> static int lin_core(const lin::Args &a, cudaStream_t st)
{
    static DeviceOnce once;
    NNCU_TRY(smem_limit(once, lin::core_kernel<T, STATES>, 4 * lin::CoreSmem(lin::DIM_MAX, lin::DIM_MAX).floats));
    CUDA_TRY(launch_k(lin::core_kernel<T, STATES>, dim3(a.B * a.H, STATES ? a.n_seg - 1 : a.n_seg), dim3(256),
                      4 * lin::CoreSmem(a.da, a.dc).floats, st, a));
    KERNEL_CHECK();
    return NNCU_OK;
}

template <int DA, int DC, bool STATES, int TERMS> static int lin_mma_launch(const lin::Args &a, cudaStream_t st)
{
    static DeviceOnce once;
    NNCU_TRY(smem_limit(once, lin::mma_kernel<DA, DC, STATES, TERMS>, lin::MmaSmem<DA, DC>::BYTES));
    CUDA_TRY(launch_k(lin::mma_kernel<DA, DC, STATES, TERMS>, dim3(a.B * a.H, STATES ? a.n_seg - 1 : a.n_seg), dim3(256),
                      lin::MmaSmem<DA, DC>::BYTES, st, a));
    KERNEL_CHECK();
    return NNCU_OK;
}

template <int DA, int DC> static int lin_mma_sized(const lin::Args &a, cudaStream_t st)
{
    if (a.s_end) {
        if (a.n_seg > 1)
            NNCU_TRY((lin_mma_launch<DA, DC, true, 3>(a, st)));
        return lin_mma_launch<DA, DC, false, 3>(a, st);
    }
    if (a.n_seg > 1)
        NNCU_TRY((lin_mma_launch<DA, DC, true, 2>(a, st)));
    return lin_mma_launch<DA, DC, false, 2>(a, st);
}

// head sizes go up to the next of 32, 64 and 128, zeros beyond their own
static int lin_mma(const lin::Args &a, cudaStream_t st)
{
    auto with = [&](auto da) {
        constexpr int DA = decltype(da)::value;
        return a.dc <= 32 ? lin_mma_sized<DA, 32>(a, st) : a.dc <= 64 ? lin_mma_sized<DA, 64>(a, st) : lin_mma_sized<DA, 128>(a, st);
    };
    return a.da <= 32 ? with(std::integral_constant<int, 32>()) : a.da <= 64 ? with(std::integral_constant<int, 64>())
                                                                            : with(std::integral_constant<int, 128>());
}

// rows laid out in 16-byte pieces
static bool lin_pieces(const lin::Args &a)
{
    return a.da % 8 == 0 && a.dc % 8 == 0 && a.lda % 8 == 0 && a.ldb % 8 == 0 && a.ldc % 8 == 0 && a.ldo % 2 == 0 && aligned(a.a, 16) &&
           aligned(a.b, 16) && aligned(a.c, 16) && aligned(a.o, 4);
}

// one pass of the form at the head of linear_attention.cuh
template <typename T> static int lin_run(const lin::Args &a, cudaStream_t st)
{
    if (a.T <= lin::STEP_TOKENS) {
        const bool wide = a.dc % 4 == 0 && aligned(a.s0, 16) && aligned(a.s_end, 16);
        return wide ? lin_step<T, 4>(a, st) : lin_step<T, 1>(a, st);
    }
    if (sizeof(T) == 2 && lin_pieces(a))
        return lin_mma(a, st);
    if (a.n_seg > 1)
        NNCU_TRY((lin_core<T, true>(a, st)));
    return lin_core<T, false>(a, st);
}

static int lin_any(const nncu_linear_attn_shape *s, const lin::Args &a, cudaStream_t st)
{
    return s->dtype_bf16 ? lin_run<bf16>(a, st) : lin_run<float>(a, st);
}

extern "C" {

int nncu_linear_attention_workspace(const nncu_linear_attn_shape *s, int backward, size_t *bytes_out)
{
    NNCU_TRY(lin_check(s));
    if (!bytes_out)
        return nncu_fail(NNCU_ERR_INVALID, "null argument");
    (void)backward;
    *bytes_out = lin_need(s);
    return NNCU_OK;
}

int nncu_linear_attention_forward(const nncu_linear_attn_shape *s, const void *q, const void *k, const void *v, const float *decay_host,
                                  const int32_t *len, const float *state_in, void *out, float *state_out, void *workspace,
                                  size_t workspace_bytes, void *cuda_stream)
{
    NNCU_TRY(lin_check(s));
    if (!q || !k || !v || !out)
        return nncu_fail(NNCU_ERR_INVALID, "null tensor");
    NNCU_TRY(lin_common(s, decay_host, workspace, workspace_bytes));
    if (out == q || out == k || out == v)
        return nncu_fail(NNCU_ERR_INVALID, "linear attention: the result cannot go over q, k or v");
    NNCU_TRY(elements_aligned({q, k, v, out}, s->dtype_bf16 ? 2 : 4));
    NNCU_TRY(elements_aligned({len, state_in, state_out}, 4));
    NNCU_TRY(on_device({q, k, v, len, state_in, out, state_out, lin_need(s) ? workspace : nullptr}));
    lin::Args a = lin_args(s, decay_host, len, workspace);
    const long long wk = (long long)s->n_head * s->d_key, wv = (long long)s->n_head * s->d_value;
    a.a = q; a.b = k; a.c = v; a.o = out;
    a.lda = s->ld_q ? s->ld_q : wk; a.ldb = s->ld_k ? s->ld_k : wk; a.ldc = s->ld_v ? s->ld_v : wv; a.ldo = s->ld_out ? s->ld_out : wv;
    a.da = s->d_key; a.dc = s->d_value;
    a.s0 = state_in; a.s_end = state_out;
    a.e1 = 1;
    a.s_state = a.s_pair = s->scale;
    a.s_in = 1.0f;
    ChainScope chain;
    return lin_any(s, a, (cudaStream_t)cuda_stream);
}

int nncu_linear_attention_backward(const nncu_linear_attn_shape *s, const void *q, const void *k, const void *v, const float *decay_host,
                                   const int32_t *len, const float *state_in, const void *dout, const float *dstate_out, void *dq,
                                   void *dk, void *dv, float *dstate_in, void *workspace, size_t workspace_bytes, void *cuda_stream)
{
    NNCU_TRY(lin_check(s));
    if (!q || !k || !v || !dout || !dq || !dk || !dv)
        return nncu_fail(NNCU_ERR_INVALID, "null tensor");
    NNCU_TRY(lin_common(s, decay_host, workspace, workspace_bytes));
    for (const void *to : {dq, dk, dv})
        if (to == q || to == k || to == v || to == dout || (to == dq) + (to == dk) + (to == dv) > 1)
            return nncu_fail(NNCU_ERR_INVALID, "linear attention: a gradient needs a place of its own");
    NNCU_TRY(elements_aligned({q, k, v, dout, dq, dk, dv}, s->dtype_bf16 ? 2 : 4));
    NNCU_TRY(elements_aligned({len, state_in, dstate_out, dstate_in}, 4));
    NNCU_TRY(on_device({q, k, v, len, state_in, dout, dstate_out, dq, dk, dv, dstate_in, lin_need(s) ? workspace : nullptr}));
    const long long wk = (long long)s->n_head * s->d_key, wv = (long long)s->n_head * s->d_value;
    const long long lq = s->ld_q ? s->ld_q : wk, lk = s->ld_k ? s->ld_k : wk, lv = s->ld_v ? s->ld_v : wv, lo = s->ld_out ? s->ld_out : wv;
    ChainScope chain;
    cudaStream_t st = (cudaStream_t)cuda_stream;
    const lin::Args base = lin_args(s, decay_host, len, workspace);
    lin::Args a = base;
    a.a = dout; a.lda = lo; a.b = v; a.ldb = lv; a.c = k; a.ldc = lk; a.o = dq; a.ldo = lq;
    a.da = s->d_value; a.dc = s->d_key;
    a.s0 = state_in; a.s0_t = 1;
    a.e1 = 1;
    a.s_state = a.s_pair = s->scale;
    a.s_in = 1.0f;
    NNCU_TRY(lin_any(s, a, st));
    a = base;
    a.reverse = 1;
    a.e2 = 1;
    a.s_state = 1.0f;
    a.s_pair = a.s_in = s->scale;
    a.s0 = dstate_out;
    lin::Args d = a;
    a.a = v; a.lda = lv; a.b = dout; a.ldb = lo; a.c = q; a.ldc = lq; a.o = dk; a.ldo = lk;
    a.da = s->d_value; a.dc = s->d_key; a.s0_t = 1;
    NNCU_TRY(lin_any(s, a, st));
    // last: dstate_in may lie where dstate_out lies
    d.a = k; d.lda = lk; d.b = q; d.ldb = lq; d.c = dout; d.ldc = lo; d.o = dv; d.ldo = lv;
    d.da = s->d_key; d.dc = s->d_value; d.s_end = dstate_in;
    return lin_any(s, d, st);
}

} // extern "C"
