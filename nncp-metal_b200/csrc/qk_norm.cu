// qk_norm.cu -- head norms with the position rotation behind the C ABI: checks of arguments, widths, launches.
#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>

#include "qk_norm.cuh"
#include "op_checks.h"

static int qk_check(const nncu_qk_norm_shape *s)
{
    if (!s || s->n_rows < 1 || s->n_head < 1 || s->n_head_k < 0 || s->d_key < 2 || (s->d_key & 1) || s->d_rot < 0 ||
        (s->d_rot & 1) || s->d_rot > s->d_key || !(s->eps >= 0.0f) || !isfinite(s->eps) || (s->d_rot && !(s->rope_base > 0.0f && isfinite(s->rope_base))))
        return nncu_fail(NNCU_ERR_INVALID, "qk norm: bad shape");
    if (s->d_key > NNCU_QK_NORM_DIM_MAX || s->n_head > NNCU_QK_NORM_HEADS_MAX || s->n_head_k > NNCU_QK_NORM_HEADS_MAX || s->n_rows > 1 << 30)
        return nncu_fail(NNCU_ERR_RANGE, "qk norm: d_key over %d, more than %d heads or too many rows", NNCU_QK_NORM_DIM_MAX, NNCU_QK_NORM_HEADS_MAX);
    const long long wq = (long long)s->n_head * s->d_key, wk = (long long)s->n_head_k * s->d_key;
    if ((s->ld_q && s->ld_q < wq) || (s->ld_q_out && s->ld_q_out < wq) || (s->ld_k && s->ld_k < wk) || (s->ld_k_out && s->ld_k_out < wk))
        return nncu_fail(NNCU_ERR_INVALID, "qk norm: a row pitch is less than the row");
    return NNCU_OK;
}

// Rows that a CTA takes at a time: four rounds of heads for its eight warps (a lane holds eight pairs or so), or as many as
// leave two CTAs an SM.
static int qk_rows_per(const nncu_qk_norm_shape *s)
{
    const int per_warp = std::max(1, 32 * 16 / s->d_key), kinds = s->n_head_k ? 2 : 1;
    int n = 1;
    while (n < qkn::ROWS_MAX && n * s->n_head < 32 * per_warp && (n * s->n_head < 8 * per_warp || (long long)ceil_div(s->n_rows, 2 * n) * kinds >= 2 * SMS))
        n *= 2;
    return n;
}
static int qk_blocks(const nncu_qk_norm_shape *s, bool back)
{
    const int blocks = ceil_div(s->n_rows, qk_rows_per(s)), kinds = s->n_head_k ? 2 : 1;
    return std::min(blocks, (back ? 2 : 8) * SMS / kinds); // backward: each leaves a partial sum of dgain
}

static qkn::Args qk_args(const nncu_qk_norm_shape *s, const void *q, const void *k, const float *gain_q, const float *gain_k, const int32_t *pos)
{
    qkn::Args a;
    memset(&a, 0, sizeof(a));
    a.x[0] = q; a.x[1] = k;
    a.gain[0] = gain_q; a.gain[1] = gain_k;
    a.pos = pos;
    const long long wq = (long long)s->n_head * s->d_key, wk = (long long)s->n_head_k * s->d_key;
    a.ldx[0] = s->ld_q ? s->ld_q : (int)wq; a.ldx[1] = s->ld_k ? s->ld_k : (int)wk;
    a.ldy[0] = s->ld_q_out ? s->ld_q_out : (int)wq; a.ldy[1] = s->ld_k_out ? s->ld_k_out : (int)wk;
    a.heads[0] = s->n_head; a.heads[1] = s->n_head_k;
    a.N = s->n_rows; a.d = s->d_key; a.rot = s->d_rot; a.eps = s->eps;
    a.rows_per = qk_rows_per(s);
    for (int i = 0; i < 2; i++)
        a.inverse[i] = a.heads[i] > 1 ? (uint32_t)(((1ull << 32) + a.heads[i] - 1) / a.heads[i]) : 0;
    // pair by pair in 64 bits behind the point: one power for all of them
    const long double step = s->d_rot ? powl((long double)s->rope_base, -2.0L / s->d_rot) : 1.0L;
    long double turn = 1.0L / 6.283185307179586476925L;
    for (int i = 0; i < s->d_rot / 2; i++, turn *= step)
        a.turns[i] = (double)turn;
    return a;
}

template <typename T, int W, int NG, bool BACK> static int qk_launch(const nncu_qk_norm_shape *s, qkn::Args &a, cudaStream_t st)
{
    a.lanes = 1;
    while (a.lanes * W * NG < a.d / 2)
        a.lanes *= 2;
    const size_t smem = sizeof(float) * (size_t)(a.rows_per + (BACK ? 9 : 1)) * a.d;
    const dim3 grid(qk_blocks(s, BACK), s->n_head_k ? 2 : 1);
    if (s->adjacent)
        CUDA_TRY(launch_k(qkn::kernel<T, W, NG, true, BACK>, grid, dim3(256), smem, st, a));
    else
        CUDA_TRY(launch_k(qkn::kernel<T, W, NG, false, BACK>, grid, dim3(256), smem, st, a));
    KERNEL_CHECK();
    return NNCU_OK;
}

// Accesses of w values: the widest that pairs, pitches and addresses allow.  A head of 256 values fits the 32 lanes
// of a warp at every width.
template <typename T, bool BACK> static int qk_any(const nncu_qk_norm_shape *s, qkn::Args &a, cudaStream_t st)
{
    int w = 16 / (int)sizeof(T);
    auto fits = [&]() {
        bool ok = a.d / 2 % w == 0 && a.rot / 2 % w == 0;
        for (int i = 0; i < 2; i++)
            if (a.heads[i])
                ok = ok && a.ldx[i] % w == 0 && a.ldy[i] % w == 0 && aligned(a.x[i], w * sizeof(T)) && aligned(a.y[i], w * sizeof(T)) &&
                     aligned(a.dy[i], w * sizeof(T));
        return ok;
    };
    while (w > 1 && !fits())
        w /= 2;
    if constexpr (sizeof(T) == 2)
        if (w == 8)
            return qk_launch<T, 8, 1, BACK>(s, a, st);
    return w == 4 ? qk_launch<T, 4, 1, BACK>(s, a, st) : w == 2 ? qk_launch<T, 2, 2, BACK>(s, a, st) : qk_launch<T, 1, 4, BACK>(s, a, st);
}

// Results lie over an input only where every value is written by the thread that has read it: over the same rows
static int qk_places(const qkn::Args &a)
{
    for (int i = 0; i < 2; i++) {
        const void *y = a.y[i], *x = a.x[i], *dy = a.dy[i];
        if (!y)
            continue;
        const int ldy = a.dy[i] ? a.ldx[i] : a.ldy[i]; // pitch of y: of the results, or backward of x
        if ((y == x && ldy != a.ldx[i]) || (y == dy && ldy != a.ldy[i]) || y == a.y[1 - i] || y == a.x[1 - i] || y == a.dy[1 - i])
            return nncu_fail(NNCU_ERR_INVALID, "qk norm: results in place need the pitch of their inputs, and a place each");
    }
    return NNCU_OK;
}

extern "C" {

int nncu_qk_norm_rope_forward(const nncu_qk_norm_shape *s, const void *q, const void *k, const float *gain_q, const float *gain_k,
                              const int32_t *pos, void *q_out, void *k_out, void *cuda_stream)
{
    NNCU_TRY(qk_check(s));
    if (!q || !q_out || (s->n_head_k && (!k || !k_out)) || (s->d_rot && !pos))
        return nncu_fail(NNCU_ERR_INVALID, "null tensor");
    qkn::Args a = qk_args(s, q, s->n_head_k ? k : nullptr, gain_q, gain_k, pos);
    a.y[0] = q_out; a.y[1] = s->n_head_k ? k_out : nullptr;
    NNCU_TRY(qk_places(a));
    NNCU_TRY(elements_aligned({a.x[0], a.x[1], a.y[0], a.y[1]}, s->dtype_bf16 ? 2 : 4));
    NNCU_TRY(elements_aligned({gain_q, gain_k, pos}, 4));
    NNCU_TRY(on_device({a.x[0], a.x[1], gain_q, gain_k, pos, a.y[0], a.y[1]}));
    ChainScope chain;
    return s->dtype_bf16 ? qk_any<bf16, false>(s, a, (cudaStream_t)cuda_stream) : qk_any<float, false>(s, a, (cudaStream_t)cuda_stream);
}

int nncu_qk_norm_rope_workspace(const nncu_qk_norm_shape *s, size_t *bytes_out)
{
    NNCU_TRY(qk_check(s));
    if (!bytes_out)
        return nncu_fail(NNCU_ERR_INVALID, "null argument");
    *bytes_out = sizeof(float) * 2 * (size_t)s->d_key * qk_blocks(s, true);
    return NNCU_OK;
}

int nncu_qk_norm_rope_backward(const nncu_qk_norm_shape *s, const void *q, const void *k, const float *gain_q, const float *gain_k,
                               const int32_t *pos, const void *dq_out, const void *dk_out, void *dq, void *dk, float *dgain_q,
                               float *dgain_k, void *workspace, size_t workspace_bytes, void *cuda_stream)
{
    size_t need = 0;
    NNCU_TRY(nncu_qk_norm_rope_workspace(s, &need));
    if (!q || !dq_out || !dq || (s->n_head_k && (!k || !dk_out || !dk)) || (s->d_rot && !pos))
        return nncu_fail(NNCU_ERR_INVALID, "null tensor");
    if ((dgain_q && !gain_q) || (dgain_k && (!gain_k || !s->n_head_k)))
        return nncu_fail(NNCU_ERR_INVALID, "qk norm: the gradient of a gain that is not there");
    const bool gains = dgain_q || dgain_k;
    if (gains && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return nncu_fail(NNCU_ERR_INVALID, "qk norm: a workspace of %zu bytes that begins at a multiple of 16 is needed", need);
    qkn::Args a = qk_args(s, q, s->n_head_k ? k : nullptr, gain_q, gain_k, pos);
    a.dy[0] = dq_out; a.dy[1] = s->n_head_k ? dk_out : nullptr;
    a.y[0] = dq; a.y[1] = s->n_head_k ? dk : nullptr;
    a.part = gains ? (float *)workspace : nullptr;
    NNCU_TRY(qk_places(a));
    NNCU_TRY(elements_aligned({a.x[0], a.x[1], a.dy[0], a.dy[1], a.y[0], a.y[1]}, s->dtype_bf16 ? 2 : 4));
    NNCU_TRY(elements_aligned({gain_q, gain_k, pos, dgain_q, dgain_k}, 4));
    NNCU_TRY(on_device({a.x[0], a.x[1], a.dy[0], a.dy[1], gain_q, gain_k, pos, a.y[0], a.y[1], dgain_q, dgain_k, a.part}));
    ChainScope chain;
    cudaStream_t st = (cudaStream_t)cuda_stream;
    NNCU_TRY((s->dtype_bf16 ? qk_any<bf16, true>(s, a, st) : qk_any<float, true>(s, a, st)));
    if (gains) {
        CUDA_TRY(launch_k(qkn::gain_kernel, dim3(ceil_div(2 * s->d_key, 8)), dim3(256), 0, st, (const float *)a.part, qk_blocks(s, true), s->d_key,
                          dgain_q, dgain_k));
        KERNEL_CHECK();
    }
    return NNCU_OK;
}

} // extern "C"
