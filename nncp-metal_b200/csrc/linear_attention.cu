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
// twice, and pay where one CTA for each (stream, head) would leave most SMs without work.  Parts of one chunk while there are
// 16 at most, of two behind that, since each goes through the sums of all before it (1 x 2 pairs of 1000 tokens of 128, bf16,
// in 4, 8 and 16 parts: 42, 27 and 24 us; one pair of 4096 of 64 in 16, 32 and 64: 21.5, 20.4 and 26.2).
static void lin_parts(const nncu_linear_attn_shape *s, int roles, int *n_seg, int *seg)
{
    const long long ctas = (long long)s->n_streams * s->n_head * roles;
    const int chunk = s->dtype_bf16 ? lin::TC : lin::FC, chunks = ceil_div(s->seg_len, chunk);
    // fp32: an SM takes three CTAs of head size 64 and one of 128
    const int most = std::max(s->d_key, s->d_value), want = s->dtype_bf16 ? SMS : SMS * (most <= 64 ? 3 : 1);
    const int n = (int)std::min<long long>(std::max<long long>(want / ctas, 1), std::max(std::min(chunks, 16), chunks / 2));
    int each = ceil_div(chunks, n);
    // a chunk of the first pass takes 0.6 of one of the second, both passes together a chunk more (two chunks of 64 tokens, 8
    // pairs of 64: 7.6 us in one part, 8.2 in two; three 9.8, in three parts 8.6)
    if (8ll * each + 5 > 5ll * chunks)
        each = chunks;
    *seg = each * chunk;
    *n_seg = ceil_div(chunks, each);
}

// floats of a state in a workspace: the tensor-core kernel's, head sizes up to the next of 32, 64 and 128 and four
// groups of 16 rows
static int lin_slot(const nncu_linear_attn_shape *s)
{
    auto up = [](int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; };
    const int k = up(s->d_key), v = up(s->d_value);
    return std::max(std::max(k, 64) * v, std::max(v, 64) * k); // [d_key][d_value] and the other way round
}

static size_t lin_need(const nncu_linear_attn_shape *s, int roles)
{
    if (s->seg_len <= lin::STEP_TOKENS)
        return 0;
    int n_seg, seg;
    lin_parts(s, roles, &n_seg, &seg);
    return n_seg > 1 ? sizeof(float) * (size_t)roles * s->n_streams * s->n_head * (n_seg + 1) * lin_slot(s) : 0;
}

static int lin_common(const nncu_linear_attn_shape *s, int roles, const float *decay_host, const void *workspace, size_t workspace_bytes)
{
    if (!decay_host)
        return nncu_fail(NNCU_ERR_INVALID, "null tensor");
    for (int h = 0; h < s->n_head; h++)
        if (!(decay_host[h] > 0.0f && decay_host[h] <= 1.0f))
            return nncu_fail(NNCU_ERR_INVALID, "linear attention: the decay of head %d is not in (0, 1]", h);
    const size_t need = lin_need(s, roles);
    if (need > workspace_bytes || (need && (!workspace || !aligned(workspace, 16))))
        return nncu_fail(NNCU_ERR_INVALID, "linear attention: a workspace of %zu bytes that begins at a multiple of 16 is needed", need);
    return NNCU_OK;
}

static lin::Args lin_args(const nncu_linear_attn_shape *s, int roles, const float *decay_host, const int32_t *len, void *workspace)
{
    lin::Args a;
    memset(&a, 0, sizeof(a));
    a.len = len;
    a.B = s->n_streams; a.H = s->n_head; a.T = s->seg_len;
    lin_parts(s, roles, &a.n_seg, &a.seg);
    a.slot = lin_slot(s);
    for (int i = 0; i < roles; i++)
        a.role[i].parts = (float *)workspace + (size_t)i * a.B * a.H * (a.n_seg + 1) * a.slot;
    for (int h = 0; h < s->n_head; h++) {
        a.rate[h] = (float)log2((double)decay_host[h]);
        a.decay[h] = decay_host[h];
    }
    return a;
}

// A state goes out where it came in, or somewhere else altogether
static bool lin_apart(const nncu_linear_attn_shape *s, const float *from, const float *to)
{
    const size_t n = (size_t)s->n_streams * s->n_head * s->d_key * s->d_value;
    return !from || !to || from + n <= to || to + n <= from;
}

template <typename T, int VEC> static int lin_step(const lin::Args &a, int roles, int dc, cudaStream_t st)
{
    CUDA_TRY(launch_k(lin::step_kernel<T, VEC>, dim3(a.B * a.H, ceil_div(dc, 8 * VEC), roles), dim3(128), 0, st, a));
    KERNEL_CHECK();
    return NNCU_OK;
}

template <typename T, bool STATES> static int lin_core(const lin::Args &a, int roles, cudaStream_t st)
{
    static DeviceOnce once;
    NNCU_TRY(smem_limit(once, lin::core_kernel<T, STATES>, 4 * lin::CoreSmem(lin::DIM_MAX, lin::DIM_MAX).floats));
    int floats = 0;
    for (int i = 0; i < roles; i++)
        floats = std::max(floats, lin::CoreSmem(a.role[i].da, a.role[i].dc).floats);
    CUDA_TRY(launch_k(lin::core_kernel<T, STATES>, dim3(a.B * a.H, STATES ? a.n_seg - 1 : a.n_seg, roles), dim3(256), 4 * floats, st, a));
    KERNEL_CHECK();
    return NNCU_OK;
}

template <bool STATES> static int lin_quad(const lin::Args &a, int roles, cudaStream_t st)
{
    static DeviceOnce once;
    NNCU_TRY(smem_limit(once, lin::quad_kernel<STATES>, 4 * lin::QuadSmem(lin::DIM_MAX, lin::DIM_MAX).floats));
    int floats = 0;
    for (int i = 0; i < roles; i++)
        floats = std::max(floats, lin::QuadSmem(a.role[i].da, a.role[i].dc).floats);
    CUDA_TRY(launch_k(lin::quad_kernel<STATES>, dim3(a.B * a.H, STATES ? a.n_seg - 1 : a.n_seg, roles), dim3(32 * ceil_div(a.role[0].dc, 16)), 4 * floats, st, a));
    KERNEL_CHECK();
    return NNCU_OK;
}

template <int DA, int DC, bool STATES, bool TMA, bool TWO> static int lin_mma_launch(const lin::MmaArgs &m, int roles, cudaStream_t st)
{
    constexpr int bytes = lin::MmaSmem<DA, DC, TWO>::BYTES;
    static DeviceOnce once;
    NNCU_TRY(smem_limit(once, lin::mma_kernel<DA, DC, STATES, TMA, TWO>, bytes));
    CUDA_TRY(launch_k(lin::mma_kernel<DA, DC, STATES, TMA, TWO>, dim3(m.p.B * m.p.H, m.p.n_seg, roles), dim3(4 * DC), bytes, st, m));
    KERNEL_CHECK();
    return NNCU_OK;
}

// 64 tokens x `cols` values of one head of rows [T*B][ld]
static int lin_map(const lin::Args &a, const void *rows, long long ld, int d, int cols, CUtensorMap *out)
{
    tc::EncodeTiledFn fn = tc::encode_fn();
    if (!fn)
        return nncu_fail(NNCU_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)a.H, (cuuint64_t)a.B, (cuuint64_t)a.T};
    const cuuint64_t strides[3] = {(cuuint64_t)d * 2, (cuuint64_t)ld * 2, (cuuint64_t)ld * 2 * a.B};
    const cuuint32_t box[4] = {(cuuint32_t)std::min(cols, 64), 1, 1, lin::TC}, each[4] = {1, 1, 1, 1};
    const CUresult rc = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(rows), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           cols == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? NNCU_OK : nncu_fail(NNCU_ERR_CUDA, "cuTensorMapEncodeTiled failed: %d", (int)rc);
}

template <int DA, int DC, bool TWO> static int lin_mma_sized(const lin::Args &a, int roles, cudaStream_t st)
{
    lin::MmaArgs m;
    m.p = a;
    if (a.T <= lin::TC)
        return lin_mma_launch<DA, DC, false, false, TWO>(m, roles, st);
    for (int i = 0; i < roles; i++) {
        const lin::Role &q = a.role[i];
        NNCU_TRY(lin_map(a, q.a, q.lda, q.da, DA, &m.map[i][0]));
        NNCU_TRY(lin_map(a, q.b, q.ldb, q.da, DA, &m.map[i][1]));
        NNCU_TRY(lin_map(a, q.c, q.ldc, q.dc, DC, &m.map[i][2]));
        if (q.a2)
            NNCU_TRY(lin_map(a, q.a2, q.lda2, q.dc, DC, &m.map[i][3]));
    }
    if (a.n_seg > 1)
        NNCU_TRY((lin_mma_launch<DA, DC, true, true, false>(m, roles, st)));
    return lin_mma_launch<DA, DC, false, true, TWO>(m, roles, st);
}

// head sizes go up to the next of 32, 64 and 128, zeros beyond their own
static int lin_mma(const lin::Args &a, int roles, cudaStream_t st)
{
    const int dc = a.role[0].dc, da = a.role[0].da;
    if (a.role[0].a2)
        return lin_mma_sized<64, 64, true>(a, roles, st);
    auto with = [&](auto size) {
        constexpr int DA = decltype(size)::value;
        return dc <= 32 ? lin_mma_sized<DA, 32, false>(a, roles, st) : dc <= 64 ? lin_mma_sized<DA, 64, false>(a, roles, st) : lin_mma_sized<DA, 128, false>(a, roles, st);
    };
    return da <= 32 ? with(std::integral_constant<int, 32>()) : da <= 64 ? with(std::integral_constant<int, 64>())
                                                                         : with(std::integral_constant<int, 128>());
}

// rows laid out in 16-byte pieces, and pitches that a tensor map takes
static bool lin_pieces(const lin::Role &q, long long B)
{
    for (long long ld : {q.lda, q.ldb, q.ldc, q.ldo})
        if (ld % 8 != 0 || ld * B * 2 >= 1ll << 40)
            return false;
    return q.da % 8 == 0 && q.dc % 8 == 0 && aligned(q.a, 16) && aligned(q.b, 16) && aligned(q.c, 16) && aligned(q.o, 16) && aligned(q.s0, 8) &&
           aligned(q.s_end, 8) && (!q.a2 || (q.lda2 % 8 == 0 && q.ldo2 % 8 == 0 && q.lda2 * B * 2 < 1ll << 40 && aligned(q.a2, 16) && aligned(q.o2, 16)));
}

// the same for fp32 rows, which need no tensor map
static bool lin_quads(const lin::Role &q)
{
    return q.da % 4 == 0 && q.dc % 4 == 0 && q.lda % 4 == 0 && q.ldb % 4 == 0 && q.ldc % 4 == 0 && q.ldo % 4 == 0 && aligned(q.a, 16) &&
           aligned(q.b, 16) && aligned(q.c, 16) && aligned(q.o, 16);
}

// Roles of the same head sizes, side by side in one launch, in the form at the head of linear_attention.cuh
template <typename T> static int lin_run(const lin::Args &a, int roles, cudaStream_t st)
{
    bool pieces = sizeof(T) == 2, quads = sizeof(T) == 4, wide = true;
    for (int i = 0; i < roles; i++) {
        const lin::Role &q = a.role[i];
        pieces = pieces && lin_pieces(q, a.B);
        quads = quads && lin_quads(q);
        wide = wide && q.dc % 4 == 0 && aligned(q.s0, 16) && aligned(q.s_end, 16);
    }
    if (a.T <= lin::STEP_TOKENS)
        return wide ? lin_step<T, 4>(a, roles, a.role[0].dc, st) : lin_step<T, 1>(a, roles, a.role[0].dc, st);
    if (pieces)
        return lin_mma(a, roles, st);
    if constexpr (sizeof(T) == 4)
        if (quads) {
            if (a.n_seg > 1)
                NNCU_TRY(lin_quad<true>(a, roles, st));
            return lin_quad<false>(a, roles, st);
        }
    if (a.n_seg > 1)
        NNCU_TRY((lin_core<T, true>(a, roles, st)));
    return lin_core<T, false>(a, roles, st);
}

static int lin_any(const nncu_linear_attn_shape *s, const lin::Args &a, int roles, cudaStream_t st)
{
    return s->dtype_bf16 ? lin_run<bf16>(a, roles, st) : lin_run<float>(a, roles, st);
}

extern "C" {

int nncu_linear_attention_workspace(const nncu_linear_attn_shape *s, int backward, size_t *bytes_out)
{
    NNCU_TRY(lin_check(s));
    if (!bytes_out)
        return nncu_fail(NNCU_ERR_INVALID, "null argument");
    *bytes_out = std::max(lin_need(s, 1), backward ? lin_need(s, 3) : 0);
    return NNCU_OK;
}

int nncu_linear_attention_forward(const nncu_linear_attn_shape *s, const void *q, const void *k, const void *v, const float *decay_host,
                                  const int32_t *len, const float *state_in, void *out, float *state_out, void *workspace,
                                  size_t workspace_bytes, void *cuda_stream)
{
    NNCU_TRY(lin_check(s));
    if (!q || !k || !v || !out)
        return nncu_fail(NNCU_ERR_INVALID, "null tensor");
    NNCU_TRY(lin_common(s, 1, decay_host, workspace, workspace_bytes));
    if (out == q || out == k || out == v)
        return nncu_fail(NNCU_ERR_INVALID, "linear attention: the result cannot go over q, k or v");
    if (state_in != state_out && !lin_apart(s, state_in, state_out))
        return nncu_fail(NNCU_ERR_INVALID, "linear attention: the states overlap");
    NNCU_TRY(elements_aligned({q, k, v, out}, s->dtype_bf16 ? 2 : 4));
    NNCU_TRY(elements_aligned({len, state_in, state_out}, 4));
    NNCU_TRY(on_device({q, k, v, len, state_in, out, state_out, lin_need(s, 1) ? workspace : nullptr}));
    lin::Args args = lin_args(s, 1, decay_host, len, workspace);
    lin::Role &a = args.role[0];
    const long long wk = (long long)s->n_head * s->d_key, wv = (long long)s->n_head * s->d_value;
    a.a = q; a.b = k; a.c = v; a.o = out;
    a.lda = s->ld_q ? s->ld_q : wk; a.ldb = s->ld_k ? s->ld_k : wk; a.ldc = s->ld_v ? s->ld_v : wv; a.ldo = s->ld_out ? s->ld_out : wv;
    a.da = s->d_key; a.dc = s->d_value;
    a.s0 = state_in; a.s_end = state_out;
    a.e1 = 1;
    a.s_state = a.s_pair = s->scale;
    a.s_in = 1.0f;
    ChainScope chain;
    return lin_any(s, args, 1, (cudaStream_t)cuda_stream);
}

int nncu_linear_attention_backward(const nncu_linear_attn_shape *s, const void *q, const void *k, const void *v, const float *decay_host,
                                   const int32_t *len, const float *state_in, const void *dout, const float *dstate_out, void *dq,
                                   void *dk, void *dv, float *dstate_in, void *workspace, size_t workspace_bytes, void *cuda_stream)
{
    NNCU_TRY(lin_check(s));
    if (!q || !k || !v || !dout || !dq || !dk || !dv)
        return nncu_fail(NNCU_ERR_INVALID, "null tensor");
    NNCU_TRY(lin_common(s, 3, decay_host, workspace, workspace_bytes));
    for (const void *to : {dq, dk, dv})
        if (to == q || to == k || to == v || to == dout || (to == dq) + (to == dk) + (to == dv) > 1)
            return nncu_fail(NNCU_ERR_INVALID, "linear attention: a gradient needs a place of its own");
    if ((dstate_in != dstate_out && !lin_apart(s, dstate_out, dstate_in)) || !lin_apart(s, state_in, dstate_in))
        return nncu_fail(NNCU_ERR_INVALID, "linear attention: the states overlap");
    NNCU_TRY(elements_aligned({q, k, v, dout, dq, dk, dv}, s->dtype_bf16 ? 2 : 4));
    NNCU_TRY(elements_aligned({len, state_in, dstate_out, dstate_in}, 4));
    NNCU_TRY(on_device({q, k, v, len, state_in, dout, dstate_out, dq, dk, dv, dstate_in, lin_need(s, 3) ? workspace : nullptr}));
    const long long wk = (long long)s->n_head * s->d_key, wv = (long long)s->n_head * s->d_value;
    const long long lq = s->ld_q ? s->ld_q : wk, lk = s->ld_k ? s->ld_k : wk, lv = s->ld_v ? s->ld_v : wv, lo = s->ld_out ? s->ld_out : wv;
    ChainScope chain;
    cudaStream_t st = (cudaStream_t)cuda_stream;
    lin::Args all = lin_args(s, 3, decay_host, len, workspace);
    // the longest first: dv carries the third term
    lin::Role &rv = all.role[0], &rq = all.role[1], &rk = all.role[2];
    rq.a = dout; rq.lda = lo; rq.b = v; rq.ldb = lv; rq.c = k; rq.ldc = lk; rq.o = dq; rq.ldo = lq;
    rk.a = v; rk.lda = lv; rk.b = dout; rk.ldb = lo; rk.c = q; rk.ldc = lq; rk.o = dk; rk.ldo = lk;
    rv.a = k; rv.lda = lk; rv.b = q; rv.ldb = lq; rv.c = dout; rv.ldc = lo; rv.o = dv; rv.ldo = lv;
    rq.da = rk.da = s->d_value; rq.dc = rk.dc = s->d_key; rv.da = s->d_key; rv.dc = s->d_value;
    rq.s0 = state_in; rk.s0 = rv.s0 = dstate_out;
    rq.s0_t = rk.s0_t = 1;
    rv.s_end = dstate_in;
    rq.e1 = rk.e2 = rv.e2 = 1;
    rk.reverse = rv.reverse = 1;
    rq.s_state = rq.s_pair = rk.s_pair = rv.s_pair = rk.s_in = rv.s_in = s->scale;
    rq.s_in = rk.s_state = rv.s_state = 1.0f;
    // bf16 rows in 16-byte pieces, head sizes from 33 to 64: dk beside dv, from the same tiles and the same state, where three
    // CTAs for each (stream, head) are more than the two an SM that run in one round (128 pairs of 2048 tokens, backward 185 ->
    // 155 us, 256 of 512 89 -> 80; 32 pairs of 1024 40 -> 62), and where different head sizes would make two launches
    const int least = std::min(s->d_key, s->d_value), most = std::max(s->d_key, s->d_value);
    if (s->dtype_bf16 && s->seg_len > lin::STEP_TOKENS && least > 32 && most <= 64 &&
        (3ll * s->n_streams * s->n_head * all.n_seg > 2 * SMS || s->d_key != s->d_value)) {
        lin::Args two = all;
        lin::Role &both = two.role[0];
        both.a2 = v; both.lda2 = lv; both.o2 = dk; both.ldo2 = lk;
        if (lin_pieces(both, s->n_streams) && lin_pieces(rq, s->n_streams))
            return lin_any(s, two, 2, st);
    }
    // one launch for all three, or dv behind the others: where its head sizes are other than theirs, and where
    // dstate_in lies over the dstate_out that they read
    if (s->d_key == s->d_value && lin_apart(s, dstate_out, dstate_in))
        return lin_any(s, all, 3, st);
    lin::Args two = all;
    two.role[0] = rq;
    two.role[1] = rk;
    NNCU_TRY(lin_any(s, two, 2, st));
    return lin_any(s, all, 1, st);
}

} // extern "C"
