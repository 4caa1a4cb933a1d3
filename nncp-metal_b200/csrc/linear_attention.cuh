// linear_attention.cuh -- attention whose memory is a matrix that decays at each head's own rate.
//
//   S_t = l S_{t-1} + k_t^T v_t        o_t = scale q_t S_t        (l in (0, 1], one for each head)
//
// Over a run of n tokens that begins with state S, rows counted from 0,
//
//   o_i = scale (l^(i+1) q_i S + sum_{j<=i} l^(i-j) (q_i . k_j) v_j),   S' = l^n S + sum_j l^(n-1-j) k_j^T v_j,
//
// so a sequence is taken chunk by chunk: inside a chunk products of tiles, between chunks the state.  The
// adjoint has the same form three times over:
//
//   dq: rows (dout, v, k) with the states S^T, in the sequence's order
//   dv: rows (k, q, dout) with the states dS, from the last token to the first
//   dk: rows (v, dout, q) with the states dS^T, from the last token to the first
//
// Every kernel here therefore takes rows a, b, c and a state [da][dc] and gives
//
//   o_i = s_state l^(i+e1) a_i S + s_pair sum_{j<=i} l^(i-j) (a_i . b_j) c_j,
//   S'  = l^n S + s_in sum_j l^(n-1-j+e2) b_j^T c_j
//
// with e1 = 1, e2 = 0 in the sequence's order and e1 = 0, e2 = 1 in the reverse one.
#pragma once
#include "warp_mma.cuh"

namespace lin {

constexpr int HEADS_MAX = NNCU_LINEAR_ATTN_HEADS_MAX;
constexpr int DIM_MAX = NNCU_LINEAR_ATTN_DIM_MAX;

struct Args {
    const void *a, *b, *c;
    void *o;             // NULL: states only
    const float *s0;     // state before the first token, [B][H][da][dc] or, where s0_t, [B][H][dc][da]; NULL: zeros
    float *s_end;        // state behind the last token, [B][H][da][dc]; NULL: not wanted
    float *parts;        // [B*H][n_seg][da*dc]: slot 0 the state before the first token, slot g what part g - 1 adds up to
    const int32_t *len;  // tokens of each stream; NULL: T
    long long lda, ldb, ldc, ldo; // elements from row to row
    int B, H, T, da, dc;
    int reverse, s0_t, e1, e2;
    float s_state, s_pair, s_in;
    int n_seg;           // parts a stream's tokens are cut into
    int seg;             // tokens in a part
    float rate[HEADS_MAX]; // log2 of each head's decay
};

// l^n; l^0 is 1 whatever l
__device__ __forceinline__ float power(float rate, int n) { return exp2f(rate * (float)n); }

// Where a stream's token u (counted in the kernel's order) lies, and how many there are
struct Rows {
    long long first, step; // rows
    int n;
    __device__ __forceinline__ Rows(const Args &p, int b)
    {
        n = p.len ? min(max(p.len[b], 0), p.T) : p.T;
        step = p.reverse ? -(long long)p.B : p.B;
        first = (p.reverse ? (long long)(n - 1) * p.B : 0) + b;
    }
    __device__ __forceinline__ long long row(int u) const { return first + step * u; }
};

// rows of the result behind a stream's end are zeros: those of them that part g is to write
template <typename T>
__device__ __forceinline__ void zero_behind(const Args &p, const Rows &rows, int b, int h, int g, int tid, int nthr)
{
    const int lo = max(rows.n, g * p.seg), hi = g == p.n_seg - 1 ? p.T : min(p.T, (g + 1) * p.seg);
    T *o = reinterpret_cast<T *>(p.o) + (size_t)h * p.dc;
    for (long long i = tid; i < (long long)(hi - lo) * p.dc; i += nthr)
        o[((long long)(lo + i / p.dc) * p.B + b) * p.ldo + i % p.dc] = from_f<T>(0.0f);
}

__device__ __forceinline__ float state_at(const Args &p, const float *s, int i, int c)
{
    return p.s0_t ? s[(size_t)c * p.da + i] : s[(size_t)i * p.dc + c];
}

// Element (i, c) of the state that part g begins with, from the sums of the parts before it
__device__ __forceinline__ float start_at(const Args &p, size_t pair, int g, int i, int c, float l_seg)
{
    const size_t nn = (size_t)p.da * p.dc;
    if (p.n_seg == 1)
        return p.s0 ? state_at(p, p.s0 + pair * nn, i, c) : 0.0f;
    const float *at = p.parts + pair * p.n_seg * nn + (size_t)i * p.dc + c;
    float s = at[0];
    for (int k = 1; k <= g; k++)
        s = fmaf(l_seg, s, at[k * nn]);
    return s;
}

// ---------------- CUDA cores: fp32, and bf16 whose rows are not laid out in 16-byte pieces ----------------
//
// A CTA of 256 threads goes through one part of one (stream, head) in chunks of 32 tokens; the tiles and the
// state are fp32 in shared memory, a thread takes 4 x 4 results at a time.  Bound by shared-memory reads: five loads
// for sixteen multiply-adds.

constexpr int FC = 32; // tokens in a chunk

struct CoreSmem {
    int da4, dc4, ld_a, ld_c, b, c, s, p, w, floats;
    __host__ __device__ CoreSmem(int da, int dc)
    {
        da4 = (da + 3) & ~3; dc4 = (dc + 3) & ~3;
        ld_a = da4 + 4; ld_c = dc4 + 4; // rows four banks on
        b = FC * ld_a; c = b + FC * ld_a; s = c + FC * ld_c; p = s + da4 * ld_c; w = p + FC * (FC + 1);
        floats = w + 2 * (FC + 2);
    }
};

template <typename T>
__device__ __forceinline__ void core_load(float *dst, int ld, int d4, int d, const void *src, long long ldr, int h, const Rows &rows, int u0, int n)
{
    const T *base = reinterpret_cast<const T *>(src) + (size_t)h * d;
    for (int i = threadIdx.x; i < FC * d4; i += 256) {
        const int r = i / d4, x = i % d4;
        dst[r * ld + x] = r < n && x < d ? to_f(base[rows.row(u0 + r) * ldr + x]) : 0.0f;
    }
}

// STATES: the first pass over a sequence in several parts: what each part but the last adds to the state
template <typename T, bool STATES>
__global__ void __launch_bounds__(256) core_kernel(const __grid_constant__ Args p)
{
    extern __shared__ __align__(16) float smf[];
    const CoreSmem sm(p.da, p.dc);
    float *As = smf, *Bs = smf + sm.b, *Cs = smf + sm.c, *Ss = smf + sm.s, *Ps = smf + sm.p, *pw = smf + sm.w, *wt = pw + FC + 2;
    const int tid = threadIdx.x;
    const size_t pair = blockIdx.x;
    const int g = blockIdx.y, b = (int)(pair / p.H), h = (int)(pair % p.H);
    const float rate = p.rate[h];
    pdl_trigger();
    pdl_wait();
    const Rows rows(p, b);
    const size_t nn = (size_t)p.da * p.dc;
    const int begin = g * p.seg, end = min(rows.n, begin + p.seg);
    const float l_seg = power(rate, p.seg);
    for (int i = tid; i < FC + 2; i += 256)
        pw[i] = power(rate, i);
    for (int i = tid; i < sm.da4 * sm.dc4; i += 256) {
        const int x = i / sm.dc4, y = i % sm.dc4;
        float s = 0.0f;
        if (x < p.da && y < p.dc) {
            if (!STATES)
                s = start_at(p, pair, g, x, y, l_seg);
            else if (g == 0) { // the state before the first token is kept: s_end may lie where it lies
                p.parts[pair * p.n_seg * nn + (size_t)x * p.dc + y] = p.s0 ? state_at(p, p.s0 + pair * nn, x, y) : 0.0f;
            }
        }
        Ss[x * sm.ld_c + y] = s;
    }
    if (!STATES && p.o)
        zero_behind<T>(p, rows, b, h, g, tid, 256);
    for (int u0 = begin; u0 < end; u0 += FC) {
        const int n = min(FC, end - u0);
        __syncthreads();
        if (!STATES)
            core_load<T>(As, sm.ld_a, sm.da4, p.da, p.a, p.lda, h, rows, u0, n);
        core_load<T>(Bs, sm.ld_a, sm.da4, p.da, p.b, p.ldb, h, rows, u0, n);
        core_load<T>(Cs, sm.ld_c, sm.dc4, p.dc, p.c, p.ldc, h, rows, u0, n);
        for (int i = tid; i < FC; i += 256)
            wt[i] = i < n ? p.s_in * pw[n - 1 - i + p.e2] : 0.0f;
        __syncthreads();
        if (!STATES) {
            for (int k = 0; k < FC * FC / 256; k++) {
                const int i = tid / 8, j = tid % 8 + 8 * k;
                float s = 0.0f;
                if (j <= i) {
                    for (int x = 0; x < sm.da4; x += 4) {
                        const float4 u = *reinterpret_cast<const float4 *>(As + i * sm.ld_a + x), v = *reinterpret_cast<const float4 *>(Bs + j * sm.ld_a + x);
                        s = fmaf(u.x, v.x, fmaf(u.y, v.y, fmaf(u.z, v.z, fmaf(u.w, v.w, s))));
                    }
                    s *= p.s_pair * pw[i - j];
                }
                Ps[i * (FC + 1) + j] = s;
            }
            __syncthreads();
            for (int it = tid; it < FC / 4 * (sm.dc4 / 4); it += 256) {
                const int i0 = it / (sm.dc4 / 4) * 4, c0 = it % (sm.dc4 / 4) * 4;
                float acc[4][4] = {};
                for (int x = 0; x < p.da; x++) {
                    const float4 s = *reinterpret_cast<const float4 *>(Ss + x * sm.ld_c + c0);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float u = As[(i0 + r) * sm.ld_a + x];
                        acc[r][0] = fmaf(u, s.x, acc[r][0]); acc[r][1] = fmaf(u, s.y, acc[r][1]);
                        acc[r][2] = fmaf(u, s.z, acc[r][2]); acc[r][3] = fmaf(u, s.w, acc[r][3]);
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float f = p.s_state * pw[i0 + r + p.e1];
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        acc[r][c] *= f;
                }
                for (int j = 0; j < min(i0 + 4, n); j++) {
                    const float4 s = *reinterpret_cast<const float4 *>(Cs + j * sm.ld_c + c0);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float u = Ps[(i0 + r) * (FC + 1) + j];
                        acc[r][0] = fmaf(u, s.x, acc[r][0]); acc[r][1] = fmaf(u, s.y, acc[r][1]);
                        acc[r][2] = fmaf(u, s.z, acc[r][2]); acc[r][3] = fmaf(u, s.w, acc[r][3]);
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (i0 + r < n) {
                        T *o = reinterpret_cast<T *>(p.o) + rows.row(u0 + i0 + r) * p.ldo + (size_t)h * p.dc + c0;
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            if (c0 + c < p.dc)
                                o[c] = from_f<T>(acc[r][c]);
                    }
            }
            __syncthreads();
        }
        const float l_n = pw[n];
        for (int it = tid; it < (sm.da4 / 4) * (sm.dc4 / 4); it += 256) {
            const int x0 = it / (sm.dc4 / 4) * 4, c0 = it % (sm.dc4 / 4) * 4;
            float acc[4][4] = {};
            for (int j = 0; j < n; j++) {
                const float4 s = *reinterpret_cast<const float4 *>(Cs + j * sm.ld_c + c0);
                const float w = wt[j];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float u = w * Bs[j * sm.ld_a + x0 + r];
                    acc[r][0] = fmaf(u, s.x, acc[r][0]); acc[r][1] = fmaf(u, s.y, acc[r][1]);
                    acc[r][2] = fmaf(u, s.z, acc[r][2]); acc[r][3] = fmaf(u, s.w, acc[r][3]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    float *s = Ss + (x0 + r) * sm.ld_c + c0 + c;
                    *s = fmaf(l_n, *s, acc[r][c]);
                }
        }
    }
    __syncthreads();
    // behind the last token; a stream without tokens ends in part 0
    float *to = STATES ? p.parts + (pair * p.n_seg + g + 1) * nn
                       : (p.s_end && begin < max(rows.n, 1) && max(rows.n, 1) <= begin + p.seg ? p.s_end + pair * nn : nullptr);
    if (to)
        for (int i = tid; i < p.da * p.dc; i += 256)
            to[i] = Ss[i / p.dc * sm.ld_c + i % p.dc];
}

// ---------------- a few tokens: the recurrence itself ----------------
//
// A CTA of four warps takes 8 * VEC columns of one (stream, head)'s state into registers, sixteen rows side by side, and
// goes through the tokens one after the other.  Bound by HBM: the state once in and once out, all of a thread's
// loads in flight together.

constexpr int STEP_TOKENS = 8;

template <typename T, int VEC>
__global__ void __launch_bounds__(128) step_kernel(const __grid_constant__ Args p)
{
    constexpr int COLS = 8 * VEC, MOST = DIM_MAX / 16;
    __shared__ float As[STEP_TOKENS][DIM_MAX], Bs[STEP_TOKENS][DIM_MAX], Cs[STEP_TOKENS][COLS], red[STEP_TOKENS][4][COLS];
    const int tid = threadIdx.x, cg = tid & 7, rl = tid >> 3;
    const size_t pair = blockIdx.x;
    const int b = (int)(pair / p.H), h = (int)(pair % p.H), c0 = blockIdx.y * COLS;
    const float l = exp2f(p.rate[h]);
    pdl_trigger();
    pdl_wait();
    const Rows rows(p, b);
    const size_t nn = (size_t)p.da * p.dc;
    float s[MOST][VEC];
#pragma unroll
    for (int k = 0; k < MOST; k++) {
        const int x = rl + 16 * k, c = c0 + cg * VEC;
#pragma unroll
        for (int v = 0; v < VEC; v++)
            s[k][v] = 0.0f;
        if (p.s0 && x < p.da && c < p.dc) {
            const float *s0 = p.s0 + pair * nn;
            if (VEC == 4 && !p.s0_t) {
                const float4 f = *reinterpret_cast<const float4 *>(s0 + (size_t)x * p.dc + c);
                s[k][0] = f.x; s[k][1 % VEC] = f.y; s[k][2 % VEC] = f.z; s[k][3 % VEC] = f.w;
            } else {
#pragma unroll
                for (int v = 0; v < VEC; v++)
                    s[k][v] = state_at(p, s0, x, c + v);
            }
        }
    }
    const T *a = reinterpret_cast<const T *>(p.a) + (size_t)h * p.da, *bb = reinterpret_cast<const T *>(p.b) + (size_t)h * p.da,
            *cc = reinterpret_cast<const T *>(p.c) + (size_t)h * p.dc;
    for (int u = 0; u < rows.n; u++) {
        const long long row = rows.row(u);
        if (tid < p.da) {
            As[u][tid] = to_f(a[row * p.lda + tid]);
            Bs[u][tid] = p.s_in * to_f(bb[row * p.ldb + tid]);
        }
        if (tid < COLS)
            Cs[u][tid] = c0 + tid < p.dc ? to_f(cc[row * p.ldc + c0 + tid]) : 0.0f;
    }
    __syncthreads();
    const float before = p.e1 ? l : 1.0f, behind = p.e2 ? l : 1.0f, s_out = p.s_state;
    for (int u = 0; u < rows.n; u++) {
        float acc[VEC], cv[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            acc[v] = 0.0f;
            cv[v] = Cs[u][cg * VEC + v];
        }
#pragma unroll
        for (int k = 0; k < MOST; k++) {
            const int x = rl + 16 * k;
            if (x < p.da) {
                const float av = As[u][x], bv = Bs[u][x];
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    s[k][v] = fmaf(before, s[k][v], bv * cv[v]);
                    acc[v] = fmaf(av, s[k][v], acc[v]);
                    s[k][v] *= behind;
                }
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            acc[v] += __shfl_xor_sync(0xffffffffu, acc[v], 8);
            acc[v] += __shfl_xor_sync(0xffffffffu, acc[v], 16);
            if ((tid & 31) < 8)
                red[u][tid >> 5][cg * VEC + v] = acc[v];
        }
    }
    if (p.s_end) {
#pragma unroll
        for (int k = 0; k < MOST; k++) {
            const int x = rl + 16 * k, c = c0 + cg * VEC;
            if (x < p.da && c < p.dc) {
                float *to = p.s_end + pair * nn + (size_t)x * p.dc + c;
                if (VEC == 4)
                    *reinterpret_cast<float4 *>(to) = make_float4(s[k][0], s[k][1 % VEC], s[k][2 % VEC], s[k][3 % VEC]);
                else
                    to[0] = s[k][0];
            }
        }
    }
    __syncthreads();
    if (p.o) {
        T *o = reinterpret_cast<T *>(p.o) + (size_t)h * p.dc;
        for (int i = tid; i < p.T * COLS; i += 128) {
            const int u = i / COLS, x = i % COLS;
            if (c0 + x >= p.dc)
                continue;
            if (u < rows.n)
                o[rows.row(u) * p.ldo + c0 + x] = from_f<T>(s_out * (red[u][0][x] + red[u][1][x] + red[u][2][x] + red[u][3][x]));
            else // behind the stream's end
                o[((long long)u * p.B + b) * p.ldo + c0 + x] = from_f<T>(0.0f);
        }
    }
}

} // namespace lin
