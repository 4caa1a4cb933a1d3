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

// ---------------- bf16 on warp-level tensor-core products ----------------
//
// A CTA of eight warps goes through one part of one (stream, head) in chunks of 64 tokens.  Warp (r, hc) takes rows
// 16 r .. 16 r + 15 of a chunk and half hc of the columns of c; of the state it owns the same columns of rows 16 r .. (and
// 16 (r + 4) .. of 128) in fp32 accumulators.  The results need all of the state: it goes through shared memory in bf16,
// one rounding, as the pair weights P have one; products of a decayed b with c, which the state adds up, are kept to
// 24 bits by three bf16 terms of the decayed value, so that the state is an fp32 sum of fp32 products.  The next chunk's
// tiles are fetched under the present chunk, and one barrier a chunk hands over tiles and state.

constexpr int TC = 64; // tokens in a chunk

template <int DA, int DC> struct MmaSmem {
    static constexpr int LA = DA + 8, LC = DC + 8;            // pitches: rows four banks on
    static constexpr int A = 0, B = A + 2 * TC * LA * 2, C = B + 2 * TC * LA * 2, S = C + 2 * TC * LC * 2,
                         W = S + 2 * DA * LC * 2, BYTES = W + (2 * TC + 8) * 4;
};

// 64 rows of a matrix as a tile, zeros behind row n and column d
template <int D>
__device__ __forceinline__ void tile_load(bf16 *dst, const bf16 *src, long long ldr, int d, const Rows &rows, int u0, int n)
{
    constexpr int CPR = D / 8;
    for (int i = threadIdx.x; i < TC * CPR; i += 256) {
        const int r = i / CPR, x = i % CPR * 8;
        const bool ok = r < n && x < d;
        fa::cp16(dst + r * (D + 8) + x, ok ? src + rows.row(u0 + r) * ldr + x : src, ok);
    }
}

// a pair of bf16 values times their weights as three bf16 terms that add up to 24 bits of them
__device__ __forceinline__ void split3(uint32_t v, float w0, float w1, uint32_t &hi, uint32_t &mid, uint32_t &lo)
{
    float x = __uint_as_float(v << 16) * w0, y = __uint_as_float(v & 0xffff0000u) * w1;
    hi = fa::pack2(x, y);
    x -= __uint_as_float(hi << 16);
    y -= __uint_as_float(hi & 0xffff0000u);
    mid = fa::pack2(x, y);
    lo = fa::pack2(x - __uint_as_float(mid << 16), y - __uint_as_float(mid & 0xffff0000u));
}

// TERMS: 3, or 2 where no state is a result (17 bits of a decayed value are more than the rounding behind them keeps)
template <int DA, int DC, bool STATES, int TERMS>
__global__ void __launch_bounds__(256) mma_kernel(const __grid_constant__ Args p)
{
    using SM = MmaSmem<DA, DC>;
    constexpr int LA = SM::LA, LC = SM::LC, NT = DC / 16, MT = DA > 64 ? DA / 64 : 1, KS = DA / 16;
    extern __shared__ __align__(16) unsigned char smb[];
    bf16 *As = reinterpret_cast<bf16 *>(smb + SM::A), *Bs = reinterpret_cast<bf16 *>(smb + SM::B),
         *Cs = reinterpret_cast<bf16 *>(smb + SM::C), *Ss = reinterpret_cast<bf16 *>(smb + SM::S);
    float *wts = reinterpret_cast<float *>(smb + SM::W), *pw16 = wts + 2 * TC; // weights of full and last chunks; l^16m
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, t = lane & 3;
    // the two warps of a scheduler take rows r and 3 - r: the triangle is dealt evenly
    const int hc = warp >> 2, r = hc ? 3 - (warp & 3) : warp & 3;
    const size_t pair = blockIdx.x;
    const int g = blockIdx.y, b = (int)(pair / p.H), h = (int)(pair % p.H);
    const float rate = p.rate[h];
    pdl_trigger();
    pdl_wait();
    const Rows rows(p, b);
    const size_t nn = (size_t)p.da * p.dc;
    const int begin = g * p.seg, end = min(rows.n, begin + p.seg), total = max(end - begin, 0), chunks = (total + TC - 1) / TC;
    const bf16 *ga = reinterpret_cast<const bf16 *>(p.a) + (size_t)h * p.da, *gb = reinterpret_cast<const bf16 *>(p.b) + (size_t)h * p.da,
               *gc = reinterpret_cast<const bf16 *>(p.c) + (size_t)h * p.dc;
    auto fetch = [&](int k) {
        const int u0 = begin + k * TC, n = end - u0, buf = k & 1;
        if (!STATES)
            tile_load<DA>(As + buf * TC * LA, ga, p.lda, p.da, rows, u0, n);
        tile_load<DA>(Bs + buf * TC * LA, gb, p.ldb, p.da, rows, u0, n);
        tile_load<DC>(Cs + buf * TC * LC, gc, p.ldc, p.dc, rows, u0, n);
        fa::cp_commit();
    };
    if (chunks)
        fetch(0);
    const int n_last = total - (chunks - 1) * TC;
    if (tid < TC)
        wts[tid] = p.s_in * power(rate, TC - 1 - tid + p.e2);
    else if (tid < 2 * TC)
        wts[tid] = tid - TC < n_last ? p.s_in * power(rate, n_last - 1 - (tid - TC) + p.e2) : 0.0f;
    else if (tid < 2 * TC + 4)
        pw16[tid - 2 * TC] = power(rate, 16 * (tid - 2 * TC));

    // the state: element c of s[m][n] is row 16 (r + 4 m) + gq + 8 (c >> 1), column hc * DC / 2 + 8 n + 2 t + (c & 1)
    float s[MT][NT][4];
    const float l_seg = power(rate, p.seg), l_full = power(rate, TC), l_last = power(rate, n_last);
    const bool has_state = r * 16 < DA; // of 32 rows the warps r = 2, 3 own none
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int x = 16 * (r + 4 * m) + gq + 8 * (c >> 1), y = hc * (DC / 2) + 8 * n + 2 * t + (c & 1);
                s[m][n][c] = 0.0f;
                if (x < p.da && y < p.dc) {
                    if (!STATES)
                        s[m][n][c] = start_at(p, pair, g, x, y, l_seg);
                    else if (g == 0) // the state before the first token is kept: s_end may lie where it lies
                        p.parts[pair * p.n_seg * nn + (size_t)x * p.dc + y] = p.s0 ? state_at(p, p.s0 + pair * nn, x, y) : 0.0f;
                }
            }
    auto publish = [&](int buf) {
        if (!STATES && has_state)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    bf16 *to = Ss + buf * DA * LC + (16 * (r + 4 * m) + gq) * LC + hc * (DC / 2) + 8 * n + 2 * t;
                    *reinterpret_cast<uint32_t *>(to) = fa::pack2(s[m][n][0], s[m][n][1]);
                    *reinterpret_cast<uint32_t *>(to + 8 * LC) = fa::pack2(s[m][n][2], s[m][n][3]);
                }
    };
    publish(0);
    if (!STATES && p.o)
        zero_behind<bf16>(p, rows, b, h, g, tid, 256);

    // weights of pairs 16 rows apart and on the diagonal, of this thread's elements of two 8-key groups
    float apart[2][4], diag[2][4];
    const float f_a = p.s_state * power(rate, 16 * r + gq + p.e1), f_b = p.s_state * power(rate, 16 * r + gq + 8 + p.e1);
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int d = gq + 8 * (c >> 1) - 8 * n - 2 * t - (c & 1);
            apart[n][c] = p.s_pair * power(rate, 16 + d);
            diag[n][c] = d >= 0 ? p.s_pair * power(rate, d) : 0.0f;
        }

    for (int k = 0; k < chunks; k++) {
        const int buf = k & 1, u0 = begin + k * TC, n = min(TC, end - u0);
        const bool last = k == chunks - 1;
        fa::cp_wait<0>();
        __syncthreads(); // this chunk's tiles and state stand; the other buffers are free
        if (!last)
            fetch(k + 1);
        const bf16 *At = As + buf * TC * LA, *Bt = Bs + buf * TC * LA, *Ct = Cs + buf * TC * LC + hc * (DC / 2),
                   *St = Ss + buf * DA * LC + hc * (DC / 2);
        float o[NT][4];
        if (!STATES) {
#pragma unroll
            for (int x = 0; x < NT; x++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    o[x][c] = 0.0f;
            uint32_t aq[KS][4];
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                fa::ldsm4(aq[ks], At + (16 * r + (lane & 15)) * LA + ks * 16 + (lane >> 4) * 8);
#pragma unroll
                for (int x = 0; x < NT; x += 2) {
                    uint32_t f[4];
                    fa::ldsm4t(f, St + (ks * 16 + (lane & 15)) * LC + x * 8 + (lane >> 4) * 8);
                    fa::mma(o[x], aq[ks], f[0], f[1]);
                    fa::mma(o[x + 1], aq[ks], f[2], f[3]);
                }
            }
#pragma unroll
            for (int x = 0; x < NT; x++) {
                o[x][0] *= f_a; o[x][1] *= f_a;
                o[x][2] *= f_b; o[x][3] *= f_b;
            }
#pragma unroll
            for (int pc = 0; pc < 4; pc++) {
                if (pc > r)
                    break;
                float w[2][4] = {};
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t f[4];
                    fa::ldsm4(f, Bt + (pc * 16 + (lane & 7) + (lane >> 4) * 8) * LA + ks * 16 + ((lane >> 3) & 1) * 8);
                    fa::mma(w[0], aq[ks], f[0], f[1]);
                    fa::mma(w[1], aq[ks], f[2], f[3]);
                }
                if (pc == r) {
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            w[x][c] = gq + 8 * (c >> 1) >= 8 * x + 2 * t + (c & 1) ? w[x][c] * diag[x][c] : 0.0f;
                } else {
                    const float f = pw16[r - pc - 1];
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            w[x][c] *= f * apart[x][c];
                }
                const uint32_t pf[4] = {fa::pack2(w[0][0], w[0][1]), fa::pack2(w[0][2], w[0][3]), fa::pack2(w[1][0], w[1][1]),
                                        fa::pack2(w[1][2], w[1][3])};
#pragma unroll
                for (int x = 0; x < NT; x += 2) {
                    uint32_t f[4];
                    fa::ldsm4t(f, Ct + (pc * 16 + (lane & 15)) * LC + x * 8 + (lane >> 4) * 8);
                    fa::mma(o[x], pf, f[0], f[1]);
                    fa::mma(o[x + 1], pf, f[2], f[3]);
                }
            }
            // rows out: a lane's column pairs
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
                const int i = 16 * r + gq + 4 * c;
                bf16 *to = reinterpret_cast<bf16 *>(p.o) + (i < n ? rows.row(u0 + i) * p.ldo : 0) + (size_t)h * p.dc + hc * (DC / 2) + 2 * t;
#pragma unroll
                for (int x = 0; x < NT; x++)
                    if (i < n && hc * (DC / 2) + 8 * x < p.dc)
                        *reinterpret_cast<uint32_t *>(to + 8 * x) = fa::pack2(o[x][c], o[x][c + 1]);
            }
        }
        if (last && !STATES && !p.s_end)
            break;
        // the state behind the chunk
        const float l_n = last ? l_last : l_full, *wt = wts + (last ? TC : 0);
        if (has_state) {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int x = 0; x < NT; x++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        s[m][x][c] *= l_n;
#pragma unroll
            for (int ks = 0; ks < TC / 16; ks++) {
                const float2 w0 = *reinterpret_cast<const float2 *>(wt + ks * 16 + 2 * t), w8 = *reinterpret_cast<const float2 *>(wt + ks * 16 + 8 + 2 * t);
                uint32_t hi[MT][4], mid[MT][4], lo[MT][4];
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    uint32_t f[4];
                    fa::ldsm4t(f, Bt + (ks * 16 + (lane & 7) + (lane >> 4) * 8) * LA + 16 * (r + 4 * m) + ((lane >> 3) & 1) * 8);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        split3(f[e], e < 2 ? w0.x : w8.x, e < 2 ? w0.y : w8.y, hi[m][e], mid[m][e], lo[m][e]);
                }
#pragma unroll
                for (int x = 0; x < NT; x += 2) {
                    uint32_t f[4];
                    fa::ldsm4t(f, Ct + (ks * 16 + (lane & 15)) * LC + x * 8 + (lane >> 4) * 8);
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        fa::mma(s[m][x], hi[m], f[0], f[1]);
                        fa::mma(s[m][x + 1], hi[m], f[2], f[3]);
                        fa::mma(s[m][x], mid[m], f[0], f[1]);
                        fa::mma(s[m][x + 1], mid[m], f[2], f[3]);
                        if (TERMS > 2) {
                            fa::mma(s[m][x], lo[m], f[0], f[1]);
                            fa::mma(s[m][x + 1], lo[m], f[2], f[3]);
                        }
                    }
                }
            }
        }
        if (!last)
            publish(buf ^ 1);
    }
    float *to = STATES ? p.parts + (pair * p.n_seg + g + 1) * nn
                       : (p.s_end && begin < max(rows.n, 1) && max(rows.n, 1) <= begin + p.seg ? p.s_end + pair * nn : nullptr);
    if (to && has_state)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int x = 0; x < NT; x++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int i = 16 * (r + 4 * m) + gq + 8 * (c >> 1), y = hc * (DC / 2) + 8 * x + 2 * t + (c & 1);
                    if (i < p.da && y < p.dc)
                        to[(size_t)i * p.dc + y] = s[m][x][c];
                }
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
