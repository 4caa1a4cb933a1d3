// qk_norm.cuh -- queries and keys normed for each head and rotated by their positions in one pass.
//
//   x^ = x / sqrt(mean(x^2) + eps),  n = x^ gain,  y = R(pos) n
//
// R turns the pairs (i, i + d_rot / 2) -- or (2i, 2i + 1) -- of the first d_rot values by pos base^(-2i / d_rot).  The
// adjoint turns back: u = R(-pos) dy, dgain = sum u x^, w = u gain, dx = (w - x^ mean(w x^)) / sqrt(mean(x^2) + eps).
//
// Bound by HBM: every value once in and once out (forward), twice in and once out (backward).  A head's row lies in
// the registers of G neighbouring lanes, each with both members of its pairs, so that neither the rotation nor a
// second look at x costs memory; sines and cosines are taken once for a row and all its heads.  Angles are
// reduced in 64 bits: positions of a large file leave no digit of an fp32 angle behind the point.
#pragma once
#include "warp_mma.cuh"

namespace qkn {

constexpr int DIM_MAX = NNCU_QK_NORM_DIM_MAX;

struct Args {
    const void *x[2];    // queries, keys
    const void *dy[2];   // gradients of the results
    void *y[2];          // results, or gradients of x
    const float *gain[2];
    const int32_t *pos;  // of each row; below 0: the row is padding
    float *part;         // [grid][2][d] partial sums of dgain
    long long ldx[2], ldy[2];
    int heads[2];
    int N, d, rot, adjacent, lanes, rows_per; // lanes: of a head (a power of two)
    float eps;
    double turns[DIM_MAX / 2]; // of pair i from one position to the next
};

template <typename T, int W> __device__ __forceinline__ void take(float (&v)[W], const T *p)
{
#pragma unroll
    for (int i = 0; i < W; i++)
        v[i] = to_f(p[i]);
}
template <typename T, int W> __device__ __forceinline__ void load(float (&v)[W], const T *p)
{
    if constexpr (sizeof(T) * W == 16) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        take<T, W>(v, reinterpret_cast<const T *>(&u));
    } else if constexpr (sizeof(T) * W == 8) {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        take<T, W>(v, reinterpret_cast<const T *>(&u));
    } else if constexpr (sizeof(T) * W == 4) {
        const uint32_t u = *reinterpret_cast<const uint32_t *>(p);
        take<T, W>(v, reinterpret_cast<const T *>(&u));
    } else {
        take<T, W>(v, p);
    }
}
template <typename T, int W> __device__ __forceinline__ void store(T *p, const float (&v)[W])
{
    struct __align__(16) { T t[W]; } o;
#pragma unroll
    for (int i = 0; i < W; i++)
        o.t[i] = from_f<T>(v[i]);
    if constexpr (sizeof(T) * W == 16)
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(&o);
    else if constexpr (sizeof(T) * W == 8)
        *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(&o);
    else if constexpr (sizeof(T) * W == 4)
        *reinterpret_cast<uint32_t *>(p) = *reinterpret_cast<const uint32_t *>(&o);
    else
#pragma unroll
        for (int i = 0; i < W; i++)
            p[i] = o.t[i];
}

// Where a lane's pairs p0 .. p0 + W - 1 lie in a head's row: two runs of W values.  Pairs behind the rotated ones are
// halves of what is left, or neighbours too.
template <int W> struct Place {
    int lo, hi;
    __device__ __forceinline__ Place(const Args &a, int p0)
    {
        if (a.adjacent) {
            lo = 2 * p0;
            hi = lo + W;
        } else if (p0 < a.rot / 2) {
            lo = p0;
            hi = p0 + a.rot / 2;
        } else {
            lo = p0 + a.rot / 2;
            hi = lo + (a.d - a.rot) / 2;
        }
    }
};

// the W pairs of a lane turned by the angles at cs; to: +1 there, -1 back.  x[0], x[1]: the two runs
template <int W> __device__ __forceinline__ void turn(float (&x)[2][W], const float2 *cs, bool adjacent, float to)
{
#pragma unroll
    for (int k = 0; k < W; k++) {
        const float c = cs[k].x, s = to * cs[k].y;
        if (adjacent) { // pair k: values 2k, 2k + 1 of both runs in a row
            float &a = x[2 * k / W][2 * k % W], &b = x[(2 * k + 1) / W][(2 * k + 1) % W];
            const float u = a * c - b * s;
            b = b * c + a * s;
            a = u;
        } else {
            const float u = x[0][k] * c - x[1][k] * s;
            x[1][k] = x[1][k] * c + x[0][k] * s;
            x[0][k] = u;
        }
    }
}

// cosines and sines of rows r0 .. r0 + n - 1: [n][rot / 2]
__device__ __forceinline__ void angles(const Args &a, float2 *cs, int r0, int n, int tid, int nthr)
{
    const int half = a.rot / 2;
    for (int i = tid; i < n * half; i += nthr) {
        const double t = (double)a.pos[r0 + i / half] * a.turns[i % half];
        float s, c;
        sincospif((float)(2.0 * (t - rint(t))), &s, &c);
        cs[i] = make_float2(c, s);
    }
}

// A lane has NG groups of W pairs, a group's neighbours in the neighbouring lanes
template <typename T, int W, int NG, bool BACK>
__global__ void __launch_bounds__(256) kernel(const __grid_constant__ Args a)
{
    extern __shared__ __align__(16) float sh[];
    float2 *cs = reinterpret_cast<float2 *>(sh);
    float *red = sh + a.rows_per * a.rot; // backward: [8 warps][d]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.lanes, per_warp = 32 / G;
    const int half = a.rot / 2;
    int p0[NG], lo[NG], hi[NG];
    bool mine[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
        p0[g] = ((lane & (G - 1)) + g * G) * W;
        mine[g] = p0[g] < a.d / 2;
        const Place<W> at(a, mine[g] ? p0[g] : 0);
        lo[g] = at.lo;
        hi[g] = at.hi;
    }
    const float inv_d = 1.0f / (float)a.d;
    pdl_trigger();
    pdl_wait();
    float acc[BACK ? 2 : 1][NG][2][W] = {};
    for (int r0 = blockIdx.x * a.rows_per; r0 < a.N; r0 += gridDim.x * a.rows_per) {
        const int n = min(a.rows_per, a.N - r0);
        if (half) {
            __syncthreads();
            angles(a, cs, r0, n, tid, 256);
            __syncthreads();
        }
#pragma unroll
        for (int what = 0; what < 2; what++) {
            const int H = a.heads[what];
            float gain[NG][2][W];
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int k = 0; k < W; k++)
                        gain[g][j][k] = a.gain[what] && mine[g] ? a.gain[what][(j ? hi[g] : lo[g]) + k] : 1.0f;
            // a warp's heads are neighbours; all its lanes go through every round (shuffles)
            for (int i0 = warp * per_warp; i0 < n * H; i0 += 8 * per_warp) {
                const int i = i0 + lane / G, r = i < n * H ? i / H : 0, h = i < n * H ? i % H : 0;
                const long long row = r0 + r;
                const bool real = i < n * H, live = real && (!a.pos || a.pos[row] >= 0);
                const T *px = reinterpret_cast<const T *>(a.x[what]) + row * a.ldx[what] + (size_t)h * a.d;
                const T *pd = reinterpret_cast<const T *>(a.dy[what]) + row * a.ldy[what] + (size_t)h * a.d;
                float x[NG][2][W] = {}, u[NG][2][W] = {};
                float sq = 0.0f;
#pragma unroll
                for (int g = 0; g < NG; g++)
                    if (live && mine[g]) {
                        load<T, W>(x[g][0], px + lo[g]);
                        load<T, W>(x[g][1], px + hi[g]);
                        if (BACK) {
                            load<T, W>(u[g][0], pd + lo[g]);
                            load<T, W>(u[g][1], pd + hi[g]);
                        }
                    }
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int k = 0; k < W; k++)
                        sq += x[g][0][k] * x[g][0][k] + x[g][1][k] * x[g][1][k];
                for (int o = G / 2; o > 0; o >>= 1)
                    sq += __shfl_xor_sync(0xffffffffu, sq, o);
                const float rs = rsqrtf(sq * inv_d + a.eps);
                if (!BACK) {
#pragma unroll
                    for (int g = 0; g < NG; g++) {
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int k = 0; k < W; k++)
                                u[g][j][k] = x[g][j][k] * rs * gain[g][j][k];
                        if (p0[g] < half)
                            turn<W>(u[g], cs + r * half + p0[g], a.adjacent, 1.0f);
                    }
                } else {
                    float dot = 0.0f;
#pragma unroll
                    for (int g = 0; g < NG; g++) {
                        if (p0[g] < half)
                            turn<W>(u[g], cs + r * half + p0[g], a.adjacent, -1.0f);
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int k = 0; k < W; k++) {
                                x[g][j][k] *= rs;
                                acc[what][g][j][k] += u[g][j][k] * x[g][j][k];
                                u[g][j][k] *= gain[g][j][k];
                                dot += u[g][j][k] * x[g][j][k];
                            }
                    }
                    for (int o = G / 2; o > 0; o >>= 1)
                        dot += __shfl_xor_sync(0xffffffffu, dot, o);
                    dot *= inv_d;
#pragma unroll
                    for (int g = 0; g < NG; g++)
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int k = 0; k < W; k++)
                                u[g][j][k] = rs * (u[g][j][k] - x[g][j][k] * dot);
                }
                // padding: x and u are zeros, and so are the results (eps may be 0)
                T *py = reinterpret_cast<T *>(a.y[what]) + row * (BACK ? a.ldx[what] : a.ldy[what]) + (size_t)h * a.d;
#pragma unroll
                for (int g = 0; g < NG; g++)
                    if (real && mine[g]) {
                        if (!live)
#pragma unroll
                            for (int k = 0; k < W; k++)
                                u[g][0][k] = u[g][1][k] = 0.0f;
                        store<T, W>(py + lo[g], u[g][0]);
                        store<T, W>(py + hi[g], u[g][1]);
                    }
            }
        }
    }
    if (BACK && a.part) {
        // the CTA's sums: lanes of the same pairs, then warps in order
#pragma unroll
        for (int what = 0; what < 2; what++) {
            __syncthreads();
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int k = 0; k < W; k++) {
                        float s = acc[BACK ? what : 0][g][j][k];
                        for (int o = G; o < 32; o <<= 1)
                            s += __shfl_xor_sync(0xffffffffu, s, o);
                        if (lane < G && mine[g])
                            red[warp * a.d + (j ? hi[g] : lo[g]) + k] = s;
                    }
            __syncthreads();
            for (int i = tid; i < a.d; i += 256) {
                float s = 0.0f;
                for (int w = 0; w < 8; w++)
                    s += red[w * a.d + i];
                a.part[((size_t)blockIdx.x * 2 + what) * a.d + i] = s;
            }
        }
    }
}

// dgain of queries and keys: the CTAs' sums, eight strands in a fixed order
__global__ void __launch_bounds__(256) gain_kernel(const float *__restrict__ part, int n_parts, int d, float *dgain_q, float *dgain_k)
{
    __shared__ float red[8][32];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), strand = threadIdx.x >> 5;
    pdl_trigger();
    pdl_wait();
    float s = 0.0f;
    if (col < 2 * d)
        for (int i = strand; i < n_parts; i += 8)
            s += part[(size_t)i * 2 * d + col];
    red[strand][threadIdx.x & 31] = s;
    __syncthreads();
    if (strand == 0 && col < 2 * d) {
        s = red[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < 8; k++)
            s += red[k][threadIdx.x];
        float *to = col < d ? dgain_q : dgain_k;
        if (to)
            to[col < d ? col : col - d] = s;
    }
}

} // namespace qkn
