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
    uint32_t inverse[2]; // ceil(2^32 / heads); 0 for one head
    int N, d, rot, adjacent, lanes, rows_per; // lanes: of a head (a power of two)
    float eps;
    double turns[DIM_MAX / 2]; // of pair i from one position to the next
};

// W values as they lie in memory
template <int BYTES> struct Raw;
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<2> { typedef uint16_t type; };
template <typename T, int W> using raw_t = typename Raw<sizeof(T) * W>::type;

template <typename T, int W> __device__ __forceinline__ void take(float (&v)[W], const raw_t<T, W> &u)
{
    const T *p = reinterpret_cast<const T *>(&u);
#pragma unroll
    for (int i = 0; i < W; i++)
        v[i] = to_f(p[i]);
}
template <typename T, int W> __device__ __forceinline__ raw_t<T, W> put(const float (&v)[W])
{
    raw_t<T, W> u;
    T *p = reinterpret_cast<T *>(&u);
#pragma unroll
    for (int i = 0; i < W; i++)
        p[i] = from_f<T>(v[i]);
    return u;
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

// Cosines and sines of rows r0 .. r0 + n - 1, [n][rot / 2], and which of them are no padding
__device__ __forceinline__ void angles(const Args &a, float2 *cs, int *live, int r0, int n, int tid)
{
    const int half = a.rot / 2;
    for (int i = tid; i < n * half; i += 256) {
        const double t = (double)a.pos[r0 + i / half] * a.turns[i % half];
        float s, c;
        sincospif((float)(2.0 * (t - rint(t))), &s, &c);
        cs[i] = make_float2(c, s);
    }
    if (tid < n)
        live[tid] = !a.pos || a.pos[r0 + tid] >= 0;
}

// A warp takes 32 / lanes heads of neighbouring places at a time, queries of the CTA's rows and then keys; the
// next ones are on their way while it computes, the first while the angles are taken.  A lane has NG groups of W pairs,
// a group's neighbours in the neighbouring lanes.
template <typename T, int W, int NG, bool BACK>
__global__ void __launch_bounds__(256, BACK ? 2 : 3) kernel(const __grid_constant__ Args a)
{
    extern __shared__ __align__(16) float sh[];
    __shared__ int live[8];
    float2 *cs = reinterpret_cast<float2 *>(sh);
    float *gains = sh + a.rows_per * a.rot, *red = gains + 2 * a.d; // backward: red [8 warps][d]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.lanes, per_warp = 32 / G, sub = lane / G;
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
    pdl_wait();
    for (int i = tid; i < 2 * a.d; i += 256) {
        const float *from = a.gain[i >= a.d];
        gains[i] = from ? from[i >= a.d ? i - a.d : i] : 1.0f;
    }
    float acc[BACK ? 2 : 1][NG][2][W] = {};
    struct Item {
        raw_t<T, W> x[NG][2], dy[BACK ? NG : 1][2];
        long long at; // where the result goes
        int r, what;
        bool real;
    };
    for (int r0 = blockIdx.x * a.rows_per; r0 < a.N; r0 += gridDim.x * a.rows_per) {
        const int n = min(a.rows_per, a.N - r0);
        const int rounds_q = (n * a.heads[0] + per_warp - 1) / per_warp, rounds = rounds_q + (n * a.heads[1] + per_warp - 1) / per_warp;
        auto fetch = [&](int round) {
            Item it;
            it.what = round >= rounds_q;
            const int H = a.heads[it.what], i = (round - (it.what ? rounds_q : 0)) * per_warp + sub;
            it.real = i < n * H;
            it.r = it.real ? (H == 1 ? i : (int)__umulhi((uint32_t)i, a.inverse[it.what])) : 0;
            const long long row = r0 + it.r, col = (long long)(it.real ? i - it.r * H : 0) * a.d;
            const T *px = reinterpret_cast<const T *>(a.x[it.what]) + row * a.ldx[it.what] + col;
            const T *pd = reinterpret_cast<const T *>(a.dy[it.what]) + row * a.ldy[it.what] + col;
            it.at = row * (BACK ? a.ldx[it.what] : a.ldy[it.what]) + col;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                it.x[g][0] = it.x[g][1] = raw_t<T, W>();
                if (BACK)
                    it.dy[BACK ? g : 0][0] = it.dy[BACK ? g : 0][1] = raw_t<T, W>();
                if (it.real && mine[g]) {
                    it.x[g][0] = *reinterpret_cast<const raw_t<T, W> *>(px + lo[g]);
                    it.x[g][1] = *reinterpret_cast<const raw_t<T, W> *>(px + hi[g]);
                    if (BACK) {
                        it.dy[BACK ? g : 0][0] = *reinterpret_cast<const raw_t<T, W> *>(pd + lo[g]);
                        it.dy[BACK ? g : 0][1] = *reinterpret_cast<const raw_t<T, W> *>(pd + hi[g]);
                    }
                }
            }
            return it;
        };
        Item next = {};
        if (warp < rounds)
            next = fetch(warp);
        __syncthreads();
        angles(a, cs, live, r0, n, tid);
        __syncthreads();
#pragma unroll 1
        for (int round = warp; round < rounds; round += 8) { // all lanes of a warp go through every round (shuffles)
            const Item it = next;
            if (round + 8 < rounds)
                next = fetch(round + 8);
            const bool alive = it.real && live[it.r];
            const float *gain = gains + it.what * a.d;
            const float2 *turns = cs + it.r * half;
            float x[NG][2][W], u[NG][2][W];
            float sq = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    take<T, W>(x[g][j], it.x[g][j]);
                    if (BACK)
                        take<T, W>(u[g][j], it.dy[BACK ? g : 0][j]);
                    if (!alive) // padding: zeros, whatever lies there
#pragma unroll
                        for (int k = 0; k < W; k++)
                            x[g][j][k] = u[g][j][k] = 0.0f;
#pragma unroll
                    for (int k = 0; k < W; k++)
                        sq += x[g][j][k] * x[g][j][k];
                }
            for (int o = G / 2; o > 0; o >>= 1)
                sq += __shfl_xor_sync(0xffffffffu, sq, o);
            const float rs = alive ? rsqrtf(sq * inv_d + a.eps) : 0.0f;
            if (!BACK) {
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    if (!mine[g])
                        continue;
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int k = 0; k < W; k++)
                            u[g][j][k] = x[g][j][k] * rs * gain[(j ? hi[g] : lo[g]) + k];
                    if (p0[g] < half)
                        turn<W>(u[g], turns + p0[g], a.adjacent, 1.0f);
                }
            } else {
                float dot = 0.0f;
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    if (!mine[g])
                        continue;
                    if (p0[g] < half)
                        turn<W>(u[g], turns + p0[g], a.adjacent, -1.0f);
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int k = 0; k < W; k++) {
                            x[g][j][k] *= rs;
                            const float ux = u[g][j][k] * x[g][j][k];
                            acc[0][g][j][k] += it.what ? 0.0f : ux;
                            acc[BACK ? 1 : 0][g][j][k] += it.what ? ux : 0.0f;
                            u[g][j][k] *= gain[(j ? hi[g] : lo[g]) + k];
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
            T *py = reinterpret_cast<T *>(a.y[it.what]) + it.at;
#pragma unroll
            for (int g = 0; g < NG; g++)
                if (it.real && mine[g]) {
                    *reinterpret_cast<raw_t<T, W> *>(py + lo[g]) = alive ? put<T, W>(u[g][0]) : raw_t<T, W>();
                    *reinterpret_cast<raw_t<T, W> *>(py + hi[g]) = alive ? put<T, W>(u[g][1]) : raw_t<T, W>();
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

// dgain of queries and keys: the CTAs' sums, eight columns a CTA, 32 strands in a fixed order
__global__ void __launch_bounds__(256) gain_kernel(const float *__restrict__ part, int n_parts, int d, float *dgain_q, float *dgain_k)
{
    __shared__ float red[32][9];
    const int x = threadIdx.x & 7, strand = threadIdx.x >> 3, col = blockIdx.x * 8 + x;
    pdl_wait();
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (col < 2 * d)
        for (int i = strand; i < n_parts; i += 128)
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + 32 * k < n_parts)
                    s[k] += part[(size_t)(i + 32 * k) * 2 * d + col];
    red[strand][x] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (strand == 0 && col < 2 * d) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; k++)
            sum += red[k][x];
        float *to = col < d ? dgain_q : dgain_k;
        if (to)
            to[col < d ? col : col - d] = sum;
    }
}

} // namespace qkn
