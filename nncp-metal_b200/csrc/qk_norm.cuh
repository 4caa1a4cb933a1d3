// qk_norm.cuh -- queries and keys normed for each head and rotated by their positions in one pass.
//
//   x^ = x / sqrt(mean(x^2) + eps),  n = x^ gain,  y = R(pos) n
//
// R turns the pairs (i, i + d_rot / 2) -- or (2i, 2i + 1) -- of the first d_rot values by pos base^(-2i / d_rot).  The
// adjoint turns back: u = R(-pos) dy, dgain = sum u x^, w = u gain, dx = (w - x^ mean(w x^)) / sqrt(mean(x^2) + eps).
//
// The bytes are every value once in and once out (forward), twice in and once out (backward).  A head's row lies in
// the registers of G neighbouring lanes, each with both members of its pairs, so that neither the rotation nor a
// second look at x costs memory; sines and cosines are taken once for a row and all its heads.  Angles are
// reduced in 64 bits: positions of a large file leave no digit of an fp32 angle behind the point.
//
// Bound by the issue of instructions, some 20 for a value and pass, and by the waits for shared memory and shuffles between
// them: 16384 rows of 16 + 16 heads of 64, bf16, forward 29.8 us (134 MB, 4.5 TB/s), backward with gains 47.4 (201 MB, 4.2).
// Gains and angles as they come, four lanes to a bank, took 33.2 and 48.3.
#pragma once
#include "warp_mma.cuh"

namespace qkn {

constexpr int DIM_MAX = NNCU_QK_NORM_DIM_MAX;
constexpr int ROWS_MAX = 32; // rows of a CTA at a time

struct Args {
    const void *x[2];    // queries, keys
    const void *dy[2];   // gradients of the results
    void *y[2];          // results, or gradients of x
    const float *gain[2];
    const int32_t *pos;  // of each row; below 0: the row is padding
    float *part;         // [grid][2][d] partial sums of dgain
    int ldx[2], ldy[2];
    int heads[2];
    uint32_t inverse[2]; // ceil(2^32 / heads); 0 for one head
    int N, d, rot, lanes, rows_per; // lanes: of a head (a power of two)
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
    if constexpr (sizeof(T) == 2 && W > 1) {
        const uint32_t *p = reinterpret_cast<const uint32_t *>(&u);
#pragma unroll
        for (int i = 0; i < W; i += 2) {
            v[i] = __uint_as_float(p[i / 2] << 16);
            v[i + 1] = __uint_as_float(p[i / 2] & 0xffff0000u);
        }
    } else {
        const T *p = reinterpret_cast<const T *>(&u);
#pragma unroll
        for (int i = 0; i < W; i++)
            v[i] = to_f(p[i]);
    }
}
template <typename T, int W> __device__ __forceinline__ raw_t<T, W> put(const float (&v)[W])
{
    raw_t<T, W> u;
    if constexpr (sizeof(T) == 2 && W > 1) {
        uint32_t *p = reinterpret_cast<uint32_t *>(&u);
#pragma unroll
        for (int i = 0; i < W; i += 2)
            p[i / 2] = fa::pack2(v[i], v[i + 1]);
    } else {
        T *p = reinterpret_cast<T *>(&u);
#pragma unroll
        for (int i = 0; i < W; i++)
            p[i] = from_f<T>(v[i]);
    }
    return u;
}

// Where a lane's pairs p0 .. p0 + W - 1 lie in a head's row: two runs of W values.  Pairs behind the rotated ones are
// halves of what is left, or neighbours too.
template <int W, bool ADJACENT> struct Place {
    int lo, hi;
    __device__ __forceinline__ Place(const Args &a, int p0)
    {
        if (ADJACENT) {
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

// A lane's N floats of shared memory; four at a time where they lie so, `apart` floats from four to four: the lanes' fours
// stand side by side, and a warp's read touches each bank once
template <int N, bool QUADS> __device__ __forceinline__ void floats(float (&v)[N], const float *p, int apart)
{
    if constexpr (QUADS) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(p + i / 4 * apart);
            v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            v[i] = p[i];
    }
}

// Where pair p's angle lies among a row's, n lanes of W pairs: two pairs of each lane, then the next two
template <int W> __device__ __forceinline__ int angle_at(int p, int n)
{
    const int k = p % W;
    return W < 2 ? p : (k / 2 * n + p / W) * 2 + k % 2;
}

// the W pairs of a lane turned by the angles at cs (cosine, sine); TO: +1 there, -1 back.  x[0], x[1]: the two runs
template <int W, int TO, bool ADJACENT> __device__ __forceinline__ void turn(float (&x)[2][W], const float2 *cs, int n)
{
    float at[2 * W];
    floats<2 * W, (W >= 2)>(at, reinterpret_cast<const float *>(cs), 4 * n);
    if constexpr (ADJACENT) { // pair k: values 2k, 2k + 1 of both runs in a row
#pragma unroll
        for (int k = 0; k < W; k++) {
            const float c = at[2 * k], s = TO * at[2 * k + 1];
            float &a = x[2 * k / W][2 * k % W], &b = x[(2 * k + 1) / W][(2 * k + 1) % W];
            const float u = a * c - b * s;
            b = b * c + a * s;
            a = u;
        }
    } else {
#pragma unroll
        for (int k = 0; k < W; k++) {
            const float c = at[2 * k], s = TO * at[2 * k + 1], u = x[0][k] * c - x[1][k] * s;
            x[1][k] = x[1][k] * c + x[0][k] * s;
            x[0][k] = u;
        }
    }
}

// Cosines and sines of rows r0 .. r0 + n - 1, [n][d / 2] (one and zero for pairs that are only normed), and which of them
// are no padding
template <int W> __device__ __forceinline__ void angles(const Args &a, float2 *cs, int *live, int r0, int n, int tid)
{
    const int half = a.d / 2;
    for (int i = tid; i < n * half; i += 256) {
        const int r = i / half, p = i - r * half;
        float s = 0.0f, c = 1.0f;
        if (2 * p < a.rot) {
            const double t = (double)a.pos[r0 + r] * a.turns[p];
            sincospif((float)(2.0 * (t - rint(t))), &s, &c);
        }
        cs[r * half + angle_at<W>(p, half / W)] = make_float2(c, s);
    }
    if (tid < n)
        live[tid] = !a.pos || a.pos[r0 + tid] >= 0;
}

// CTAs of blockIdx.y 0 take queries, of 1 keys.  A warp takes 32 / lanes heads of neighbouring places at a time; the next
// ones are on their way while it computes, the first while the angles are taken.  A lane has NG groups of W pairs, a
// group's neighbours in the neighbouring lanes.
template <typename T, int W, int NG, bool ADJACENT, bool BACK>
__global__ void __launch_bounds__(256, BACK ? 2 : 4) kernel(const __grid_constant__ Args a)
{
    extern __shared__ __align__(16) float sh[];
    __shared__ int live[ROWS_MAX];
    float2 *cs = reinterpret_cast<float2 *>(sh);
    float *gain = sh + a.rows_per * a.d, *red = gain + a.d; // backward: red [8 warps][d]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.lanes, per_warp = 32 / G, sub = lane / G;
    const int what = blockIdx.y, H = a.heads[what], ldx = a.ldx[what], ldy = a.ldy[what], half = a.d / 2;
    const uint32_t inverse = a.inverse[what];
    const T *gx = reinterpret_cast<const T *>(a.x[what]), *gd = reinterpret_cast<const T *>(a.dy[what]);
    T *gy = reinterpret_cast<T *>(a.y[what]);
    int p0[NG], lo[NG], hi[NG];
    bool mine[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
        p0[g] = ((lane & (G - 1)) + g * G) * W;
        mine[g] = p0[g] < half;
        const Place<W, ADJACENT> at(a, mine[g] ? p0[g] : 0);
        lo[g] = at.lo;
        hi[g] = at.hi;
    }
    const float inv_d = 1.0f / (float)a.d;
    pdl_wait();
    const int n_lanes = half / W;
    if (tid < G) // runs one behind the other; in each the lanes' first fours, then their second fours
#pragma unroll
        for (int g = 0; g < NG; g++)
            if (mine[g])
#pragma unroll
                for (int k = 0; k < W; k++) {
                    const int to = W < 4 ? p0[g] + k : (k / 4 * n_lanes + p0[g] / W) * 4 + k % 4;
                    gain[to] = a.gain[what] ? a.gain[what][lo[g] + k] : 1.0f;
                    gain[half + to] = a.gain[what] ? a.gain[what][hi[g] + k] : 1.0f;
                }
    float acc[NG][2][W] = {};
    struct Item {
        raw_t<T, W> x[NG][2], dy[BACK ? NG : 1][2];
        long long at; // where the result goes
        int r;
        bool real;
    };
    for (int r0 = blockIdx.x * a.rows_per; r0 < a.N; r0 += gridDim.x * a.rows_per) {
        const int n = min(a.rows_per, a.N - r0), heads = n * H;
        auto fetch = [&](int i0) {
            Item it;
            const int i = i0 + sub;
            it.real = i < heads;
            it.r = !it.real ? 0 : H == 1 ? i : (int)__umulhi((uint32_t)i, inverse);
            const int col = it.real ? (i - it.r * H) * a.d : 0;
            const long long atx = (long long)(r0 + it.r) * ldx + col, aty = (long long)(r0 + it.r) * ldy + col;
            it.at = BACK ? atx : aty;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                it.x[g][0] = it.x[g][1] = raw_t<T, W>();
                if (BACK)
                    it.dy[BACK ? g : 0][0] = it.dy[BACK ? g : 0][1] = raw_t<T, W>();
                if (it.real && mine[g]) {
                    it.x[g][0] = *reinterpret_cast<const raw_t<T, W> *>(gx + atx + lo[g]);
                    it.x[g][1] = *reinterpret_cast<const raw_t<T, W> *>(gx + atx + hi[g]);
                    if (BACK) {
                        it.dy[BACK ? g : 0][0] = *reinterpret_cast<const raw_t<T, W> *>(gd + aty + lo[g]);
                        it.dy[BACK ? g : 0][1] = *reinterpret_cast<const raw_t<T, W> *>(gd + aty + hi[g]);
                    }
                }
            }
            return it;
        };
        Item next = {};
        if (warp * per_warp < heads)
            next = fetch(warp * per_warp);
        __syncthreads();
        angles<W>(a, cs, live, r0, n, tid);
        __syncthreads();
#pragma unroll 1
        for (int i0 = warp * per_warp; i0 < heads; i0 += 8 * per_warp) { // all lanes of a warp go through every round (shuffles)
            Item it = next;
            if (i0 + 8 * per_warp < heads)
                next = fetch(i0 + 8 * per_warp);
            const bool alive = it.real && live[it.r]; // lanes without a head add nothing to dgain: no root of their zeros is taken
            const bool all_alive = __all_sync(0xffffffffu, alive);
            if (!all_alive && !alive) // padding: zeros, whatever lies there
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    it.x[g][0] = it.x[g][1] = raw_t<T, W>();
                    if (BACK)
                        it.dy[BACK ? g : 0][0] = it.dy[BACK ? g : 0][1] = raw_t<T, W>();
                }
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
#pragma unroll
                    for (int k = 0; k < W; k++)
                        sq += x[g][j][k] * x[g][j][k];
                }
            for (int o = G / 2; o > 0; o >>= 1)
                sq += __shfl_xor_sync(0xffffffffu, sq, o);
            const float rs = alive ? rsqrtf(sq * inv_d + a.eps) : 0.0f;
            float dot = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                if (NG > 1 && !mine[g])
                    continue;
                const int p = mine[g] ? p0[g] : 0;
                if (BACK)
                    turn<W, -1, ADJACENT>(u[g], turns + (W < 2 ? p : p / W * 2), n_lanes);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float by[W];
                    floats<W, (W >= 4)>(by, gain + j * half + (W < 4 ? p : p / W * 4), 4 * n_lanes);
#pragma unroll
                    for (int k = 0; k < W; k++) {
                        x[g][j][k] *= rs;
                        if (BACK) {
                            acc[g][j][k] = fmaf(u[g][j][k], x[g][j][k], acc[g][j][k]);
                            u[g][j][k] *= by[k];
                            dot = fmaf(u[g][j][k], x[g][j][k], dot);
                        } else {
                            u[g][j][k] = x[g][j][k] * by[k];
                        }
                    }
                }
                if (!BACK)
                    turn<W, 1, ADJACENT>(u[g], turns + (W < 2 ? p : p / W * 2), n_lanes);
            }
            if (BACK) {
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
            T *py = gy + it.at;
#pragma unroll
            for (int g = 0; g < NG; g++)
                if (it.real && mine[g]) {
                    raw_t<T, W> out[2] = {put<T, W>(u[g][0]), put<T, W>(u[g][1])};
                    if (!all_alive && !alive)
                        out[0] = out[1] = raw_t<T, W>();
                    *reinterpret_cast<raw_t<T, W> *>(py + lo[g]) = out[0];
                    *reinterpret_cast<raw_t<T, W> *>(py + hi[g]) = out[1];
                }
        }
    }
    if (BACK && a.part) {
        // the CTA's sums: lanes of the same pairs, then warps in order
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int k = 0; k < W; k++) {
                    float s = acc[g][j][k];
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

// dgain of queries and keys: the CTAs' sums, eight columns a CTA, 32 strands in a fixed order
__global__ void __launch_bounds__(256) gain_kernel(const float *__restrict__ part, int n_parts, int d, float *dgain_q, float *dgain_k)
{
    __shared__ float red[32][9];
    const int x = threadIdx.x & 7, strand = threadIdx.x >> 3, col = blockIdx.x * 8 + x;
    const bool wanted = col < 2 * d && (col < d ? dgain_q : dgain_k);
    pdl_wait();
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (wanted)
        for (int i = strand; i < n_parts; i += 128)
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + 32 * k < n_parts)
                    s[k] += part[(size_t)(i + 32 * k) * 2 * d + col];
    red[strand][x] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (strand == 0 && wanted) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; k++)
            sum += red[k][x];
        (col < d ? dgain_q : dgain_k)[col < d ? col : col - d] = sum;
    }
}

} // namespace qkn
