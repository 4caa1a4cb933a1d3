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
#include <type_traits>

#include "copy_ring.h"
#include "gemm_tc.cuh"
#include "warp_mma.cuh"

namespace lin {

constexpr int HEADS_MAX = NNCU_LINEAR_ATTN_HEADS_MAX;
constexpr int DIM_MAX = NNCU_LINEAR_ATTN_DIM_MAX;

// one set of rows and its state
struct Role {
    const void *a, *b, *c;
    void *o;
    const float *s0;     // state before the first token, [B][H][da][dc] or, where s0_t, [B][H][dc][da]; NULL: zeros
    float *s_end;        // state behind the last token, [B][H][da][dc]; NULL: not wanted
    float *parts;        // [B*H][n_seg + 1][slot]: slot 0 the state before the first token, slot g what part g - 1 adds up to
    const void *a2;      // not NULL: a second result of the same rows and state (kernels of two results)
    void *o2;
    long long lda, ldb, ldc, ldo, lda2, ldo2; // elements from row to row
    int da, dc, reverse, s0_t, e1, e2;
    float s_state, s_pair, s_in;
};

struct Args {
    Role role[3];        // blockIdx.z says which
    const int32_t *len;  // tokens of each stream; NULL: T
    int B, H, T;
    int n_seg;           // parts a stream's tokens are cut into
    int seg;             // tokens in a part
    int slot;            // floats of a state in parts
    float rate[HEADS_MAX]; // log2 of each head's decay
    float decay[HEADS_MAX];
};

// l^n; l^0 is 1 whatever l
__device__ __forceinline__ float power(float rate, int n) { return exp2f(rate * (float)n); }

// Where a stream's token u (counted in the kernel's order) lies, and how many there are
struct Rows {
    long long first, step; // rows
    int n;
    __device__ __forceinline__ Rows(const Args &p, const Role &q, int b)
    {
        n = p.len ? min(max(p.len[b], 0), p.T) : p.T;
        step = q.reverse ? -(long long)p.B : p.B;
        first = (q.reverse ? (long long)(n - 1) * p.B : 0) + b;
    }
    __device__ __forceinline__ long long row(int u) const { return first + step * u; }
};

// rows of the result behind a stream's end are zeros: those of them that part g is to write, a warp a row
template <typename T>
__device__ __forceinline__ void zero_behind(const Args &p, void *out, long long ldo, int d, const Rows &rows, int b, int h, int g, int warp,
                                            int warps, int lane)
{
    const int hi = g == p.n_seg - 1 ? p.T : min(p.T, (g + 1) * p.seg);
    for (int t = max(rows.n, g * p.seg) + warp; t < hi; t += warps) {
        T *o = reinterpret_cast<T *>(out) + ((long long)t * p.B + b) * ldo + (size_t)h * d;
        for (int i = lane; i < d; i += 32)
            o[i] = from_f<T>(0.0f);
    }
}

__device__ __forceinline__ float state_at(const Role &q, const float *s, int i, int c)
{
    return q.s0_t ? s[(size_t)c * q.da + i] : s[(size_t)i * q.dc + c];
}

// Whether the last token of a stream of n is in part g: the state behind it is the stream's.  A stream without tokens
// ends in part 0.
__device__ __forceinline__ bool ends_in(const Args &p, int n, int g) { return g * p.seg < max(n, 1) && max(n, 1) <= g * p.seg + p.seg; }

// ---------------- CUDA cores: rows that are not laid out in 16-byte pieces ----------------
//
// A CTA of 256 threads goes through one part of one (stream, head) in chunks of 32 tokens; tiles and state are fp32 in
// shared memory, a thread takes 2 x 2 pair weights and 4 x 4 results or 8 x 4 elements of the state at a time.  Bound by
// latency: values come one by one, and a chunk is loaded before it is computed.  8 x 8 pairs of 512 tokens of 62, fp32,
// forward: 91 us.

constexpr int FC = 32; // tokens in a chunk

struct CoreSmem {
    int da4, dc4, ld_a, ld_c, tile, b, c, s, p, w, floats;
    __host__ __device__ CoreSmem(int da, int dc)
    {
        da4 = (da + 3) & ~3; dc4 = (dc + 3) & ~3;
        ld_a = da4 + 4; ld_c = dc4 + 4; // rows four banks on
        b = FC * ld_a; c = b + FC * ld_a; tile = c + FC * ld_c;
        s = tile; p = s + da4 * ld_c; w = p + FC * (FC + 4);
        floats = w + 2 * (FC + 2);
    }
};

// 32 rows of a matrix as a tile, zeros behind row n and column d
template <typename T>
__device__ __forceinline__ void core_load(float *dst, int ld, int d4, int d, const void *src, long long ldr, int h, const Rows &rows, int u0, int n)
{
    const T *base = reinterpret_cast<const T *>(src) + (size_t)h * d;
    for (int i = threadIdx.x; i < FC * d4; i += 256) {
        const int r = i / d4, x = i - r * d4;
        dst[r * ld + x] = r < n && x < d ? to_f(base[rows.row(u0 + r) * ldr + x]) : 0.0f;
    }
}

__device__ __forceinline__ float4 quad(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ void add4(float4 &s, float u, const float4 &v)
{
    s.x = fmaf(u, v.x, s.x); s.y = fmaf(u, v.y, s.y); s.z = fmaf(u, v.z, s.z); s.w = fmaf(u, v.w, s.w);
}
__device__ __forceinline__ float dot4(const float4 &u, const float4 &v, float s)
{
    return fmaf(u.x, v.x, fmaf(u.y, v.y, fmaf(u.z, v.z, fmaf(u.w, v.w, s))));
}

// STATES: the first pass over a sequence in several parts: what each part but the last adds to the state
template <typename T, bool STATES>
__global__ void __launch_bounds__(256) core_kernel(const __grid_constant__ Args p)
{
    extern __shared__ __align__(16) float smf[];
    const Role &q = p.role[blockIdx.z];
    const CoreSmem sm(q.da, q.dc);
    float *Ss = smf + sm.s, *Ps = smf + sm.p, *pw = smf + sm.w, *wt = pw + FC + 2;
    constexpr int LP = FC + 4;
    const int tid = threadIdx.x;
    const size_t pair = blockIdx.x;
    const int g = blockIdx.y, b = (int)(pair / p.H), h = (int)(pair % p.H);
    const float rate = p.rate[h];
    pdl_wait();
    const Rows rows(p, q, b);
    const size_t nn = (size_t)q.da * q.dc;
    const int begin = g * p.seg, end = min(rows.n, begin + p.seg);
    float *As = smf, *Bs = As + sm.b, *Cs = As + sm.c;
    const float l_seg = power(rate, p.seg);
    for (int i = tid; i < FC + 2; i += 256)
        pw[i] = power(rate, i);
    const int c4 = sm.dc4 / 4;
    for (int i = tid; i < sm.da4 * sm.dc4; i += 256) {
        const int x = i / sm.dc4, y = i - x * sm.dc4;
        float s = 0.0f;
        if (x < q.da && y < q.dc) {
            float *part = q.parts + pair * (p.n_seg + 1) * p.slot + (size_t)x * q.dc + y;
            const float first = q.s0 && (p.n_seg == 1 || (STATES && g == 0)) ? state_at(q, q.s0 + pair * nn, x, y) : 0.0f;
            if (STATES && g == 0) // the state before the first token is kept: s_end may lie where it lies
                *part = first;
            if (!STATES) {
                s = p.n_seg == 1 ? first : part[0];
                for (int k = 1; k <= g; k++)
                    s = fmaf(l_seg, s, part[(size_t)k * p.slot]);
            }
        }
        Ss[x * sm.ld_c + y] = s;
    }
    if (!STATES)
        zero_behind<T>(p, q.o, q.ldo, q.dc, rows, b, h, g, tid >> 5, 8, tid & 31);
    for (int u0 = begin; u0 < end; u0 += FC) {
        const int n = min(FC, end - u0);
        __syncthreads(); // the chunk before has been read
        if (!STATES)
            core_load<T>(As, sm.ld_a, sm.da4, q.da, q.a, q.lda, h, rows, u0, n);
        core_load<T>(Bs, sm.ld_a, sm.da4, q.da, q.b, q.ldb, h, rows, u0, n);
        core_load<T>(Cs, sm.ld_c, sm.dc4, q.dc, q.c, q.ldc, h, rows, u0, n);
        __syncthreads();
        if (tid < FC)
            wt[tid] = tid < n ? q.s_in * pw[n - 1 - tid + q.e2] : 0.0f;
        if (!STATES) {
            {
                const int i0 = tid / 16, j0 = tid % 16; // rows i0, i0 + 16, keys j0, j0 + 16
                float w[2][2] = {};
                for (int x = 0; x < sm.da4; x += 4) {
                    const float4 a0 = quad(As + i0 * sm.ld_a + x), a1 = quad(As + (i0 + 16) * sm.ld_a + x);
                    const float4 b0 = quad(Bs + j0 * sm.ld_a + x), b1 = quad(Bs + (j0 + 16) * sm.ld_a + x);
                    w[0][0] = dot4(a0, b0, w[0][0]);
                    w[1][0] = dot4(a1, b0, w[1][0]);
                    w[1][1] = dot4(a1, b1, w[1][1]);
                }
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int v = 0; v < 2; v++) {
                        const int i = i0 + 16 * u, j = j0 + 16 * v;
                        Ps[i * LP + j] = j <= i ? w[u][v] * q.s_pair * pw[i - j] : 0.0f;
                    }
            }
            __syncthreads();
            constexpr int R = 4;
            for (int it = tid; it < FC / R * c4; it += 256) {
                const int i0 = it / c4 * R, c0 = (it - it / c4 * c4) * 4;
                float4 o[R];
#pragma unroll
                for (int r = 0; r < R; r++)
                    o[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                // four columns of the R rows at u against four rows of four columns at v
                auto product = [&](const float *u, int ldu, const float *v) {
                    const float4 v0 = quad(v), v1 = quad(v + sm.ld_c), v2 = quad(v + 2 * sm.ld_c), v3 = quad(v + 3 * sm.ld_c);
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        const float4 w = quad(u + r * ldu);
                        add4(o[r], w.x, v0); add4(o[r], w.y, v1); add4(o[r], w.z, v2); add4(o[r], w.w, v3);
                    }
                };
                for (int x = 0; x < sm.da4; x += 4)
                    product(As + i0 * sm.ld_a + x, sm.ld_a, Ss + x * sm.ld_c + c0);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const float f = q.s_state * pw[i0 + r + q.e1];
                    o[r].x *= f; o[r].y *= f; o[r].z *= f; o[r].w *= f;
                }
                for (int j = 0; j < min(i0 + R, n); j += 4) // weights behind the row are zeros, and so are rows behind the last
                    product(Ps + i0 * LP + j, LP, Cs + j * sm.ld_c + c0);
#pragma unroll
                for (int r = 0; r < R; r++)
                    if (i0 + r < n) {
                        T *to = reinterpret_cast<T *>(q.o) + rows.row(u0 + i0 + r) * q.ldo + (size_t)h * q.dc + c0;
                        const float v[4] = {o[r].x, o[r].y, o[r].z, o[r].w};
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            if (c0 + c < q.dc)
                                to[c] = from_f<T>(v[c]);
                    }
            }
        }
        __syncthreads(); // the state has been read, the weights stand
        if (!STATES && u0 + FC >= end && !q.s_end)
            break;
        const float l_n = pw[n];
        // R rows of the state at a time, eight where that leaves work for every thread
        auto carry = [&](auto size) {
            constexpr int R = decltype(size)::value;
            for (int it = tid; it < sm.da4 / R * c4; it += 256) {
                const int x0 = it / c4 * R, c0 = (it - it / c4 * c4) * 4;
                float4 add[R];
#pragma unroll
                for (int r = 0; r < R; r++)
                    add[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                for (int j = 0; j < n; j++) {
                    const float4 v = quad(Cs + j * sm.ld_c + c0);
                    const float w = wt[j];
#pragma unroll
                    for (int r = 0; r < R; r += 4) {
                        const float4 u = quad(Bs + j * sm.ld_a + x0 + r);
                        add4(add[r], w * u.x, v); add4(add[r + 1], w * u.y, v);
                        add4(add[r + 2], w * u.z, v); add4(add[r + 3], w * u.w, v);
                    }
                }
#pragma unroll
                for (int r = 0; r < R; r++) {
                    float4 *s = reinterpret_cast<float4 *>(Ss + (x0 + r) * sm.ld_c + c0);
                    float4 now = *s;
                    now.x = fmaf(l_n, now.x, add[r].x); now.y = fmaf(l_n, now.y, add[r].y);
                    now.z = fmaf(l_n, now.z, add[r].z); now.w = fmaf(l_n, now.w, add[r].w);
                    *s = now;
                }
            }
        };
        if (sm.da4 % 8 == 0 && sm.da4 / 8 * c4 >= 256)
            carry(std::integral_constant<int, 8>());
        else
            carry(std::integral_constant<int, 4>());
    }
    __syncthreads();
    float *to = STATES ? q.parts + (pair * (p.n_seg + 1) + g + 1) * p.slot : (q.s_end && ends_in(p, rows.n, g) ? q.s_end + pair * nn : nullptr);
    if (to)
        for (int i = tid; i < q.da * q.dc; i += 256)
            to[i] = Ss[i / q.dc * sm.ld_c + i % q.dc];
}

// ---------------- fp32 on warp-level tensor-core products ----------------
//
// A CTA goes through one part of one (stream, head) in chunks of 32 tokens, rows in 16-byte pieces copied asynchronously, the
// next chunk's under the present one.  An fp32 value is two tf32 values of 11 bits and a rest of 2^-22 of it at most; a
// product of two takes three tf32 products (high by high in one sum, the mixed ones in another), the fourth is below 2^-22 too.
// Each warp has sixteen columns of the results and of the state, so that a split left factor serves four products of tiles.  The
// state stays in shared memory in fp32: what a chunk adds to it has sums of its own, since products cut the sum that they
// are added to.
//
// Tiles [token][value] lie with rows four banks on where products take them by rows (a, b) and eight banks on where by
// columns (c, the state): a fragment's 32 words touch 32 banks.  Only b as the state's left factor goes two to a bank.
//
// Bound by the chain of a chunk's phases: of 14800 cycles at head size 128 the products take 7600 at the rate that this
// instruction reaches (277 TFLOP/s), the pair weights, which three warps compute, 3500, the next rows' copies 1200.
// 8 x 8 pairs of 512 tokens of 64, forward: 37.5 us (on CUDA cores 70.6), with the backward pass 118 (257); 4 x 8 of
// 1024 tokens of 128: 105 (228) and 371 (673).  Bulk copies of a row each instead of 16 bytes a thread: 57 us for 37.5.

struct QuadSmem {
    int da16, dc16, ld_a, ld_c, tile, b, c, s, p, w, floats;
    __host__ __device__ QuadSmem(int da, int dc)
    {
        da16 = (da + 15) & ~15; dc16 = (dc + 15) & ~15;
        ld_a = da16 + 4; ld_c = dc16 + 8;
        b = FC * ld_a; c = b + FC * ld_a; tile = c + FC * ld_c;
        s = 2 * tile; p = s + da16 * ld_c; w = p + FC * (FC + 4);
        floats = w + FC + 4;
    }
};

// This thread's fours of a matrix that all threads of a CTA go through: column x of rows r, r + step, ...
struct Fours {
    int r, x, step;
    __device__ __forceinline__ explicit Fours(int columns)
    {
        const int n = columns / 4;
        step = blockDim.x / n;
        r = threadIdx.x / n;
        x = (threadIdx.x - r * n) * 4;
        if (r >= step) // threads of no whole row
            r = 1 << 30;
    }
};

// 32 rows of a matrix as a tile, zeros behind row n and column d
__device__ __forceinline__ void quad_load(float *dst, int ld, const Fours &f, int d, const void *src, long long ldr, int h, const Rows &rows, int u0, int n)
{
    if (f.r >= FC)
        return;
    const float *base = reinterpret_cast<const float *>(src) + (size_t)h * d + (f.x < d ? f.x : 0), *from = base + rows.row(u0 + f.r) * ldr;
    const long long step = f.step * rows.step * ldr;
    for (int r = f.r; r < FC; r += f.step, from += step)
        fa::cp16(dst + r * ld + f.x, r < n ? from : base, r < n && f.x < d);
}

struct Two {
    uint32_t hi, lo;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ explicit Two(float x)
    {
        hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u; // to the nearest: halves go up
        lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
    }
};
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 x 16 sums, column groups x = 0, 1
struct Sums {
    float big[2][4], small[2][4];
    __device__ __forceinline__ Sums()
    {
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                big[x][c] = small[x][c] = 0.0f;
    }
    __device__ __forceinline__ void add(const Two (&a)[4], const Two (&b)[2][2])
    {
#pragma unroll
        for (int x = 0; x < 2; x++)
            mma_tf32(small[x], a[0].lo, a[1].lo, a[2].lo, a[3].lo, b[x][0].hi, b[x][1].hi);
#pragma unroll
        for (int x = 0; x < 2; x++)
            mma_tf32(big[x], a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[x][0].hi, b[x][1].hi);
#pragma unroll
        for (int x = 0; x < 2; x++)
            mma_tf32(small[x], a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[x][0].lo, b[x][1].lo);
    }
    __device__ __forceinline__ float sum(int x, int c) const { return big[x][c] + small[x][c]; }
};
// fragments: at is this lane's first value; `row` and `k` go from row (column) to row and from one contracted place to the next
__device__ __forceinline__ void left16(Two (&a)[4], const float *at, int row, int k)
{
    a[0] = Two(at[0]);
    a[1] = Two(at[8 * row]);
    a[2] = Two(at[4 * k]);
    a[3] = Two(at[8 * row + 4 * k]);
}
__device__ __forceinline__ void right16(Two (&b)[2][2], const float *at, int column, int k)
{
#pragma unroll
    for (int x = 0; x < 2; x++) {
        b[x][0] = Two(at[8 * x * column]);
        b[x][1] = Two(at[8 * x * column + 4 * k]);
    }
}

// A warp for each sixteen columns of c.  Parts hold states as [da16][dc16].
template <bool STATES> __global__ void __launch_bounds__(256) quad_kernel(const __grid_constant__ Args p)
{
    extern __shared__ __align__(16) float smf[];
    const Role &q = p.role[blockIdx.z];
    const QuadSmem sm(q.da, q.dc);
    float *Ss = smf + sm.s, *Ps = smf + sm.p, *pw = smf + sm.w;
    constexpr int LP = FC + 4;
    const int tid = threadIdx.x, thr = blockDim.x, warp = tid >> 5, lane = tid & 31, g4 = lane >> 2, t = lane & 3, y0 = 16 * warp;
    const size_t pair = blockIdx.x;
    const int g = blockIdx.y, b = (int)(pair / p.H), h = (int)(pair % p.H);
    const float rate = p.rate[h];
    const int a_steps = (q.da + 7) / 8;
    const Fours fours_a(sm.da16), fours_c(sm.dc16);
    pdl_wait();
    const Rows rows(p, q, b);
    const size_t nn = (size_t)q.da * q.dc;
    const int begin = g * p.seg, end = min(rows.n, begin + p.seg);
    auto fetch = [&](int u0, float *to) {
        const int n = end - u0;
        if (!STATES)
            quad_load(to, sm.ld_a, fours_a, q.da, q.a, q.lda, h, rows, u0, n);
        quad_load(to + sm.b, sm.ld_a, fours_a, q.da, q.b, q.ldb, h, rows, u0, n);
        quad_load(to + sm.c, sm.ld_c, fours_c, q.dc, q.c, q.ldc, h, rows, u0, n);
        fa::cp_commit();
    };
    if (begin < end)
        fetch(begin, smf);
    const float l_seg = power(rate, p.seg);
    for (int i = tid; i < FC + 2; i += thr)
        pw[i] = power(rate, i);
    // the state before this part, several rows at a time on their way
    float *parts = p.n_seg > 1 ? q.parts + pair * (p.n_seg + 1) * p.slot : nullptr;
    constexpr int WAY = 8;
    for (int x0 = fours_c.r; x0 < sm.da16; x0 += WAY * fours_c.step) {
        float4 s[WAY];
#pragma unroll
        for (int i = 0; i < WAY; i++) {
            const int x = x0 + i * fours_c.step;
            s[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (q.s0 && (p.n_seg == 1 || (STATES && g == 0)) && x < q.da && fours_c.x < q.dc) {
                const float *s0 = q.s0 + pair * nn;
                s[i] = make_float4(state_at(q, s0, x, fours_c.x), state_at(q, s0, x, fours_c.x + 1), state_at(q, s0, x, fours_c.x + 2),
                                   state_at(q, s0, x, fours_c.x + 3));
            }
        }
        if (p.n_seg > 1 && (!STATES || g == 0))
            for (int k = 0; k <= g; k++) {
#pragma unroll
                for (int i = 0; i < WAY; i++) {
                    const int x = x0 + i * fours_c.step;
                    if (x < sm.da16) {
                        float4 *at = reinterpret_cast<float4 *>(parts + (size_t)k * p.slot + (size_t)x * sm.dc16 + fours_c.x);
                        if (STATES) { // the state before the first token is kept: s_end may lie where it lies
                            *at = s[i];
                            s[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        } else {
                            const float4 f = *at;
                            s[i].x = fmaf(l_seg, s[i].x, f.x); s[i].y = fmaf(l_seg, s[i].y, f.y);
                            s[i].z = fmaf(l_seg, s[i].z, f.z); s[i].w = fmaf(l_seg, s[i].w, f.w);
                        }
                    }
                }
            }
#pragma unroll
        for (int i = 0; i < WAY; i++)
            if (x0 + i * fours_c.step < sm.da16)
                *reinterpret_cast<float4 *>(Ss + (x0 + i * fours_c.step) * sm.ld_c + fours_c.x) = s[i];
    }
    if (!STATES)
        zero_behind<float>(p, q.o, q.ldo, q.dc, rows, b, h, g, warp, thr >> 5, lane);
    int turn = 0;
    for (int u0 = begin; u0 < end; u0 += FC, turn ^= 1) {
        const int n = min(FC, end - u0);
        const float *As = smf + turn * sm.tile, *Bs = As + sm.b, *Cs = As + sm.c + y0 + g4;
        fa::cp_wait<0>();
        __syncthreads(); // this chunk's tiles and the state stand, the chunk before has been read
        if (u0 + FC < end)
            fetch(u0 + FC, smf + (turn ^ 1) * sm.tile);
        Two left[4], right[2][2];
        if (!STATES) {
            for (int it = warp; it < 3; it += thr >> 5) { // pair weights: sixteen rows by sixteen keys that are not all behind them
                const int m = it > 0, k16 = it > 1;
                const float *at = As + (16 * m + g4) * sm.ld_a + t, *bt = Bs + (16 * k16 + g4) * sm.ld_a + t;
                Sums w;
#pragma unroll 2
                for (int ks = 0; ks < a_steps; ks++) {
                    left16(left, at + 8 * ks, sm.ld_a, 1);
                    right16(right, bt + 8 * ks, sm.ld_a, 1);
                    w.add(left, right);
                }
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int i = 16 * m + g4 + 4 * (c & 2), j = 16 * k16 + 8 * x + 2 * t + (c & 1);
                        Ps[i * LP + j] = j <= i ? w.sum(x, c) * q.s_pair * pw[i - j] : 0.0f;
                    }
            }
            // what the state gives
            Sums o[2];
            const float *at = As + g4 * sm.ld_a + t, *st = Ss + t * sm.ld_c + y0 + g4;
#pragma unroll 2
            for (int ks = 0; ks < a_steps; ks++) {
                right16(right, st + 8 * ks * sm.ld_c, 1, sm.ld_c);
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    left16(left, at + 16 * m * sm.ld_a + 8 * ks, sm.ld_a, 1);
                    o[m].add(left, right);
                }
            }
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float l = q.s_state * pw[16 * m + g4 + 4 * (c & 2) + q.e1];
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        o[m].big[x][c] *= l;
                        o[m].small[x][c] *= l;
                    }
                }
            __syncthreads(); // the weights stand, the state has been read
#pragma unroll
            for (int ks = 0; ks < FC / 8; ks++) {
                right16(right, Cs + (8 * ks + t) * sm.ld_c, 1, sm.ld_c);
#pragma unroll
                for (int m = 0; m < 2; m++)
                    if (ks < 2 * m + 2) {
                        left16(left, Ps + (16 * m + g4) * LP + 8 * ks + t, LP, 1);
                        o[m].add(left, right);
                    }
            }
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int c = 0; c < 4; c += 2) {
                    const int i = 16 * m + g4 + 4 * c;
                    if (i < n) {
                        float *to = reinterpret_cast<float *>(q.o) + rows.row(u0 + i) * q.ldo + (size_t)h * q.dc + y0 + 2 * t;
#pragma unroll
                        for (int x = 0; x < 2; x++)
                            if (y0 + 8 * x + 2 * t < q.dc)
                                *reinterpret_cast<float2 *>(to + 8 * x) = make_float2(o[m].sum(x, c), o[m].sum(x, c + 1));
                    }
                }
            if (u0 + FC >= end && !q.s_end)
                break;
        }
        const float l_n = pw[n];
        Two weighted[FC / 8][2][2];
#pragma unroll
        for (int ks = 0; ks < FC / 8; ks++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int j = 8 * ks + t + 4 * c;
                const float w = j < n ? q.s_in * pw[n - 1 - j + q.e2] : 0.0f;
#pragma unroll
                for (int x = 0; x < 2; x++)
                    weighted[ks][x][c] = Two(w * Cs[j * sm.ld_c + 8 * x]);
            }
#pragma unroll 1
        for (int x0 = 0; x0 < q.da; x0 += 16) {
            Sums add;
#pragma unroll
            for (int ks = 0; ks < FC / 8; ks++) {
                left16(left, Bs + (8 * ks + t) * sm.ld_a + x0 + g4, 1, sm.ld_a);
                add.add(left, weighted[ks]);
            }
#pragma unroll
            for (int c = 0; c < 4; c += 2)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    float2 *s = reinterpret_cast<float2 *>(Ss + (x0 + g4 + 4 * c) * sm.ld_c + y0 + 8 * x + 2 * t);
                    const float2 now = *s;
                    *s = make_float2(fmaf(l_n, now.x, add.sum(x, c)), fmaf(l_n, now.y, add.sum(x, c + 1)));
                }
        }
    }
    __syncthreads();
    if (STATES) {
        for (int x = fours_c.r; x < sm.da16; x += fours_c.step)
            *reinterpret_cast<float4 *>(parts + (size_t)(g + 1) * p.slot + (size_t)x * sm.dc16 + fours_c.x) = quad(Ss + x * sm.ld_c + fours_c.x);
    } else if (q.s_end && ends_in(p, rows.n, g) && fours_c.x < q.dc) {
        for (int x = fours_c.r; x < q.da; x += fours_c.step) {
            float *to = q.s_end + pair * nn + (size_t)x * q.dc + fours_c.x;
            const float4 f = quad(Ss + x * sm.ld_c + fours_c.x);
            to[0] = f.x; to[1] = f.y; to[2] = f.z; to[3] = f.w;
        }
    }
}

// ---------------- bf16 on warp-level tensor-core products ----------------
//
// A CTA of 4 CG warps goes through one part of one (stream, head) in chunks of 64 tokens.  Warp (r, cg) takes rows
// 16 r .. 16 r + 15 of a chunk and 32 columns of c, the cg-th; of the state it owns the same columns of rows 16 r ..
// (and 16 (r + 4) .. of 128) in fp32 accumulators.  The results need all of the state: it goes through shared memory as two
// bf16 terms, and so do the pair weights P.  What 16 bits leave out, 2^-16 of each, is far below a result's own rounding;
// with one term each the errors against 64 bits were 2.35e-3 of the results instead of the 1.66e-3 of that rounding
// (128 pairs of 2048 tokens of 64, forward: 62.7 us, now 77).  Products of a decayed b with c, which the state adds up, are
// kept to 24 bits by three bf16 terms of the decayed value, so that the state is an fp32 sum of fp32 products.  Pair weights
// and terms are the same for the CG warps of the same rows: each computes every CG-th and they meet at a barrier of their own.
//
// Tiles come by TMA, 64 tokens x 64 (32) values of a head a copy, from a map of (value, head, stream, token): what lies beyond
// a head's values or the sequence arrives as zeros.  One thread asks for the next chunk's under the present chunk; a
// barrier hands over tiles and state, another one frees the state's place when all have read it (in the middle
// of the chunk that one is no faster).  In the reverse order a chunk's row i is the tile's row 63 - i.
//
// Bound by the chain of a chunk's phases (weights, what the state gives, products with c, the state to the next chunk) in
// too few warps to hide it: the tensor pipe is active 40 to 55 % of the time (of single chunks 23), shared memory 33 to 46, an
// instruction issues in 29 to 43.  8 x 16 pairs of 2048 tokens of 64, forward and backward: 231 us, 50 GFLOP of the chunk form's
// products, in two or three terms but for the pair weights, 218 TFLOP/s of the 550 that this instruction reaches; the bytes
// alone 41.5 us.  2 x 8 pairs of 4096 tokens of 128, forward, in eight parts: 77 us (both passes), bytes 10.5.

constexpr int TC = 64; // tokens in a chunk

struct __align__(64) MmaArgs {
    CUtensorMap map[3][4]; // of a, b, c, a2 of each role
    Args p;
};

template <int DA, int DC, bool TWO> struct MmaSmem {
    static constexpr int TA = TC * DA * 2, TB = TC * DC * 2, LC = DC + 8; // tiles; pitch of the state, rows four banks on
    static constexpr int MT = DA > 64 ? DA / 64 : 1;
    static constexpr int SL = DA * LC * 2, XP = 10 * 512; // a term of the state, of the pair weights
    static constexpr int XS = 4 * 4 * MT * 3 * 512;       // the decayed values' terms
    static constexpr int A = 0, B = A + 2 * TA, C = B + 2 * TA, A2 = C + 2 * TB, S = A2 + (TWO ? TB : 0), P = S + 2 * SL, SP = P + 2 * XP, W = SP + XS,
                         BAR = W + (2 * TC + 8) * 4, BYTES = BAR + 32 + 1024; // the tiles begin at a multiple of 1024
    static_assert(BYTES <= SMEM_MOST && (DA > 64 || DC > 64 || 2 * (BYTES + 1024) <= SMEM_MOST + 1024), "");
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int h, int b, int t)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(h), "r"(b), "r"(t)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_at(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm4t_at(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
// Byte offset of 16-byte piece c of row r in a tile of D values a row: blocks of 64 columns, rows of 128 bytes, piece c at
// c ^ (r % 8); with 32 columns rows of 64 bytes and piece c at c ^ (r / 2 % 4).  Flipping bits 1 and 2 of c flips bits 5
// and 6 of the offset; 16 rows on, the pieces lie in the same order.
template <int D> __device__ __forceinline__ uint32_t tile_at(int r, int c)
{
    if constexpr (D == 32)
        return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
    else
        return (uint32_t)((c >> 3) * (TC * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
template <int D> struct Rows16 { static constexpr int BYTES = D == 32 ? 16 * 64 : 16 * 128; };

// 64 tokens of one head from time t0 on as TMA lays them, zeros outside [0, n) and behind value d.  src: the head's first row
template <int D, int THR> __device__ __forceinline__ void tile_copy(uint32_t dst, const bf16 *src, long long pitch, int d, int t0, int n)
{
    constexpr int CPR = D / 8, ROWS = THR / CPR; // pieces of a row, rows at a time: a multiple of eight, so that pieces keep their order
    static_assert(ROWS % 8 == 0, "");
    const int r = threadIdx.x / CPR, x = threadIdx.x % CPR;
    const bf16 *from = src + (t0 + r) * pitch + x * 8;
    dst += tile_at<D>(r, x);
#pragma unroll
    for (int i = 0; i < (TC + ROWS - 1) / ROWS; i++, from += ROWS * pitch, dst += ROWS * (D == 32 ? 64 : 128)) {
        const int t = t0 + r + i * ROWS;
        const bool in = t >= 0 && t < n && x * 8 < d;
        if (TC % ROWS == 0 || r < TC)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(in ? from : src), "r"(in ? 16 : 0) : "memory");
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

// a pair of values as two bf16 terms each: 16 bits of them
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo)
{
    hi = fa::pack2(x, y);
    lo = fa::pack2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}

// TMA: tiles come by tensor maps; otherwise (streams of one chunk, where there is nothing to fetch ahead and twelve maps
// for a step cost the host 6 us) all threads copy 16 bytes at a time.
// TWO: roles with a2 have a second result,
//   o2_i = s_state l^(i+e1) a2_i S^T + s_pair sum_{j<=i} l^(i-j) (a2_i . c_j) b_j,
// from the same tiles of b and c and the same state: dk beside dv.  It is computed behind the first one, in the same room for pair
// weights, and a2 has one place, filled again while the next chunk computes its first result: so two such CTAs share an SM.
template <int DA, int DC, bool STATES, bool TMA, bool TWO>
__global__ void __launch_bounds__(4 * DC, DA <= 64 && DC <= 64 ? 2 : 1) mma_kernel(const __grid_constant__ MmaArgs args)
{
    using SM = MmaSmem<DA, DC, TWO>;
    constexpr int LC = SM::LC, NT = 4, MT = SM::MT, KS = DA / 16, THR = 4 * DC, CG = DC / 32;
    extern __shared__ __align__(16) unsigned char smraw[];
    __shared__ int abort_s, flag;
    unsigned char *sm = smraw + ((1024u - (fa::smem_addr(smraw) & 1023u)) & 1023u);
    const uint32_t base = fa::smem_addr(sm), bar = base + SM::BAR;
    bf16 *Ss = reinterpret_cast<bf16 *>(sm + SM::S);
    float *wts = reinterpret_cast<float *>(sm + SM::W), *pw16 = wts + 2 * TC; // weights of full and last chunks; l^16m
    const Args &p = args.p;
    const Role &q = p.role[blockIdx.z];
    const CUtensorMap *maps = args.map[blockIdx.z];
    const bool two = TWO && !STATES && q.a2;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, t = lane & 3;
    // a scheduler's warps take rows r and 3 - r in turn: the triangle is dealt evenly
    const int cg = warp >> 2, r = cg & 1 ? 3 - (warp & 3) : warp & 3;
    const size_t pair = blockIdx.x;
    const int g = blockIdx.y, b = (int)(pair / p.H), h = (int)(pair % p.H);
    const float rate = p.rate[h];
    if constexpr (TMA) {
        if (tid == 0) {
            abort_s = 0;
            tc::mbar_init(bar, 1);
            tc::mbar_init(bar + 8, 1);
            tc::mbar_init(bar + 16, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
    pdl_wait(); // no early trigger: successors resident beside these CTAs cost more than their launch (128 pairs of 2048 tokens 110 -> 78 us)
    const Rows rows(p, q, b);
    const size_t nn = (size_t)q.da * q.dc;
    if (STATES && !q.s_end && g == p.n_seg - 1) // nobody asks for the last part's sum
        return;
    const int begin = g * p.seg, end = min(rows.n, begin + p.seg), total = max(end - begin, 0), chunks = (total + TC - 1) / TC;
    bool ok = true; // the CTA's waits; behind one that ran out results are NaN and nothing more is asked for
    CopyRing chunk_ring(2), a2_ring(1); // thread 0's
    auto fetch = [&](int k) {
        const int u0 = begin + k * TC, buf = k & 1, t0 = q.reverse ? rows.n - TC - u0 : u0;
        if constexpr (!TMA) {
            if (!STATES)
                tile_copy<DA, THR>(base + SM::A + buf * SM::TA, reinterpret_cast<const bf16 *>(q.a) + b * q.lda + h * q.da, p.B * q.lda, q.da, t0, rows.n);
            tile_copy<DA, THR>(base + SM::B + buf * SM::TA, reinterpret_cast<const bf16 *>(q.b) + b * q.ldb + h * q.da, p.B * q.ldb, q.da, t0, rows.n);
            tile_copy<DC, THR>(base + SM::C + buf * SM::TB, reinterpret_cast<const bf16 *>(q.c) + b * q.ldc + h * q.dc, p.B * q.ldc, q.dc, t0, rows.n);
            if (two)
                tile_copy<DC, THR>(base + SM::A2, reinterpret_cast<const bf16 *>(q.a2) + b * q.lda2 + h * q.dc, p.B * q.lda2, q.dc, t0, rows.n);
            fa::cp_commit();
        } else if (tid == 0 && ok) {
            const uint32_t full = bar + 8 * buf;
            chunk_ring.asked++;
            tc::mbar_expect_tx(full, (STATES ? 1 : 2) * SM::TA + SM::TB);
#pragma unroll
            for (int x = 0; x < DA; x += 64) {
                if (!STATES)
                    tma_load_4d(base + SM::A + buf * SM::TA + x * TC * 2, &maps[0], full, x, h, b, t0);
                tma_load_4d(base + SM::B + buf * SM::TA + x * TC * 2, &maps[1], full, x, h, b, t0);
            }
#pragma unroll
            for (int x = 0; x < DC; x += 64)
                tma_load_4d(base + SM::C + buf * SM::TB + x * TC * 2, &maps[2], full, x, h, b, t0);
        }
    };
    auto fetch2 = [&](int k) { // a2, when the chunk before has read its place
        if (TMA && two && tid == 0 && ok) {
            const int u0 = begin + k * TC, t0 = q.reverse ? rows.n - TC - u0 : u0;
            a2_ring.asked++;
            tc::mbar_expect_tx(bar + 16, SM::TB);
#pragma unroll
            for (int x = 0; x < DC; x += 64)
                tma_load_4d(base + SM::A2 + x * TC * 2, &maps[3], bar + 16, x, h, b, t0);
        }
    };
    if (chunks) {
        fetch(0);
        fetch2(0);
    }

    // the state: element c of s[m][n] is row 16 (r + 4 m) + gq + 8 (c >> 1), column 32 cg + 8 n + 2 t + (c & 1); in
    // parts it lies as the threads hold it
    float s[MT][NT][4];
    const bool has_state = r * 16 < DA; // of 32 rows the warps r = 2, 3 own none
    const bool first = p.n_seg == 1 || (STATES && g == 0);
    float4 *part = reinterpret_cast<float4 *>(q.parts + pair * (p.n_seg + 1) * p.slot) + tid;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
            s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.0f;
    if (first && q.s0) {
        const float *from = q.s0 + pair * nn + (q.s0_t ? (32 * cg + 2 * t) * q.da + 16 * r + gq : (16 * r + gq) * q.dc + 32 * cg + 2 * t);
        const int row = q.s0_t ? 1 : q.dc, col = q.s0_t ? q.da : 1;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int c = 0; c < 4; c += 2)
                    if (16 * (r + 4 * m) + gq + 4 * c < q.da && 32 * cg + 8 * n + 2 * t < q.dc) {
                        const float *at = from + (64 * m + 4 * c) * row + 8 * n * col;
                        if (q.s0_t) {
                            s[m][n][c] = at[0];
                            s[m][n][c + 1] = at[col];
                        } else {
                            const float2 f = *reinterpret_cast<const float2 *>(at);
                            s[m][n][c] = f.x;
                            s[m][n][c + 1] = f.y;
                        }
                    }
    }
    const int n_last = total - (chunks - 1) * TC;
    const float l_seg = power(rate, p.seg), l_full = power(rate, TC), l_last = power(rate, n_last);
    if (tid < TC) {
        wts[tid] = q.s_in * power(rate, TC - 1 - tid + q.e2);
        wts[tid + TC] = tid < n_last ? q.s_in * power(rate, n_last - 1 - tid + q.e2) : 0.0f;
    } else if (tid < TC + 4) {
        pw16[tid - TC] = power(rate, 16 * (tid - TC));
    }
    // weights of pairs on the diagonal and 16 rows from it, of this thread's elements of two 8-key groups: row - key is
    // d + 8 j with j = (c >> 1) - n from -1 to 1, less c & 1
    float apart[3][2], diag[3][2], f_a = 0.0f, f_b = 0.0f;
    if (!STATES) {
        f_a = q.s_state * power(rate, 16 * r + gq + q.e1);
        f_b = q.s_state * power(rate, 16 * r + gq + 8 + q.e1);
#pragma unroll
        for (int j = 0; j < 3; j++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int d = gq - 2 * t - c + 8 * (j - 1);
                apart[j][c] = q.s_pair * power(rate, 16 + d);
                diag[j][c] = q.s_pair * power(rate, max(d, 0));
            }
    }
    // fragments of the tiles: this lane's rows of sixteen, in the chunk's order
    auto row_of = [&](int i) { return q.reverse ? TC - 1 - i : i; };
    const int step_a = (q.reverse ? -1 : 1) * Rows16<DA>::BYTES, step_c = (q.reverse ? -1 : 1) * Rows16<DC>::BYTES;
    const int l15 = lane & 15, lrow = (lane & 7) + (lane >> 4) * 8, lhi = lane >> 4, lmid = (lane >> 3) & 1;
    const uint32_t a_at = base + SM::A + tile_at<DA>(row_of(16 * r + l15), lhi);          // rows r of a, values 16 ks: ^ ks << 5
    const uint32_t b_at = base + SM::B + tile_at<DA>(row_of(lrow), lmid);                  // rows 0 .. 15 of b, the same
    const uint32_t bt_at = base + SM::B + tile_at<DA>(row_of(lrow), 2 * r % (DA / 8) + lmid); // transposed: values 16 r
    const uint32_t c_at = base + SM::C + tile_at<DC>(row_of(l15), 4 * cg + lhi);           // transposed: rows 0 .. 15 of c
    const uint32_t s_at = base + SM::S + (l15 * LC + 32 * cg + lhi * 8) * 2;
    uint4 *pairs = reinterpret_cast<uint4 *>(sm + SM::P) + r * (r + 1) / 2 * 32 + lane;        // fragments of this warp's rows, keys not behind them
    uint4 *terms = reinterpret_cast<uint4 *>(sm + SM::SP) + r * 4 * MT * 3 * 32 + lane;
    if (p.n_seg > 1) {
        if (STATES) {
            if (g == 0) // the state before the first token is kept: s_end may lie where it lies
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        part[(m * NT + n) * THR] = make_float4(s[m][n][0], s[m][n][1], s[m][n][2], s[m][n][3]);
                        s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.0f;
                    }
        } else {
#pragma unroll 1
            for (int k = 0; k <= g; k++, part += p.slot / 4)
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const float4 f = part[(m * NT + n) * THR];
                        s[m][n][0] = fmaf(l_seg, s[m][n][0], f.x); s[m][n][1] = fmaf(l_seg, s[m][n][1], f.y);
                        s[m][n][2] = fmaf(l_seg, s[m][n][2], f.z); s[m][n][3] = fmaf(l_seg, s[m][n][3], f.w);
                    }
        }
    }
    // fp32 values that lie as the state does, out
    auto state_out = [&](const float (&x)[MT][NT][4]) {
        float *to = q.s_end + pair * nn;
        if (has_state)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int c = 0; c < 4; c += 2) {
                        const int i = 16 * (r + 4 * m) + gq + 4 * c, y = 32 * cg + 8 * n + 2 * t;
                        if (i < q.da && y < q.dc)
                            *reinterpret_cast<float2 *>(to + i * q.dc + y) = make_float2(x[m][n][c], x[m][n][c + 1]);
                    }
    };
    // Of several parts the last one's sum stands in the slot behind the others, exact to the third term: the state behind the
    // last token is known before the first chunk, and the chunks need no third term.
    const bool ends = q.s_end && ends_in(p, rows.n, g), follows = STATES || (q.s_end && p.n_seg == 1); // follows: s is a result
    if (!STATES && ends && p.n_seg > 1) {
        const float l_total = power(rate, total);
        float x[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float4 f = part[(m * NT + n) * THR]; // behind the loop above: slot g + 1
                x[m][n][0] = fmaf(l_total, s[m][n][0], f.x); x[m][n][1] = fmaf(l_total, s[m][n][1], f.y);
                x[m][n][2] = fmaf(l_total, s[m][n][2], f.z); x[m][n][3] = fmaf(l_total, s[m][n][3], f.w);
            }
        state_out(x);
    }
    auto publish = [&]() {
        if (!STATES && has_state)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int c = 0; c < 4; c += 2) {
                        bf16 *to = Ss + (16 * (r + 4 * m) + gq + 4 * c) * LC + 32 * cg + 8 * n + 2 * t;
                        uint32_t hi, lo;
                        split2(s[m][n][c], s[m][n][c + 1], hi, lo);
                        *reinterpret_cast<uint32_t *>(to) = hi;
                        *reinterpret_cast<uint32_t *>(to + DA * LC) = lo;
                    }
    };
    publish();
    if (!STATES)
        zero_behind<bf16>(p, q.o, q.ldo, q.dc, rows, b, h, g, warp, THR / 32, lane);
    if (two)
        zero_behind<bf16>(p, q.o2, q.ldo2, q.da, rows, b, h, g, warp, THR / 32, lane);

    for (int k = 0; k < chunks; k++) {
        const int buf = k & 1, u0 = begin + k * TC, n = min(TC, end - u0);
        const bool last = k == chunks - 1;
        if constexpr (TMA)
            ok = ok && tc::mbar_wait(bar + 8 * buf, chunk_ring.parity(k), &abort_s, &flag, 81);
        else
            fa::cp_wait<0>();
        if (TMA && n < TC && p.len && !q.reverse) // rows behind the stream's end hold anything: the tile's are zeros
            for (int i = tid; i < (TC - n) * (DA / 8 + DC / 8); i += THR) {
                const int row = n + i / (DA / 8 + DC / 8), x = i % (DA / 8 + DC / 8);
                unsigned char *to = sm + (x < DA / 8 ? SM::B + buf * SM::TA + tile_at<DA>(row, x) : SM::C + buf * SM::TB + tile_at<DC>(row, x - DA / 8));
                *reinterpret_cast<uint4 *>(to) = make_uint4(0u, 0u, 0u, 0u);
            }
        // this chunk's tiles and state stand; the other buffers are free
        if constexpr (TMA)
            ok = __syncthreads_and(ok);
        else
            __syncthreads();
        if (!last)
            fetch(k + 1);
        const uint32_t At = a_at + buf * SM::TA, Bt = b_at + buf * SM::TA, Tt = bt_at + buf * SM::TA, Ct = c_at + buf * SM::TB;
        const bool carries = has_state && (follows || !last); // the state behind the chunk is of use
        const float *wt = wts + (last ? TC : 0);
        float o[NT][4];
        auto row_barrier = [&]() { // the warps of these rows
            if constexpr (CG > 1)
                asm volatile("bar.sync %0, %1;" ::"r"(1 + r), "n"(32 * CG) : "memory");
            else
                __syncwarp();
        };
        auto row_agree = [&](bool x) { // the same, and whether x holds in all of them
            uint32_t all;
            asm volatile("{\n\t.reg .pred p, q;\n\t"
                         "setp.ne.u32 p, %1, 0;\n\t"
                         "bar.red.and.pred q, %2, %3, p;\n\t"
                         "selp.u32 %0, 1, 0, q;\n\t}"
                         : "=r"(all)
                         : "r"((uint32_t)x), "r"(1 + r), "n"(32 * CG)
                         : "memory");
            return all != 0;
        };
        // pair weights of every CG-th sixteen keys, for all warps of these rows: rows `u` against the tile's rows at v
        auto weights = [&](const uint32_t (&u)[KS][4], uint32_t v, int step) {
#pragma unroll
            for (int i = 0; i < 4 / CG; i++) {
                const int pc = cg + i * CG;
                if (pc > r)
                    break;
                float w[2][4] = {};
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t f[4];
                    ldsm4_at(f, ((v ^ ((ks & 3) << 5)) + (ks >> 2) * (TC * 128)) + pc * step);
                    fa::mma(w[0], u[ks], f[0], f[1]);
                    fa::mma(w[1], u[ks], f[2], f[3]);
                }
                if (pc == r) {
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            w[x][c] = gq + 8 * (c >> 1) >= 8 * x + 2 * t + (c & 1) ? w[x][c] * diag[(c >> 1) - x + 1][c & 1] : 0.0f;
                } else {
                    const float f = pw16[r - pc - 1];
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            w[x][c] *= f * apart[(c >> 1) - x + 1][c & 1];
                }
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    split2(w[e >> 1][e % 2 * 2], w[e >> 1][e % 2 * 2 + 1], hi[e], lo[e]);
                pairs[pc * 32] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                pairs[pc * 32 + SM::XP / 16] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        };
        // what the pair weights of keys 16 ks .. give, f: the products' right factors
        auto paired = [&](float (&x)[NT][4], int ks, const uint32_t (&f)[NT / 2][4]) {
#pragma unroll
            for (int term = 0; term < 2; term++) {
                const uint4 u = pairs[ks * 32 + term * (SM::XP / 16)];
                const uint32_t pf[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < NT; i++)
                    fa::mma(x[i], pf, f[i / 2][i % 2 * 2], f[i / 2][i % 2 * 2 + 1]);
            }
        };
        auto decayed = [&](float (&x)[NT][4]) {
#pragma unroll
            for (int i = 0; i < NT; i++) {
                x[i][0] *= f_a; x[i][1] *= f_a;
                x[i][2] *= f_b; x[i][3] *= f_b;
            }
        };
        // rows out: a quad's 32 columns in four pieces of 16 bytes
        auto rows_out = [&](const float (&x)[NT][4], void *out, long long ldo, int d) {
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
                const int i = 16 * r + gq + 4 * c;
                bf16 *to = reinterpret_cast<bf16 *>(out) + (i < n ? rows.row(u0 + i) * ldo : 0) + (size_t)h * d + 32 * cg;
                uint32_t v[4];
#pragma unroll
                for (int k = 0; k < NT; k++)
                    v[k] = ok ? fa::pack2(x[k][c], x[k][c + 1]) : 0x7fff7fffu; // NaN behind a wait that ran out
                fa::quad_transpose(v, t);
                if (i < n && 32 * cg + 8 * t < d)
                    *reinterpret_cast<uint4 *>(to + 8 * t) = make_uint4(v[0], v[1], v[2], v[3]);
            }
        };
        if (!STATES) {
            uint32_t aq[KS][4];
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                ldsm4_at(aq[ks], (At ^ ((ks & 3) << 5)) + (ks >> 2) * (TC * 128));
            weights(aq, Bt, step_a);
            // what the state gives
#pragma unroll
            for (int x = 0; x < NT; x++)
                o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int x = 0; x < NT; x += 2)
#pragma unroll
                    for (int term = 0; term < 2; term++) {
                        uint32_t f[4];
                        ldsm4t_at(f, s_at + term * SM::SL + (ks * 16 * LC + x * 8) * 2);
                        fa::mma(o[x], aq[ks], f[0], f[1]);
                        fa::mma(o[x + 1], aq[ks], f[2], f[3]);
                    }
            decayed(o);
        }
        // decayed values of every CG-th sixteen tokens, in three terms
        if (carries) {
#pragma unroll
            for (int i = 0; i < 4 / CG; i++) {
                const int ks = cg + i * CG;
                const float2 w0 = *reinterpret_cast<const float2 *>(wt + ks * 16 + 2 * t), w8 = *reinterpret_cast<const float2 *>(wt + ks * 16 + 8 + 2 * t);
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    uint32_t f[4], hi[4], mid[4], lo[4];
                    ldsm4t_at(f, Tt + m * (TC * 128) + ks * step_a);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        split3(f[e], e < 2 ? w0.x : w8.x, e < 2 ? w0.y : w8.y, hi[e], mid[e], lo[e]);
                    uint4 *to = terms + (ks * MT + m) * 96;
                    to[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    to[32] = make_uint4(mid[0], mid[1], mid[2], mid[3]);
                    to[64] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            }
        }
        row_barrier();
        // the third term where a state is a result; elsewhere the state is a factor, of which 16 bits are kept
        const bool third = follows && q.s_end;
        // what the chunk adds has sums of its own: products cut the sum they are added to, the state is rounded
        float add[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int x = 0; x < NT; x++)
                add[m][x][0] = add[m][x][1] = add[m][x][2] = add[m][x][3] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < TC / 16; ks++) {
            uint32_t f[NT / 2][4];
#pragma unroll
            for (int x = 0; x < NT; x += 2)
                ldsm4t_at(f[x / 2], (Ct ^ (x << 4)) + ks * step_c);
            if (!STATES && ks <= r)
                paired(o, ks, f);
            if (carries) {
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int term = 0; term < 3; term++)
                        if (term < 2 || third) {
                            const uint4 u = terms[(ks * MT + m) * 96 + term * 32];
                            const uint32_t bf[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                            for (int x = 0; x < NT; x++)
                                fa::mma(add[m][x], bf, f[x / 2][x % 2 * 2], f[x / 2][x % 2 * 2 + 1]);
                        }
            }
        }
        const float l_n = last ? l_last : l_full;
        if (carries)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int x = 0; x < NT; x++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        s[m][x][c] = fmaf(l_n, s[m][x][c], add[m][x][c]);
        if (!STATES)
            rows_out(o, q.o, q.ldo, q.dc);
        if constexpr (TWO && !STATES) {
            static_assert(DA == DC, "");
            if (two) {
                if constexpr (TMA)
                    ok = ok && tc::mbar_wait(bar + 16, a2_ring.parity(k), &abort_s, &flag, 83);
                ok = row_agree(ok); // and the first result's pair weights have been read
                uint32_t aq[KS][4];
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
                    ldsm4_at(aq[ks], ((a_at - SM::A + SM::A2) ^ ((ks & 3) << 5)) + (ks >> 2) * (TC * 128));
                weights(aq, b_at - SM::B + SM::C + buf * SM::TB, step_c);
#pragma unroll
                for (int x = 0; x < NT; x++)
                    o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
#pragma unroll
                    for (int x = 0; x < NT; x += 2)
#pragma unroll
                        for (int term = 0; term < 2; term++) { // the state's rows are columns here
                            uint32_t f[4];
                            ldsm4_at(f, base + SM::S + term * SM::SL + ((32 * cg + 8 * x + lrow) * LC + ks * 16 + lmid * 8) * 2);
                            fa::mma(o[x], aq[ks], f[0], f[1]);
                            fa::mma(o[x + 1], aq[ks], f[2], f[3]);
                        }
                decayed(o);
                row_barrier();
#pragma unroll
                for (int ks = 0; ks < TC / 16; ks++)
                    if (ks <= r) {
                        uint32_t f[NT / 2][4];
#pragma unroll
                        for (int x = 0; x < NT; x += 2)
                            ldsm4t_at(f[x / 2], ((c_at - SM::C + SM::B + buf * SM::TA) ^ (x << 4)) + ks * step_a);
                        paired(o, ks, f);
                    }
                rows_out(o, q.o2, q.ldo2, q.da);
            }
        }
        if (!last) {
            if (!STATES)
                __syncthreads(); // the state of this chunk has been read: its place is free, and that of a2
            fetch2(k + 1);
            publish();
        }
    }
    if (!ok) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int x = 0; x < NT; x++)
                s[m][x][0] = s[m][x][1] = s[m][x][2] = s[m][x][3] = NAN;
        // copies in flight land before the CTA leaves
        chunk_ring.each_open([&](int place, int parity) { tc::mbar_wait(bar + 8 * place, parity, &abort_s, &flag, 81, tc::DRAIN_TRIES); });
        a2_ring.each_open([&](int, int parity) { tc::mbar_wait(bar + 16, parity, &abort_s, &flag, 83, tc::DRAIN_TRIES); });
    }
    if (STATES) {
        part += (size_t)(g + 1) * (p.slot / 4);
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int x = 0; x < NT; x++)
                part[(m * NT + x) * THR] = make_float4(s[m][x][0], s[m][x][1], s[m][x][2], s[m][x][3]);
    } else if (ends && p.n_seg == 1) {
        state_out(s);
    }
}

// ---------------- a few tokens: the recurrence itself ----------------
//
// A CTA of four warps takes 8 * VEC columns of one (stream, head)'s state into registers, sixteen rows side by side, and
// goes through the tokens one after the other.  Bound by HBM: the state once in and once out, all of a thread's
// loads in flight together.  One token of 128 x 8 states of 64 x 64, 34 MB: 7.3 us, 4.7 TB/s; of 4 x 4 of 32 x 32 2.6 us,
// the latency of a launch and of one load behind another.

constexpr int STEP_TOKENS = 8;

template <typename T, int VEC>
__global__ void __launch_bounds__(128) step_kernel(const __grid_constant__ Args p)
{
    constexpr int COLS = 8 * VEC, MOST = DIM_MAX / 16;
    __shared__ float As[STEP_TOKENS][DIM_MAX], Bs[STEP_TOKENS][DIM_MAX], Cs[STEP_TOKENS][COLS], red[STEP_TOKENS][4][COLS];
    const Role &q = p.role[blockIdx.z];
    const int tid = threadIdx.x, cg = tid & 7, rl = tid >> 3;
    const size_t pair = blockIdx.x;
    const int b = (int)(pair / p.H), h = (int)(pair % p.H), c0 = blockIdx.y * COLS;
    const float l = p.decay[h]; // itself: what a power of its logarithm is off by adds up over the calls that carry a state
    pdl_trigger();
    pdl_wait();
    const Rows rows(p, q, b);
    const size_t nn = (size_t)q.da * q.dc;
    float s[MOST][VEC];
#pragma unroll
    for (int k = 0; k < MOST; k++) {
        const int x = rl + 16 * k, c = c0 + cg * VEC;
#pragma unroll
        for (int v = 0; v < VEC; v++)
            s[k][v] = 0.0f;
        if (q.s0 && x < q.da && c < q.dc) {
            const float *s0 = q.s0 + pair * nn;
            if (VEC == 4 && !q.s0_t) {
                const float4 f = *reinterpret_cast<const float4 *>(s0 + (size_t)x * q.dc + c);
                s[k][0] = f.x; s[k][1 % VEC] = f.y; s[k][2 % VEC] = f.z; s[k][3 % VEC] = f.w;
            } else {
#pragma unroll
                for (int v = 0; v < VEC; v++)
                    s[k][v] = state_at(q, s0, x, c + v);
            }
        }
    }
    const T *a = reinterpret_cast<const T *>(q.a) + (size_t)h * q.da, *bb = reinterpret_cast<const T *>(q.b) + (size_t)h * q.da,
            *cc = reinterpret_cast<const T *>(q.c) + (size_t)h * q.dc;
    for (int u = 0; u < rows.n; u++) {
        const long long row = rows.row(u);
        if (tid < q.da) {
            As[u][tid] = to_f(a[row * q.lda + tid]);
            Bs[u][tid] = q.s_in * to_f(bb[row * q.ldb + tid]);
        }
        if (tid < COLS)
            Cs[u][tid] = c0 + tid < q.dc ? to_f(cc[row * q.ldc + c0 + tid]) : 0.0f;
    }
    __syncthreads();
    const float before = q.e1 ? l : 1.0f, behind = q.e2 ? l : 1.0f, s_out = q.s_state;
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
            if (x < q.da) {
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
    if (q.s_end) {
#pragma unroll
        for (int k = 0; k < MOST; k++) {
            const int x = rl + 16 * k, c = c0 + cg * VEC;
            if (x < q.da && c < q.dc) {
                float *to = q.s_end + pair * nn + (size_t)x * q.dc + c;
                if (VEC == 4)
                    *reinterpret_cast<float4 *>(to) = make_float4(s[k][0], s[k][1 % VEC], s[k][2 % VEC], s[k][3 % VEC]);
                else
                    to[0] = s[k][0];
            }
        }
    }
    __syncthreads();
    {
        T *o = reinterpret_cast<T *>(q.o) + (size_t)h * q.dc;
        for (int i = tid; i < p.T * COLS; i += 128) {
            const int u = i / COLS, x = i % COLS;
            if (c0 + x >= q.dc)
                continue;
            if (u < rows.n)
                o[rows.row(u) * q.ldo + c0 + x] = from_f<T>(s_out * (red[u][0][x] + red[u][1][x] + red[u][2][x] + red[u][3][x]));
            else // behind the stream's end
                o[((long long)u * p.B + b) * q.ldo + c0 + x] = from_f<T>(0.0f);
        }
    }
}

} // namespace lin
