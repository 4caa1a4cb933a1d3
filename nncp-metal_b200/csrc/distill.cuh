// distill.cuh -- the loss of a student against a teacher's top logits and the coded symbol, and its gradient.
//
//   q = softmax(top / tau) over the entries that are there,  p_tau = softmax(z / tau),  p = softmax(z)
//   L = w [(1 - share) (lse(z) - z_target) + share tau^2 sum_k q_k (ln q_k - ln p_tau(id_k))]
//   dL/dz = w [(1 - share) (p - 1_target) + share tau (p_tau - sum_k q_k 1_{id_k})]
//
// Bound by HBM: the logits once in, the gradient once out.  A row of up to 16384 logits lies in the registers of one
// CTA from the first read to the gradient; longer rows are read again.  With d = z - max,
// T1 = sum_k e_k (top_k - maxtop - d_k) / tau and e_k = exp((top_k - maxtop) / tau) the teacher's term is
// T1 / sum e - ln sum e + ln sum exp(d / tau): two reductions over a row, one of maxima and one of sums.
//
// Exponentials are what an SM has least of: sixteen a cycle, and two a logit and pass take half of the time that HBM
// needs.  At a temperature of 1, 2, 3 or 4 exp(d) is that power of exp(d / tau): one exponential a logit and one register
// for it from the sums to the gradient, and two rows of 16384 to an SM instead of one.
//
// The gradient is written dense first; the few entries that the target and the teacher name are computed again whole and
// written over it, so that each value is rounded once.
#pragma once
#include "warp_mma.cuh"

namespace distill {

constexpr int TOP_MAX = NNCU_DISTILL_TOP_MAX;

struct Args {
    const void *z;
    const int32_t *ids;     // [N][K]
    const float *top;       // [N][K]
    const int32_t *targets; // [N], may be NULL (no target anywhere)
    const float *weight;    // [N], may be NULL (ones)
    float *loss;            // [N]
    float *lse;             // [N][2]: of z and of z / tau
    void *dz;
    long long ldz, lddz;
    int N, V, K, K4;        // K4: K up to the next multiple of four
    int power;              // exp(d) is this power of exp(d / tau); 0: neither 1 to 4
    float share, tau, inv_tau;
};

enum { LOSS = 1, GRAD = 2 }; // what a launch gives; GRAD alone takes the sums from lse

// block-wide reductions of a few values at once; every thread gets the results
template <int THR, int N_, bool MAX> __device__ __forceinline__ void reduce(float (&v)[N_], float *red)
{
    constexpr int WARPS = THR / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < N_; i++)
        v[i] = MAX ? warp_max(v[i]) : warp_sum(v[i]);
    __syncthreads(); // red may still be read
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N_; i++)
            red[i * WARPS + warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N_; i++) {
        float s = red[i * WARPS + lane % WARPS];
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) {
            const float u = __shfl_xor_sync(0xffffffffu, s, o);
            s = MAX ? fmaxf(s, u) : s + u;
        }
        v[i] = s;
    }
}

template <typename T> __device__ __forceinline__ float4 load4(const T *p)
{
    if constexpr (sizeof(T) == 4)
        return *reinterpret_cast<const float4 *>(p);
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ void store4(T *p, float4 v)
{
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4 *>(p) = v;
    else
        *reinterpret_cast<uint2 *>(p) = make_uint2(fa::pack2(v.x, v.y), fa::pack2(v.z, v.w));
}

// exp(d) from exp(d / tau)
__device__ __forceinline__ float to_power(float e, int power)
{
    const float e2 = e * e;
    return power == 1 ? e : power == 2 ? e2 : power == 3 ? e2 * e : e2 * e2;
}

// PER groups of four logits a thread; PER = 0: a row of any length, read again for each use.  TWO: exp(d) and
// exp(d / tau) are apart.  Groups begin at multiples of four elements in memory, `shift` logits before the row's first where
// that lies between: whole groups go in one access, the row's ends one by one.
template <typename TZ, typename TG, int WHAT, int THR, int PER, bool TWO>
__global__ void __launch_bounds__(THR, PER > 0 && !TWO && (WHAT & LOSS) ? 1024 / THR : 1) kernel(const __grid_constant__ Args a)
{
    constexpr bool KEEP = PER > 0;
    constexpr int E = KEEP ? PER : 1;
    extern __shared__ __align__(16) float sh[]; // of the teacher's entries: symbols, e, the student's logits
    __shared__ float red[4 * THR / 32];
    int32_t *sid = reinterpret_cast<int32_t *>(sh);
    float *se = sh + a.K4, *sz = se + a.K4;
    const int tid = threadIdx.x, V = a.V, K = a.K;
    const long long r = blockIdx.x;
    pdl_wait();
    const TZ *z = reinterpret_cast<const TZ *>(a.z) + r * a.ldz;
    TG *dz = reinterpret_cast<TG *>(a.dz) + r * a.lddz;
    const int shift = (int)(reinterpret_cast<uintptr_t>(z) / sizeof(TZ) % 4);
    auto each = [&](auto f) { // f(slot, first logit)
        if constexpr (KEEP) {
#pragma unroll
            for (int k = 0; k < PER; k++)
                f(k, (k * THR + tid) * 4 - shift);
        } else {
#pragma unroll 4
            for (int i = tid * 4 - shift; i < V; i += THR * 4)
                f(0, i);
        }
    };
    float x[E][4], y[TWO ? E : 1][4];
    auto read = [&](float (&v)[4], int i) {
        if (i >= 0 && i + 4 <= V) {
            const float4 f = load4<TZ>(z + i);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++)
                v[c] = i + c >= 0 && i + c < V ? to_f(z[i + c]) : -INFINITY;
        }
    };
    if constexpr (KEEP)
        each([&](int k, int i) { read(x[k], i); });
    const float w = a.weight ? a.weight[r] : 1.0f;
    const int target = a.targets ? a.targets[r] : -1;
    const bool known = target >= 0 && target < V;
    // the teacher's entries
    float most[2] = {-INFINITY, -INFINITY};
    for (int k = tid; k < a.K4; k += THR) {
        const int id = k < K ? a.ids[r * K + k] : -1;
        const bool there = id >= 0 && id < V;
        sid[k] = there ? id : -1;
        se[k] = there ? a.top[r * K + k] : -INFINITY;
        sz[k] = there ? to_f(z[id]) : 0.0f;
        most[1] = fmaxf(most[1], se[k]);
    }
    const float z_target = known ? to_f(z[target]) : 0.0f;
    auto nothing = [&]() { // a row without weight, or whose mask leaves no symbol
        if (WHAT & LOSS) {
            if (tid == 0) {
                a.loss[r] = 0.0f;
                if (a.lse)
                    a.lse[2 * r] = a.lse[2 * r + 1] = -INFINITY;
            }
        }
        if (WHAT & GRAD)
            for (int i = tid; i < V; i += THR)
                dz[i] = from_f<TG>(0.0f);
    };
    if (w == 0.0f) {
        nothing();
        return;
    }
    float lse = 0.0f, lse_tau = 0.0f, m = 0.0f, inv_l = 0.0f, inv_l_tau = 0.0f;
    if constexpr (WHAT & LOSS)
        each([&](int k, int i) {
            if constexpr (!KEEP)
                read(x[k], i);
            most[0] = fmaxf(fmaxf(fmaxf(most[0], x[k][0]), fmaxf(x[k][1], x[k][2])), x[k][3]);
        });
    reduce<THR, 2, true>(most, red);
    const float mq = most[1];
    float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f}; // of exp(d), of exp(d / tau), of e, T1
    if constexpr (WHAT & LOSS) {
        m = most[0];
        if (m == -INFINITY) {
            nothing();
            return;
        }
        const float f = 1.4426950408889634f * a.inv_tau, from = -m * f;
        each([&](int k, int i) {
            if constexpr (!KEEP)
                read(x[k], i);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float e = exp2f(fmaf(x[k][c], f, from));
                if constexpr (TWO) {
                    x[k][c] = __expf(x[k][c] - m);
                    y[k][c] = e;
                    sums[0] += x[k][c];
                } else {
                    x[k][c] = e;
                    sums[0] += to_power(e, a.power);
                }
                sums[1] += e;
            }
        });
    }
    for (int k = tid; k < a.K4; k += THR) {
        const float d = se[k] - mq, e = sid[k] >= 0 ? expf(d * a.inv_tau) : 0.0f;
        if (e > 0.0f) {
            sums[2] += e;
            if constexpr (WHAT & LOSS)
                sums[3] += e * (d - (sz[k] - m)) * a.inv_tau;
        }
        se[k] = e > 0.0f ? e : 0.0f;
    }
    reduce<THR, 4, false>(sums, red); // its barriers also let the entries be read by all
    pdl_trigger();
    const bool taught = sums[2] > 0.0f;
    if constexpr (WHAT & LOSS) {
        inv_l = 1.0f / sums[0];
        inv_l_tau = 1.0f / sums[1];
        if (tid == 0) {
            float loss = 0.0f;
            if (known && a.share != 1.0f)
                loss += (1.0f - a.share) * (logf(sums[0]) - (z_target - m));
            if (taught && a.share != 0.0f)
                loss += a.share * a.tau * a.tau * (sums[3] / sums[2] + logf(sums[1] / sums[2]));
            a.loss[r] = w * loss;
            if (a.lse) {
                a.lse[2 * r] = m + logf(sums[0]);
                a.lse[2 * r + 1] = m * a.inv_tau + logf(sums[1]);
            }
        }
    } else {
        lse = a.lse[2 * r];
        lse_tau = a.lse[2 * r + 1];
        if (lse == -INFINITY) {
            nothing();
            return;
        }
    }
    if constexpr (WHAT & GRAD) {
        const float f = known ? w * (1.0f - a.share) : 0.0f, f_tau = taught ? w * a.share * a.tau : 0.0f;
        const float g = f * inv_l, g_tau = f_tau * inv_l_tau;
        // f p + f_tau p_tau of one logit
        auto both = [&](float zv) {
            if constexpr (WHAT & LOSS)
                return g * __expf(zv - m) + g_tau * __expf((zv - m) * a.inv_tau);
            else
                return f * __expf(zv - lse) + f_tau * __expf(zv * a.inv_tau - lse_tau);
        };
        const bool whole = reinterpret_cast<uintptr_t>(dz) / sizeof(TG) % 4 == shift; // the groups are groups there too
        each([&](int k, int i) {
            float o[4];
            if constexpr (KEEP && (WHAT & LOSS)) {
#pragma unroll
                for (int c = 0; c < 4; c++)
                    o[c] = TWO ? g * x[k][c] + g_tau * y[TWO ? k : 0][c] : g * to_power(x[k][c], a.power) + g_tau * x[k][c];
            } else {
                float v[4];
                read(v, i);
#pragma unroll
                for (int c = 0; c < 4; c++)
                    o[c] = both(v[c]);
            }
            if (whole && i >= 0 && i + 4 <= V)
                store4<TG>(dz + i, make_float4(o[0], o[1], o[2], o[3]));
            else
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (i + c >= 0 && i + c < V)
                        dz[i + c] = from_f<TG>(o[c]);
        });
        __syncthreads(); // the named entries go over the dense ones
        const float inv_e = taught ? f_tau / sums[2] : 0.0f;
        for (int k = tid; k <= K; k += THR) {
            const int id = k < K ? sid[k] : (known ? target : -1);
            if (id < 0)
                continue;
            float off = 0.0f; // of all entries that name this symbol; the first of them writes
            bool first = true;
            for (int j = 0; j < a.K4; j += 4) {
                const int4 s = *reinterpret_cast<const int4 *>(sid + j);
                const float4 e = *reinterpret_cast<const float4 *>(se + j);
                off += s.x == id ? e.x : 0.0f;
                off += s.y == id ? e.y : 0.0f;
                off += s.z == id ? e.z : 0.0f;
                off += s.w == id ? e.w : 0.0f;
                first = first && !((s.x == id && j < k) || (s.y == id && j + 1 < k) || (s.z == id && j + 2 < k) || (s.w == id && j + 3 < k));
            }
            if (first)
                dz[id] = from_f<TG>(both(k < K ? sz[k] : z_target) - (id == target ? f : 0.0f) - off * inv_e);
        }
    }
}

} // namespace distill
