// distill.cuh -- the loss of a student against a teacher's top logits and the coded symbol, and its gradient.
//
//   q = softmax(top / tau) over the entries that are there,  p_tau = softmax(z / tau),  p = softmax(z)
//   L = w [(1 - share) (lse(z) - z_target) + share tau^2 sum_k q_k (ln q_k - ln p_tau(id_k))]
//   dL/dz = w [(1 - share) (p - 1_target) + share tau (p_tau - sum_k q_k 1_{id_k})]
//
// Bound by HBM: the logits once in, the gradient once out.  A row of up to 16384 logits lies in the registers of one
// CTA, both exponentials with it, from the first read to the gradient; longer rows are read again.  With d = z - max,
// T1 = sum_k e_k (top_k - maxtop - d_k) / tau and e_k = exp((top_k - maxtop) / tau) the teacher's term is
// T1 / sum e - ln sum e + ln sum exp(d / tau): two reductions over a row, one of maxima and one of sums.
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
    int N, V, K;
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
    if constexpr (WARPS > 1) {
        __syncthreads(); // red may still be read
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N_; i++)
                red[i * WARPS + warp] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N_; i++) {
            float s = red[i * WARPS];
            for (int w = 1; w < WARPS; w++)
                s = MAX ? fmaxf(s, red[i * WARPS + w]) : s + red[i * WARPS + w];
            v[i] = s;
        }
    }
}

template <typename T, int VEC> __device__ __forceinline__ void load(float (&v)[VEC], const T *p)
{
    if constexpr (VEC == 1) {
        v[0] = to_f(*p);
    } else if constexpr (sizeof(T) == 4) {
        const float4 f = *reinterpret_cast<const float4 *>(p);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
        v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
    }
}
template <typename T, int VEC> __device__ __forceinline__ void store(T *p, const float (&v)[VEC])
{
    if constexpr (VEC == 1)
        *p = from_f<T>(v[0]);
    else if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else
        *reinterpret_cast<uint2 *>(p) = make_uint2(fa::pack2(v[0], v[1]), fa::pack2(v[2], v[3]));
}

// PER groups of VEC logits a thread; PER = 0: a row of any length, read again for each use
template <typename TZ, typename TG, int WHAT, int THR, int VEC, int PER>
__global__ void __launch_bounds__(THR) kernel(const __grid_constant__ Args a)
{
    constexpr bool KEEP = PER > 0;
    constexpr int E = KEEP ? PER : 1;
    extern __shared__ __align__(16) float sh[]; // ids, then e of the teacher's entries
    __shared__ float red[4 * THR / 32];
    int32_t *sid = reinterpret_cast<int32_t *>(sh);
    float *se = sh + a.K;
    const int tid = threadIdx.x, V = a.V, K = a.K;
    const long long r = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    const float w = a.weight ? a.weight[r] : 1.0f;
    const TZ *z = reinterpret_cast<const TZ *>(a.z) + r * a.ldz;
    TG *dz = reinterpret_cast<TG *>(a.dz) + r * a.lddz;
    auto each = [&](auto f) { // f(slot, first logit)
        if constexpr (KEEP) {
#pragma unroll
            for (int k = 0; k < PER; k++)
                f(k, (k * THR + tid) * VEC);
        } else {
            for (int i = tid * VEC; i < V; i += THR * VEC)
                f(0, i);
        }
    };
    auto nothing = [&]() { // a row without weight, or whose mask leaves no symbol
        if (WHAT & LOSS) {
            if (tid == 0) {
                a.loss[r] = 0.0f;
                if (a.lse)
                    a.lse[2 * r] = a.lse[2 * r + 1] = -INFINITY;
            }
        }
        if (WHAT & GRAD) {
            for (int i = tid; i < V; i += THR)
                dz[i] = from_f<TG>(0.0f);
        }
    };
    if (w == 0.0f) {
        nothing();
        return;
    }
    // the teacher's entries
    float most[2] = {-INFINITY, -INFINITY};
    for (int k = tid; k < K; k += THR) {
        const int id = a.ids[r * K + k];
        const bool there = id >= 0 && id < V;
        sid[k] = there ? id : -1;
        se[k] = there ? a.top[r * K + k] : -INFINITY;
        most[1] = fmaxf(most[1], se[k]);
    }
    float x[E][VEC], y[E][VEC];
    auto read = [&](int k, int i) {
        if (i + VEC <= V)
            load<TZ, VEC>(x[k], z + i);
        else
#pragma unroll
            for (int v = 0; v < VEC; v++)
                x[k][v] = i + v < V ? to_f(z[i + v]) : -INFINITY;
    };
    float lse = 0.0f, lse_tau = 0.0f, m = 0.0f, inv_l = 0.0f, inv_l_tau = 0.0f;
    if constexpr (WHAT & LOSS) {
        each([&](int k, int i) {
            read(k, i);
#pragma unroll
            for (int v = 0; v < VEC; v++)
                most[0] = fmaxf(most[0], x[k][v]);
        });
    } else if constexpr (KEEP) {
        each([&](int k, int i) { read(k, i); });
    }
    reduce<THR, 2, true>(most, red);
    const float mq = most[1];
    float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f}; // of exp(d), of exp(d / tau), of e, T1
    if constexpr (WHAT & LOSS) {
        m = most[0];
        if (m == -INFINITY) {
            nothing();
            return;
        }
        each([&](int k, int i) {
            if constexpr (!KEEP)
                read(k, i);
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                const float d = x[k][v] - m;
                x[k][v] = __expf(d);
                y[k][v] = a.tau == 1.0f ? x[k][v] : __expf(d * a.inv_tau);
                sums[0] += x[k][v];
                sums[1] += y[k][v];
            }
        });
    }
    for (int k = tid; k < K; k += THR) {
        const float d = se[k] - mq, e = sid[k] >= 0 ? expf(d * a.inv_tau) : 0.0f;
        if (e > 0.0f) {
            sums[2] += e;
            if constexpr (WHAT & LOSS)
                sums[3] += e * (d - (to_f(z[sid[k]]) - m)) * a.inv_tau;
        }
        se[k] = e > 0.0f ? e : 0.0f;
    }
    reduce<THR, 4, false>(sums, red); // its barriers also let se be read by all
    const int target = a.targets ? a.targets[r] : -1;
    const bool known = target >= 0 && target < V, taught = sums[2] > 0.0f;
    if constexpr (WHAT & LOSS) {
        lse = m + logf(sums[0]);
        lse_tau = m * a.inv_tau + logf(sums[1]);
        inv_l = 1.0f / sums[0];
        inv_l_tau = 1.0f / sums[1];
        if (tid == 0) {
            float loss = 0.0f;
            if (known && a.share != 1.0f)
                loss += (1.0f - a.share) * (logf(sums[0]) - (to_f(z[target]) - m));
            if (taught && a.share != 0.0f)
                loss += a.share * a.tau * a.tau * (sums[3] / sums[2] + logf(sums[1] / sums[2]));
            a.loss[r] = w * loss;
            if (a.lse) {
                a.lse[2 * r] = lse;
                a.lse[2 * r + 1] = lse_tau;
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
        // f p + f_tau p_tau of one logit, as the dense pass gives it
        auto both = [&](float zv) {
            if constexpr (WHAT & LOSS)
                return f * inv_l * __expf(zv - m) + f_tau * inv_l_tau * __expf((zv - m) * a.inv_tau);
            else
                return f * __expf(zv - lse) + f_tau * __expf(zv * a.inv_tau - lse_tau);
        };
        each([&](int k, int i) {
            if constexpr (!KEEP)
                read(k, i);
            float o[VEC];
#pragma unroll
            for (int v = 0; v < VEC; v++)
                o[v] = KEEP && (WHAT & LOSS) ? f * inv_l * x[k][v] + f_tau * inv_l_tau * y[k][v] : both(x[k][v]);
            if (i + VEC <= V)
                store<TG, VEC>(dz + i, o);
            else
#pragma unroll
                for (int v = 0; v < VEC; v++)
                    if (i + v < V)
                        dz[i + v] = from_f<TG>(o[v]);
        });
        __syncthreads(); // the named entries go over the dense ones
        const float inv_e = taught ? f_tau / sums[2] : 0.0f;
        for (int k = tid; k <= K; k += THR) {
            const int id = k < K ? sid[k] : (known ? target : -1);
            if (id < 0)
                continue;
            float off = 0.0f; // of all entries that name this symbol; the first of them writes
            bool first = true;
            for (int j = 0; j < K; j++)
                if (sid[j] == id) {
                    first = first && j >= k;
                    off += se[j];
                }
            if (first)
                dz[id] = from_f<TG>(both(to_f(z[id])) - (id == target ? f : 0.0f) - off * inv_e);
        }
    }
}

} // namespace distill
