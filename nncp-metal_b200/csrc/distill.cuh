// distill.cuh -- the loss of a student against a teacher's top logits and the coded symbol, and its gradient.
//
//   q = softmax(top / tau) over the entries that are there,  p_tau = softmax(z / tau),  p = softmax(z)
//   L = w [(1 - share) (lse(z) - z_target) + share tau^2 sum_k q_k (ln q_k - ln p_tau(id_k))]
//   dL/dz = w [(1 - share) (p - 1_target) + share tau (p_tau - sum_k q_k 1_{id_k})]
//
// With u = z log2(e) / tau - R for a whole number R next to the row's largest (so that no rounding of a shift is in
// every term), e = 2^u and l = sum e:  p_tau = e / l,  ln p_tau = u ln 2 - ln l,  and with e_k = exp((top_k - maxtop) / tau)
// the teacher's term is sum_k e_k ((top_k - maxtop) / tau - u_k ln 2) / sum e_k - ln sum e_k + ln l.  Two reductions over a
// row, one of maxima and one of sums.
//
// The bytes are the logits once in, the gradient once out.  A CTA stays and takes every gridDim.x-th row; the rows behind come
// by bulk copy into `slots` places in shared memory while one is gone through three times there: maximum, sums,
// gradient.  (A row that is loaded, reduced twice and stored in turn leaves HBM idle most of the time: 2048 rows of 16384
// logits, loss and gradient, took 69 us with a row in the registers of a CTA.)  What of a row does not lie in whole
// 16-byte pieces, at its two ends, is a thread's each.  2048 rows of 16384 fp32 logits with a bf16 gradient, 64 entries a
// row: 46 us, 201 MB at 4.4 TB/s.  Nothing is full: instructions issue in 58 % of the cycles (25 for a logit, 11 of them in the
// three passes, the rest a row's own: the wait for it, reductions, entries); a row of 64 KB leaves an SM three CTAs of one place
// each, which wait for their copies and at barriers for the warps with entries.
//
// Exponentials are what an SM has least of, sixteen a cycle.  Where tau is 1 or 2, or one of the terms is not there, p
// is 2^u or its square over their sum: one exponential a logit and pass instead of two.
//
// The gradient is written dense first; the few entries that the target and the teacher name are computed again whole and
// written over it, so that each value is rounded once.
#pragma once
#include <type_traits>

#include "copy_ring.h"
#include "gemm_tc.cuh"
#include "warp_mma.cuh"

namespace distill {

constexpr int TOP_MAX = NNCU_DISTILL_TOP_MAX;
constexpr int THREADS_MAX = 512, SLOTS_MAX = 4;
constexpr int PLACES = 1024; // by which entries that name the same symbol are found
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

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
    int N, V, K, K4;        // K4: entries and the target, up to a multiple of four
    int slots, slot_bytes;
    float share, tau, inv_tau;
};

enum { LOSS = 1, GRAD = 2 }; // what a launch gives; GRAD alone takes the sums from lse
enum { FAR_ROW = 2 };
// how p follows from e: itself, its square, or an exponential of its own
enum { SAME = 1, SQUARE = 2, APART = 0 };

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// the larger, NaN where one of them is: a row of nothing but NaN is no row of nothing but -inf
__device__ __forceinline__ float most_of(float x, float y)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
    return m;
}
__device__ __forceinline__ float warp_most(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v = most_of(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// block-wide reductions of a few values at once behind one barrier; every thread gets the results, and whether all are ok
template <int N_, bool MAX> __device__ __forceinline__ bool reduce(float (&v)[N_], float *red, bool ok = true)
{
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < N_; i++)
        v[i] = MAX ? warp_most(v[i]) : warp_sum(v[i]);
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N_; i++)
            red[i * 16 + warp] = v[i];
    if (MAX)
        ok = __syncthreads_and(ok);
    else
        __syncthreads();
#pragma unroll
    for (int i = 0; i < N_; i++)
        v[i] = red[i * 16 + (lane & (warps - 1))]; // warps: a power of two, 16 at most
    for (int o = warps / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N_; i++) {
            const float u = __shfl_xor_sync(0xffffffffu, v[i], o);
            v[i] = MAX ? most_of(v[i], u) : v[i] + u;
        }
    return ok;
}

template <typename T> __device__ __forceinline__ void load4(float (&v)[4], const T *p)
{
    if constexpr (sizeof(T) == 4) {
        const float4 f = *reinterpret_cast<const float4 *>(p);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
        v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
    }
}
template <typename T> __device__ __forceinline__ void store4(T *p, const float (&v)[4])
{
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else
        *reinterpret_cast<uint2 *>(p) = make_uint2(fa::pack2(v[0], v[1]), fa::pack2(v[2], v[3]));
}

// A CTA's entries of one row: the teacher's, and behind them the target, whose e is 0
struct Entries {
    int32_t *id;
    float *e, *z;
};

// What the symbols that entries name are computed again from
struct Kept {
    float g, g_tau, inv_e, f, shift, shift1; // of what p is over, of e, of e_k; the target's; shifts of e and p, or of a row that is far, its base
    int target, any;                        // any: 0 nothing, 1, or FAR_ROW
    void *dz;
};

// RING: rows through shared memory; otherwise rows too long for it are read from global memory each time, one to a CTA.
//
// LATE: what the entries' symbols get is computed while the next row is on its way, from what the warps have kept, and not
// before the dense gradient: for CTAs of several rows (2048 of 16384 fp32 logits: 48.5 -> 46.3 us; at one row a CTA there is
// nothing to wait for, 650 of 9208 bf16 logits, loss and gradient apart: 13.05 -> 13.65).
//
// Two barriers a row.  What one row leaves for behind a barrier -- the named entries over its dense gradient, its place in the
// ring for the next copy -- is done behind the first one of the next row; entries and partial sums lie in two
// places that rows take in turn.
template <typename TZ, typename TG, int WHAT, int HARD, bool RING, bool LATE>
__global__ void __launch_bounds__(THREADS_MAX, 2) kernel(const __grid_constant__ Args a)
{
    extern __shared__ __align__(128) unsigned char ring[]; // rows, then twice the entries: symbols, e, the student's logits
    __shared__ float red[2][6 * 16];
    __shared__ __align__(8) uint64_t bars[SLOTS_MAX];
    __shared__ int abort_s, flag;
    __shared__ Kept kept[LATE ? THREADS_MAX / 32 : 1]; // each warp's of the row before
    __shared__ __align__(4) uint16_t last[PLACES], many[PLACES]; // of the entries of a place: one of them; the row in which it had several
    const int tid = threadIdx.x, thr = blockDim.x, V = a.V, K = a.K;
    const uint32_t bar0 = fa::smem_addr(bars), ring0 = fa::smem_addr(ring);
    if (RING && tid == 0) {
        abort_s = 0;
        for (int i = 0; i < a.slots; i++)
            tc::mbar_init(bar0 + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    for (int i = tid; i < PLACES / 2; i += thr)
        reinterpret_cast<uint32_t *>(many)[i] = 0xffffffffu;
    __syncthreads();
    pdl_wait();
    bool ok = true; // the CTA's waits; behind one that ran out results are NaN and nothing more is asked for
    // the whole pieces of row r: logits [lo, hi)
    auto pieces = [&](const TZ *z, int &lo, int &hi) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(z);
        lo = min(V, (int)(-at & 15) / (int)sizeof(TZ));
        hi = max(lo, V - (int)((at + (size_t)V * sizeof(TZ)) & 15) / (int)sizeof(TZ));
    };
    CopyRing ring_of(max(a.slots, 1)); // thread 0's: places are filled in turn
    auto fetch = [&](int slot, long long r) {
        if (RING && tid == 0 && ok && r < a.N) {
            const TZ *z = reinterpret_cast<const TZ *>(a.z) + r * a.ldz;
            int lo, hi;
            pieces(z, lo, hi);
            const uint32_t bytes = (uint32_t)(hi - lo) * sizeof(TZ), bar = bar0 + 8 * slot;
            ring_of.asked++;
            tc::mbar_expect_tx(bar, bytes);
            if (bytes)
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ring0 + slot * a.slot_bytes),
                             "l"(z + lo), "r"(bytes), "r"(bar)
                             : "memory");
        }
    };
    // what a row needs beside its logits, one row ahead
    struct Side {
        float w, top, lse, lse_tau;
        int target, id;
    };
    auto side = [&](long long r) {
        Side s;
        s.w = a.weight ? a.weight[r] : 1.0f;
        s.target = a.targets ? a.targets[r] : -1;
        s.id = tid < K ? a.ids[r * K + tid] : -1;
        s.top = tid < K ? a.top[r * K + tid] : 0.0f;
        if constexpr (!(WHAT & LOSS)) {
            s.lse = a.lse[2 * r];
            s.lse_tau = a.lse[2 * r + 1];
        }
        return s;
    };
    const float scale = LOG2E * a.inv_tau;
    const bool defer = K + 1 <= 2 * thr; // a thread keeps two entries at most
    const int warp_at = tid & ~31;
    const bool names = (WHAT & GRAD) && defer && warp_at <= K;
    if (LATE && names && tid == warp_at)
        kept[tid >> 5].any = 0;
    auto soft_at = [&](float v, float shift) { return ex2(fmaf(v, scale, -shift)); };
    auto hard_at = [&](float v, float e, float shift1) { return HARD == SAME ? e : HARD == SQUARE ? e * e : ex2(fmaf(v, LOG2E, -shift1)); };
    auto entries = [&](int turn) {
        Entries en;
        en.id = reinterpret_cast<int32_t *>(ring + a.slots * a.slot_bytes) + turn * 3 * a.K4;
        en.e = reinterpret_cast<float *>(en.id) + a.K4;
        en.z = en.e + a.K4;
        return en;
    };
    // The gradient of the symbol of entry k: f less at the target, and inv_e times the sum of e over all entries that
    // name it.  The first of them writes.  Entries alone in their place are alone.
    auto named = [&](const Kept &of, const Entries &en, uint16_t round, int k, TG *&to, float &value) {
        const int id = k <= K ? en.id[k] : -1;
        to = nullptr;
        if (id < 0)
            return;
        float off = en.e[k];
        bool first = true;
        if (many[(unsigned)id % PLACES] == round) {
            off = 0.0f;
#pragma unroll 1
            for (int j = 0; j < a.K4; j += 4) {
                const int4 like = *reinterpret_cast<const int4 *>(en.id + j);
                if (like.x == id || like.y == id || like.z == id || like.w == id)
                    for (int i = j; i < j + 4; i++)
                        if (en.id[i] == id) {
                            off += en.e[i];
                            first = first && i >= k;
                        }
            }
        }
        if (first) {
            const bool far = of.any == FAR_ROW;
            const float z = far ? en.z[k] - of.shift : en.z[k], e = soft_at(z, far ? 0.0f : of.shift);
            to = reinterpret_cast<TG *>(of.dz) + id;
            value = (HARD == SAME ? (of.g + of.g_tau) * e : fmaf(of.g, hard_at(z, e, of.shift1), of.g_tau * e)) - (id == of.target ? of.f : 0.0f) -
                    off * of.inv_e;
        }
    };
    long long r = blockIdx.x;
    for (int i = 0; i < a.slots; i++)
        fetch(i, r + (long long)i * gridDim.x);
    Side next = side(r);
    int slot = 0, parity = 0, turn = 0; // slot, parity: those of row after row in ring_of's order
    TG *late[2] = {nullptr, nullptr}; // entries of the row before, to be written behind a barrier
    float late_value[2];
    uint16_t round = 0;
    auto named_two = [&](const Kept &of, const Entries &en, uint16_t round) {
        named(of, en, round, tid, late[0], late_value[0]);
        if (warp_at + thr <= K)
            named(of, en, round, tid + thr, late[1], late_value[1]);
    };
    auto named_before = [&]() { // the entries of the row before
        if (LATE && names) {
            __syncwarp();
            const Kept of = kept[tid >> 5];
            if (of.any)
                named_two(of, entries(turn ^ 1), round - 1);
        }
    };
    for (; r < a.N; r += gridDim.x, turn ^= 1, round++) {
        const Side now = next;
        if (r + gridDim.x < a.N)
            next = side(r + gridDim.x);
        const TZ *z = reinterpret_cast<const TZ *>(a.z) + r * a.ldz;
        TG *dz = reinterpret_cast<TG *>(a.dz) + r * a.lddz;
        int lo, hi;
        pieces(z, lo, hi);
        const TZ *row = RING ? reinterpret_cast<const TZ *>(ring + slot * a.slot_bytes) : z + lo; // logit lo + i at row[i]
        const int pieces4 = (hi - lo) / 4, edge = tid < lo ? tid : tid < lo + V - hi ? hi + tid - lo : -1; // a logit at one of the ends
        const float z_edge = edge >= 0 ? to_f(z[edge]) : -INFINITY;
        named_before(); // while this row is on its way
        if (RING)
            ok = ok && tc::mbar_wait(bar0 + 8 * slot, parity, &abort_s, &flag, 82);
        const float w = now.w;
        // Saved sums are logs of them above zero: of a row far from it they keep too few digits (2^-24 of 64 is what a
        // probability may be off by), and it is gone through from the beginning
        const bool whole_way = (WHAT & LOSS) || (w != 0.0f && now.lse != -INFINITY && !(fmaxf(fabsf(now.lse), fabsf(now.lse_tau)) <= 64.0f));
        const bool known = now.target >= 0 && now.target < V;
        const Entries en = entries(turn);
        float most[2] = {z_edge, -INFINITY};
#pragma unroll 1
        for (int k = tid; k < a.K4; k += thr) {
            const int id = k == K ? now.target : k > K ? -1 : k < thr ? now.id : a.ids[r * K + k];
            const bool there = id >= 0 && id < V;
            const float top = there && k < K ? (k < thr ? now.top : a.top[r * K + k]) : -INFINITY;
            en.id[k] = there ? id : -1;
            if ((WHAT & GRAD) && there)
                last[(unsigned)id % PLACES] = (uint16_t)k;
            en.e[k] = top;
            en.z[k] = !there ? 0.0f : to_f(RING && id >= lo && id < hi ? row[id - lo] : z[id]);
            most[1] = most_of(most[1], top);
        }
        if (whole_way) {
#pragma unroll 4
            for (int i = tid; i < pieces4; i += thr) {
                float v[4];
                load4<TZ>(v, row + 4 * i);
                most[0] = most_of(most_of(most[0], most_of(v[0], v[1])), most_of(v[2], v[3]));
            }
        }
        ok = reduce<2, true>(most, red[turn], ok);
        if (!ok) // what lies in the row's place may be another's
            most[0] = NAN;
        // behind the barrier: what the row before has left
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if ((WHAT & GRAD) && late[i])
                *late[i] = from_f<TG>(late_value[i]);
            late[i] = nullptr;
        }
        if (a.slots > 1 && r != blockIdx.x)
            fetch(slot ? slot - 1 : a.slots - 1, r + (long long)(a.slots - 1) * gridDim.x);
        const float m = whole_way ? most[0] : now.lse_tau * a.tau, mq = most[1];
        const bool none = w == 0.0f || ((WHAT & LOSS) ? most[0] : now.lse) == -INFINITY; // no weight, or a mask that leaves no symbol
        if (LATE && names && tid == warp_at)
            kept[tid >> 5].any = !none;
        if (none) {
            if ((WHAT & LOSS) && tid == 0) {
                a.loss[r] = 0.0f;
                if (a.lse)
                    a.lse[2 * r] = a.lse[2 * r + 1] = -INFINITY;
            }
            if constexpr (WHAT & GRAD)
                for (int i = tid; i < V; i += thr)
                    dz[i] = from_f<TG>(0.0f);
        } else {
            const bool asked = a.share != 0.0f && mq != -INFINITY; // the teacher, who knows of a symbol
            float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f}; // of what p is over, of e, of e_k, the teacher's
            // where the largest logit times the scale has no digits behind the point left (all logits at a type's lowest
            // value, say), logits are taken from it; elsewhere that subtraction would be an instruction a logit and pass
            const bool far = whole_way && !(fabsf(m) * fmaxf(scale, LOG2E) < 1048576.0f);
            const float base = far ? m : 0.0f;
            // by saved sums, p's exponents count from its own: lse_tau tau is up to tau ln V above it
            const float shift = far ? 0.0f : rintf(m * scale), shift1 = far ? 0.0f : rintf((whole_way ? m : now.lse) * LOG2E);
            auto soft = [&](float v) { return soft_at(v, shift); };
            auto hard = [&](float v, float e) { return hard_at(v, e, shift1); };
            auto sum_up = [&](auto is_far) {
                constexpr bool FAR = decltype(is_far)::value;
                constexpr int AHEAD = FAR ? 1 : 4;
#pragma unroll AHEAD
                for (int i = tid; i < pieces4; i += thr) {
                    float v[4];
                    load4<TZ>(v, row + 4 * i);
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const float x = FAR ? v[c] - base : v[c], e = soft(x);
                        sums[1] += e;
                        if constexpr (HARD != SAME)
                            sums[0] += hard(x, e);
                    }
                }
                const float x = z_edge - base, e = soft(x);
                sums[1] += e;
                if constexpr (HARD != SAME)
                    sums[0] += hard(x, e);
            };
            if (whole_way) {
                if (far)
                    sum_up(std::true_type());
                else
                    sum_up(std::false_type());
            }
            // ln 2 u = (z - m) / tau + this
            const float above = fmaf(m - base, scale, -shift) * LN2;
#pragma unroll 1
            for (int k = tid; k < a.K4; k += thr) {
                const float d = (en.e[k] - mq) * a.inv_tau, e = k < K && en.id[k] >= 0 && asked ? expf(d) : 0.0f;
                if (e != 0.0f) { // NaN too
                    sums[2] += e;
                    if constexpr (WHAT & LOSS)
                        sums[3] += e * (d - fmaf(en.z[k] - m, a.inv_tau, above));
                }
                en.e[k] = e;
                if ((WHAT & GRAD) && en.id[k] >= 0 && last[(unsigned)en.id[k] % PLACES] != k)
                    many[(unsigned)en.id[k] % PLACES] = round;
            }
            reduce<4, false>(sums, red[turn] + 2 * 16); // its barrier also lets the entries be read by all
            if constexpr (HARD == SAME)
                sums[0] = sums[1];
            const bool taught = !(sums[2] <= 0.0f);
            if ((WHAT & LOSS) && tid == thr - 1) {
                // p's shift, and what is above the largest logit's
                const float whole = HARD == APART ? shift1 : HARD * shift, over = fmaf(m - base, HARD == APART ? LOG2E : HARD * scale, -whole) * LN2;
                float loss = 0.0f;
                if (known && a.share != 1.0f)
                    loss += (1.0f - a.share) * (logf(sums[0]) - (en.z[K] - m) - over);
                if (taught)
                    loss += a.share * a.tau * a.tau * (sums[3] / sums[2] + logf(sums[1] / sums[2]));
                a.loss[r] = w * loss;
                if (a.lse) {
                    a.lse[2 * r] = base + fmaf(whole, LN2, logf(sums[0]));
                    a.lse[2 * r + 1] = base * a.inv_tau + fmaf(shift, LN2, logf(sums[1]));
                }
            }
            if constexpr (WHAT & GRAD) {
                const float f = known ? w * (1.0f - a.share) : 0.0f, f_tau = taught ? w * a.share * a.tau : 0.0f;
                float g, g_tau; // of what p is over, of e
                if (whole_way) {
                    g = __fdividef(f, sums[0]);
                    g_tau = __fdividef(f_tau, sums[1]);
                } else {
                    g = f * ex2(fmaf(-now.lse, LOG2E, HARD == APART ? shift1 : HARD * shift));
                    g_tau = f_tau * ex2(fmaf(-now.lse_tau, LOG2E, shift));
                    if (!ok)
                        g = g_tau = NAN;
                }
                const float inv_e = taught ? __fdividef(f_tau, sums[2]) : 0.0f;
                auto both = [&](float v) {
                    const float e = soft(v);
                    return HARD == SAME ? (g + g_tau) * e : HARD == SQUARE ? e * fmaf(g, e, g_tau) : fmaf(g, hard(v, e), g_tau * e);
                };
                const Kept of = {g, g_tau, inv_e, f, far ? base : shift, shift1, now.target, far ? FAR_ROW : 1, dz};
                if (names) {
                    if (!LATE)
                        named_two(of, entries(turn), round);
                    else if (tid == warp_at)
                        kept[tid >> 5] = of;
                }
                TG *to = dz + lo;
                auto dense = [&](auto is_far) {
                    constexpr bool FAR = decltype(is_far)::value;
                    constexpr int AHEAD = FAR ? 1 : 4;
                    if (reinterpret_cast<uintptr_t>(to) % (4 * sizeof(TG)) == 0) {
#pragma unroll AHEAD
                        for (int i = tid; i < pieces4; i += thr) {
                            float v[4];
                            load4<TZ>(v, row + 4 * i);
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                v[c] = both(FAR ? v[c] - base : v[c]);
                            store4<TG>(to + 4 * i, v);
                        }
                    } else {
#pragma unroll AHEAD
                        for (int i = tid; i < hi - lo; i += thr)
                            to[i] = from_f<TG>(both(to_f(row[i]) - (FAR ? base : 0.0f)));
                    }
                };
                if (far)
                    dense(std::true_type());
                else
                    dense(std::false_type());
                if (edge >= 0)
                    dz[edge] = from_f<TG>(both(z_edge - base));
                if (!defer) {
                    __syncthreads();
                    for (int k = tid; k <= K; k += thr) {
                        TG *at;
                        float value;
                        named(of, en, round, k, at, value);
                        if (at)
                            *at = from_f<TG>(value);
                    }
                }
            }
        }
        if (a.slots == 1) { // no place for a row ahead
            __syncthreads();
            fetch(0, r + gridDim.x);
        }
        if (++slot >= a.slots) {
            slot = 0;
            parity ^= 1;
        }
    }
    if constexpr (WHAT & GRAD) {
        named_before();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (late[i])
                *late[i] = from_f<TG>(late_value[i]);
    }
    if (RING && !ok) // copies in flight land before the CTA leaves
        ring_of.each_open([&](int place, int parity) { tc::mbar_wait(bar0 + 8 * place, parity, &abort_s, &flag, 82, tc::DRAIN_TRIES); });
}

} // namespace distill
