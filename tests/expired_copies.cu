// Linear attention and distillation with waits for copies that give up: those of one thread, or of all, for phases of one
// parity, or of both.  What a CTA waits for before it leaves is waited for as usual.
#include <cstdarg>
#include <cstdio>

#include "common.cuh"
#include "gemm_tc.cuh"
namespace tc {
__device__ int expired_thread, expired_parity; // -1: all; expired_parity 2: none
__device__ __forceinline__ bool expired_wait(uint32_t bar, uint32_t parity, volatile int *abort_s, int *err_flag, int code, uint32_t tries = WAIT_TRIES)
{
    if (tries != DRAIN_TRIES && (expired_thread < 0 || expired_thread == (int)threadIdx.x) && (expired_parity < 0 || expired_parity == (int)parity))
        return false;
    return mbar_wait(bar, parity, abort_s, err_flag, code, tries);
}
} // namespace tc
#define mbar_wait expired_wait
#include "distill.cuh"
#include "linear_attention.cu"

thread_local char g_nncu_err[512] = "";
unsigned long long g_nncu_launches = 0;
GemmProfiler *g_nncu_prof = nullptr;
thread_local int g_nncu_edges = 0;
int nncu_fail(int code, const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_nncu_err, sizeof(g_nncu_err), fmt, ap);
    va_end(ap);
    return code;
}

extern "C" const char *nncu_last_error(void) { return g_nncu_err; }
extern "C" int expire(int thread, int parity)
{
    CUDA_TRY(cudaDeviceSynchronize());
    CUDA_TRY(cudaMemcpyToSymbol(tc::expired_thread, &thread, sizeof(int)));
    CUDA_TRY(cudaMemcpyToSymbol(tc::expired_parity, &parity, sizeof(int)));
    return NNCU_OK;
}

// nncu_distill_* in fp32 at temperature 2 with a share of the teacher, on `grid` CTAs with `slots` places each
template <int WHAT, bool LATE> static int run(const distill::Args &a, int grid)
{
    static DeviceOnce once;
    NNCU_TRY(smem_limit(once, distill::kernel<float, float, WHAT, distill::SQUARE, true, LATE>, 200 * 1024));
    CUDA_TRY(launch_k(distill::kernel<float, float, WHAT, distill::SQUARE, true, LATE>, dim3(grid), dim3(128),
                      (size_t)a.slots * a.slot_bytes + 2 * 3 * 4 * a.K4, 0, a));
    KERNEL_CHECK();
    return NNCU_OK;
}
extern "C" int expired_distill(int what, int late, int grid, int slots, int N, int V, int K, const float *z, const int32_t *ids, const float *top,
                               const int32_t *targets, float *loss, float *lse, float *dz)
{
    distill::Args a = {};
    a.z = z; a.ids = ids; a.top = top; a.targets = targets; a.loss = loss; a.lse = lse; a.dz = dz;
    a.ldz = a.lddz = V;
    a.N = N; a.V = V; a.K = K; a.K4 = (K + 1 + 3) & ~3;
    a.slots = slots; a.slot_bytes = (V * 4 + 31) & ~15;
    a.share = 0.5f; a.tau = 2.0f; a.inv_tau = 0.5f;
    using namespace distill;
    if (what == LOSS)
        return run<LOSS, false>(a, grid);
    if (what == GRAD)
        return late ? run<GRAD, true>(a, grid) : run<GRAD, false>(a, grid);
    return late ? run<LOSS | GRAD, true>(a, grid) : run<LOSS | GRAD, false>(a, grid);
}
