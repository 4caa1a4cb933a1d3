// warp_mma.cuh -- what kernels on warp-level tensor-core instructions (mma.sync m16n8k16) share: fragment
// loads, the product, asynchronous 16-byte copies and the way of a fragment back to memory.
#pragma once
#include "common.cuh"

namespace fa {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const bf16 *p)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_addr(p)));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const bf16 *p)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_addr(p)));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
                 "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void cp16(void *dst, const void *src, bool valid)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 4 x 4 transpose of 32-bit values over the four lanes of a quad: lane t ends with what lane u held in
// v[t] at v[u] (turns four 4-byte column pairs per lane into one 16-byte run per lane)
__device__ __forceinline__ void quad_transpose(uint32_t (&v)[4], int t)
{
    const bool o1 = t & 1, o2 = t & 2;
    uint32_t a = o1 ? v[0] : v[1], b = o1 ? v[2] : v[3];
    a = __shfl_xor_sync(0xffffffffu, a, 1);
    b = __shfl_xor_sync(0xffffffffu, b, 1);
    if (o1) { v[0] = a; v[2] = b; } else { v[1] = a; v[3] = b; }
    a = o2 ? v[0] : v[2];
    b = o2 ? v[1] : v[3];
    a = __shfl_xor_sync(0xffffffffu, a, 2);
    b = __shfl_xor_sync(0xffffffffu, b, 2);
    if (o2) { v[0] = a; v[1] = b; } else { v[2] = a; v[3] = b; }
}

inline __host__ __device__ bool aligned_to(const void *p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// One row of a warp tile out as bf16: lane t of the quad holds columns nt * 8 + 2t, + 1 of the N / 8
// column groups in x[nt][c], x[nt][c + 1].  Rows of 32 columns and more leave in 16-byte pieces where the
// destination is aligned to them (WIDE).
template <bool WIDE, int NT> __device__ __forceinline__ void store_row(bf16 *dst, const float (&x)[NT][4], int c, int t, bool act)
{
    if constexpr (WIDE && NT % 4 == 0) {
#pragma unroll
        for (int n4 = 0; n4 < NT; n4 += 4) {
            uint32_t v[4];
#pragma unroll
            for (int u = 0; u < 4; u++)
                v[u] = pack2(x[n4 + u][c], x[n4 + u][c + 1]);
            quad_transpose(v, t);
            if (act)
                *reinterpret_cast<uint4 *>(dst + (n4 + t) * 8) = make_uint4(v[0], v[1], v[2], v[3]);
        }
    } else {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
            if (act)
                *reinterpret_cast<uint32_t *>(dst + nt * 8 + 2 * t) = pack2(x[nt][c], x[nt][c + 1]);
    }
}

} // namespace fa
