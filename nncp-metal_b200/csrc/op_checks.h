// op_checks.h -- checks that the isolated operators make of their tensors.
#pragma once
#include <initializer_list>

#include "attention_deal.h"
#include "common.cuh"

using attn::SMS;

static inline bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Every tensor lies in memory of the current device (or in managed memory): a host address, or one of another
// device, would fault in the kernel.
static inline int on_device(std::initializer_list<const void *> tensors)
{
    int dev = -1;
    CUDA_TRY(cudaGetDevice(&dev));
    for (const void *t : tensors) {
        if (!t)
            continue;
        cudaPointerAttributes at;
        CUDA_TRY(cudaPointerGetAttributes(&at, t));
        if (at.type != cudaMemoryTypeManaged && (at.type != cudaMemoryTypeDevice || at.device != dev))
            return nncu_fail(NNCU_ERR_INVALID, "a tensor does not lie in the memory of device %d, the current one", dev);
    }
    return NNCU_OK;
}

static inline int elements_aligned(std::initializer_list<const void *> tensors, size_t bytes)
{
    for (const void *t : tensors)
        if (!aligned(t, bytes))
            return nncu_fail(NNCU_ERR_INVALID, "a tensor does not begin at a multiple of its element size");
    return NNCU_OK;
}
