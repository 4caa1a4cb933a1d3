// copy_ring.h -- asynchronous copies into places that take turns, a barrier each: which phase of which barrier a copy
// completes.  Plain C++, so that the order can be checked without a GPU.
#pragma once

#ifdef __CUDACC__
#define RING_HD __host__ __device__
#else
#define RING_HD
#endif

// Copies are asked for in order, the j-th into place j % places.
struct CopyRing {
    int places;
    int asked = 0; // so far, by the thread that asks
    RING_HD explicit CopyRing(int n) : places(n) {}
    RING_HD int place(int j) const { return j % places; }
    RING_HD int parity(int j) const { return j / places & 1; }
    // The copies that may be on their way still when no more are asked for: the last one into each place.  f(place, parity).
    template <typename F> RING_HD void each_open(F f) const
    {
        for (int j = asked > places ? asked - places : 0; j < asked; j++)
            f(place(j), parity(j));
    }
};
