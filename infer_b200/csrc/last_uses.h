// Which phases of a ring's barriers nobody has waited for yet when the loop around it ends.
#pragma once

#ifdef __CUDACC__
#define IB_HD __host__ __device__ __forceinline__
#else
#define IB_HD inline
#endif

namespace ib {

// A ring of `slots` barriers: use u is of barrier u % slots and completes its phase u / slots; a loop of `uses` uses waits, before use u, for use u - slots.
// wait(barrier, parity) is called for the uses that are left, oldest first, and ends the rest by false. For arrivals from another CTA: once these waits have
// returned, every one has landed, so that the CTA may end.
template <typename Wait> IB_HD bool last_uses(int uses, int slots, Wait&& wait) {
    for (int u = uses > slots ? uses - slots : 0; u < uses; u++)
        if (!wait(u % slots, unsigned(u / slots) & 1u)) return false;
    return true;
}

}  // namespace ib
