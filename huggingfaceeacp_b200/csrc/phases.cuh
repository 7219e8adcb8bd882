// The phases of an mbarrier, counted. Plain C++, so that it is tested without a GPU.
#pragma once

#ifdef __CUDACC__
#define HFK_BOTH __host__ __device__
#else
#define HFK_BOTH
#endif

namespace hfk
{
// The parity that a wait for the last of `begun` uses names (at least one): use n is
// phase n, and a wait with the other parity returns at once, whatever is in flight.
HFK_BOTH constexpr unsigned last_parity(int begun)
{
    return (unsigned) (begun - 1) & 1;
}
} // namespace hfk
