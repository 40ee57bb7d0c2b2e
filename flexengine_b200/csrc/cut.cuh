// Which way to go from a step of a row's tokens to the one that holds a limit (sampling_filtered.cu).  Plain C++ too, so that it can be tried without a GPU.
#pragma once

#ifdef __CUDACC__
#define FE_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define FE_HOST_DEVICE inline
#endif

namespace fe {

// -1: the limit is reached before the step, 1: it is not reached with it, 0: it lies in it.  ``before`` and ``here``: what the steps before
// and the step hold, in tokens or in mass.  The sum of the two is rounded once, as the next step's ``before`` is: then 1 here is never followed by -1 there.
// (Each rounded by itself, 1772367175443750147 and 501071425968473999 against 2273438601411224320 gave 1, and their sum -1: a walk without end.)
FE_HOST_DEVICE int cut_way(unsigned long long before, unsigned long long here, double limit) {
    if ((double)before >= limit) return -1;
    return (double)(before + here) < limit ? 1 : 0;
}

}  // namespace fe
