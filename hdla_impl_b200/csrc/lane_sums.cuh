// Which of N sums a lane ends up with after scatter_sum (selective_scan.cuh) over M lanes, whose numbers differ in the bits
// from `low` on, and which lane stores it.  Plain C++, so that the lanes can be enumerated on the host.
#pragma once

#ifdef __CUDACC__
#define HDLA_LANES __host__ __device__ __forceinline__
#else
#define HDLA_LANES inline
#endif

namespace hdla {

// the first of the lane's max(1, N / M) sums
template <int N, int M>
HDLA_LANES int scatter_at(int lane, int low) {
    int n = N, at = 0;
    for (int m = 1; m < M; m <<= 1)
        if (n > 1) {
            n >>= 1;
            if (lane & (m * low)) at += n;
        }
    return at;
}
// Whether the lane is the one that stores them: with more lanes than sums (M > N) several lanes hold the same sum, and a sum
// that is added to memory must be added by one of them.
template <int N, int M>
HDLA_LANES bool scatter_owner(int lane, int low) {
    int n = N;
    for (int m = 1; m < M; m <<= 1) {
        if (n > 1) n >>= 1;
        else if (lane & (m * low)) return false;
    }
    return true;
}

}  // namespace hdla
