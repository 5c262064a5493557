// Ragged batches: tokens cu[s] .. cu[s + 1] - 1 of a packed array are sequence s's.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hba {
namespace ragged {

// Tokens of sequence s: the first one's place and how many (cu is clamped to the
// packed array, so a wrong one reads nothing outside it).
__device__ __forceinline__ int tokens(const int32_t *cu, int s, int T, int &first) {
    first = max(0, min(T, cu[s]));
    return max(0, min(T, cu[s + 1]) - first);
}

// The sequence and the place in it of workgroup `slot`, where sequence s has
// count(s) workgroups; -1 past the last.  Every thread of a workgroup of 256
// calls it: thread i counts the i-th of 256 runs of sequences, a scan over the
// threads finds the run, and its thread walks it.
template <class F> __device__ __forceinline__ int find(int slot, int Bd, const F &count, int &place) {
    __shared__ int wsum[4], found[2];
    const int tid = threadIdx.x, lane = tid & 63;
    const int per = (Bd + 255) / 256, s0 = min(tid * per, Bd), s1 = min(s0 + per, Bd);
    int mine = 0;
    for (int s = s0; s < s1; ++s) mine += count(s);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(upto, o, 64);
        if (lane >= o) upto += x;
    }
    if (lane == 63) wsum[tid >> 6] = upto;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    for (int i = 0; i < (tid >> 6); ++i) upto += wsum[i];
    int at = upto - mine;
    if (slot >= at && slot < upto) {
        int s = s0, c = 0;
        for (; s < s1; ++s) {
            c = count(s);
            if (slot < at + c) break;
            at += c;
        }
        found[0] = s;
        found[1] = slot - at;
    }
    __syncthreads();
    place = found[1];
    return __builtin_amdgcn_readfirstlane(found[0]);
}

// The sequence of token t (the last s with cu[s] <= t).
__device__ __forceinline__ int sequence(const int32_t *cu, int Bd, int t) {
    int lo = 0, hi = Bd - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

}  // namespace ragged
}  // namespace hba
