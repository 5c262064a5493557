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
// count(s) workgroups; -1 past the last.  Every thread of a workgroup of NT
// calls it: thread i counts the i-th of NT runs of sequences, a scan over the
// threads finds the run, and its thread walks it.
template <int NT = 256, class F> __device__ __forceinline__ int find(int slot, int Bd, const F &count, int &place) {
    __shared__ int wsum[NT / 64], found[2];
    const int tid = threadIdx.x, lane = tid & 63;
    const int per = (Bd + NT - 1) / NT, s0 = min(tid * per, Bd), s1 = min(s0 + per, Bd);
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

// The sum of count(s) over sequences 0 .. n - 1, by a workgroup of NT threads.
template <int NT, class F> __device__ __forceinline__ int total(int n, const F &count) {
    __shared__ int wsum[NT / 64];
    int mine = 0;
    for (int s = threadIdx.x; s < n; s += NT) mine += count(s);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) mine += __shfl_xor(mine, o, 64);
    __syncthreads();   // an earlier call's sums are read
    if (threadIdx.x % 64 == 0) wsum[threadIdx.x / 64] = mine;
    __syncthreads();
    mine = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) mine += wsum[w];
    return __builtin_amdgcn_readfirstlane(mine);
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
