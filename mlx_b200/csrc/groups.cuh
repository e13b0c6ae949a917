// The tables that the kernels of products grouped by expert make of the offsets in device memory.
#pragma once
#include <cstdint>

namespace luxcuda {

// Whole block, behind the wait for the kernel that wrote the offsets; ends with a barrier.  off[e], e <= experts: the experts' first rows, cut to
// [0, rows]; first[e]: how many pieces of work the experts before e have, pieces(n) of them for n rows.  Offsets that rise have `most` pieces
// at most (below 2^30); where others would have more, the rest is left out.
template <class Pieces>
__device__ __forceinline__ void group_tables(int* off, int* first, const int* offsets, int experts, int rows, int most, const Pieces& pieces) {
    for (int e = threadIdx.x; e <= experts; e += blockDim.x) off[e] = min(max(__ldcg(offsets + e), 0), rows);
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int before = 0;
        if (lane == 0) first[0] = 0;
        for (int e0 = 0; e0 < experts; e0 += 32) {
            const int e = e0 + lane, n = e < experts ? off[e + 1] - off[e] : 0;
            int sum = n > 0 ? min(pieces(n), most) : 0;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum = min(sum + v, most);
            }
            sum = min(sum + before, most);
            if (e < experts) first[e + 1] = sum;
            before = __shfl_sync(0xffffffffu, sum, 31);
        }
    }
    __syncthreads();
}

}  // namespace luxcuda
