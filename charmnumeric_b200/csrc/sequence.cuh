// Device helpers shared by the sequence model operators: element conversions, wide loads and
// stores, and sums over a warp or a block.
#pragma once
#include <cuda_fp16.h>

#include <cstdint>

namespace cn {
namespace seq {

// accumulator type of an element type
template <typename T> struct Acc { using type = float; };
template <> struct Acc<double> { using type = double; };

__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }

// one rounding to the nearest value of the element type
template <typename T> __device__ __forceinline__ T narrow(typename Acc<T>::type v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements, moved as one access of V * sizeof(T) bytes (a power of two up to 16, aligned)
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

template <typename A>
__device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename A>
__device__ __forceinline__ A warp_max(A v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const A w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
}

// Sum over a block of whole warps, in every thread, always in the same order: a butterfly in each
// warp (both partners add the same two values), then the warps' sums in the order of the warps.
// `sm` has one entry per warp and may be used again behind the next barrier.
template <typename A>
__device__ __forceinline__ A block_sum(A v, A* sm) {
    v = warp_sum(v);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    A t = 0;
    for (int w = 0; w < warps; ++w) t += sm[w];
    return t;
}

}  // namespace seq
}  // namespace cn
