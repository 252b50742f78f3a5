// Short causal convolution along time, one filter per channel, with a carried state.
//
//   y[b,t,c] = act(bias[c] + sum_j w[c,j] X[b, t-k+1+j, c])
//
// X continues x to negative times with the state, the k - 1 inputs before the first.  The new state
// is the last k - 1 rows of X; behind the end of a sequence y is 0.
#include <algorithm>

#include "cn_types.hpp"
#include "sequence.cuh"
#include "sequence.hpp"

namespace cn {

using namespace seq;

namespace {

template <typename T>
__global__ void __launch_bounds__(256) causal_conv_kernel(CausalConvArgs a) {
    using A = typename Acc<T>::type;
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.d) return;
    for (int64_t b = blockIdx.z; b < a.b; b += gridDim.z) {
    const int64_t end = a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.t) : a.t;
    const T* x = (const T*)a.x + b * a.t * a.d + c;
    const T* st = a.state ? (const T*)a.state + b * (a.k - 1) * a.d + c : nullptr;
    auto input = [&](int64_t t) -> T {
        if (t >= 0) return x[t * a.d];
        return st ? st[(t + a.k - 1) * a.d] : narrow<T>(A(0));
    };
    T* ns = (T*)a.new_state + b * (a.k - 1) * a.d + c;
    T keep[kMaxConvWidth - 1];
    if (blockIdx.y == 0)
        for (int j = 0; j < a.k - 1; ++j) keep[j] = input(end - a.k + 1 + j);
    for (int64_t t = blockIdx.y; t < a.t; t += gridDim.y) {
        A s = a.bias ? widen(((const T*)a.bias)[c]) : A(0);
        if (t < end) {
            for (int j = 0; j < a.k; ++j) s += widen(((const T*)a.weight)[c * a.k + j]) * widen(input(t - a.k + 1 + j));
            if (a.silu) s = s / (A(1) + exp(-s));
        }
        ((T*)a.y)[(b * a.t + t) * a.d + c] = t < end ? narrow<T>(s) : narrow<T>(A(0));
    }
    if (blockIdx.y == 0)
        for (int j = 0; j < a.k - 1; ++j) ns[j * a.d] = keep[j];
    }
}

}  // namespace

cudaError_t launch_causal_conv(const CausalConvArgs& a, int sm_count, cudaStream_t s) {
    (void)sm_count;
    const dim3 grid((unsigned)((a.d + 255) / 256), (unsigned)std::max<int64_t>(1, std::min<int64_t>(a.t, 1024)), (unsigned)std::min<int64_t>(a.b, 65535));
    switch (a.dtype) {
        case DT_F16: causal_conv_kernel<__half><<<grid, 256, 0, s>>>(a); break;
        case DT_F32: causal_conv_kernel<float><<<grid, 256, 0, s>>>(a); break;
        case DT_F64: causal_conv_kernel<double><<<grid, 256, 0, s>>>(a); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace cn
