// Selective state space scan.
//
//   dt = softplus(delta[b,t,c] + delta_bias[c])
//   h[b,c,n] <- exp(dt A[c,n]) h[b,c,n] + dt B[b,t,g,n] x[b,t,c]
//   y[b,t,c] = (sum_n C[b,t,g,n] h[b,c,n] + D[c] x[b,t,c]) z / (1 + exp(-z))
//
// Behind the end of a sequence the states stay and y is 0.
#include <algorithm>

#include "cn_types.hpp"
#include "sequence.cuh"
#include "sequence.hpp"

namespace cn {

using namespace seq;

namespace {

// log(1 + e^v) without overflow
template <typename A>
__device__ __forceinline__ A softplus(A v) {
    return (v > 0 ? v : A(0)) + log1p(exp(-fabs(v)));
}

// One warp per channel and sequence, its lanes the states.
template <typename T>
__global__ void __launch_bounds__(128) selective_scan_kernel(SelectiveScanArgs a) {
    using A = typename Acc<T>::type;
    constexpr int kPer = kMaxScanStates / 32;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (at >= a.b * a.d) return;
    const int64_t b = at / a.d, c = at - b * a.d;
    const int lane = threadIdx.x & 31;
    const int64_t end = a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.t) : a.t;
    const int64_t bn = (int64_t)a.groups * a.n, g0 = c / (a.d / a.groups) * a.n;
    A h[kPer], decay[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int n = lane + 32 * i;
        h[i] = n < a.n && a.state ? ((const A*)a.state)[at * a.n + n] : A(0);
        decay[i] = n < a.n ? ((const A*)a.A)[c * a.n + n] : A(0);
    }
    const A skip = a.D ? ((const A*)a.D)[c] : A(0), db = a.delta_bias ? ((const A*)a.delta_bias)[c] : A(0);
    for (int64_t t = 0; t < a.t; ++t) {
        const int64_t i = (b * a.t + t) * a.d + c;
        A y = 0;
        if (t < end) {
            const A x = widen(((const T*)a.x)[i]);
            A dt = widen(((const T*)a.delta)[i]) + db;
            if (a.softplus) dt = softplus(dt);
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int n = lane + 32 * j;
                if (n >= a.n) continue;
                const int64_t k = (b * a.t + t) * bn + g0 + n;
                h[j] = exp(dt * decay[j]) * h[j] + dt * x * widen(((const T*)a.B)[k]);
                y += widen(((const T*)a.C)[k]) * h[j];
            }
            y = warp_sum(y) + skip * x;
            if (a.z) {
                const A z = widen(((const T*)a.z)[i]);
                y *= z / (A(1) + exp(-z));
            }
        }
        if (lane == 0) ((T*)a.y)[i] = narrow<T>(y);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int n = lane + 32 * i;
        if (n < a.n) ((A*)a.new_state)[at * a.n + n] = h[i];
    }
}

}  // namespace

size_t selective_scan_workspace(const SelectiveScanArgs& a, int sm_count) {
    (void)a;
    (void)sm_count;
    return 0;
}

cudaError_t launch_selective_scan(const SelectiveScanArgs& a, int sm_count, cudaStream_t s) {
    (void)sm_count;
    const int64_t blocks = (a.b * a.d + 3) / 4;
    if (blocks >= (1LL << 31)) return cudaErrorInvalidValue;
    switch (a.dtype) {
        case DT_F16: selective_scan_kernel<__half><<<(int)blocks, 128, 0, s>>>(a); break;
        case DT_F32: selective_scan_kernel<float><<<(int)blocks, 128, 0, s>>>(a); break;
        case DT_F64: selective_scan_kernel<double><<<(int)blocks, 128, 0, s>>>(a); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace cn
