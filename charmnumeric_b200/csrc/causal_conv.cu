// Short causal convolution along time, one filter per channel, with a carried state.
//
//   y[b,t,c] = act(bias[c] + sum_j w[c,j] X[b, t-k+1+j, c])
//
// X continues x to negative times with the state, the k - 1 inputs before the first.  The new state
// is the last k - 1 rows of X; behind the end of a sequence y is 0.
//
// Bound by HBM: x is read and y written once.  A thread has V neighbouring channels (four where the channels
// allow, two of 64 bits) and walks a run of steps with the last inputs in registers, so that an input is
// loaded once but for the k - 1 in front of a run; eight steps' inputs are requested together.
// 4 x 4096 x 4096 channels, width 4, in 16 bits, full lengths, with state, bias and silu (268 MB, floor 41 us): 63.5 us,
// 67.4 with the new state's inputs held in registers from the start; widths 5, 6, 7, 8 at 2048 steps 47, 49, 51, 62 us
// (floor 20; 53 for the first three by the kernel of width 8).  In 32 bits 95 us (floor 82).
// Ways that were slower, in one comparison in which the form before took 59 us: eight channels and four steps
// together, which hold more of the registers for fewer blocks an SM, 92; four and four 62; runs of 64 steps as 32;
// 16 steps together and partial groups with a condition on every step 83 and more.
// 96 single tokens of 4100 channels in 32 bits: 12.3 to 6.2 us, most of it the launch.
#include <algorithm>

#include "cn_types.hpp"
#include "sequence.cuh"
#include "sequence.hpp"

namespace cn {

using namespace seq;

namespace {

constexpr int kThreads = 128;

// v / (1 + e^-v).  For 16 and 32 bits by the hardware's 2^x and 1 / x: a relative error of some 2^-22 and that of the
// 32-bit argument, |v| 2^-24, where the logistic is small; below what k products and sums of 32 bits leave in v.
__device__ __forceinline__ float silu(float v) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * v));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return v * r;
}
__device__ __forceinline__ double silu(double v) { return v / (1.0 + exp(-v)); }

// K: the width.  Every width has its own kernel: a filter that is filled up with zeros multiplies inputs that it
// does not reach, and 0 times an infinity is NaN.  Five blocks an SM where the filters and inputs leave the
// registers for it.  TOGETHER: steps whose inputs are requested together, 8, or 1 for single tokens (with the
// others' registers and code 10.2 instead of 6.2 us).
template <typename T, int V, int K, int TOGETHER>
__global__ void __launch_bounds__(kThreads, TOGETHER == 1 ? 1 : K <= 4 && sizeof(T) <= 4 ? 5 : 3) causal_conv_kernel(CausalConvArgs a, int64_t run, int64_t runs) {
    using A = typename Acc<T>::type;
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x, across = a.d / V;
    if (id >= across * runs) return;
    const int64_t c = id % across * V, t0 = id / across * run, t1 = min(t0 + run, a.t);
    A w[K][V], bias[V];
    if constexpr (V * sizeof(T) >= 8 && K < kMaxConvWidth) {
        // the filters of V channels are K pieces of V values
        T f[K * V];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const Pack<T, V> p = *(const Pack<T, V>*)((const T*)a.weight + c * K + i * V);
#pragma unroll
            for (int v = 0; v < V; ++v) f[i * V + v] = p.v[v];
        }
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) w[j][v] = widen(f[v * K + j]);
    } else {
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) w[j][v] = widen(((const T*)a.weight)[(c + v) * K + j]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) bias[v] = a.bias ? widen(((const T*)a.bias)[c + v]) : A(0);
    Pack<T, V> zero;
#pragma unroll
    for (int v = 0; v < V; ++v) zero.v[v] = narrow<T>(A(0));

    for (int64_t b = blockIdx.y; b < a.b; b += gridDim.y) {
        const int64_t end = a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.t) : a.t;
        const T* const xs = (const T*)a.x + b * a.t * a.d + c;
        const T* const before = a.state ? (const T*)a.state + b * (K - 1) * a.d + c : nullptr;
        T* const ys = (T*)a.y + b * a.t * a.d + c;
        T* const after = (T*)a.new_state + b * (K - 1) * a.d + c;
        auto input = [&](int64_t t) -> Pack<T, V> {
            if (t >= 0) return *(const Pack<T, V>*)(xs + t * a.d);
            return before ? *(const Pack<T, V>*)(before + (t + K - 1) * a.d) : zero;
        };
        // the first run's threads carry the state: for a single step, where it may be the same array, read before
        // and written behind everything else; for longer ones read there too, which holds no registers
        Pack<T, V> keep[K - 1];
        auto carry = [&]() {
#pragma unroll
            for (int j = 0; j < K - 1; ++j) keep[j] = input(end - K + 1 + j);
        };
        if (TOGETHER == 1 && t0 == 0) carry();
        const int64_t live = min(t1, end);
        int64_t t = t0;
        if (t < live) {
            A win[K - 1][V];
            Pack<T, V> first[K - 1];
            if (t0 >= K - 1) {
#pragma unroll
                for (int j = 0; j < K - 1; ++j) first[j] = *(const Pack<T, V>*)(xs + (t0 - K + 1 + j) * a.d);
            } else {
#pragma unroll
                for (int j = 0; j < K - 1; ++j) first[j] = input(t0 - K + 1 + j);
            }
#pragma unroll
            for (int j = 0; j < K - 1; ++j)
#pragma unroll
                for (int v = 0; v < V; ++v) win[j][v] = widen(first[j].v[v]);
            auto step = [&](const Pack<T, V>& p, T* to) {
                Pack<T, V> y;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const A x = widen(p.v[v]);
                    A s = bias[v];
#pragma unroll
                    for (int j = 0; j < K - 1; ++j) s += w[j][v] * win[j][v];
                    s += w[K - 1][v] * x;
#pragma unroll
                    for (int j = 0; j < K - 2; ++j) win[j][v] = win[j + 1][v];
                    win[K - 2][v] = x;
                    y.v[v] = narrow<T>(a.silu ? silu(s) : s);
                }
                *(Pack<T, V>*)to = y;
            };
            const T* from = xs + t * a.d;
            T* to = ys + t * a.d;
            if constexpr (TOGETHER == 1) {
                for (; t < live; ++t, from += a.d, to += a.d) step(*(const Pack<T, V>*)from, to);
            } else {
                Pack<T, V> p[TOGETHER];
                for (; t + TOGETHER <= live; t += TOGETHER) {
#pragma unroll
                    for (int i = 0; i < TOGETHER; ++i, from += a.d) p[i] = *(const Pack<T, V>*)from;
#pragma unroll
                    for (int i = 0; i < TOGETHER; ++i, to += a.d) step(p[i], to);
                }
                // the last few, together too
                const int rest = (int)(live - t);
#pragma unroll
                for (int i = 0; i < TOGETHER - 1; ++i, from += a.d)
                    if (i < rest) p[i] = *(const Pack<T, V>*)from;
#pragma unroll
                for (int i = 0; i < TOGETHER - 1; ++i, to += a.d)
                    if (i < rest) step(p[i], to);
                t = live;
            }
        }
        for (; t < t1; ++t) *(Pack<T, V>*)(ys + t * a.d) = zero;
        if (t0 == 0) {
            if (TOGETHER != 1) carry();
#pragma unroll
            for (int j = 0; j < K - 1; ++j) *(Pack<T, V>*)(after + j * a.d) = keep[j];
        }
    }
}

template <typename T, int V, int K>
cudaError_t conv(const CausalConvArgs& a, int sm_count, cudaStream_t s) {
    // Runs long enough that the k - 1 inputs in front of them are a small part (32 steps and more),
    // as long as every SM has 16 warps; shorter ones down to 8 steps to get there
    const int64_t across = a.d / V, threads = (int64_t)sm_count * 512;
    int64_t run = 32;
    while (run > 8 && across * a.b * ((a.t + run - 1) / run) < threads) run /= 2;
    const int64_t runs = std::max<int64_t>((a.t + run - 1) / run, 1), blocks = (across * runs + kThreads - 1) / kThreads;
    if (blocks >= (1LL << 31)) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)blocks, (unsigned)std::min<int64_t>(a.b, 65535));
    if (a.t == 1) causal_conv_kernel<T, V, K, 1><<<grid, kThreads, 0, s>>>(a, run, runs);
    else causal_conv_kernel<T, V, K, 8><<<grid, kThreads, 0, s>>>(a, run, runs);
    return cudaGetLastError();
}

template <typename T, int V>
cudaError_t conv(const CausalConvArgs& a, int sm_count, cudaStream_t s) {
    switch (a.k) {
        case 2: return conv<T, V, 2>(a, sm_count, s);
        case 3: return conv<T, V, 3>(a, sm_count, s);
        case 4: return conv<T, V, 4>(a, sm_count, s);
        case 5: return conv<T, V, 5>(a, sm_count, s);
        case 6: return conv<T, V, 6>(a, sm_count, s);
        case 7: return conv<T, V, 7>(a, sm_count, s);
        case kMaxConvWidth: return conv<T, V, kMaxConvWidth>(a, sm_count, s);
        default: return cudaErrorInvalidValue;
    }
}

template <typename T>
cudaError_t conv(const CausalConvArgs& a, int sm_count, cudaStream_t s) {
    constexpr int V = sizeof(T) == 8 ? 2 : 4;
    if (a.d % V == 0) return conv<T, V>(a, sm_count, s);
    if (V > 2 && a.d % 2 == 0) return conv<T, 2>(a, sm_count, s);
    return conv<T, 1>(a, sm_count, s);
}

}  // namespace

cudaError_t launch_causal_conv(const CausalConvArgs& a, int sm_count, cudaStream_t s) {
    switch (a.dtype) {
        case DT_F16: return conv<__half>(a, sm_count, s);
        case DT_F32: return conv<float>(a, sm_count, s);
        case DT_F64: return conv<double>(a, sm_count, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace cn
