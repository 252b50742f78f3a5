// Launchers of the sequence model operators: root-mean-square norm, short causal convolution,
// selective state space scan, sampling, and the conversions of the storage types.  Every launcher
// enqueues on the given stream, allocates nothing and returns the CUDA status of the launch.
//
// Arrays are dense and row-major.  `dtype` is that of the activations (DT_F16, DT_F32 or DT_F64);
// sums, statistics and states are held in the accumulator type: float for DT_F16 and DT_F32,
// double for DT_F64.  A null pointer stands for an operand that was left out.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace cn {

// h = x + residual; r = 1 / sqrt(mean(h^2) + eps); y = h r weight.
struct RmsNormArgs {
    const void* x = nullptr;
    const void* residual = nullptr;
    const void* weight = nullptr;
    void* y = nullptr;              // dtype, or int8 codes where group > 0
    void* scale = nullptr;          // accumulator type, one per row and group of columns
    void* h = nullptr;              // the sum, where there is a residual
    int64_t rows = 0, n = 0;
    int64_t group = 0;              // columns per scale of the 8-bit output; 0: y in dtype
    double eps = 0;
    int dtype = 0;
};
cudaError_t launch_rms_norm(const RmsNormArgs& a, int sm_count, cudaStream_t s);

// y[b,t,c] = act(bias[c] + sum_j weight[c,j] X[b,t-k+1+j,c]), X = state for negative times.
struct CausalConvArgs {
    const void* x = nullptr;        // (b, t, d)
    const void* weight = nullptr;   // (d, k)
    const void* bias = nullptr;     // (d)
    const void* state = nullptr;    // (b, k-1, d): the inputs before the first
    const int* lengths = nullptr;   // (b): tokens of each sequence, clipped to [0, t]
    void* y = nullptr;
    void* new_state = nullptr;      // (b, k-1, d); may be `state` itself where t == 1
    int64_t b = 0, t = 0, d = 0;
    int k = 0;
    bool silu = false;
    int dtype = 0;
};
cudaError_t launch_causal_conv(const CausalConvArgs& a, int sm_count, cudaStream_t s);
constexpr int kMaxConvWidth = 8;

// h[b,c,n] <- exp(dt A[c,n]) h + dt B[b,t,g,n] x[b,t,c];  y = sum_n C[b,t,g,n] h + D[c] x,
// times z sigmoid(z); dt = softplus(delta + delta_bias) or the sum itself; g = c / (d / groups).
struct SelectiveScanArgs {
    const void* x = nullptr;           // (b, t, d)
    const void* delta = nullptr;       // (b, t, d)
    const void* A = nullptr;           // (d, n), accumulator type
    const void* B = nullptr;           // (b, t, groups n)
    const void* C = nullptr;           // (b, t, groups n)
    const void* D = nullptr;           // (d), accumulator type
    const void* z = nullptr;           // (b, t, d)
    const void* delta_bias = nullptr;  // (d), accumulator type
    const void* state = nullptr;       // (b, d, n), accumulator type
    const int* lengths = nullptr;      // (b)
    void* y = nullptr;                 // (b, t, d)
    void* new_state = nullptr;         // (b, d, n); may be `state` itself where t == 1
    int64_t b = 0, t = 0, d = 0;
    int n = 0, groups = 1;
    bool softplus = true;
    int dtype = 0;
    void* workspace = nullptr;         // selective_scan_workspace() bytes
};
constexpr int kMaxScanStates = 256;
size_t selective_scan_workspace(const SelectiveScanArgs& a, int sm_count);
cudaError_t launch_selective_scan(const SelectiveScanArgs& a, int sm_count, cudaStream_t s);

// A parameter of the sampler: one value, or one of each row.
struct RowParam {
    const void* data = nullptr;
    int dtype = 0;      // DT_F32, DT_F64 or DT_I32
    double value = 0;   // where data is null
};
struct SampleArgs {
    const void* logits = nullptr;   // (rows, v)
    const void* u = nullptr;        // (rows)
    int u_dtype = 0;                // DT_F32 or DT_F64
    RowParam temperature, top_k, top_p, min_p;
    int* token = nullptr;           // (rows)
    void* logp = nullptr;           // (rows), accumulator type
    int64_t rows = 0, v = 0;
    int dtype = 0;
};
constexpr int64_t kMaxVocabulary = 1LL << 24;
cudaError_t launch_sample(const SampleArgs& a, int sm_count, cudaStream_t s);

// out = in converted to `to`, times scale[row, column / group] where there is a scale (of `scale_dtype`).
struct ConvertArgs {
    const void* in = nullptr;
    void* out = nullptr;
    const void* scale = nullptr;
    int from = 0, to = 0, scale_dtype = 0;
    int64_t rows = 0, n = 0, group = 1;
};
cudaError_t launch_convert(const ConvertArgs& a, int sm_count, cudaStream_t s);

}  // namespace cn
