// Root-mean-square norm of rows, with the addition of a residual and an 8-bit output, and the
// conversions that the storage types need.
//
//   h = x + residual,   r = 1 / sqrt(mean(h^2) + eps),   y = h r w
//
// In 8 bits a group of columns is held as codes q and one scale:  with v = h w and a = max |v|,
//   q = rint(v (127 / a)),   scale = a r / 127,   value = q scale.
// r cancels out of q, so the codes depend on no sum and no order.  a = 0: codes and scale 0; a
// infinite or NaN: codes 0 and scale NaN, so that every value of the group is NaN.
#include <algorithm>
#include <type_traits>

#include "cn_types.hpp"
#include "sequence.cuh"
#include "sequence.hpp"

namespace cn {

using namespace seq;

namespace {

template <typename T>
__global__ void __launch_bounds__(256) rms_norm_kernel(RmsNormArgs a) {
    using A = typename Acc<T>::type;
    __shared__ A sm[8];
    const int64_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.n;
    const T* res = a.residual ? (const T*)a.residual + row * a.n : nullptr;
    const T* w = (const T*)a.weight;
    A s = 0;
    for (int64_t i = threadIdx.x; i < a.n; i += 256) {
        A h = widen(x[i]);
        if (res) h += widen(res[i]);
        s += h * h;
    }
    s = block_sum(s, sm);
    const A r = A(1) / sqrt(s / (A)a.n + (A)a.eps);
    if (a.group == 0) {
        for (int64_t i = threadIdx.x; i < a.n; i += 256) {
            A h = widen(x[i]);
            if (res) {
                h += widen(res[i]);
                ((T*)a.h)[row * a.n + i] = narrow<T>(h);
            }
            ((T*)a.y)[row * a.n + i] = narrow<T>(h * r * (w ? widen(w[i]) : A(1)));
        }
        return;
    }
    const int64_t groups = (a.n + a.group - 1) / a.group;
    const int lane = threadIdx.x & 31;
    for (int64_t g = threadIdx.x >> 5; g < groups; g += 8) {
        const int64_t i0 = g * a.group, i1 = min(i0 + a.group, a.n);
        A most = 0;
        bool nan = false;
        for (int64_t i = i0 + lane; i < i1; i += 32) {
            A h = widen(x[i]);
            if (res) {
                h += widen(res[i]);
                ((T*)a.h)[row * a.n + i] = narrow<T>(h);
            }
            const A v = fabs(w ? h * widen(w[i]) : h);
            nan |= v != v;
            most = v > most ? v : most;
        }
        most = warp_max(most);
        const bool bad = __any_sync(0xffffffffu, nan) || isinf(most);
        const A f = most > 0 && !bad ? A(127) / most : A(0);
        for (int64_t i = i0 + lane; i < i1; i += 32) {
            A h = widen(x[i]);
            if (res) h += widen(res[i]);
            const A v = w ? h * widen(w[i]) : h;
            ((signed char*)a.y)[row * a.n + i] = bad ? 0 : (signed char)(int)rint(v * f);
        }
        if (lane == 0) ((A*)a.scale)[row * groups + g] = bad ? (A)NAN : most * r / A(127);
    }
}

// ---- conversions ------------------------------------------------------------------------------------

// one rounding, as the C conversion between the two types; 16 bits are reached from 64
template <typename To, typename From>
__device__ __forceinline__ To convert(From v) {
    if constexpr (std::is_same<From, __half>::value) return convert<To>(__half2float(v));
    else if constexpr (std::is_same<To, __half>::value) return __double2half((double)v);
    else return (To)v;
}

template <typename From, typename To>
__global__ void __launch_bounds__(256) convert_kernel(const From* in, To* out, int64_t size) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256)
        out[i] = convert<To>(in[i]);
}

template <typename To, typename S>
__global__ void __launch_bounds__(256)
dequantize_kernel(const signed char* in, const S* scale, To* out, int64_t rows, int64_t n, int64_t group, int64_t groups) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / n, col = i - row * n;
        out[i] = narrow<To>((typename Acc<To>::type)((S)in[i] * scale[row * groups + col / group]));
    }
}

template <typename From>
cudaError_t convert_from(const ConvertArgs& a, int grid, cudaStream_t s) {
    const int64_t size = a.rows * a.n;
    const From* in = (const From*)a.in;
    switch (a.to) {
        case DT_F32: convert_kernel<<<grid, 256, 0, s>>>(in, (float*)a.out, size); break;
        case DT_F64: convert_kernel<<<grid, 256, 0, s>>>(in, (double*)a.out, size); break;
        case DT_I32: convert_kernel<<<grid, 256, 0, s>>>(in, (int*)a.out, size); break;
        case DT_I64: convert_kernel<<<grid, 256, 0, s>>>(in, (long long*)a.out, size); break;
        case DT_F16: convert_kernel<<<grid, 256, 0, s>>>(in, (__half*)a.out, size); break;
        case DT_I8: convert_kernel<<<grid, 256, 0, s>>>(in, (signed char*)a.out, size); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

template <typename To>
cudaError_t dequantize_to(const ConvertArgs& a, int grid, cudaStream_t s) {
    const int64_t groups = (a.n + a.group - 1) / a.group;
    if (a.scale_dtype == DT_F64)
        dequantize_kernel<<<grid, 256, 0, s>>>((const signed char*)a.in, (const double*)a.scale, (To*)a.out, a.rows, a.n, a.group, groups);
    else
        dequantize_kernel<<<grid, 256, 0, s>>>((const signed char*)a.in, (const float*)a.scale, (To*)a.out, a.rows, a.n, a.group, groups);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rms_norm(const RmsNormArgs& a, int sm_count, cudaStream_t s) {
    (void)sm_count;
    if (a.rows >= (1LL << 31)) return cudaErrorInvalidValue;
    const int grid = (int)a.rows;
    switch (a.dtype) {
        case DT_F16: rms_norm_kernel<__half><<<grid, 256, 0, s>>>(a); break;
        case DT_F32: rms_norm_kernel<float><<<grid, 256, 0, s>>>(a); break;
        case DT_F64: rms_norm_kernel<double><<<grid, 256, 0, s>>>(a); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_convert(const ConvertArgs& a, int sm_count, cudaStream_t s) {
    const int grid = (int)std::min<int64_t>((a.rows * a.n + 255) / 256, (int64_t)sm_count * 16);
    if (grid < 1) return cudaSuccess;
    if (a.scale) {
        switch (a.to) {
            case DT_F32: return dequantize_to<float>(a, grid, s);
            case DT_F64: return dequantize_to<double>(a, grid, s);
            case DT_F16: return dequantize_to<__half>(a, grid, s);
            default: return cudaErrorInvalidValue;
        }
    }
    switch (a.from) {
        case DT_F32: return convert_from<float>(a, grid, s);
        case DT_F64: return convert_from<double>(a, grid, s);
        case DT_I32: return convert_from<int>(a, grid, s);
        case DT_I64: return convert_from<long long>(a, grid, s);
        case DT_F16: return convert_from<__half>(a, grid, s);
        case DT_I8: return convert_from<signed char>(a, grid, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace cn
