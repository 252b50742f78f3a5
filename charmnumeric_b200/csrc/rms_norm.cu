// Root-mean-square norm of rows, with the addition of a residual and an 8-bit output, and the
// conversions that the storage types need.
//
//   h = x + residual,   r = 1 / sqrt(mean(h^2) + eps),   y = h r w
//
// In 8 bits a group of columns is held as codes q and one scale:  with v = h w and a = max |v|,
//   q = rint(v ((1 / a) 127)),   scale = a r / 127,   value = q scale.
// r cancels out of q, so the codes depend on no sum and no order.  a = 0, or so small that 1 / a
// overflows: codes and scale 0; a infinite or NaN: codes 0 and scale NaN, so that every value of the
// group is NaN.
#include <algorithm>
#include <type_traits>

#include "cn_types.hpp"
#include "sequence.cuh"
#include "sequence.hpp"

namespace cn {

using namespace seq;

namespace {

// A row is read once and stays in registers: W warps have a row, a thread R pieces of V neighbouring
// values (16 bytes), W * 32 pieces apart.  Bound by HBM.  One warp a row for short rows (no barrier;
// four rows a block), up to 32 for long ones; rows longer than that are read twice, the second time
// from L2.  Pieces begin at 16-byte borders of the arrays, which all have the same ones: where n is no
// multiple of V a row's first and last piece are partly its neighbours' (WHOLE = false) and are moved
// value by value.
// 8192 rows of 4096 in 16 bits with a residual: 268 MB in 44 us, 6.1 TB/s (93 % of a copy's rate).
// 1531 rows of 5003 in 32 bits, odd places: 24.8 us, 123 MB.
template <typename T, int V, int R, int W, bool RESIDUAL, bool WHOLE>
struct Row {
    using A = typename Acc<T>::type;
    int64_t base;            // of the row in its array
    int n, first;            // column of this thread's first value; before column 0 for some first pieces
    Pack<T, V> x[R], r[RESIDUAL ? R : 1];

    __device__ __forceinline__ int at(int i) const { return first + i * (W * 32 * V); }
    __device__ __forceinline__ bool any(int i) const { return at(i) < n; }
    __device__ __forceinline__ bool all(int i) const { return WHOLE || (at(i) >= 0 && at(i) + V <= n); }
    __device__ __forceinline__ bool has(int i, int j) const { return WHOLE || (at(i) + j >= 0 && at(i) + j < n); }

    // piece i of an array of rows; what is not the row's is left as it is
    template <typename U>
    __device__ __forceinline__ void get(Pack<U, V>& to, const U* from, int i) const {
        if (all(i)) {
            to = *(const Pack<U, V>*)(from + base + at(i));
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (has(i, j)) to.v[j] = from[base + at(i) + j];
        }
    }
    template <typename U>
    __device__ __forceinline__ void put(const Pack<U, V>& from, U* to, int i) const {
        if (all(i)) {
            *(Pack<U, V>*)(to + base + at(i)) = from;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (has(i, j)) to[base + at(i) + j] = from.v[j];
        }
    }
    __device__ __forceinline__ void load(const RmsNormArgs& a, int64_t row, int tid) {
        base = row * a.n;
        n = (int)a.n;
        first = tid * V - (WHOLE ? 0 : (int)(base % V));
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (!any(i)) break;
            get(x[i], (const T*)a.x, i);
            if (RESIDUAL) get(r[i], (const T*)a.residual, i);
        }
    }
    // columns of the weight, which begin at other borders than a row's
    __device__ __forceinline__ void weight(A (&w)[V], const RmsNormArgs& a, int i) const {
        if (WHOLE && a.weight) {
            const Pack<T, V> v = *(const Pack<T, V>*)((const T*)a.weight + at(i));
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = widen(v.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = a.weight && has(i, j) ? widen(((const T*)a.weight)[at(i) + j]) : A(1);
        }
    }
    __device__ __forceinline__ A sum(int i, int j) const {
        const A v = widen(x[i].v[j]);
        return RESIDUAL ? v + widen(r[i].v[j]) : v;
    }
};

// the factor from values to codes; 0 where the codes are
template <typename A>
__device__ __forceinline__ A code_factor(A most) {
    const A f = A(1) / most * A(127);
    return most > 0 && most < (A)INFINITY && f < (A)INFINITY ? f : A(0);
}
template <typename A>
__device__ __forceinline__ A scale_of(A most, A factor, A r) {
    return !(most < (A)INFINITY) ? (A)NAN : factor > 0 ? most * r / A(127) : A(0);
}

template <typename A>
__device__ __forceinline__ A root(A squares, const RmsNormArgs& a) {
    return A(1) / sqrt(squares / (A)a.n + (A)a.eps);
}

template <typename T, int V, int R, int W, bool RESIDUAL, bool WHOLE>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) rms_norm_kernel(RmsNormArgs a) {
    using A = typename Acc<T>::type;
    const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;
    Row<T, V, R, W, RESIDUAL, WHOLE> in;
    in.load(a, row, W == 1 ? threadIdx.x & 31 : threadIdx.x);
    A s = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (!in.any(i)) break;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const A h = in.sum(i, j);
            if (in.has(i, j)) s += h * h;
        }
    }
    if (W == 1) {
        s = warp_sum(s);
    } else {
        __shared__ A sm[W];
        s = block_sum(s, sm);
    }
    const A r = root(s, a);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (!in.any(i)) break;
        Pack<T, V> y, h;
        A w[V];
        in.weight(w, a, i);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const A v = in.sum(i, j);
            h.v[j] = narrow<T>(v);
            y.v[j] = narrow<T>(v * r * w[j]);
        }
        in.put(y, (T*)a.y, i);
        if (RESIDUAL) in.put(h, (T*)a.h, i);
    }
}

// The larger of a value (of at least 0, or NaN) and |v|, where NaN is the largest: as integers the bits are
// in that order.
__device__ __forceinline__ float most_of(float most, float v) {
    return __uint_as_float(max(__float_as_uint(most), __float_as_uint(v) & 0x7fffffffu));
}
__device__ __forceinline__ double most_of(double most, double v) {
    return __longlong_as_double(max(__double_as_longlong(most), __double_as_longlong(v) & 0x7fffffffffffffffLL));
}

// v f, rounded to the nearest whole number of -127 to 127.  Added to 1.5 2^23 (2^52) the number is in the
// last bits; no product may go into that sum.
__device__ __forceinline__ signed char code_of(float v, float f) {
    return (signed char)__float_as_uint(__fadd_rn(__fmul_rn(v, f), 12582912.0f));
}
__device__ __forceinline__ signed char code_of(double v, double f) {
    return (signed char)__double_as_longlong(__dadd_rn(__dmul_rn(v, f), 6755399441055744.0));
}

// The same with the 8-bit output.  The lanes that share a group of columns find its largest value
// together: G lanes for groups of G pieces (a power of two up to a warp), or the whole block for one
// scale a row (G = 0).  h is stored, and h w kept, before the row's sum is known.
// 8192 rows of 4096 in 16 bits with a residual, groups of 128: 235 MB in 47 us, 5.0 TB/s; the issue slots are
// three quarters busy with roundings and maxima.
template <typename T, int V, int R, int W, int G, bool RESIDUAL, bool WHOLE>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) rms_norm_8_kernel(RmsNormArgs a) {
    using A = typename Acc<T>::type;
    const int tid = W == 1 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;
    Row<T, V, R, W, RESIDUAL, WHOLE> in;
    in.load(a, row, tid);
    A s = 0, most[R], v[R][V];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        most[i] = 0;
        if (in.any(i)) {
            A w[V];
            Pack<T, V> h;
            in.weight(w, a, i);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const A x = in.sum(i, j);
                h.v[j] = narrow<T>(x);
                v[i][j] = x * w[j];
                if (!in.has(i, j)) continue;
                s += x * x;
                most[i] = most_of(most[i], v[i][j]);
            }
            if (RESIDUAL) in.put(h, (T*)a.h, i);
        }
    }
    __shared__ A sm[W], sm_most[W];
    if (G == 0) {
#pragma unroll
        for (int i = 1; i < R; ++i) most[0] = most_of(most[0], most[i]);
    }
#pragma unroll
    for (int i = 0; i < (G == 0 ? 1 : R); ++i)
#pragma unroll
        for (int o = (G == 0 ? 16 : G / 2); o > 0; o >>= 1) most[i] = most_of(most[i], __shfl_xor_sync(0xffffffffu, most[i], o));
    if (G == 0 && W > 1 && (tid & 31) == 0) sm_most[tid >> 5] = most[0];
    s = W == 1 ? warp_sum(s) : block_sum(s, sm);    // its barrier covers sm_most
    if (G == 0) {
        if (W > 1)
#pragma unroll
            for (int i = 0; i < W; ++i) most[0] = most_of(most[0], sm_most[i]);
#pragma unroll
        for (int i = 1; i < R; ++i) most[i] = most[0];
    }
    const A r = root(s, a);
    const int64_t groups = (a.n + a.group - 1) / a.group;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (!in.any(i)) break;
        const A f = code_factor(most[i]);
        Pack<signed char, V> q;
#pragma unroll
        for (int j = 0; j < V; ++j) q.v[j] = f > 0 ? code_of(v[i][j], f) : (signed char)0;
        in.put(q, (signed char*)a.y, i);
        if (G == 0 ? tid == 0 && i == 0 : tid % (G ? G : 1) == 0)
            ((A*)a.scale)[row * groups + (G == 0 ? 0 : in.at(i) / (int)a.group)] = scale_of(most[i], f, r);
    }
}

// Any length, any group, any alignment; a block a row, which is read again for the results.  The simple kernel, value by
// value and a warp a group: 8192 rows of 4096 in 16 bits with a residual and their values, groups of 100 226 us, of 512
// 138, 4097 columns in groups of 128 199 (82 for groups of 128 in registers); 256 rows of 70000 in 32 bits with one scale
// 2482, of which one warp a row has most.
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_long_kernel(RmsNormArgs a) {
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
    const A r = root(s, a);
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
        for (int64_t i = i0 + lane; i < i1; i += 32) {
            A h = widen(x[i]);
            if (res) {
                h += widen(res[i]);
                ((T*)a.h)[row * a.n + i] = narrow<T>(h);
            }
            most = most_of(most, w ? h * widen(w[i]) : h);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = most_of(most, __shfl_xor_sync(0xffffffffu, most, o));
        const A f = code_factor(most);
        for (int64_t i = i0 + lane; i < i1; i += 32) {
            A h = widen(x[i]);
            if (res) h += widen(res[i]);
            const A v = w ? h * widen(w[i]) : h;
            ((signed char*)a.y)[row * a.n + i] = f > 0 ? code_of(v, f) : (signed char)0;
        }
        if (lane == 0) ((A*)a.scale)[row * groups + g] = scale_of(most, f, r);
    }
}

// ---- variants ---------------------------------------------------------------------------------------------

template <typename T, int V, int R, int W, bool WHOLE>
cudaError_t launch_row(const RmsNormArgs& a, cudaStream_t s) {
    const unsigned blocks = (unsigned)(W == 1 ? (a.rows + 3) / 4 : a.rows), threads = W == 1 ? 128 : W * 32;
    if (a.residual) rms_norm_kernel<T, V, R, W, true, WHOLE><<<blocks, threads, 0, s>>>(a);
    else rms_norm_kernel<T, V, R, W, false, WHOLE><<<blocks, threads, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int V, int R, int W, int G, bool WHOLE>
cudaError_t launch_row_8(const RmsNormArgs& a, cudaStream_t s) {
    const unsigned blocks = (unsigned)(W == 1 ? (a.rows + 3) / 4 : a.rows), threads = W == 1 ? 128 : W * 32;
    if (a.residual) rms_norm_8_kernel<T, V, R, W, G, true, WHOLE><<<blocks, threads, 0, s>>>(a);
    else rms_norm_8_kernel<T, V, R, W, G, false, WHOLE><<<blocks, threads, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_long(const RmsNormArgs& a, cudaStream_t s) {
    rms_norm_long_kernel<T><<<(unsigned)a.rows, 256, 0, s>>>(a);
    return cudaGetLastError();
}

// One warp for up to 4 pieces a thread, else as few warps (4 to 32) as hold the row in 4, in 3 where that
// does: threads without a piece cost (1531 rows of 5003 floats: 28.0 us in 4 by 16 warps, 24.8 in 3).
template <typename T, bool WHOLE>
cudaError_t by_length(const RmsNormArgs& a, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int64_t pieces = (a.n + V - 1) / V + !WHOLE;
    if (pieces <= 32) return launch_row<T, V, 1, 1, WHOLE>(a, s);
    if (pieces <= 128) return launch_row<T, V, 4, 1, WHOLE>(a, s);
    if (pieces <= 256) return launch_row<T, V, 2, 4, WHOLE>(a, s);
    if (pieces <= 384) return launch_row<T, V, 3, 4, WHOLE>(a, s);
    if (pieces <= 512) return launch_row<T, V, 4, 4, WHOLE>(a, s);
    if (pieces <= 768) return launch_row<T, V, 3, 8, WHOLE>(a, s);
    if (pieces <= 1024) return launch_row<T, V, 4, 8, WHOLE>(a, s);
    if (pieces <= 1536) return launch_row<T, V, 3, 16, WHOLE>(a, s);
    if (pieces <= 2048) return launch_row<T, V, 4, 16, WHOLE>(a, s);
    if (pieces <= 4096) return launch_row<T, V, 4, 32, WHOLE>(a, s);
    return launch_long<T>(a, s);
}

template <typename T, int G, bool WHOLE>
cudaError_t by_length_8(const RmsNormArgs& a, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int64_t pieces = (a.n + V - 1) / V + !WHOLE;
    if (pieces <= 128) return launch_row_8<T, V, 4, 1, G, WHOLE>(a, s);
    if (pieces <= 512) return launch_row_8<T, V, 4, 4, G, WHOLE>(a, s);
    if (pieces <= 1024) return launch_row_8<T, V, 4, 8, G, WHOLE>(a, s);
    if (pieces <= 2048) return launch_row_8<T, V, 4, 16, G, WHOLE>(a, s);
    return launch_long<T>(a, s);
}

template <typename T>
cudaError_t rms_norm(const RmsNormArgs& a, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool whole = a.n % V == 0;
    if (a.group == 0) return whole ? by_length<T, true>(a, s) : by_length<T, false>(a, s);
    if (a.group >= a.n) return whole ? by_length_8<T, 0, true>(a, s) : by_length_8<T, 0, false>(a, s);
    // groups of a power of two of pieces are shared by neighbouring lanes
    if (whole && a.group == 4 * V) return by_length_8<T, 4, true>(a, s);
    if (whole && a.group == 8 * V) return by_length_8<T, 8, true>(a, s);
    if (whole && a.group == 16 * V) return by_length_8<T, 16, true>(a, s);
    if (whole && a.group == 32 * V) return by_length_8<T, 32, true>(a, s);
    return launch_long<T>(a, s);
}

// ---- conversions ------------------------------------------------------------------------------------

// one rounding, as the C conversion between the two types; 16 bits are reached from 64
template <typename To, typename From>
__device__ __forceinline__ To convert(From v) {
    if constexpr (std::is_same<From, __half>::value) return convert<To>(__half2float(v));
    else if constexpr (std::is_same<To, __half>::value) return __double2half((double)v);
    else return (To)v;
}

// four values a thread and turn: one access of up to 16 (or two) bytes a value
template <typename From, typename To>
__global__ void __launch_bounds__(256) convert_kernel(const From* in, To* out, int64_t size) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i + 4 <= size) {
        Pack<From, 4> v;
        if constexpr (sizeof(From) == 8) {
            *(Pack<From, 2>*)&v.v[0] = *(const Pack<From, 2>*)(in + i);
            *(Pack<From, 2>*)&v.v[2] = *(const Pack<From, 2>*)(in + i + 2);
        } else {
            v = *(const Pack<From, 4>*)(in + i);
        }
        Pack<To, 4> w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w.v[j] = convert<To>(v.v[j]);
        if constexpr (sizeof(To) == 8) {
            *(Pack<To, 2>*)(out + i) = *(Pack<To, 2>*)&w.v[0];
            *(Pack<To, 2>*)(out + i + 2) = *(Pack<To, 2>*)&w.v[2];
        } else {
            *(Pack<To, 4>*)(out + i) = w;
        }
    } else {
        for (int64_t k = i; k < size; ++k) out[k] = convert<To>(in[k]);
    }
}

// code * scale, rounded once.  Into fewer bits than a product of the scale's type has, the product is first cut to the
// neighbour whose last bit is 1 where it is not exact: that one lies on the same side of every border between values
// of the narrower type (an infinite product compares as exact).  8 bits times 24 are exact in 64.
template <typename To, typename S> struct Value;
template <> struct Value<float, float> {
    __device__ __forceinline__ static float of(signed char q, float f) { return (float)q * f; }
};
template <> struct Value<double, float> {
    __device__ __forceinline__ static double of(signed char q, float f) { return (double)q * (double)f; }
};
template <> struct Value<__half, float> {
    __device__ __forceinline__ static __half of(signed char q, float f) {
        const float p = __fmul_rz((float)q, f);
        return __float2half_rn(fabsf(__fmaf_rn((float)q, f, -p)) > 0 ? __uint_as_float(__float_as_uint(p) | 1u) : p);
    }
};
template <typename To> struct Value<To, double> {
    __device__ __forceinline__ static To of(signed char q, double f) {
        const double p = __dmul_rz((double)q, f);
        const double odd = fabs(__fma_rn((double)q, f, -p)) > 0 ? __longlong_as_double(__double_as_longlong(p) | 1) : p;
        if constexpr (std::is_same<To, __half>::value) return __double2half(odd);
        else return (To)odd;
    }
};
template <> struct Value<double, double> {
    __device__ __forceinline__ static double of(signed char q, double f) { return (double)q * f; }
};

// Values of codes: V neighbouring codes of a row and group a thread, rows down blockIdx.y, four of them on
// their way at once; bound by HBM.  8192 rows of 4096 to 32 bits: 169 MB in 35 us, 4.8 TB/s (most of it stores).
template <typename To, typename S, int V>
__global__ void __launch_bounds__(256)
dequantize_kernel(const signed char* in, const S* scale, To* out, int64_t rows, int64_t n, int64_t group, int64_t groups) {
    constexpr int kRows = 4, kWide = 16 / sizeof(To) < V ? 16 / sizeof(To) : V;
    const int64_t col = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * V;
    if (col >= n) return;
    const int64_t g = col / group, down = (int64_t)gridDim.y * blockDim.y;
    for (int64_t row0 = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; row0 < rows; row0 += kRows * down) {
        Pack<signed char, V> q[kRows];
        S f[kRows];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int64_t row = row0 + k * down;
            if (row < rows) {
                q[k] = *(const Pack<signed char, V>*)(in + row * n + col);
                f[k] = scale[row * groups + g];
            }
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int64_t row = row0 + k * down;
            if (row >= rows) break;
#pragma unroll
            for (int j = 0; j < V; j += kWide) {
                Pack<To, kWide> v;
#pragma unroll
                for (int m = 0; m < kWide; ++m) v.v[m] = Value<To, S>::of(q[k].v[j + m], f[k]);
                *(Pack<To, kWide>*)(out + row * n + col + j) = v;
            }
        }
    }
}

template <typename From>
cudaError_t convert_from(const ConvertArgs& a, cudaStream_t s) {
    const int64_t size = a.rows * a.n, blocks = (size + 1023) / 1024;
    if (blocks >= (1LL << 31)) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned)blocks;
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

template <typename To, typename S, int V>
cudaError_t dequantize(const ConvertArgs& a, int sm_count, cudaStream_t s) {
    const int64_t groups = (a.n + a.group - 1) / a.group, pieces = (a.n + V - 1) / V;
    int across = 32;
    while (across < 256 && across < pieces) across *= 2;
    const int down = 256 / across;
    const int64_t bx = (pieces + across - 1) / across;
    if (bx >= (1LL << 31)) return cudaErrorInvalidValue;
    // enough blocks for 16 an SM, each over several rows
    const int64_t by = std::max<int64_t>(1, std::min<int64_t>({(a.rows + down - 1) / down, (int64_t)sm_count * 16 / bx, 65535}));
    dequantize_kernel<To, S, V><<<dim3((unsigned)bx, (unsigned)by), dim3(across, down), 0, s>>>(
        (const signed char*)a.in, (const S*)a.scale, (To*)a.out, a.rows, a.n, a.group, groups);
    return cudaGetLastError();
}

template <typename To, typename S>
cudaError_t dequantize(const ConvertArgs& a, int sm_count, cudaStream_t s) {
    const bool whole = a.group >= a.n;
    // as many codes as make one 16-byte store
    constexpr int V = 16 / sizeof(To);
    if (a.n % V == 0 && (whole || a.group % V == 0)) return dequantize<To, S, V>(a, sm_count, s);
    return dequantize<To, S, 1>(a, sm_count, s);
}

template <typename To>
cudaError_t dequantize_to(const ConvertArgs& a, int sm_count, cudaStream_t s) {
    return a.scale_dtype == DT_F64 ? dequantize<To, double>(a, sm_count, s) : dequantize<To, float>(a, sm_count, s);
}

}  // namespace

cudaError_t launch_rms_norm(const RmsNormArgs& a, int sm_count, cudaStream_t s) {
    (void)sm_count;
    if (a.rows >= (1LL << 31)) return cudaErrorInvalidValue;
    switch (a.dtype) {
        case DT_F16: return rms_norm<__half>(a, s);
        case DT_F32: return rms_norm<float>(a, s);
        case DT_F64: return rms_norm<double>(a, s);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_convert(const ConvertArgs& a, int sm_count, cudaStream_t s) {
    if (a.rows * a.n < 1) return cudaSuccess;
    if (a.scale) {
        switch (a.to) {
            case DT_F32: return dequantize_to<float>(a, sm_count, s);
            case DT_F64: return dequantize_to<double>(a, sm_count, s);
            case DT_F16: return dequantize_to<__half>(a, sm_count, s);
            default: return cudaErrorInvalidValue;
        }
    }
    switch (a.from) {
        case DT_F32: return convert_from<float>(a, s);
        case DT_F64: return convert_from<double>(a, s);
        case DT_I32: return convert_from<int>(a, s);
        case DT_I64: return convert_from<long long>(a, s);
        case DT_F16: return convert_from<__half>(a, s);
        case DT_I8: return convert_from<signed char>(a, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace cn
