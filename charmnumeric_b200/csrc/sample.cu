// Sampling of one token per row from given random numbers, with temperature, top-k, top-p and min-p.
//
// With x the row's logits and e_i = exp((x_i - max x) / temperature):
//   top-k keeps the k largest x (ties: the lowest indices);
//   top-p keeps, of these in descending order (ties: ascending index), every token before which the
//   sum of e is below top_p times the sum of all of them;
//   min-p keeps, of these, e_i >= min_p.
// A temperature that is not above 0 keeps the first of the largest logits alone.
// The token is the first in index order whose running sum of kept e exceeds u times their total.
//
// The sums are held as 64-bit integers, rint(e 2^s) with s such that no row overflows: they do not
// depend on the order of the additions, so every way of splitting a row gives the same token, and
// the first two filters come down to one border in the order of the logits, (key, number of ties kept).
// NaN counts as -infinity.  Equal infinities differ by 0, so a row with +infinities draws among them.
#include <algorithm>

#include "cn_types.hpp"
#include "sequence.cuh"
#include "sequence.hpp"

namespace cn {

using namespace seq;

namespace {

typedef unsigned long long u64;

// Integers in the order of the values; -0 and 0 are one value, NaN the lowest.
template <typename A> struct Order;
template <> struct Order<float> {
    using Key = unsigned int;
    static constexpr int kBits = 32;
    __device__ static Key key(float x) {
        if (!(x == x)) x = -INFINITY;
        const unsigned int u = __float_as_uint(x + 0.0f);
        return u >> 31 ? ~u : u | 0x80000000u;
    }
    __device__ static float value(Key k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }
};
template <> struct Order<double> {
    using Key = u64;
    static constexpr int kBits = 64;
    __device__ static Key key(double x) {
        if (!(x == x)) x = -INFINITY;
        const u64 u = (u64)__double_as_longlong(x + 0.0);
        return u >> 63 ? ~u : u | (1ULL << 63);
    }
    __device__ static double value(Key k) { return __longlong_as_double((long long)(k >> 63 ? k & ~(1ULL << 63) : ~k)); }
};

__device__ __forceinline__ double row_param(const RowParam& p, int64_t row) {
    if (!p.data) return p.value;
    if (p.dtype == DT_I32) return (double)((const int*)p.data)[row];
    return p.dtype == DT_F64 ? ((const double*)p.data)[row] : (double)((const float*)p.data)[row];
}

constexpr int kThreads = 1024;

// exclusive prefix sum over the block, in the order of the threads
__device__ __forceinline__ u64 block_prefix(u64 v, u64* sm, u64* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 w = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += w;
    }
    __syncthreads();
    if (lane == 31) sm[warp] = s;
    __syncthreads();
    u64 before = 0, all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) before += sm[w];
        all += sm[w];
    }
    *total = all;
    return before + s - v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a, int shift) {
    using A = typename Acc<T>::type;
    using O = Order<A>;
    using Key = typename O::Key;
    __shared__ u64 sm[kThreads / 32];
    const int64_t row = blockIdx.x, v = a.v;
    const T* x = (const T*)a.logits + row * v;
    auto key_at = [&](int64_t i) { return O::key(widen(x[i])); };
    auto sum_of = [&](auto&& f) {
        u64 s = 0;
        for (int64_t i = threadIdx.x; i < v; i += kThreads) s += f(key_at(i));
        __syncthreads();
        return block_sum(s, sm);
    };

    // the largest key, bit by bit from the top: some key is at least the candidate
    Key top = 0;
    for (int bit = O::kBits - 1; bit >= 0; --bit) {
        const Key cand = top | ((Key)1 << bit);
        if (sum_of([&](Key k) -> u64 { return k >= cand; })) top = cand;
    }
    const A most = O::value(top);
    if (most == -INFINITY) {
        if (threadIdx.x == 0) {
            a.token[row] = -1;
            ((A*)a.logp)[row] = -INFINITY;
        }
        return;
    }
    const A temp = (A)row_param(a.temperature, row);
    const bool greedy = !(temp > 0);
    const A unit = (A)(1ULL << shift);
    auto weight = [&](Key k) -> A {
        const A x = O::value(k);
        return k == top ? A(1) : greedy || x == -INFINITY ? A(0) : exp((x - most) / temp);
    };
    auto mass = [&](Key k) -> u64 { return (u64)rint(weight(k) * unit); };

    // the border: keys above `edge` are kept, and the first `ties` of those equal to it
    Key edge = greedy ? top : 0;
    u64 ties = greedy ? 1 : ~0ULL;
    const double kk = row_param(a.top_k, row);
    if (!greedy && kk >= 1 && kk < (double)v) {
        const u64 k = (u64)kk;
        for (int bit = O::kBits - 1; bit >= 0; --bit) {
            const Key cand = edge | ((Key)1 << bit);
            if (sum_of([&](Key q) -> u64 { return q >= cand; }) >= k) edge = cand;
        }
        ties = k - sum_of([&](Key q) -> u64 { return q > edge; });
    }
    const double pp = row_param(a.top_p, row);
    if (!greedy && pp < 1) {
        // sum of the kept weights from `from` up; tied keys at the border count `ties` times
        auto kept_from = [&](Key from) {
            u64 s = sum_of([&](Key q) -> u64 { return q >= from && q > edge ? mass(q) : 0; });
            if (edge >= from && ties != ~0ULL) s += ties * mass(edge);
            return s;
        };
        const double want = ceil(pp * (double)kept_from(0));
        const u64 need = want >= 1 ? (u64)want : 1;
        Key border = 0;
        for (int bit = O::kBits - 1; bit >= 0; --bit) {
            const Key cand = border | ((Key)1 << bit);
            if (kept_from(cand) >= need) border = cand;
        }
        const u64 above = border == ~(Key)0 ? 0 : kept_from(border + 1);
        const u64 m = mass(border);
        u64 some = m ? (need - above + m - 1) / m : 1;
        if (border == edge && some > ties) some = ties;
        edge = border;
        ties = some;
    }
    const A least = (A)fmin(row_param(a.min_p, row), 1.0);  // the largest logit stays

    // the draw: consecutive pieces of the row, one per thread
    const int64_t piece = (v + kThreads - 1) / kThreads;
    const int64_t i0 = min((int64_t)threadIdx.x * piece, v), i1 = min(i0 + piece, v);
    u64 tied = 0, all;
    for (int64_t i = i0; i < i1; ++i) tied += key_at(i) == edge;
    const u64 rank = block_prefix(tied, sm, &all);
    auto walk = [&](auto&& stop) {
        u64 sum = 0, r = rank;
        for (int64_t i = i0; i < i1; ++i) {
            const Key k = key_at(i);
            const bool keep = k > edge || (k == edge && r++ < ties);
            if (!keep || !(weight(k) >= least)) continue;
            sum += mass(k);
            if (stop(sum, i)) break;
        }
        return sum;
    };
    u64 total;
    const u64 mine = walk([](u64, int64_t) { return false; });
    const u64 before = block_prefix(mine, sm, &total);
    const double u = a.u_dtype == DT_F64 ? ((const double*)a.u)[row] : (double)((const float*)a.u)[row];
    u64 aim = u > 0 ? (u >= 1 ? total : (u64)(u * (double)total)) : 0;
    if (aim >= total) aim = total - 1;
    if (before <= aim && aim < before + mine)
        walk([&](u64 sum, int64_t i) {
            if (before + sum <= aim) return false;
            a.token[row] = (int)i;
            const double e = greedy ? 0.0 : ((double)widen(x[i]) - (double)most) / (double)temp;
            ((A*)a.logp)[row] = (A)((key_at(i) == top ? 0.0 : e) - log((double)total / (double)(1ULL << shift)));
            return true;
        });
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int sm_count, cudaStream_t s) {
    (void)sm_count;
    if (a.rows >= (1LL << 31)) return cudaErrorInvalidValue;
    int shift = 62;  // v terms of at most 2^shift stay below 2^62
    while ((1LL << (62 - shift)) < a.v) --shift;
    const int grid = (int)a.rows;
    switch (a.dtype) {
        case DT_F16: sample_kernel<__half><<<grid, kThreads, 0, s>>>(a, shift); break;
        case DT_F32: sample_kernel<float><<<grid, kThreads, 0, s>>>(a, shift); break;
        case DT_F64: sample_kernel<double><<<grid, kThreads, 0, s>>>(a, shift); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace cn
