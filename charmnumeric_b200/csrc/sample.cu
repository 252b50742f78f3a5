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
// NaN counts as -infinity.  A row with +infinities draws among them alone.
//
// Nothing is sorted.  A cluster of up to 8 blocks has a row, each block a slice of it in shared memory as
// integer keys in the order of the values, read from HBM once.  A border is found by histograms: the
// first over steps of 1/32 in log2 e, the next over what the bin with the border spans in key space,
// 1024 times finer each time, until a bin is one key.  Every block adds up all blocks' histograms
// (distributed shared memory), so that one cluster barrier a round is enough.
#include <cooperative_groups.h>

#include <algorithm>

#include "cn_types.hpp"
#include "sequence.cuh"
#include "sequence.hpp"

namespace cn {

using namespace seq;
namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 2 * kThreads, kMostBlocks = 8;
constexpr int kBinsPerOctave = 32;

// Integers in the order of the values; -0 and 0 are one value, NaN the lowest.
template <typename T> struct Order;
template <> struct Order<__half> {
    using Key = unsigned int;
    using Stored = unsigned short;
    __device__ static Key key(__half x) {
        unsigned int u = __half_as_ushort(x);
        if ((u & 0x7fffu) > 0x7c00u) u = 0xfc00u;
        if (u == 0x8000u) u = 0;
        return u >> 15 ? ~u & 0xffffu : u | 0x8000u;
    }
    __device__ static float value(Key k) { return __half2float(__ushort_as_half((unsigned short)(k >> 15 ? k & 0x7fffu : ~k))); }
    // the keys next to a value's, not below and not above it
    __device__ static Key at_least(float x) { return key(__float2half_ru(x)) + 1; }
    __device__ static Key at_most(float x) { const Key k = key(__float2half_rd(x)); return k ? k - 1 : 0; }
};
template <> struct Order<float> {
    using Key = unsigned int;
    using Stored = unsigned int;
    __device__ static Key key(float x) {
        if (!(x == x)) x = -INFINITY;
        const unsigned int u = __float_as_uint(x + 0.0f);
        return u >> 31 ? ~u : u | 0x80000000u;
    }
    __device__ static float value(Key k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }
    __device__ static Key at_least(float x) { return key(x) + 1; }
    __device__ static Key at_most(float x) { const Key k = key(x); return k ? k - 1 : 0; }
};
template <> struct Order<double> {
    using Key = u64;
    using Stored = u64;
    __device__ static Key key(double x) {
        if (!(x == x)) x = -INFINITY;
        const u64 u = (u64)__double_as_longlong(x + 0.0);
        return u >> 63 ? ~u : u | (1ULL << 63);
    }
    __device__ static double value(Key k) { return __longlong_as_double((long long)(k >> 63 ? k & ~(1ULL << 63) : ~k)); }
    __device__ static Key at_least(double x) { return key(x) + 1; }
    __device__ static Key at_most(double x) { const Key k = key(x); return k ? k - 1 : 0; }
};

__device__ __forceinline__ double row_param(const RowParam& p, int64_t row) {
    if (!p.data) return p.value;
    if (p.dtype == DT_I32) return (double)((const int*)p.data)[row];
    return p.dtype == DT_F64 ? ((const double*)p.data)[row] : (double)((const float*)p.data)[row];
}

__device__ __forceinline__ float power(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ double power(double v) { return exp2(v); }

// Weights e of 0 to 1 as integers.  WIDE: 64 bits at once, rint(e 2^shift).  Else three limbs of 15 bits,
// whose sums over a slice of up to 2^15 values fit the 32 bits that shared memory can add to at once,
// and whose sum over 8 slices fits 64.
// A histogram is an array of bins of 64 bits, or three arrays of the limbs' sums.
template <bool WIDE> struct Mass;
template <> struct Mass<true> {
    static constexpr int kWords = 2;
    template <typename A> __device__ static u64 of(A e, int shift) { return (u64)rint(e * (A)(1ULL << shift)); }
    template <typename A> __device__ static void add(unsigned* bins, int bin, A e, int shift) { atomicAdd((u64*)bins + bin, of(e, shift)); }
    __device__ static void count(unsigned* bins, int bin) { atomicAdd((u64*)bins + bin, 1ULL); }
    // bins 2 i and 2 i + 1, summed over the blocks; every block begins with its own
    template <bool COUNT, typename F> __device__ static void sum(u64 (&own)[2], int i, int blocks, F&& bins_of) {
        for (int q = 0; q < blocks; ++q) {
            const Pack<u64, 2> w = ((const Pack<u64, 2>*)bins_of(q))[i];
            own[0] += w.v[0];
            own[1] += w.v[1];
        }
    }
};
template <> struct Mass<false> {
    static constexpr int kWords = 3;
    __device__ static void limbs(float e, unsigned (&l)[3]) {
        // every difference and product is exact
        const float s = e * 32768.0f;
        l[0] = (unsigned)s;
        const float t = (s - (float)l[0]) * 32768.0f;
        l[1] = (unsigned)t;
        l[2] = (unsigned)rintf((t - (float)l[1]) * 32768.0f);
    }
    __device__ static u64 of(float e, int) {
        unsigned l[3];
        limbs(e, l);
        return ((u64)l[0] << 30) + ((u64)l[1] << 15) + l[2];
    }
    __device__ static void add(unsigned* bins, int bin, float e, int) {
        unsigned l[3];
        limbs(e, l);
        if (l[0]) atomicAdd(bins + bin, l[0]);
        if (l[1]) atomicAdd(bins + kBins + bin, l[1]);
        if (l[2]) atomicAdd(bins + 2 * kBins + bin, l[2]);
    }
    __device__ static void count(unsigned* bins, int bin) { atomicAdd(bins + 2 * kBins + bin, 1u); }
    template <bool COUNT, typename F> __device__ static void sum(u64 (&own)[2], int i, int blocks, F&& bins_of) {
#pragma unroll
        for (int k = COUNT ? 2 : 0; k < 3; ++k) {
            // all blocks' values are on their way before the first is added
            Pack<unsigned, 2> w[kMostBlocks];
#pragma unroll
            for (int q = 0; q < kMostBlocks; ++q) {
                if (q < blocks) w[q] = ((const Pack<unsigned, 2>*)(bins_of(q) + k * kBins))[i];
                else w[q] = {{0, 0}};
            }
            u64 a = 0, b = 0;
#pragma unroll
            for (int q = 0; q < kMostBlocks; ++q) {
                a += w[q].v[0];
                b += w[q].v[1];
            }
            own[0] += a << 15 * (2 - k);
            own[1] += b << 15 * (2 - k);
        }
    }
};

template <typename T, bool WIDE>
struct SampleShared {
    alignas(16) unsigned bins[2][kBins * Mass<WIDE>::kWords];  // two rounds' histograms
    u64 scan[kWarps];
    u64 weight[kWarps];                                        // each warp's kept weight above the border
    u64 tied[kWarps];                                          // ... and values at the border
    typename Order<T>::Key top[kWarps], most;
    u64 before, own, extra, total;                             // what a search has found
    int found;
};

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
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const u64 t = sm[w];
        if (w < warp) before += t;
        all += t;
    }
    *total = all;
    return before + s - v;
}

// One cluster a row.  RESIDENT: a block's slice fits its shared memory; else it is read from L2 each time.
// V: values of one load.  A warp has `per_warp` neighbouring values (a multiple of 32) of the slice.
template <typename T, int V, bool WIDE, bool RESIDENT>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a, int64_t per_warp, int shift) {
    using A = typename Acc<T>::type;
    using O = Order<T>;
    using Key = typename O::Key;
    using M = Mass<WIDE>;
    extern __shared__ __align__(16) unsigned char sample_shared[];
    auto& sh = *(SampleShared<T, WIDE>*)sample_shared;
    auto* const keys = (typename O::Stored*)(sample_shared + (sizeof(SampleShared<T, WIDE>) + 15) / 16 * 16);

    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / blocks, slice = per_warp * kWarps, v = a.v;
    const int64_t s0 = min(rank * slice, v), size = min(slice, v - s0);
    const T* const x = (const T*)a.logits + row * v + s0;
    auto key_at = [&](int64_t i) -> Key { return RESIDENT ? (Key)keys[i] : O::key(x[i]); };
    const int64_t w0 = min(warp * per_warp, size), w1 = min(w0 + per_warp, size);
    // f(key, valid) on this warp's values, all lanes of the warp together
    auto each = [&](auto&& f) {
        for (int64_t i = w0 + lane; i < w1; i += 32) f(key_at(i));
    };

    // the largest key
    Key top = 0;
    if (RESIDENT) {
        for (int64_t i = (int64_t)tid * V; i < size; i += (int64_t)kThreads * V) {
            if (V == 1 || i + V <= size) {
                const Pack<T, V> p = *(const Pack<T, V>*)(x + i);
                Pack<typename O::Stored, V> q;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const Key k = O::key(p.v[j]);
                    top = k > top ? k : top;
                    q.v[j] = (typename O::Stored)k;
                }
                *(Pack<typename O::Stored, V>*)(keys + i) = q;
            } else {
                for (int64_t j = i; j < size; ++j) {
                    const Key k = O::key(x[j]);
                    top = k > top ? k : top;
                    keys[j] = (typename O::Stored)k;
                }
            }
        }
    } else {
        each([&](Key k) { top = k > top ? k : top; });
    }
    for (int i = tid; i < 2 * kBins * M::kWords; i += kThreads) (&sh.bins[0][0])[i] = 0;
    top = warp_max(top);
    if (lane == 0) sh.top[warp] = top;
    __syncthreads();
    if (tid == 0) {
        for (int w = 0; w < kWarps; ++w) top = sh.top[w] > top ? sh.top[w] : top;
        sh.most = top;
    }
    cluster.sync();
    top = 0;
    if (lane < blocks) top = *cluster.map_shared_rank(&sh.most, lane);
    top = warp_max(top);
    const A most = O::value(top);
    const A temp = (A)row_param(a.temperature, row);
    const bool none = most == -INFINITY, greedy = !(temp > 0), alone = greedy || most == INFINITY;
    // differences are taken of halves, which do not overflow
    const A half = most * A(0.5), scale = greedy ? A(0) : A(2 * 1.4426950408889634) / temp;
    auto weight = [&](Key k) -> A {
        const A e = O::value(k);
        return k == top ? A(1) : alone || e == -INFINITY ? A(0) : power((e * A(0.5) - half) * scale);
    };
    auto mass = [&](Key k) { return M::of(weight(k), shift); };

    // ---- borders ----
    // The key at which the sum over the kept values in descending order reaches a target, the sum above
    // it and its own: the number of values, or their weight.  `aim` gives the target for the sum of all.
    int turn = 0;
    Key edge = greedy ? top : 0;       // keys above the edge are kept, and the first `ties` at it
    u64 ties = greedy ? 1 : ~0ULL, tied = ~0ULL;
    struct Border { Key key; u64 above, own; };
    auto border_of = [&](auto by_weight, auto&& aim) -> Border {
        constexpr bool kWeight = decltype(by_weight)::value;
        // first round: bins of equal steps in log2 e, the last one open
        const A step = scale * kBinsPerOctave;
        auto octave_bin = [&](Key k) -> int {
            const A d = (half - O::value(k) * A(0.5)) * step;
            return k == top ? 0 : d < kBins - 1 ? (int)d : kBins - 1;
        };
        int octave = -1, down = 0;
        Key high = top, low = 0;
        u64 above = 0, target = 0;
        // a round leaves 1/1024 of the span or less: 8 are the most for 64-bit keys
        for (int round = 0; round < 12; ++round) {
            unsigned* const bins = sh.bins[turn & 1];
            each([&](Key k) {
                if (k < edge || k < low || k > high) return;
                int bin;
                if (octave < 0) {
                    bin = octave_bin(k);
                } else {
                    if (octave_bin(k) != octave) return;
                    bin = (int)((high - k) >> down);
                }
                if (kWeight) M::add(bins, bin, weight(k), shift);
                else M::count(bins, bin);
            });
            cluster.sync();
            u64 own[2] = {0, 0};
            M::template sum<!kWeight>(own, tid, blocks, [&](int q) { return cluster.map_shared_rank(bins, (rank + q) & (blocks - 1)); });
            if (tid == 0) sh.found = -1;
            u64 total;
            u64 before = above + block_prefix(own[0] + own[1], sh.scan, &total);
            if (octave < 0) target = aim(total);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (before < target && target <= before + own[i]) {
                    sh.found = 2 * tid + i;
                    sh.before = before;
                    sh.own = own[i];
                }
                before += own[i];
            }
            // the other histogram is free: all blocks have passed the barrier behind its last use
            ++turn;
            for (int i = tid; i < kBins * M::kWords; i += kThreads) sh.bins[turn & 1][i] = 0;
            __syncthreads();
            const int found = sh.found;
            if (found < 0) break;
            above = sh.before;
            const u64 mine = sh.own;
            __syncthreads();
            if (octave < 0) {
                octave = found;
                // a span that has all of the bin's keys, however the bin and the span were rounded;
                // whether a key is in the bin is for octave_bin to say
                const A wide = A(2) / step, slack = (fabs(most) + (A)(found + 1) * wide) * (sizeof(A) == 8 ? A(1e-14) : A(1e-6));
                if (found > 0) high = min(top, O::at_least(most - (A)found * wide + slack));
                if (found < kBins - 1) low = O::at_most(most - (A)(found + 1) * wide - slack);
            } else {
                high -= (Key)found << down;
                const Key span = ((Key)1 << down) - 1;
                low = high - low > span ? high - span : low;
            }
            if (low == high) return {high, above, mine};
            down = 0;
            while (((high - low) >> down) >= (Key)kBins) ++down;
        }
        return {edge, above, 0};    // not reached: a target is never above the sum of all
    };
    if (!greedy && !none) {
        const double kk = row_param(a.top_k, row);
        if (kk >= 1 && kk < (double)v) {
            const Border b = border_of(std::false_type(), [&](u64) { return (u64)kk; });
            edge = b.key;
            ties = (u64)kk - b.above;
            tied = b.own;
        }
        const double pp = row_param(a.top_p, row);
        if (pp < 1) {
            u64 need = 0;
            const Border b = border_of(std::true_type(), [&](u64 sum) {
                if (ties < tied) sum -= (tied - ties) * mass(edge);
                const double want = ceil(pp * (double)sum);
                need = want >= 1 ? min((u64)want, sum) : 1;
                return need;
            });
            const u64 m = mass(b.key), some = m ? (need - b.above + m - 1) / m : 1;
            ties = b.key == edge && ties < some ? ties : some;
            edge = b.key;
        }
    }

    // ---- the draw ----
    const A least = (A)fmin(row_param(a.min_p, row), 1.0);   // the largest logit stays
    if (!(weight(edge) >= least)) ties = 0;
    u64 mine = 0, at_edge = 0;
    each([&](Key k) {
        if (k == edge) ++at_edge;
        else if (k > edge) {
            const A e = weight(k);
            if (e >= least) mine += M::of(e, shift);
        }
    });
    mine = warp_sum(mine);
    at_edge = warp_sum(at_edge);
    if (lane == 0) {
        sh.weight[warp] = mine;
        sh.tied[warp] = at_edge;
    }
    cluster.sync();
    // every block adds up all warps' weights in the order of the values
    u64 theirs = 0, count = 0;
    if (tid < blocks * kWarps) {
        theirs = cluster.map_shared_rank(sh.weight, tid / kWarps)[tid % kWarps];
        count = cluster.map_shared_rank(sh.tied, tid / kWarps)[tid % kWarps];
    }
    u64 total, unused;
    const u64 tied_before = block_prefix(count, sh.scan, &unused);
    if (ties > tied_before) theirs += min(count, ties - tied_before) * mass(edge);
    const u64 before = block_prefix(theirs, sh.scan, &total);
    const double u = a.u_dtype == DT_F64 ? ((const double*)a.u)[row] : (double)((const float*)a.u)[row];
    u64 aim = u > 0 ? (u >= 1 ? total : (u64)(u * (double)total)) : 0;
    if (aim >= total) aim = total - 1;
    if (tid == 0) sh.found = -1;
    __syncthreads();
    if (!none && before <= aim && aim < before + theirs && tid / kWarps == rank) {
        sh.found = tid % kWarps;
        sh.before = before;
        sh.extra = tied_before;
    }
    __syncthreads();
    if (none && rank == 0 && tid == 0) {
        a.token[row] = -1;
        ((A*)a.logp)[row] = -INFINITY;
    }
    if (warp == sh.found) {
        u64 sum = sh.before, rank_of_tie = sh.extra;
        for (int64_t i0 = w0; i0 < w1; i0 += 32) {
            const int64_t i = i0 + lane;
            const Key k = i < w1 ? key_at(i) : 0;
            const unsigned equal = __ballot_sync(0xffffffffu, i < w1 && k == edge);
            const bool tie = i < w1 && k == edge && rank_of_tie + __popc(equal & ((1u << lane) - 1)) < ties;
            rank_of_tie += __popc(equal);
            u64 s = 0;
            if (tie || (i < w1 && k > edge && weight(k) >= least)) s = mass(k);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 w = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += w;
            }
            const unsigned past = __ballot_sync(0xffffffffu, sum + s > aim);
            if (past) {
                if (lane == __ffs(past) - 1) {
                    a.token[row] = (int)(s0 + i);
                    const double e = k == top ? 0.0 : ((double)O::value(k) - (double)most) / (double)temp;
                    ((A*)a.logp)[row] = (A)(e - log((double)total / (double)(1ULL << shift)));
                }
                break;
            }
            sum += __shfl_sync(0xffffffffu, s, 31);
        }
    }
    cluster.sync();    // no block's shared memory goes while another may read it
}

template <typename T, int V, bool WIDE, bool RESIDENT>
cudaError_t launch(const SampleArgs& a, int blocks, int64_t per_warp, int shift, cudaStream_t s) {
    const size_t bytes = (sizeof(SampleShared<T, WIDE>) + 15) / 16 * 16 + (RESIDENT ? (size_t)per_warp * kWarps * sizeof(typename Order<T>::Stored) : 0);
    const auto kernel = sample_kernel<T, V, WIDE, RESIDENT>;
    if (bytes > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(a.rows * blocks));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = bytes;
    config.stream = s;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim = {(unsigned)blocks, 1, 1};
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, a, per_warp, shift);
}

template <typename T>
cudaError_t sample(const SampleArgs& a, int sm_count, cudaStream_t s) {
    constexpr bool kDouble = sizeof(T) == 8;
    constexpr int64_t kSlice = kDouble ? 1 << 14 : 1 << 15;     // 64 to 128 KB of keys
    // as few blocks as hold a row, but more for few rows: their passes are shorter
    int blocks = 1;
    while (blocks < kMostBlocks && (a.v > blocks * kSlice || (a.rows * blocks * 2 <= sm_count && a.v > blocks * 4096))) blocks *= 2;
    const int64_t per_warp = ((a.v + blocks - 1) / blocks + kWarps * 32 - 1) / (kWarps * 32) * 32, slice = per_warp * kWarps;
    int shift = 62;                                             // v terms of at most 2^shift stay below 2^62
    while ((1LL << (62 - shift)) < a.v) --shift;
    if (a.rows * blocks >= (1LL << 31)) return cudaErrorInvalidValue;
    constexpr int V = 16 / sizeof(T);
    if (kDouble) {
        if (slice > kSlice) return launch<T, 1, true, false>(a, blocks, per_warp, shift, s);
        return a.v % V == 0 ? launch<T, V, true, true>(a, blocks, per_warp, shift, s) : launch<T, 1, true, true>(a, blocks, per_warp, shift, s);
    } else {
        if (slice > kSlice) return launch<T, 1, true, false>(a, blocks, per_warp, shift, s);
        return a.v % V == 0 ? launch<T, V, false, true>(a, blocks, per_warp, 45, s) : launch<T, 1, false, true>(a, blocks, per_warp, 45, s);
    }
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int sm_count, cudaStream_t s) {
    switch (a.dtype) {
        case DT_F16: return sample<__half>(a, sm_count, s);
        case DT_F32: return sample<float>(a, sm_count, s);
        case DT_F64: return sample<double>(a, sm_count, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace cn
