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
// A weight is the hardware's 2^x of a 32-bit argument (64 bits and exp2 for 64-bit logits), with a relative error of
// some 2^-22 + |log2 e| 2^-24: that of a difference of logits in 32 bits.
// The sums are held as 64-bit integers, e 2^s rounded to one, with s such that no row overflows: they do not
// depend on the order of the additions, so every way of splitting a row gives the same token, and
// the first two filters come down to one border in the order of the logits, (key, number of ties kept).
// NaN counts as -infinity.  A row with +infinities draws among them alone.
//
// Bound by latency: the bytes (a row's logits, once) are a tenth of the time or less, the rest are rounds of
// a pass over shared memory, a cluster barrier and a prefix sum, one after the other.  So:
// A cluster of up to 8 blocks has a row, each block a slice of it in shared memory as
// integer keys in the order of the values, read from HBM once.  A border is found by histograms: the
// first over steps of 1/16 in log2 e, the next over what the bin with the border spans in key space,
// 512 times finer each time, until a bin is one key or few values are left, which are ordered.  Every block adds up all blocks' histograms
// (distributed shared memory), so that one cluster barrier a round is enough.  A top-k of a few hundred
// leaves few values above a bound that is found from each thread's largest key; those are brought
// together and ordered by counting, and the rest of the work is on that list.
//
// 128 rows of 131072 in 16 bits, top-k 50, top-p 0.9, min-p 0.02: a block a row without shared memory 1592 us;
// clusters with keys in shared memory 226; histograms read in wide, coalesced pieces 136; rows looped over
// by resident clusters (a cluster starts slower than a row that follows another in it) 96; the short list 54;
// looked for by the threads that have loaded its values 51 us (floor 5).
// One row of 32768 in 32 bits with top-p 0.95: 419, 102, 27 us; the last rounds as an ordered list 20.5 us.
// 37 rows of 50021 in 32 bits with top-p 0.98: 649 to 45 us, of it the first histogram and the draw, each a
// weight for every value, 6 and 5, the barriers and prefix sums between them most of the rest.
// Slower: 1024 threads; weights of four neighbouring values made together before they are used (47 us); the
// draw's prefix sums in one warp alone (47 us).
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

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = kThreads, kMostBlocks = 8;
constexpr int kBinsPerOctave = 16, kGrain = 8, kList = kThreads;

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

// Keys of V neighbouring values.  16-bit values two at a time: a value's sign decides whether all of its
// bits or the sign alone are turned; NaN and -0 are left to the single value's routine.
template <typename T, int V>
__device__ __forceinline__ Pack<typename Order<T>::Stored, V> keys_of(const Pack<T, V>& p) {
    Pack<typename Order<T>::Stored, V> q;
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
        Pack<unsigned, V / 2> u = *(const Pack<unsigned, V / 2>*)&p;
        unsigned odd = 0;
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const unsigned w = u.v[j];
            odd |= __vcmpgtu2(w & 0x7fff7fffu, 0x7c007c00u) | __vcmpeq2(w, 0x80008000u);
            u.v[j] = w ^ ((w >> 15 & 0x00010001u) * 0x7fffu | 0x80008000u);
        }
        if (!odd) return *(const Pack<unsigned short, V>*)&u;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) q.v[j] = (typename Order<T>::Stored)Order<T>::key(p.v[j]);
    return q;
}

// whether any key of a piece is at least `from`
__device__ __forceinline__ bool any_from(const Pack<unsigned short, 8>& q, unsigned from) {
    const Pack<unsigned, 4> u = *(const Pack<unsigned, 4>*)&q;
    const unsigned both = from * 0x10001u;
    return __vcmpgeu2(u.v[0], both) | __vcmpgeu2(u.v[1], both) | __vcmpgeu2(u.v[2], both) | __vcmpgeu2(u.v[3], both);
}
__device__ __forceinline__ bool any_from(const Pack<unsigned, 4>& q, unsigned from) {
    return max(max(q.v[0], q.v[1]), max(q.v[2], q.v[3])) >= from;
}
__device__ __forceinline__ bool any_from(const Pack<u64, 2>& q, u64 from) { return q.v[0] >= from || q.v[1] >= from; }

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

// Weights e of 0 to 1 as integers.  WIDE: 64 bits at once, rint(e 2^shift).  Else floor(e 2^45) in three limbs
// of 12, 17 and 17 bits, whose sums over a slice of up to 2^15 values fit the 32 bits that shared memory can add
// to at once, and whose sum over 8 slices fits 64.
// A histogram is an array of bins of 64 bits, or three arrays of the limbs' sums.
template <bool WIDE> struct Mass;
template <> struct Mass<true> {
    static constexpr int kWords = 2;
    template <typename A> __device__ static u64 of(A e, int shift) { return (u64)rint(e * (A)(1ULL << shift)); }
    template <typename A> __device__ static void add(unsigned* bins, int bin, A e, int shift) { atomicAdd((u64*)bins + bin, of(e, shift)); }
    __device__ static void count(unsigned* bins, int bin) { atomicAdd((u64*)bins + bin, 1ULL); }
    // bin i, summed over the blocks
    template <bool COUNT, typename F> __device__ static u64 sum(int i, int blocks, F&& bins_of) {
        u64 own = 0;
        for (int q = 0; q < blocks; ++q) own += ((const u64*)bins_of(q))[i];
        return own;
    }
    // a thread's sum
    struct Sum {
        u64 s = 0;
        template <typename A> __device__ __forceinline__ void add(A e, int shift) { s += of(e, shift); }
        __device__ __forceinline__ u64 total() const { return s; }
    };
};
template <> struct Mass<false> {
    static constexpr int kWords = 3;
    struct Limbs { unsigned high, mid, low; };
    // Added to 2^12 (2^-5, 2^-22) and rounded down, a value below 1 (2^-11, 2^-28) leaves its multiple of 2^-11
    // (2^-28, 2^-45) in the last bits; what is taken off it is exact.  No branches, no conversions.
    __device__ __forceinline__ static Limbs limbs(float e) {
        const float h = __fadd_rd(e, 0x1p12f), r = __fadd_rn(e, __fadd_rn(0x1p12f, -h));
        const float m = __fadd_rd(r, 0x1p-5f), q = __fadd_rn(r, __fadd_rn(0x1p-5f, -m));
        const float l = __fadd_rd(q, 0x1p-22f);
        return {__float_as_uint(h) & 0xfffu, __float_as_uint(m) & 0x1ffffu, __float_as_uint(l) & 0x1ffffu};
    }
    __device__ __forceinline__ static u64 whole(Limbs p) { return ((u64)p.high << 34) + ((u64)p.mid << 17) + p.low; }
    __device__ static u64 of(float e, int) { return whole(limbs(e)); }
    __device__ __forceinline__ static void add(unsigned* bins, int bin, float e, int) {
        const Limbs p = limbs(e);
        if (p.high) atomicAdd(bins + bin, p.high);     // weights of 2^-11 and more
        atomicAdd(bins + kBins + bin, p.mid);
        atomicAdd(bins + 2 * kBins + bin, p.low);
    }
    __device__ static void count(unsigned* bins, int bin) { atomicAdd(bins + 2 * kBins + bin, 1u); }
    template <bool COUNT, typename F> __device__ static u64 sum(int i, int blocks, F&& bins_of) {
        // all blocks' values are on their way before the first is added
        unsigned w[COUNT ? 1 : 3][kMostBlocks];
#pragma unroll
        for (int q = 0; q < kMostBlocks; ++q)
#pragma unroll
            for (int k = 0; k < (COUNT ? 1 : 3); ++k) w[k][q] = q < blocks ? bins_of(q)[(COUNT ? 2 : k) * kBins + i] : 0;
        u64 own = 0;
#pragma unroll
        for (int k = 0; k < (COUNT ? 1 : 3); ++k) {
            u64 limb = 0;
#pragma unroll
            for (int q = 0; q < kMostBlocks; ++q) limb += w[k][q];
            own += COUNT ? limb : limb << 17 * (2 - k);
        }
        return own;
    }
    // a thread's sum, of up to 2^15 values
    struct Sum {
        Limbs s = {0, 0, 0};
        __device__ __forceinline__ void add(float e, int) {
            const Limbs p = limbs(e);
            s.high += p.high;
            s.mid += p.mid;
            s.low += p.low;
        }
        __device__ __forceinline__ u64 total() const { return whole(s); }
    };
};

template <typename T, bool WIDE>
struct SampleShared {
    alignas(16) unsigned bins[2][kBins * Mass<WIDE>::kWords];  // two rounds' histograms
    u64 scan[kWarps];
    u64 weight[kWarps];                                        // each warp's kept weight above the border
    u64 tied[kWarps];                                          // ... and values at the border
    typename Order<T>::Key top[kWarps], most;
    u64 before, own, extra;                                    // what a search has found
    typename Order<T>::Key border;
    int found;
    // a short list of values, of this block and then of the row; two rounds' counters
    int listed[2];
    alignas(16) typename Order<T>::Key list_key[kList], row_key[kList];
    int list_at[kList], row_at[kList];
    u64 row_mass[kList];
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
// V: values of one load.  A warp has `per_warp` neighbouring values (a multiple of kGrain: 16 bytes) of the slice.
template <typename T, int V, bool WIDE, bool RESIDENT>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 8 ? 1 : 2) sample_kernel(SampleArgs a, int64_t per_warp, int shift) {
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
    const int64_t slice = per_warp * kWarps, v = a.v;
    const int64_t s0 = min(rank * slice, v), size = min(slice, v - s0);
    for (int64_t row = blockIdx.x / blocks; row < a.rows; row += gridDim.x / blocks) {
        const T* const x = (const T*)a.logits + row * v + s0;
        auto key_at = [&](int64_t i) -> Key { return RESIDENT ? (Key)keys[i] : O::key(x[i]); };
        const int64_t w0 = min(warp * per_warp, size), w1 = min(w0 + per_warp, size);
        // f(key) for this warp's keys of at least `from`, which is 1 or more; in shared memory 16 bytes at a
        // time, most of which have none once a border is known to be above
        auto each = [&](Key from, auto&& f) {
            if (RESIDENT) {
                constexpr int W = 16 / sizeof(typename O::Stored);
                const typename O::Stored* const at = keys + warp * per_warp;
                for (int i = lane * W; i < (int)per_warp; i += 32 * W) {
                    const Pack<typename O::Stored, W> q = *(const Pack<typename O::Stored, W>*)(at + i);
                    if (!any_from(q, from)) continue;
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        if (q.v[j] >= from) f((Key)q.v[j]);
                }
            } else {
                for (int64_t i = w0 + lane; i < w1; i += 32) {
                    const Key k = key_at(i);
                    if (k >= from) f(k);
                }
            }
        };

        // the largest key
        Key top = 0;
        if (RESIDENT) {
            // what is left of the slice behind the row: 0, below every key
            constexpr int kTogether = 4;       // loads on their way at once
            for (int i0 = tid * V; i0 < (int)slice; i0 += kTogether * kThreads * V) {
                Pack<T, V> p[kTogether];
#pragma unroll
                for (int m = 0; m < kTogether; ++m)
                    if (i0 + m * kThreads * V < size) p[m] = *(const Pack<T, V>*)(x + i0 + m * kThreads * V);
#pragma unroll
                for (int m = 0; m < kTogether; ++m) {
                    const int i = i0 + m * kThreads * V;
                    if (i >= (int)slice) break;
                    Pack<typename O::Stored, V> q;
#pragma unroll
                    for (int j = 0; j < V; ++j) q.v[j] = 0;
                    if (i < size) q = keys_of<T, V>(p[m]);
                    *(Pack<typename O::Stored, V>*)(keys + i) = q;
#pragma unroll
                    for (int j = 0; j < V; ++j) top = q.v[j] > top ? q.v[j] : top;
                }
            }
        } else {
            each(1, [&](Key k) { top = k > top ? k : top; });
        }
        for (int i = tid; i < 2 * kBins * M::kWords; i += kThreads) (&sh.bins[0][0])[i] = 0;
        if (tid < 2) sh.listed[tid] = 0;
        const Key own_top = top;
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
        const bool none = most == -INFINITY, greedy = !(temp > 0);
        // differences are taken of halves, which do not overflow
        const A half = most * A(0.5), scale = greedy ? A(0) : A(2 * 1.4426950408889634) / temp;
        // only the largest has weight: it is infinite, or the temperature so small that its inverse is
        const bool alone = greedy || most == INFINITY || scale == INFINITY;
        // log2 of a weight, negated; infinite where the weight is 0
        auto depth = [&](Key k) -> A {
            const A e = O::value(k), d = (half - e * A(0.5)) * scale;
            return k == top ? A(0) : alone || e == -INFINITY ? (A)INFINITY : d;
        };
        auto weight = [&](Key k) { return power(-depth(k)); };
        auto mass = [&](Key k) { return M::of(weight(k), shift); };

        // ---- borders ----
        // The key at which the sum over the kept values in descending order reaches a target, the sum above
        // it and its own: the number of values, or their weight.  `aim` gives the target for the sum of all.
        int turn = 0;
        Key edge = greedy ? top : 1;       // keys above the edge are kept, and the first `ties` at it
        u64 ties = greedy ? 1 : ~0ULL, tied = ~0ULL;
        struct Border { Key key; u64 above, own; };
        // first round: bins of equal steps in log2 e, the last one open
        const A wide = A(2) / (scale * kBinsPerOctave);
        auto bin_of = [&](A depth) { return (int)fmin(depth * A(kBinsPerOctave), A(kBins - 1)); };
        auto octave_bin = [&](Key k) { return bin_of(depth(k)); };
        // keys not below and not above any of a bin, however bin and value were rounded
        auto slack_of = [&](int bin) { return (fabs(most) + (A)(bin + 1) * wide) * (sizeof(A) == 8 ? A(1e-14) : A(1e-6)); };
        auto bin_high = [&](int bin) { return bin > 0 ? min(top, O::at_least(most - (A)bin * wide + slack_of(bin))) : top; };
        auto bin_low = [&](int bin) { return bin < kBins - 1 ? max((Key)1, O::at_most(most - (A)(bin + 1) * wide - slack_of(bin))) : (Key)1; };
        // to the other histogram and counter, which are free: all blocks have passed the barrier behind their last use
        auto advance = [&]() {
            ++turn;
            for (int i = tid; i < kBins * M::kWords; i += kThreads) sh.bins[turn & 1][i] = 0;
            if (tid == 0) sh.listed[turn & 1] = 0;
            __syncthreads();
        };
        // Values listed by all blocks in this turn, behind a barrier of the cluster; this thread's is the
        // `place`th of block `from`.
        auto listed = [&](int& from, int& place) {
            const int each_of = lane < blocks ? *cluster.map_shared_rank(&sh.listed[turn & 1], lane) : 0;
            int count = 0;
#pragma unroll
            for (int q = 0; q < kMostBlocks; ++q) {
                const int theirs = __shfl_sync(0xffffffffu, each_of, q);
                if (count <= tid && tid < count + theirs) {
                    from = q;
                    place = tid - count;
                }
                count += theirs;
            }
            return count;
        };
        // Adds up all blocks' histograms of this turn, behind a barrier of the cluster; the bin in which the sum from the top reaches
        // target(sum of all), or -1; sh.before and sh.own are the sums above it and of it.
        auto search = [&](auto by_weight, u64 above, auto&& target_of) -> int {
            constexpr bool kWeight = decltype(by_weight)::value;
            unsigned* const bins = sh.bins[turn & 1];
            const u64 own = M::template sum<!kWeight>(tid, blocks, [&](int q) { return cluster.map_shared_rank(bins, (rank + q) & (blocks - 1)); });
            if (tid == 0) sh.found = -1;
            u64 total;
            const u64 before = above + block_prefix(own, sh.scan, &total);
            const u64 target = target_of(total);
            if (before < target && target <= before + own) {
                sh.found = tid;
                sh.before = before;
                sh.own = own;
            }
            advance();
            return sh.found;
        };
        auto border_of = [&](auto by_weight, Key floor, auto&& aim) -> Border {
            constexpr bool kWeight = decltype(by_weight)::value;
            int octave = -1, down = 0;
            Key high = top, low = max(floor, edge);
            u64 above = 0, target = 0;
            // The border among the listed values, one a thread (in every block): they are put in descending
            // order by counting, and their sums taken in it.
            auto in_list = [&](int count, int from, int place) -> Border {
                constexpr int W = 16 / sizeof(Key);
                const Key key = tid < count ? cluster.map_shared_rank(sh.list_key, from)[place] : 0;
                sh.row_key[tid] = key;
                if (tid == 0) sh.found = 0;
                __syncthreads();
                // greater ones are in front, and equal ones of lower threads; behind the list there are zeros
                int order = 0;
                if (tid < count) {
                    const int w0 = tid - lane;
#pragma unroll 4
                    for (int i = 0; i < w0; i += W) {
                        const Pack<Key, W> p = *(const Pack<Key, W>*)(sh.row_key + i);
#pragma unroll
                        for (int j = 0; j < W; ++j) order += p.v[j] >= key;
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += W) {
                        const Pack<Key, W> p = *(const Pack<Key, W>*)(sh.row_key + w0 + i);
#pragma unroll
                        for (int j = 0; j < W; ++j) order += (p.v[j] > key) | ((p.v[j] == key) & (i + j < lane));
                    }
#pragma unroll 4
                    for (int i = w0 + 32; i < count; i += W) {
                        const Pack<Key, W> p = *(const Pack<Key, W>*)(sh.row_key + i);
#pragma unroll
                        for (int j = 0; j < W; ++j) order += p.v[j] > key;
                    }
                }
                __syncthreads();
                sh.row_mass[tid] = 0;
                if (tid < count) sh.row_key[order] = key;
                __syncthreads();
                if (tid < count) sh.row_mass[order] = kWeight ? mass(key) : 1;
                __syncthreads();
                const u64 m = sh.row_mass[tid];
                u64 all;
                const u64 before = above + block_prefix(m, sh.scan, &all);
                if (before < target && target <= before + m) {
                    const Key k = sh.row_key[tid];
                    auto places = [&](auto&& in_front) {      // values of which this holds, which are the first ones
                        int n = 0;
                        for (int step = kList / 2; step > 0; step /= 2)
                            if (n + step <= count && in_front(sh.row_key[n + step - 1])) n += step;
                        return n < count && in_front(sh.row_key[n]) ? n + 1 : n;
                    };
                    const int greater = places([&](Key q) { return q > k; }), least = places([&](Key q) { return q >= k; });
                    sh.border = k;
                    sh.before = before - (u64)(tid - greater) * m;
                    sh.own = (u64)(least - greater) * m;
                    sh.found = 1;
                }
                advance();
                return sh.found ? Border{sh.border, sh.before, sh.own} : Border{edge, above, 0};
            };
            // a round leaves 1/256 of the span or less: 9 are the most for 64-bit keys
            for (int round = 0; round < 12; ++round) {
                unsigned* const bins = sh.bins[turn & 1];
                each(low, [&](Key k) {
                    if (k > high) return;
                    const A d = depth(k);
                    int bin = bin_of(d);
                    if (octave >= 0) {
                        if (bin != octave) return;
                        const int place = atomicAdd(&sh.listed[turn & 1], 1);
                        if (place < kList) sh.list_key[place] = k;
                        bin = (int)((high - k) >> down);
                    }
                    if (kWeight) M::add(bins, bin, power(-d), shift);
                    else M::count(bins, bin);
                });
                cluster.sync();
                if (octave >= 0) {
                    int from = 0, place = 0;
                    const int count = listed(from, place);
                    if (count <= kList) return in_list(count, from, place);      // the same in all blocks
                }
                const int found = search(by_weight, above, [&](u64 total) { return target = octave < 0 ? aim(total) : target; });
                if (found < 0) break;
                above = sh.before;
                const u64 mine = sh.own;
                // the next search writes these behind barriers that every thread passes after this
                if (octave < 0) {
                    octave = found;
                    high = bin_high(found);
                    low = max(low, bin_low(found));
                } else {
                    high -= (Key)found << down;
                    const Key span = ((Key)1 << down) - 1;
                    low = high - low > span ? high - span : low;
                }
                if (low == high) return {high, above, mine};
                const int bits = 64 - __clzll((u64)(high - low));    // of the span; bins of it have 9
                down = bits > 9 ? bits - 9 : 0;
            }
            return {edge, above, 0};    // not reached: a target is never above the sum of all
        };
        // Writes down the token that `aim_of(total)` and the sums of kept weights decide on.
        const double u = a.u_dtype == DT_F64 ? ((const double*)a.u)[row] : (double)((const float*)a.u)[row];
        auto aim_of = [&](u64 total) {
            const u64 aim = u > 0 ? (u >= 1 ? total : (u64)(u * (double)total)) : 0;
            return aim >= total ? total - 1 : aim;
        };
        auto write = [&](Key k, int at, u64 total) {
            a.token[row] = at;
            const double e = k == top ? 0.0 : ((double)O::value(k) * 0.5 - (double)most * 0.5) / (double)temp * 2.0;    // halves, as in depth()
            ((A*)a.logp)[row] = (A)(e - log((double)total / (double)(1ULL << shift)));
        };
        const A least = (A)fmin(row_param(a.min_p, row), 1.0);   // the largest logit stays
        // The first block draws from the `count` largest values of the row, one a thread: the first `k` in
        // their order, then top-p, min-p and the draw as everywhere.
        auto draw_from = [&](int count, int from, int place, int k) {
            Key key = 0;
            int at = 0;
            if (tid < count) {
                key = cluster.map_shared_rank(sh.list_key, from)[place];
                at = cluster.map_shared_rank(sh.list_at, from)[place];
                sh.row_key[tid] = key;
                sh.row_at[tid] = at;
            }
            __syncthreads();
            int order = 0;
#pragma unroll 8
            for (int i = 0; i < (tid < count ? count : 0); ++i) {
                const Key k = sh.row_key[i];
                order += (k > key) | ((k == key) & (sh.row_at[i] < at));
            }
            __syncthreads();
            if (tid < count) {
                sh.row_key[order] = key;
                sh.row_at[order] = at;
            }
            __syncthreads();
            const int kept_k = min(k, count);
            key = tid < kept_k ? sh.row_key[tid] : 0;
            at = sh.row_at[tid < kept_k ? tid : 0];
            u64 m = tid < kept_k ? mass(key) : 0, sum, total;
            const u64 before = block_prefix(m, sh.scan, &sum);
            const double pp = row_param(a.top_p, row);
            if (pp < 1) {
                const double want = ceil(pp * (double)sum);
                const u64 need = want >= 1 ? min((u64)want, sum) : 1;
                if (before >= need) m = 0;
            }
            if (tid < kept_k && !(weight(key) >= least)) m = 0;
            sh.row_mass[tid] = m;
            block_prefix(m, sh.scan, &total);
            __syncthreads();
            u64 upto = 0;
#pragma unroll 8
            for (int i = 0; i < (m ? kept_k : 0); ++i) {
                const u64 w = sh.row_mass[i];
                upto += sh.row_at[i] <= at ? w : 0;
            }
            const u64 aim = aim_of(total);
            if (m && upto - m <= aim && aim < upto) write(key, at, total);
        };
        bool short_list = false;
        if (!greedy && !none) {
            const double kk = row_param(a.top_k, row);
            if (kk >= 1 && kk < (double)v) {
                // the k-th largest of all threads' own largest keys is not above the k-th largest key: with it
                // the first histogram is of a few values instead of all
                Key floor = 1;
                if (kk <= (double)(blocks * kThreads)) {
                    if (own_top) M::count(sh.bins[turn & 1], octave_bin(own_top));
                    cluster.sync();
                    const int found = search(std::false_type(), 0, [&](u64) { return (u64)kk; });
                    if (found >= 0) floor = bin_low(found);
                    if (RESIDENT && kk <= kList / 2 && found >= 0) {
                        // most threads have loaded none
                        for (int i = tid * V; own_top >= floor && i < (int)slice; i += kThreads * V) {
                            const Pack<typename O::Stored, V> q = *(const Pack<typename O::Stored, V>*)(keys + i);
#pragma unroll
                            for (int j = 0; j < V; ++j) {
                                if (q.v[j] < floor) continue;
                                const int place = atomicAdd(&sh.listed[turn & 1], 1);
                                if (place < kList) {
                                    sh.list_key[place] = q.v[j];
                                    sh.list_at[place] = (int)s0 + i + j;
                                }
                            }
                        }
                        cluster.sync();
                        int from = 0, place = 0;
                        const int count = listed(from, place);
                        if (count <= kList) {     // the same in all blocks
                            if (rank == 0) draw_from(count, from, place, (int)kk);
                            short_list = true;
                        }
                    }
                }
                if (!short_list) {
                    const Border b = border_of(std::false_type(), floor, [&](u64) { return (u64)kk; });
                    edge = b.key;
                    ties = (u64)kk - b.above;
                    tied = b.own;
                }
            }
            const double pp = row_param(a.top_p, row);
            if (pp < 1 && !short_list) {
                u64 need = 0;
                const Border b = border_of(std::true_type(), (Key)1, [&](u64 sum) {
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
        if (!short_list) {
            if (!(weight(edge) >= least)) ties = 0;
            typename M::Sum above;
            u64 at_edge = 0;
            each(edge, [&](Key k) {
                if (k == edge) {
                    ++at_edge;
                } else {
                    const A e = weight(k);
                    if (e >= least) above.add(e, shift);
                }
            });
            const u64 mine = warp_sum(above.total());
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
            const u64 aim = aim_of(total);
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
            const int owner = sh.found;
            if (owner >= 0) {
                // the draw lies in the values of one warp of this block: all threads look for it, each in a
                // piece of neighbouring values
                const u64 first = sh.before, first_tie = sh.extra;
                const int64_t o0 = min(owner * per_warp, size), o1 = min(o0 + per_warp, size), piece = (per_warp + kThreads - 1) / kThreads;
                const int64_t i0 = min(o0 + tid * piece, o1), i1 = min(i0 + piece, o1);
                u64 equal = 0, sum = 0;
                for (int64_t i = i0; i < i1; ++i) equal += key_at(i) == edge;
                const u64 tie0 = first_tie + block_prefix(equal, sh.scan, &unused);
                auto walk = [&](auto&& stop) {
                    u64 tie = tie0, s = 0;
                    for (int64_t i = i0; i < i1; ++i) {
                        const Key k = key_at(i);
                        if (k == edge ? tie++ >= ties : k < edge || !(weight(k) >= least)) continue;
                        s += mass(k);
                        if (stop(s, i, k)) break;
                    }
                    return s;
                };
                sum = walk([](u64, int64_t, Key) { return false; });
                const u64 here = first + block_prefix(sum, sh.scan, &unused);
                if (here <= aim && aim < here + sum)
                    walk([&](u64 s, int64_t i, Key k) {
                        if (here + s <= aim) return false;
                        write(k, (int)(s0 + i), total);
                        return true;
                    });
            }
        }
        cluster.sync();    // no block's shared memory goes, or has the next row, while another may read it
    }
}

template <typename T, int V, bool WIDE, bool RESIDENT>
cudaError_t launch(const SampleArgs& a, int blocks, int64_t per_warp, int shift, int sm_count, cudaStream_t s) {
    const size_t bytes = (sizeof(SampleShared<T, WIDE>) + 15) / 16 * 16 + (RESIDENT ? (size_t)per_warp * kWarps * sizeof(typename Order<T>::Stored) : 0);
    const auto kernel = sample_kernel<T, V, WIDE, RESIDENT>;
    if (bytes > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t config = {};
    // Clusters that are resident at once, as far as registers and shared memory tell (a cluster starts
    // slower than a row that follows another in it), each with as many rows as the others.
    const int64_t each_sm = std::min<int64_t>(2, 227 * 1024 / (int64_t)(bytes + 1024));
    const int64_t most = std::max<int64_t>(sm_count * each_sm * 15 / 16 / blocks, 1), turns = (a.rows + most - 1) / most;
    config.gridDim = dim3((unsigned)((a.rows + turns - 1) / turns * blocks));
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
    const int64_t per_warp = ((a.v + blocks - 1) / blocks + kWarps * kGrain - 1) / (kWarps * kGrain) * kGrain, slice = per_warp * kWarps;
    int shift = 62;                                             // v terms of at most 2^shift stay below 2^62
    while ((1LL << (62 - shift)) < a.v) --shift;
    if (a.rows * blocks >= (1LL << 31)) return cudaErrorInvalidValue;
    constexpr int V = 16 / sizeof(T);
    if constexpr (kDouble) {
        if (slice > kSlice) return launch<T, 1, true, false>(a, blocks, per_warp, shift, sm_count, s);
        return a.v % V == 0 ? launch<T, V, true, true>(a, blocks, per_warp, shift, sm_count, s) : launch<T, 1, true, true>(a, blocks, per_warp, shift, sm_count, s);
    } else {
        if (slice > kSlice) return launch<T, 1, true, false>(a, blocks, per_warp, shift, sm_count, s);
        return a.v % V == 0 ? launch<T, V, false, true>(a, blocks, per_warp, 45, sm_count, s) : launch<T, 1, false, true>(a, blocks, per_warp, 45, sm_count, s);
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
