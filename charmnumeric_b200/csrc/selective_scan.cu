// Selective state space scan.
//
//   dt = softplus(delta[b,t,c] + delta_bias[c])
//   h[b,c,n] <- exp(dt A[c,n]) h[b,c,n] + dt B[b,t,g,n] x[b,t,c]
//   y[b,t,c] = (sum_n C[b,t,g,n] h[b,c,n] + D[c] x[b,t,c]) z / (1 + exp(-z))
//
// Behind the end of a sequence the states stay and y is 0.
//
// A prompt is bound by its exponentials, one for each (b, t, c, n): an SM's special function units
// make 16 a clock, beside which the four multiply(-add)s of a state step and the memory traffic are
// the smaller part.  So every exponential is computed once, wherever there are enough channels: a
// channel's states are spread over L lanes of a warp, which walk the whole time axis with their
// states in registers.
#include <algorithm>
#include <type_traits>

#include "cn_types.hpp"
#include "sequence.cuh"
#include "sequence.hpp"

namespace cn {

using namespace seq;

namespace {

constexpr int kThreads = 256;
constexpr int kSteps = 16;      // time steps staged in shared memory at once

// ---- arithmetic -------------------------------------------------------------------------------------

// Two values side by side.  Floats are multiplied and added in pairs by one instruction each.
template <typename A> struct alignas(2 * sizeof(A)) Two { A x, y; };

__device__ __forceinline__ unsigned long long as_bits(Two<float> v) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ Two<float> as_two(unsigned long long r) {
    Two<float> v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}
__device__ __forceinline__ Two<float> mul(Two<float> a, Two<float> b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(as_bits(a)), "l"(as_bits(b)));
    return as_two(r);
}
__device__ __forceinline__ Two<float> fma(Two<float> a, Two<float> b, Two<float> c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(as_bits(a)), "l"(as_bits(b)), "l"(as_bits(c)));
    return as_two(r);
}
__device__ __forceinline__ Two<double> mul(Two<double> a, Two<double> b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ Two<double> fma(Two<double> a, Two<double> b, Two<double> c) {
    return {::fma(a.x, b.x, c.x), ::fma(a.y, b.y, c.y)};
}

// 2^v for floats, e^v for doubles: A is scaled by `decay_scale` once
__device__ __forceinline__ float power(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ double power(double v) { return exp(v); }
template <typename A> __device__ __forceinline__ A decay_scale() { return A(1); }
template <> __device__ __forceinline__ float decay_scale<float>() { return 1.4426950408889634f; }

__device__ __forceinline__ float reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// log(1 + e^v) = max(v, 0) + log(1 + e), e = e^-|v|.  With s = e / (2 + e) <= 1/3 the logarithm is
// 2 atanh(s) = 2 (s + s^3/3 + s^5/5 + ...), which keeps its relative precision for small e; the first
// term left out is below 2^-27 of the sum.
__device__ __forceinline__ float softplus(float v) {
    const float e = power(-1.4426950408889634f * fabsf(v));
    const float s = e * reciprocal(2.0f + e), q = s * s;
    float p = 1.0f / 15.0f;
    p = fmaf(p, q, 1.0f / 13.0f);
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    return fmaxf(v, 0.0f) + 2.0f * fmaf(p * q, s, s);
}
__device__ __forceinline__ double softplus(double v) { return (v > 0 ? v : 0.0) + log1p(exp(-fabs(v))); }

__device__ __forceinline__ float gate(float z) { return z * reciprocal(1.0f + power(-1.4426950408889634f * z)); }
__device__ __forceinline__ double gate(double z) { return z / (1.0 + exp(-z)); }

// ---- prompts ------------------------------------------------------------------------------------------
//
// A block has kThreads / L channels of one sequence and group, L lanes for each; a lane has N states,
// in pairs (p L + l) 2 + {0, 1}.  The time axis is walked in tiles of kSteps.  For each tile the block
//   - computes (dt, dt x) of its channels and lays them, B and C into shared memory as floats, from
//     values that were requested a tile ahead,
//   - walks the steps; each lane lays the sum over its own states into shared memory,
//   - adds up the lanes of a channel and D x, applies the gate and stores y, channels side by side.
// One barrier a tile: two buffers alternate.  Sums through shared memory cost a store a step, and
// nothing waits for them; the halving exchanges between lanes that were here first took 3.5
// instructions a step and their latency with them.
//
// Where there are too few channels to fill the GPU, the time axis is cut into chunks.  A first pass
// (LOCAL) computes each chunk's states from zero and the sum S of its dt; the second enters a chunk with
//   h <- exp(A S_k) h + local_k   over the chunks k before it
// which costs every exponential twice.

template <typename A>
struct ScanChunks {
    int64_t length = 0;   // steps of a chunk, a multiple of kSteps
    int count = 1;
    A* local = nullptr;   // (b, count, d, n)
    A* sums = nullptr;    // (b, count, d)
};

template <typename A> struct alignas(16) Four { Two<A> x, y; };

template <typename A, int L, int N, bool LOCAL>
struct ScanShared {
    static constexpr int kChannels = kThreads / L, kPairs = N / 2;
    static constexpr int kTiles = LOCAL ? 1 : 2;
    Four<A> step[2][kChannels][kSteps + 1];                // (dt, dt), (dt x, dt x); one more against bank conflicts
    Four<A> b[2][kSteps / 2][kPairs][L];                   // the pairs of two steps
    Four<A> c[kTiles][kSteps / 2][kPairs][L];
    alignas(16) A y[kTiles][kSteps][kThreads];             // every lane's sum over its states
};

// sum of the L lanes of a channel; the pieces are read in an order that keeps the banks apart
template <int L, typename A>
__device__ __forceinline__ A lanes_sum(const A* y, int slot) {
    constexpr int V = 16 / sizeof(A) < L ? 16 / sizeof(A) : L, kPieces = L / V;
    A t = 0;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
        const int piece = (k + slot * L / 32) % kPieces;
        const Pack<A, V> v = *(const Pack<A, V>*)(y + slot * L + piece * V);
        A s = v.v[0];
#pragma unroll
        for (int j = 1; j < V; ++j) s += v.v[j];
        t += s;
    }
    return t;
}

template <typename T, int L, int N, bool LOCAL>
__global__ void __launch_bounds__(kThreads) scan_kernel(SelectiveScanArgs a, ScanChunks<typename Acc<T>::type> ck, int blocks) {
    using A = typename Acc<T>::type;
    constexpr int kChannels = kThreads / L;
    constexpr int kPairs = N / 2;
    constexpr int kOwn = (kSteps * kChannels + kThreads - 1) / kThreads;     // values of x, delta, z a thread lays down
    constexpr int kRows = kThreads / kChannels;                              // ... kRows steps apart
    constexpr int kStates = L * N;
    constexpr int kOwnB = (kSteps * kStates + kThreads - 1) / kThreads;
    constexpr int kGroup = kPairs >= 4 ? 2 : 4;                              // steps whose exponentials are made together
    extern __shared__ __align__(16) unsigned char scan_shared[];
    auto& sh = *(ScanShared<A, L, N, LOCAL>*)scan_shared;

    const int tid = threadIdx.x, lane = tid & (L - 1), own = tid / L;
    const int64_t per_group = a.d / a.groups;
    const int64_t per_blocks = blocks / a.groups;
    const int64_t b = blockIdx.x / blocks, blk = blockIdx.x % blocks;
    const int64_t g = blk / per_blocks, c0 = g * per_group + blk % per_blocks * kChannels, c1 = (g + 1) * per_group;
    const int64_t end_all = a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.t) : a.t;
    const int64_t t0 = blockIdx.y * ck.length;
    const int64_t stop = min(t0 + ck.length, a.t), end = min(stop, end_all);     // end <= t0: nothing to walk
    const int64_t bn = (int64_t)a.groups * a.n;

    // a lane's states and decays
    const int64_t c = c0 + own;
    Two<A> h[kPairs], decay[kPairs];
#pragma unroll
    for (int p = 0; p < kPairs; ++p) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = (p * L + lane) * 2 + j;
            const bool on = n < a.n && c < c1;
            const int64_t i = c * a.n + n;
            A v = 0, w = 0;
            if (on) {
                w = ((const A*)a.A)[i] * decay_scale<A>();
                if (!LOCAL && a.state) v = ((const A*)a.state)[b * a.d * a.n + i];
                if (!LOCAL)
                    for (int k = 0; k < (int)blockIdx.y; ++k) {
                        const int64_t q = (b * ck.count + k) * a.d;
                        const A s = ck.sums[q + c];
                        v = (s == 0 ? v : power(w * s) * v) + ck.local[q * a.n + i];
                    }
            }
            (j ? h[p].y : h[p].x) = v;
            (j ? decay[p].y : decay[p].x) = w;
        }
    }

    // what this thread lays down: x, delta, z of one channel, kRows steps apart, and pieces of B and C
    const int row = tid / kChannels, slot = tid % kChannels;
    const int64_t ch = c0 + slot;
    const bool mine = ch < c1 && row < kSteps;
    const A bias = mine && a.delta_bias ? ((const A*)a.delta_bias)[ch] : A(0);
    const A skip = mine && a.D ? ((const A*)a.D)[ch] : A(0);
    const int64_t first = (b * a.t + t0 + row) * a.d + ch, stride = kRows * a.d, tile = kSteps * a.d;
    const T *xs = (const T*)a.x + first, *ds = (const T*)a.delta + first, *zs = a.z ? (const T*)a.z + first : nullptr;
    T* ys = (T*)a.y + first;
    const T *bs = (const T*)a.B + (b * a.t + t0) * bn + g * a.n, *cs = (const T*)a.C + (b * a.t + t0) * bn + g * a.n;

    T rx[kOwn], rd[kOwn], rz[kOwn], rb[kOwnB], rc[kOwnB];     // requested early, used a tile later
    A px[kOwn], pz[kOwn];                                     // of the tile being walked: for the skip and the gate
    A sum = 0;                                                // LOCAL: dt summed over the chunk
    const T zero = narrow<T>(A(0));
    auto request = [&](int live) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const bool on = mine && row + i * kRows < live;
            rx[i] = on ? xs[i * stride] : zero;
            rd[i] = on ? ds[i * stride] : zero;
            if (!LOCAL) rz[i] = on && a.z ? zs[i * stride] : zero;
        }
        xs += tile;
        ds += tile;
        if (!LOCAL && a.z) zs += tile;
#pragma unroll
        for (int i = 0; i < kOwnB; ++i) {
            const int e = tid + i * kThreads, n = e % kStates, s = e / kStates;
            const bool on = s < live && n < a.n;
            rb[i] = on ? bs[s * bn + n] : zero;
            if (!LOCAL) rc[i] = on ? cs[s * bn + n] : zero;
        }
        bs += kSteps * bn;
        cs += kSteps * bn;
    };
    auto lay = [&](int live, int buf) {
        if (row < kSteps) {
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                A dt = widen(rd[i]) + bias;
                if (a.softplus) dt = softplus(dt);
                if (!mine || row + i * kRows >= live) dt = 0;
                const A dtx = dt * widen(rx[i]);
                sh.step[buf][slot][row + i * kRows] = {{dt, dt}, {dtx, dtx}};
                if (LOCAL) sum += dt;
            }
        }
#pragma unroll
        for (int i = 0; i < kOwnB; ++i) {
            const int e = tid + i * kThreads;
            if (kSteps * kStates % kThreads && e >= kSteps * kStates) break;
            const int s = e / kStates, n = e % kStates;
            const int p = n / (2 * L), l = n % (2 * L) / 2, j = (s & 1) * 2 + (n & 1);
            ((A*)&sh.b[buf][s / 2][p][l])[j] = widen(rb[i]);
            if (!LOCAL) ((A*)&sh.c[buf][s / 2][p][l])[j] = widen(rc[i]);
        }
    };

    auto walk = [&](int buf, int live, auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
        for (int s0 = 0; s0 < kSteps; s0 += kGroup) {
            if (!kWhole && s0 >= live) break;
            Two<A> e[kGroup][kPairs], term[kGroup][kPairs];
            // all of the group's exponentials and terms, which wait for no state ...
#pragma unroll
            for (int i = 0; i < kGroup; i += 2) {
                const Four<A> u = sh.step[buf][own][s0 + i], v = sh.step[buf][own][s0 + i + 1];
#pragma unroll
                for (int p = 0; p < kPairs; ++p) {
                    const Four<A> bb = sh.b[buf][(s0 + i) / 2][p][lane];
                    const Two<A> m0 = mul(u.x, decay[p]), m1 = mul(v.x, decay[p]);
                    e[i][p] = {power(m0.x), power(m0.y)};
                    e[i + 1][p] = {power(m1.x), power(m1.y)};
                    term[i][p] = mul(u.y, bb.x);
                    term[i + 1][p] = mul(v.y, bb.y);
                }
            }
            // ... then the recurrence
#pragma unroll
            for (int i = 0; i < kGroup; i += 2) {
                Two<A> y[2];
#pragma unroll
                for (int p = 0; p < kPairs; ++p) {
                    Four<A> cc;
                    if (!LOCAL) cc = sh.c[buf][(s0 + i) / 2][p][lane];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const Two<A> next = fma(e[i + k][p], h[p], term[i + k][p]);
                        // behind the end a step is left out: 0 times an infinite A is not 0
                        if (kWhole || s0 + i + k < live) h[p] = next;
                        if (!LOCAL) y[k] = p ? fma(k ? cc.y : cc.x, h[p], y[k]) : mul(k ? cc.y : cc.x, h[p]);
                    }
                }
                if (!LOCAL) {
                    sh.y[buf][s0 + i][tid] = y[0].x + y[0].y;
                    sh.y[buf][s0 + i + 1][tid] = y[1].x + y[1].y;
                }
            }
        }
    };

    auto keep = [&]() {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            px[i] = widen(rx[i]);
            if (!LOCAL) pz[i] = widen(rz[i]);
        }
    };

    if (t0 < end) {
        int live = (int)min(end - t0, (int64_t)kSteps);
        request(live);
        lay(live, 0);
        keep();
        __syncthreads();
        int buf = 0;
        for (int64_t t = t0; t < end; t += kSteps, buf ^= 1) {
            const int next = (int)min(max(end - t - kSteps, (int64_t)0), (int64_t)kSteps);
            if (next) request(next);
            if (live == kSteps) walk(buf, live, std::true_type());
            else walk(buf, live, std::false_type());
            if (next) lay(next, buf ^ 1);
            __syncthreads();
            if (!LOCAL) {
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    if (!mine || row + i * kRows >= live) continue;
                    A y = lanes_sum<L>(sh.y[buf][row + i * kRows], slot) + skip * px[i];
                    if (a.z) y *= gate(pz[i]);
                    ys[i * stride] = narrow<T>(y);
                }
                ys += tile;
            }
            if (next) keep();
            live = next;
        }
    }
    if (LOCAL) {
        // dt of a channel was summed by kRows threads: add them up in their order
        __syncthreads();
        A* const part = (A*)&sh.step;
        part[tid] = sum;
        __syncthreads();
        if (tid < kChannels && c0 + tid < c1) {
            A s = 0;
            for (int i = tid; i < kThreads; i += kChannels) s += part[i];
            ck.sums[(b * ck.count + blockIdx.y) * a.d + c0 + tid] = s;
        }
    } else {
        // rows behind the end of the sequence
        const int64_t from = max(end, t0);
        for (int64_t e = tid; e < (stop - from) * kChannels; e += kThreads) {
            const int64_t cc = c0 + e % kChannels;
            if (cc < c1) ((T*)a.y)[(b * a.t + from + e / kChannels) * a.d + cc] = zero;
        }
        if ((int)blockIdx.y != ck.count - 1) return;
    }
#pragma unroll
    for (int p = 0; p < kPairs; ++p)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = (p * L + lane) * 2 + j;
            if (n >= a.n || c >= c1) continue;
            const A v = j ? h[p].y : h[p].x;
            if (LOCAL) ck.local[((b * ck.count + blockIdx.y) * a.d + c) * a.n + n] = v;
            else ((A*)a.new_state)[(b * a.d + c) * a.n + n] = v;
        }
}

// ---- single tokens ------------------------------------------------------------------------------------
//
// The states are read and written once: a lane has V neighbouring states (16 bytes where n allows),
// `lanes` lanes a channel.  An inactive sequence's states are copied.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) scan_token_kernel(SelectiveScanArgs a, int lanes) {
    using A = typename Acc<T>::type;
    const int64_t at = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / lanes;   // b d + c
    const int lane = threadIdx.x & (lanes - 1);
    const bool on = at < a.b * a.d;
    const int64_t b = on ? at / a.d : 0, c = on ? at - b * a.d : 0;
    const bool live = on && !(a.lengths && a.lengths[b] < 1);
    const int64_t bn = (int64_t)a.groups * a.n;
    const T* const bs = (const T*)a.B + b * bn + c / (a.d / a.groups) * a.n;
    const T* const cs = (const T*)a.C + b * bn + c / (a.d / a.groups) * a.n;
    A x = 0, dt = 0, y = 0;
    if (live) {
        x = widen(((const T*)a.x)[at]);
        dt = widen(((const T*)a.delta)[at]) + (a.delta_bias ? ((const A*)a.delta_bias)[c] : A(0));
        if (a.softplus) dt = softplus(dt);
    }
    const A dtx = dt * x;
    if (on) {
        for (int n = lane * V; n < a.n; n += lanes * V) {
            Pack<A, V> h, w;
            if (a.state) h = *(const Pack<A, V>*)((const A*)a.state + at * a.n + n);
            else
#pragma unroll
                for (int j = 0; j < V; ++j) h.v[j] = 0;
            if (live) {
                w = *(const Pack<A, V>*)((const A*)a.A + c * a.n + n);
                const Pack<T, V> bb = *(const Pack<T, V>*)(bs + n), cc = *(const Pack<T, V>*)(cs + n);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    h.v[j] = power(dt * (w.v[j] * decay_scale<A>())) * h.v[j] + dtx * widen(bb.v[j]);
                    y += widen(cc.v[j]) * h.v[j];
                }
            }
            *(Pack<A, V>*)((A*)a.new_state + at * a.n + n) = h;
        }
    }
    for (int o = lanes / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (!on || lane) return;
    if (live) {
        if (a.D) y += ((const A*)a.D)[c] * x;
        if (a.z) y *= gate(widen(((const T*)a.z)[at]));
    }
    ((T*)a.y)[at] = narrow<T>(y);
}

template <typename T>
cudaError_t token(const SelectiveScanArgs& a, cudaStream_t s) {
    using A = typename Acc<T>::type;
    const int wide = sizeof(A) == 8 ? 2 : 4;
    const int v = a.n % wide == 0 ? wide : a.n % 2 == 0 ? 2 : 1;
    int lanes = 1;
    while (lanes < 32 && lanes * v < a.n) lanes *= 2;
    const int64_t blocks = (a.b * a.d * lanes + kThreads - 1) / kThreads;
    if (blocks >= (1LL << 31)) return cudaErrorInvalidValue;
    if (v == 4) scan_token_kernel<T, 4><<<(unsigned)blocks, kThreads, 0, s>>>(a, lanes);
    else if (v == 2) scan_token_kernel<T, 2><<<(unsigned)blocks, kThreads, 0, s>>>(a, lanes);
    else scan_token_kernel<T, 1><<<(unsigned)blocks, kThreads, 0, s>>>(a, lanes);
    return cudaGetLastError();
}

// ---- launches -------------------------------------------------------------------------------------------

int lanes_for(int n) { return n <= 4 ? 2 : n <= 8 ? 4 : n <= 64 ? 8 : n <= 128 ? 16 : 32; }

int64_t channel_blocks(const SelectiveScanArgs& a) {
    const int64_t channels = kThreads / lanes_for(a.n);
    return a.groups * ((a.d / a.groups + channels - 1) / channels);
}

// Chunks of the time axis: none while the channels' blocks give half of the SMs one each, since
// chunks compute every exponential twice; else as many as make two blocks an SM, of at least 64 steps.
template <typename A>
ScanChunks<A> chunks_for(const SelectiveScanArgs& a, int sm_count) {
    ScanChunks<A> ck;
    ck.length = std::max<int64_t>((a.t + kSteps - 1) / kSteps, 1) * kSteps;
    const int64_t blocks = channel_blocks(a) * a.b;
    if (2 * blocks >= sm_count || a.t < 128) return ck;
    const int64_t want = std::min<int64_t>(2 * sm_count / blocks, a.t / 64);
    ck.length = ((a.t + want - 1) / want + kSteps - 1) / kSteps * kSteps;
    ck.count = (int)((a.t + ck.length - 1) / ck.length);
    return ck;
}

template <typename T, int L, int N, bool LOCAL>
cudaError_t scan_pass(const SelectiveScanArgs& a, const ScanChunks<typename Acc<T>::type>& ck, int64_t blocks, int count, cudaStream_t s) {
    constexpr size_t bytes = sizeof(ScanShared<typename Acc<T>::type, L, N, LOCAL>);
    if (bytes > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(scan_kernel<T, L, N, LOCAL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return e;
    }
    scan_kernel<T, L, N, LOCAL><<<dim3((unsigned)(blocks * a.b), count), kThreads, bytes, s>>>(a, ck, (int)blocks);
    return cudaGetLastError();
}

template <typename T, int L, int N>
cudaError_t prompt(const SelectiveScanArgs& a, int sm_count, cudaStream_t s) {
    using A = typename Acc<T>::type;
    ScanChunks<A> ck = chunks_for<A>(a, sm_count);
    const int64_t blocks = channel_blocks(a);
    if (blocks * a.b >= (1LL << 31)) return cudaErrorInvalidValue;
    if (ck.count > 1) {
        ck.local = (A*)a.workspace;
        ck.sums = ck.local + a.b * ck.count * a.d * a.n;
        // the last chunk's states are never entered from
        const cudaError_t e = scan_pass<T, L, N, true>(a, ck, blocks, ck.count - 1, s);
        if (e != cudaSuccess) return e;
    }
    return scan_pass<T, L, N, false>(a, ck, blocks, ck.count, s);
}

template <typename T>
cudaError_t scan(const SelectiveScanArgs& a, int sm_count, cudaStream_t s) {
    if (a.t == 1) return token<T>(a, s);
    if (a.n <= 4) return prompt<T, 2, 2>(a, sm_count, s);
    if (a.n <= 8) return prompt<T, 4, 2>(a, sm_count, s);
    if (a.n <= 16) return prompt<T, 8, 2>(a, sm_count, s);
    if (a.n <= 32) return prompt<T, 8, 4>(a, sm_count, s);
    if (a.n <= 64) return prompt<T, 8, 8>(a, sm_count, s);
    if (a.n <= 128) return prompt<T, 16, 8>(a, sm_count, s);
    return prompt<T, 32, 8>(a, sm_count, s);
}

}  // namespace

size_t selective_scan_workspace(const SelectiveScanArgs& a, int sm_count) {
    if (a.t == 1) return 0;
    const int64_t count = chunks_for<float>(a, sm_count).count;
    if (count < 2) return 0;
    return (size_t)(a.b * count * a.d * (a.n + 1)) * (a.dtype == DT_F64 ? 8 : 4);
}

cudaError_t launch_selective_scan(const SelectiveScanArgs& a, int sm_count, cudaStream_t s) {
    switch (a.dtype) {
        case DT_F16: return scan<__half>(a, sm_count, s);
        case DT_F32: return scan<float>(a, sm_count, s);
        case DT_F64: return scan<double>(a, sm_count, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace cn
