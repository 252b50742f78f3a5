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
//   - walks the steps: a lane's products of C and h are summed over its states, and every kGroup steps
//     the L lanes of a channel add theirs up by halving exchanges, each ending with one step's sum,
//   - adds D x, applies the gate and stores y, channels side by side.
// One barrier a tile: two buffers alternate.
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

template <typename A, int L, int N, bool LOCAL>
struct ScanShared {
    static constexpr int kChannels = kThreads / L, kPairs = N / 2;
    static constexpr int kPitch = kChannels + 32 / L;      // lanes of a warp store to different banks
    static constexpr int kTiles = LOCAL ? 1 : 2;
    alignas(16) A step[2][kChannels][kSteps + 1][4];       // dt, dt, dt x, dt x
    alignas(16) A b[2][kSteps / 2][kPairs][L][4];          // two steps' pairs
    alignas(16) A c[kTiles][kSteps / 2][kPairs][L][4];
    A y[kTiles][kSteps][kPitch];
};

template <typename T, int L, int N, bool LOCAL>
__global__ void __launch_bounds__(kThreads) scan_kernel(SelectiveScanArgs a, ScanChunks<typename Acc<T>::type> ck, int blocks) {
    using A = typename Acc<T>::type;
    constexpr int kChannels = kThreads / L;
    constexpr int kPairs = N / 2;
    constexpr int kGroup = L < 8 ? L : 8;
    constexpr int kOwn = (kSteps * kChannels + kThreads - 1) / kThreads;
    constexpr int kStates = L * N;
    constexpr int kOwnB = (kSteps * kStates + kThreads - 1) / kThreads;
    extern __shared__ __align__(16) unsigned char scan_shared[];
    auto& sh = *(ScanShared<A, L, N, LOCAL>*)scan_shared;

    const int tid = threadIdx.x, lane = tid & (L - 1), own = tid / L;
    const int64_t per_group = a.d / a.groups;
    const int64_t per_blocks = blocks / a.groups;
    const int64_t b = blockIdx.x / blocks, blk = blockIdx.x % blocks;
    const int64_t g = blk / per_blocks, c0 = g * per_group + blk % per_blocks * kChannels, c1 = (g + 1) * per_group;
    const int64_t end_all = a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.t) : a.t;
    const int64_t t0 = blockIdx.y * ck.length;
    const int64_t stop = min(t0 + ck.length, a.t), end = min(stop, end_all);     // end < t0: nothing to walk
    const int64_t bn = (int64_t)a.groups * a.n;
    const T* const xs = (const T*)a.x + b * a.t * a.d;
    const T* const ds = (const T*)a.delta + b * a.t * a.d;
    const T* const zs = a.z ? (const T*)a.z + b * a.t * a.d : nullptr;
    const T* const bs = (const T*)a.B + b * a.t * bn + g * a.n;
    const T* const cs = (const T*)a.C + b * a.t * bn + g * a.n;

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

    // values of a tile that this thread lays down: requested early, used a tile later
    T rx[kOwn], rd[kOwn], rz[kOwn], rb[kOwnB], rc[kOwnB];
    A px[kOwn], pz[kOwn];       // the tile being walked: for the skip and the gate
    A sum = 0;                  // LOCAL: dt summed over the chunk, for the channel of slot tid % kChannels
    auto request = [&](int64_t from) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int e = tid + i * kThreads;
            const int64_t t = from + e / kChannels, ch = c0 + e % kChannels;
            const bool on = t < end && ch < c1 && e < kSteps * kChannels;
            const int64_t at = t * a.d + ch;
            rx[i] = on ? xs[at] : narrow<T>(A(0));
            rd[i] = on ? ds[at] : narrow<T>(A(0));
            if (!LOCAL) rz[i] = on && zs ? zs[at] : narrow<T>(A(0));
        }
#pragma unroll
        for (int i = 0; i < kOwnB; ++i) {
            const int e = tid + i * kThreads, n = e % kStates;
            const int64_t t = from + e / kStates;
            const bool on = t < end && n < a.n && e < kSteps * kStates;
            rb[i] = on ? bs[t * bn + n] : narrow<T>(A(0));
            if (!LOCAL) rc[i] = on ? cs[t * bn + n] : narrow<T>(A(0));
        }
    };
    auto lay = [&](int64_t from, int buf) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int e = tid + i * kThreads;
            if (kSteps * kChannels % kThreads && e >= kSteps * kChannels) break;
            const int s = e / kChannels, slot = e % kChannels;
            const bool on = from + s < end && c0 + slot < c1;
            A dt = widen(rd[i]) + (on && a.delta_bias ? ((const A*)a.delta_bias)[c0 + slot] : A(0));
            if (a.softplus) dt = softplus(dt);
            if (!on) dt = 0;
            const A x = widen(rx[i]), dtx = dt * x;
            A* const to = sh.step[buf][slot][s];
            *(Two<A>*)to = {dt, dt};
            *(Two<A>*)(to + 2) = {dtx, dtx};
            if (LOCAL) sum += dt;
        }
#pragma unroll
        for (int i = 0; i < kOwnB; ++i) {
            const int e = tid + i * kThreads;
            if (kSteps * kStates % kThreads && e >= kSteps * kStates) break;
            const int s = e / kStates, n = e % kStates;
            const int p = n / (2 * L), l = n % (2 * L) / 2, j = (s & 1) * 2 + (n & 1);
            sh.b[buf][s / 2][p][l][j] = widen(rb[i]);
            if (!LOCAL) sh.c[buf][s / 2][p][l][j] = widen(rc[i]);
        }
    };

    auto walk = [&](int buf, int live, auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
        for (int s0 = 0; s0 < kSteps; s0 += kGroup) {
            if (!kWhole && s0 >= live) break;
            A part[kGroup];
#pragma unroll
            for (int i = 0; i < kGroup; i += 2) {
                Two<A> bb[kPairs][2], cc[kPairs][2];
#pragma unroll
                for (int p = 0; p < kPairs; ++p) {
                    const A* q = sh.b[buf][(s0 + i) / 2][p][lane];
                    const Pack<A, 16 / sizeof(A)>* v = (const Pack<A, 16 / sizeof(A)>*)q;
                    Pack<A, 16 / sizeof(A)> w[sizeof(A) / 4];
#pragma unroll
                    for (int k = 0; k < (int)sizeof(A) / 4; ++k) w[k] = v[k];
                    bb[p][0] = ((Two<A>*)w)[0];
                    bb[p][1] = ((Two<A>*)w)[1];
                    if (!LOCAL) {
                        const Pack<A, 16 / sizeof(A)>* u = (const Pack<A, 16 / sizeof(A)>*)sh.c[buf][(s0 + i) / 2][p][lane];
#pragma unroll
                        for (int k = 0; k < (int)sizeof(A) / 4; ++k) w[k] = u[k];
                        cc[p][0] = ((Two<A>*)w)[0];
                        cc[p][1] = ((Two<A>*)w)[1];
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (i + k >= kGroup) break;
                    Pack<A, 16 / sizeof(A)> w[sizeof(A) / 4];
                    const Pack<A, 16 / sizeof(A)>* v = (const Pack<A, 16 / sizeof(A)>*)sh.step[buf][own][s0 + i + k];
#pragma unroll
                    for (int r = 0; r < (int)sizeof(A) / 4; ++r) w[r] = v[r];
                    const Two<A> dt = ((Two<A>*)w)[0], dtx = ((Two<A>*)w)[1];
                    Two<A> y;
#pragma unroll
                    for (int p = 0; p < kPairs; ++p) {
                        const Two<A> m = mul(dt, decay[p]);
                        const Two<A> e = {power(m.x), power(m.y)};
                        const Two<A> next = fma(e, h[p], mul(dtx, bb[p][k]));
                        // behind the end the step is left out: 0 times an infinite A is not 0
                        if (kWhole || s0 + i + k < live) h[p] = next;
                        if (!LOCAL) y = p ? fma(cc[p][k], h[p], y) : mul(cc[p][k], h[p]);
                    }
                    if (!LOCAL) part[i + k] = y.x + y.y;
                }
            }
            if (LOCAL) continue;
            // lanes at distance o exchange halves; a lane ends with the sum of step lane / (L / kGroup)
            int width = kGroup;
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) {
                if (width > 1) {
                    width /= 2;
                    const bool up = lane & o;
#pragma unroll
                    for (int i = 0; i < kGroup / 2; ++i) {
                        if (i >= width) break;
                        const A send = up ? part[i] : part[i + width], keep = up ? part[i + width] : part[i];
                        part[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
                    }
                } else {
                    part[0] += __shfl_xor_sync(0xffffffffu, part[0], o);
                }
            }
            if (lane % (L / kGroup) == 0) sh.y[buf][s0 + lane / (L / kGroup)][own] = part[0];
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
        request(t0);
        lay(t0, 0);
        keep();
        __syncthreads();
        int buf = 0;
        for (int64_t t = t0; t < end; t += kSteps, buf ^= 1) {
            const bool more = t + kSteps < end;
            if (more) request(t + kSteps);
            const int live = (int)min(end - t, (int64_t)kSteps);
            if (live == kSteps) walk(buf, live, std::true_type());
            else walk(buf, live, std::false_type());
            if (more) lay(t + kSteps, buf ^ 1);
            __syncthreads();
            if (!LOCAL) {
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    const int e = tid + i * kThreads;
                    if (kSteps * kChannels % kThreads && e >= kSteps * kChannels) break;
                    const int s = e / kChannels, slot = e % kChannels;
                    const int64_t ch = c0 + slot;
                    if (s >= live || ch >= c1) continue;
                    A y = sh.y[buf][s][slot];
                    if (a.D) y += ((const A*)a.D)[ch] * px[i];
                    if (zs) y *= gate(pz[i]);
                    ((T*)a.y)[(b * a.t + t + s) * a.d + ch] = narrow<T>(y);
                }
            }
            if (more) keep();
        }
    }
    if (LOCAL) {
        // dt of a channel was summed by kThreads / kChannels threads: add them up in their order
        __syncthreads();
        A* const part = &sh.step[0][0][0][0];
        part[tid] = sum;
        __syncthreads();
        if (tid < kChannels && c0 + tid < c1) {
            A s = 0;
            for (int i = tid; i < kThreads; i += kChannels) s += part[i];
            ck.sums[(b * ck.count + blockIdx.y) * a.d + c0 + tid] = s;
        }
    } else {
        // rows behind the end of the sequence
        for (int64_t e = tid; e < (stop - max(end, t0)) * kChannels; e += kThreads) {
            const int64_t ch = c0 + e % kChannels, t = max(end, t0) + e / kChannels;
            if (ch < c1) ((T*)a.y)[(b * a.t + t) * a.d + ch] = narrow<T>(A(0));
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
