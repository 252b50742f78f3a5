// Selective state space scan.
//
//   dt = softplus(delta[b,t,c] + delta_bias[c])
//   h[b,c,n] <- exp(dt A[c,n]) h[b,c,n] + dt B[b,t,g,n] x[b,t,c]
//   y[b,t,c] = (sum_n C[b,t,g,n] h[b,c,n] + D[c] x[b,t,c]) z / (1 + exp(-z))
//
// Behind the end of a sequence the states stay and y is 0.
//
// A prompt's floor is its exponentials, one for each (b, t, c, n): an SM's special function units
// make 16 a clock, beside which the four multiply(-add)s of a state step and the memory traffic are
// the smaller part.  So every exponential is computed once, wherever there are enough channels: a
// channel's states are spread over L lanes of a warp, which walk the whole time axis with their
// states in registers.
//
// 1 x 8192 x 4096 channels x 16 states in 16 bits, gated (floor 119 us at 1.9 GHz): a thread a channel
// 12332 us; states over lanes, tiles of 16 steps in shared memory 621; lanes' sums through shared memory
// instead of shuffles 570; walkers and helpers side by side, tiles copied ahead through a ring, sums and
// B, C in fewer bytes of shared memory 336 us.  There the issue slots are busy two
// thirds of the time and the special function units and shared memory half each: what is left is the
// instructions around an exponential (two steps' B and C widened, the term, the recurrence, C h).
// 5 x 1003 x 1537 x 16 in 32 bits, of random lengths: 1352 to 84-107 us (floor 27 at full length).
// 2 x 1000 x 500 x 12 in 64 bits: 1027 to 106 us (exponentials in FP64 instructions, twice over in chunks).
//
// Floats take the hardware's 2^x and 1 / x (errors of some 2^-22 of the value, and that of a 32-bit argument) in the
// decays, softplus and the gate: the library's functions would be several times the instructions of a step.
#include <algorithm>
#include <type_traits>

#include "cn_types.hpp"
#include "sequence.cuh"
#include "sequence.hpp"

namespace cn {

using namespace seq;

namespace {

constexpr int kThreads = 256, kHelpers = 256;

// ---- arithmetic -------------------------------------------------------------------------------------

// Two values side by side.  Floats are multiplied and added in pairs by one instruction each.
template <typename A> struct alignas(2 * sizeof(A)) Two { A x, y; };

__device__ __forceinline__ Two<float> mul(Two<float> a, Two<float> b) {
    const float2 r = __fmul2_rn({a.x, a.y}, {b.x, b.y});
    return {r.x, r.y};
}
__device__ __forceinline__ Two<float> fma(Two<float> a, Two<float> b, Two<float> c) {
    const float2 r = __ffma2_rn({a.x, a.y}, {b.x, b.y}, {c.x, c.y});
    return {r.x, r.y};
}
__device__ __forceinline__ Two<float> add(Two<float> a, Two<float> b) {
    const float2 r = __fadd2_rn({a.x, a.y}, {b.x, b.y});
    return {r.x, r.y};
}
__device__ __forceinline__ Two<double> add(Two<double> a, Two<double> b) { return {a.x + b.x, a.y + b.y}; }
template <typename A> __device__ __forceinline__ Two<A> both(A v) { return {v, v}; }
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

// e^(dt A), for steps.  A state sums the errors of its decays over as many steps as it remembers, and
// ex2.approx is on average a little low next to 0: by 0.6e-8, 1.8e-8 and 2.6e-8 of its value over
// [-0.001, 0], [-0.01, 0] and [-0.1, 0].  1e-8 more (in log2) costs nothing in a fused multiply-add, takes
// half of the error of long scans (4 x 151 x 3396 x 16: 2.4e-6 to 1.3e-6 of the states), and is too
// small to move 2^0, which has to be 1 for a step size of 0.
__device__ __forceinline__ float decay_of(float dt, float a) { return power(fmaf(dt, a, 1.44e-8f)); }
__device__ __forceinline__ double decay_of(double dt, double a) { return exp(dt * a); }

// A state v behind steps that multiply it by 2^e (e^e for doubles) in all.  The power may leave the type's range where
// the product does not, nor the steps one by one: it is then taken in two factors, a state of 0 stays 0 and an
// infinite one infinite.
template <typename A>
__device__ __forceinline__ A carried(A e, A v) {
    if (v == 0 || (fabs(v) == (A)INFINITY && fabs(e) < (A)INFINITY)) return v;
    const bool far = !(fabs(e) <= (sizeof(A) == 8 ? A(600) : A(100)));
    const A p = power(far ? e * A(0.5) : e);
    return far ? p * (p * v) : p * v;
}

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
__device__ __forceinline__ Two<float> softplus(Two<float> v) {
    const Two<float> e = {power(-1.4426950408889634f * fabsf(v.x)), power(-1.4426950408889634f * fabsf(v.y))};
    const Two<float> u = add(e, both(2.0f));
    const Two<float> s = mul(e, {reciprocal(u.x), reciprocal(u.y)}), q = mul(s, s);
    Two<float> p = both(1.0f / 15.0f);
    p = fma(p, q, both(1.0f / 13.0f));
    p = fma(p, q, both(1.0f / 11.0f));
    p = fma(p, q, both(1.0f / 9.0f));
    p = fma(p, q, both(1.0f / 7.0f));
    p = fma(p, q, both(1.0f / 5.0f));
    p = fma(p, q, both(1.0f / 3.0f));
    p = fma(mul(p, q), s, s);
    return fma(p, both(2.0f), {fmaxf(v.x, 0.0f), fmaxf(v.y, 0.0f)});
}
__device__ __forceinline__ double softplus(double v) { return (v > 0 ? v : 0.0) + log1p(exp(-fabs(v))); }
__device__ __forceinline__ Two<double> softplus(Two<double> v) { return {softplus(v.x), softplus(v.y)}; }

__device__ __forceinline__ float gate(float z) { return z * reciprocal(1.0f + power(-1.4426950408889634f * z)); }
__device__ __forceinline__ double gate(double z) { return z / (1.0 + exp(-z)); }
__device__ __forceinline__ Two<float> gate(Two<float> z) {
    const Two<float> m = mul(z, both(-1.4426950408889634f));
    const Two<float> u = add({power(m.x), power(m.y)}, both(1.0f));
    return mul(z, {reciprocal(u.x), reciprocal(u.y)});
}
__device__ __forceinline__ Two<double> gate(Two<double> z) { return {gate(z.x), gate(z.y)}; }

// ---- prompts ------------------------------------------------------------------------------------------
//
// A block has kThreads / L channels of one sequence and group.  The time axis is walked in tiles of S
// steps, by two halves of the block that work side by side, one barrier a tile:
//   - kThreads walkers, L for each channel; a walker has N states, in pairs (p L + l) 2 + {0, 1}, and
//     sums C h over its own states at every step, which goes through shared memory.  The exponentials
//     of the next steps are made before the recurrence of the present ones, which waits for them else;
//   - kThreads helpers, which copy tiles into a ring in shared memory some tiles ahead (cp.async), lay
//     (dt, dt x), B and C of the next tile down as floats, and finish the tile before: they add up the
//     lanes of each channel and D x, apply the gate and store y.
// The laid-down values and the sums have two buffers each, which alternate.
//
// Where there are too few channels to fill the GPU, the time axis is cut into chunks.  A first pass
// (LOCAL) computes each chunk's states from zero and the sum of its dt; the second enters a chunk with
//   h <- exp(A sum_k) h + local_k   over the chunks k before it
// which costs every exponential twice.

template <typename A>
struct ScanChunks {
    int64_t length = 0;   // steps of a chunk, whole tiles
    int count = 1;
    A* local = nullptr;   // (b, count, d, n)
    A* sums = nullptr;    // (b, count, d)
};

template <typename T, int L, int N, int S, bool LOCAL>
struct ScanShared {
    using A = typename Acc<T>::type;
    static constexpr int kChannels = kThreads / L, kPairs = N / 2, kStates = L * N;
    // a ring row has room for the bytes between the 16-byte border before its first value and that value
    static constexpr int kPitch = kThreads / 2 + 16;           // neighbouring steps in different banks
    static constexpr int kRow = kChannels * (int)sizeof(T) + 16, kRowB = kStates * (int)sizeof(T) + 16;
    struct Fixed {
        alignas(16) A step[2][kChannels][S + 2][2];            // dt, dt x
        // a lane's pairs of B of two steps and of C, eight values, in pieces of 16 bytes that lie side by
        // side for the lanes
        static constexpr int kPiece = 16 / (int)sizeof(T);
        alignas(16) T bc[2][S / 2][kPairs][8 / kPiece][L][kPiece];
        alignas(16) A y[2][S][kPitch];                         // L / 2 sums of each channel
        int infinite[2];                                       // an infinity or NaN beside places without a state
    };
    struct alignas(16) Stage {
        unsigned char x[S][kRow], delta[S][kRow], z[S][kRow];
        unsigned char b[S][kRowB], c[S][kRowB];
    };
    // tiles in the ring: the one to finish, the one that is walked, the one to lay down, and one or more
    // on their way, as many as let two blocks share an SM (one block of the larger kinds)
    static constexpr size_t kBudget = (sizeof(T) <= 4 && N == 2 ? 113 : 226) * 1024;
    static constexpr int kFits = sizeof(Fixed) < kBudget ? (int)((kBudget - sizeof(Fixed)) / sizeof(Stage)) : 0;
    static constexpr int kStages = kFits < 4 ? 4 : kFits > 8 ? 8 : kFits;
    Fixed f;
    Stage ring[kStages];
    static_assert(sizeof(Fixed) + kStages * sizeof(Stage) <= 227 * 1024, "shared memory of an SM");
};

// sum of K numbers of a channel; the pieces are read in an order that keeps the banks apart
template <int K, typename A>
__device__ __forceinline__ A lanes_sum(const A* y, int slot) {
    constexpr int V = 16 / (int)sizeof(A) < K ? 16 / (int)sizeof(A) : K, kPieces = K / V;
    A t = 0;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
        const int piece = (k + slot * K / 32) % kPieces;
        const Pack<A, V> v = *(const Pack<A, V>*)(y + slot * K + piece * V);
        A s = v.v[0];
#pragma unroll
        for (int j = 1; j < V; ++j) s += v.v[j];
        t = k ? t + s : s;
    }
    return t;
}

// V values in accesses of 16 bytes, `apart` values from one to the next
template <int V, typename A>
__device__ __forceinline__ Pack<A, V> load_shared(const A* p, int apart) {
    constexpr int W = 16 / (int)sizeof(A);
    Pack<A, V> r;
#pragma unroll
    for (int i = 0; i < V / W; ++i) *(Pack<A, W>*)&r.v[i * W] = *(const Pack<A, W>*)(p + i * apart);
    return r;
}

// Rows are copied into the ring in pieces of 16 bytes where every row begins at a 16-byte border, else
// of 8 (64-bit values) or 4: from the 4-byte border before a row's first value to the one behind its
// last.  16-bit values of an odd place begin in the middle of a piece; the values around a row belong
// to the array or to the room that every array has around it.
//
// FILLED: all of the kStates places have states, or it does not matter (LOCAL: y is not made).  Places without one have
// A, B and C of 0 and stay 0 while everything is finite.  With an infinite dt or x they would not, and go into y as
// NaN: the helpers look for that, and from then on these places are kept at 0 (1 x 4096 x 4096 x 12 in 16 bits
// 195 us without looking, 201 with it, 222 with these places kept at 0 all the time).
template <typename T, int L, int N, int S, bool LOCAL, bool FILLED>
__global__ void __launch_bounds__(kThreads + kHelpers, sizeof(T) <= 4 && N == 2 ? 2 : 1) scan_kernel(SelectiveScanArgs a, ScanChunks<typename Acc<T>::type> ck, int blocks, int piece) {
    using A = typename Acc<T>::type;
    using Shared = ScanShared<T, L, N, S, LOCAL>;
    constexpr int kChannels = Shared::kChannels, kPairs = Shared::kPairs, kStates = Shared::kStates, kStages = Shared::kStages;
    constexpr int kAhead = kStages - 2;                                      // tiles requested ahead of the walked one
    constexpr int kRows = kHelpers / kChannels;                              // a helper's steps are kRows apart
    constexpr int kOwn = (S + kRows - 1) / kRows;
    constexpr int kOwnB = (S * kStates + kHelpers - 1) / kHelpers;
    constexpr int kGroup = kPairs >= 4 || sizeof(A) == 8 ? 2 : 4, kGroups = S / kGroup;   // steps whose exponentials are made together
    constexpr int kMade = sizeof(A) == 8 ? 1 : 2;                            // groups in registers; two of doubles are too many
    extern __shared__ __align__(16) unsigned char scan_shared[];
    auto& all = *(Shared*)scan_shared;
    auto& sh = all.f;

    const int tid = threadIdx.x < kThreads ? threadIdx.x : threadIdx.x - kThreads;   // among the walkers, or the helpers
    const int64_t per_group = a.d / a.groups;
    const int64_t per_blocks = blocks / a.groups;
    const int64_t b = blockIdx.x / blocks, blk = blockIdx.x % blocks;
    const int64_t g = blk / per_blocks, c0 = g * per_group + blk % per_blocks * kChannels;
    const int channels = (int)min((g + 1) * per_group - c0, (int64_t)kChannels);
    const int64_t end_all = a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.t) : a.t;
    const int64_t t0 = blockIdx.y * ck.length;
    const int64_t stop = min(t0 + ck.length, a.t), end = min(stop, end_all);
    const int64_t steps = max(end - t0, (int64_t)0);
    const int tiles = (int)((steps + S - 1) / S), last = (int)(steps - (int64_t)(tiles - 1) * S);
    auto live_of = [&](int tile) { return tile == tiles - 1 ? last : S; };

    // the same for all threads of a warp, which the shuffle lets the compiler know
    if (__shfl_sync(0xffffffffu, (int)threadIdx.x, 0) < kThreads) {
        // ---- walkers ----
        const int lane = tid & (L - 1), own = tid / L;
        const int64_t c = c0 + own;
        Two<A> h[kPairs], decay[kPairs];
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = (p * L + lane) * 2 + j;
                const bool on = n < a.n && own < channels;
                const int64_t i = c * a.n + n;
                A v = 0, w = 0;
                if (on) {
                    w = ((const A*)a.A)[i] * decay_scale<A>();
                    if (!LOCAL && a.state) v = ((const A*)a.state)[b * a.d * a.n + i];
                    if (!LOCAL)
                        for (int k = 0; k < (int)blockIdx.y; ++k) {
                            const int64_t q = (b * ck.count + k) * a.d;
                            const A s = ck.sums[q + c];
                            v = (s == 0 ? v : carried(w * s, v)) + ck.local[q * a.n + i];
                        }
                }
                (j ? h[p].y : h[p].x) = v;
                (j ? decay[p].y : decay[p].x) = w;
            }
        }
        const int states = a.n - 2 * lane;
        auto walk = [&](int buf, int live, auto whole) {
            constexpr bool kWhole = decltype(whole)::value;
            Two<A> e[kMade][kGroup][kPairs], term[kMade][kGroup][kPairs], cc[kMade][kGroup][kPairs];
            // a group's exponentials and terms, which wait for no state
            auto make = [&](int from, int q) {
#pragma unroll
                for (int i = 0; i < kGroup; i += 2) {
                    const Pack<A, 4> u = load_shared<4>(&sh.step[buf][own][from + i][0], 16 / (int)sizeof(A));
#pragma unroll
                    for (int p = 0; p < kPairs; ++p) {
                        const Pack<T, 8> w = load_shared<8>(&sh.bc[buf][(from + i) / 2][p][0][lane][0], 16 * L / (int)sizeof(T));
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const A dt = u.v[2 * k], dtx = u.v[2 * k + 1];
                            e[q][i + k][p] = {decay_of(dt, decay[p].x), decay_of(dt, decay[p].y)};
                            term[q][i + k][p] = {dtx * widen(w.v[2 * k]), dtx * widen(w.v[2 * k + 1])};
                            if (!LOCAL) cc[q][i + k][p] = {widen(w.v[4 + 2 * k]), widen(w.v[5 + 2 * k])};
                        }
                    }
                }
            };
            if (kMade == 2) make(0, 0);
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                const int from = k * kGroup, q = k & (kMade - 1);
                if (!kWhole && from >= live) break;
                if (kMade == 1) make(from, 0);
                else if (k + 1 < kGroups) make(from + kGroup, q ^ 1);
#pragma unroll
                for (int i = 0; i < kGroup; i += 2) {
                    A sum[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        Two<A> y = {0, 0};
#pragma unroll
                        for (int p = 0; p < kPairs; ++p) {
                            const Two<A> next = fma(e[q][i + j][p], h[p], term[q][i + j][p]);
                            // behind the end a step is left out: 0 times an infinite A is not 0
                            if (kWhole || (from + i + j < live && (FILLED || 2 * L * p < states))) h[p].x = next.x;
                            if (kWhole || (from + i + j < live && (FILLED || 2 * L * p + 1 < states))) h[p].y = next.y;
                            if (!LOCAL) y = p ? fma(cc[q][i + j][p], h[p], y) : mul(cc[q][i + j][p], h[p]);
                        }
                        sum[j] = y.x + y.y;
                    }
                    if (!LOCAL) {
                        // neighbours exchange: even lanes keep the first step, odd ones the second
                        const bool odd = lane & 1;
                        const A other = __shfl_xor_sync(0xffffffffu, odd ? sum[0] : sum[1], 1);
                        sh.y[buf][from + i + odd][own * (L / 2) + lane / 2] = (odd ? sum[1] : sum[0]) + other;
                    }
                }
            }
        };
        __syncthreads();
        bool finite = true;      // so far, where it matters
        for (int i = 0; i < tiles; ++i) {
            if (!FILLED) finite = finite && !__shfl_sync(0xffffffffu, sh.infinite[i & 1], 0);
            if (live_of(i) == S && finite) walk(i & 1, S, std::true_type());
            else walk(i & 1, live_of(i), std::false_type());
            __syncthreads();
        }
#pragma unroll
        for (int p = 0; p < kPairs; ++p)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = (p * L + lane) * 2 + j;
                if (n >= a.n || own >= channels) continue;
                const A v = j ? h[p].y : h[p].x;
                if (LOCAL) ck.local[((b * ck.count + blockIdx.y) * a.d + c) * a.n + n] = v;
                else if ((int)blockIdx.y == ck.count - 1) ((A*)a.new_state)[(b * a.d + c) * a.n + n] = v;
            }
        if (LOCAL) __syncthreads();
        return;
    }

    // ---- helpers ----
    // Everything that is the same in every tile is computed here once; in the tiles a helper's time is
    // its instructions.
    const int row = tid / kChannels, slot = tid % kChannels;
    const bool on = slot < channels;
    const A bias = on && a.delta_bias ? ((const A*)a.delta_bias)[c0 + slot] : A(0);
    const A skip = on && a.D ? ((const A*)a.D)[c0 + slot] : A(0);
    const int64_t bn = (int64_t)a.groups * a.n;
    const int64_t base = (b * a.t + t0) * a.d + c0, base_b = (b * a.t + t0) * bn + g * a.n;
    // bytes between the border that a row is copied from and its first value: a tile has an even number
    // of rows, so they are the same in every tile
    auto lead = [&](int64_t element) { return piece == 4 ? (int)(element * (int)sizeof(T)) & 3 : 0; };

    // what this thread copies: one column of pieces of x, delta, z, B or C, and every `copy_rows`th row
    const int cols = ((channels * (int)sizeof(T) + (piece == 4 && sizeof(T) == 2 ? 2 : 0)) + piece - 1) / piece;
    const int cols_b = ((a.n * (int)sizeof(T) + (piece == 4 && sizeof(T) == 2 ? 2 : 0)) + piece - 1) / piece;
    const int all_cols = 3 * cols + 2 * cols_b;
    const unsigned ring = (unsigned)__cvta_generic_to_shared(&all.ring[0]);
    const int copy_rows = max(kHelpers / all_cols, 1), most_cols = (all_cols + kHelpers - 1) / kHelpers;
    struct Column { const unsigned char* from; unsigned to; int64_t pitch; unsigned row_bytes; };
    auto column_of = [&](int k) {
        Column q;
        const bool bc = k >= 3 * cols;
        const int which = bc ? 3 + (k - 3 * cols) / cols_b : k / cols, at = (bc ? (k - 3 * cols) % cols_b : k % cols) * piece;
        const void* array = which == 0 ? a.x : which == 1 ? a.delta : which == 2 ? a.z : which == 3 ? a.B : a.C;
        q.from = array && k < all_cols && !(LOCAL && (which == 2 || which == 4))
                     ? (const unsigned char*)array + (bc ? base_b : base) * (int)sizeof(T) + at : nullptr;
        q.pitch = (bc ? bn : a.d) * (int)sizeof(T);
        q.row_bytes = bc ? Shared::kRowB : Shared::kRow;
        q.to = ring + (unsigned)(which < 3 ? which * S * Shared::kRow : 3 * S * Shared::kRow + (which - 3) * S * Shared::kRowB) + at;
        return q;
    };
    const int first_row = most_cols > 1 ? 0 : tid / all_cols;
    const Column column = column_of(most_cols > 1 ? tid : first_row < copy_rows ? tid % all_cols : all_cols);
    const unsigned char* column_from = column.from + (column.from ? first_row * column.pitch : 0);
    int requested = 0;
    unsigned request_at = 0;                      // stage of the tile requested next, as an offset
    auto copy_column = [&](const Column& q, const unsigned char* from, int live) {
        const uintptr_t border = ~(uintptr_t)(piece - 1);
        const int64_t step = copy_rows * q.pitch;
        unsigned to = q.to + request_at + first_row * q.row_bytes;
        for (int r = first_row; r < live; r += copy_rows) {
            const uintptr_t at = (uintptr_t)from & border;
            if (piece == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(at) : "memory");
            else if (sizeof(T) == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(at) : "memory");
            else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(at) : "memory");
            from += step;
            to += copy_rows * q.row_bytes;
        }
    };
    auto request = [&]() {
        if (requested < tiles) {
            const int live = live_of(requested);
            if (column.from) {
                copy_column(column, column_from, live);
                column_from += S * column.pitch;
            }
            for (int m = 1; m < most_cols; ++m) {   // rows of more pieces than there are helpers
                const Column q = column_of(tid + m * kHelpers);
                if (q.from) copy_column(q, q.from + (int64_t)requested * S * q.pitch, live);
            }
            ++requested;
            request_at = request_at == (kStages - 1) * sizeof(typename Shared::Stage) ? 0 : request_at + (unsigned)sizeof(typename Shared::Stage);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");   // one a tile, empty behind the last
    };
    // all but the latest kAhead - 2 requests have arrived, for this thread
    auto arrived = [&]() { asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 2) : "memory"); };

    // a helper's own values: steps row + i kRows of channel `slot`; and of B and C
    constexpr int kOwnPairs = (kOwn + 1) / 2;
    unsigned own_at[kOwn], own_b[kOwnB];          // places in a stage's x, B
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const int s = min(row + i * kRows, S - 1);
        own_at[i] = (unsigned)(s * Shared::kRow + lead(base + s * a.d) + slot * (int)sizeof(T));
    }
#pragma unroll
    for (int i = 0; i < kOwnB; ++i) {
        const int e = min(tid + i * kHelpers, S * kStates - 1), s = e / kStates, n = min(e % kStates, a.n - 1);
        own_b[i] = (unsigned)(3 * S * Shared::kRow + s * Shared::kRowB + lead(base_b + s * bn) + n * (int)sizeof(T));
    }
    const unsigned char *lay_at = (const unsigned char*)&all.ring[0], *finish_at = lay_at;
    const unsigned char* const wrap = lay_at + (kStages - 1) * sizeof(typename Shared::Stage);
    auto next_stage = [&](const unsigned char*& at) { at = at == wrap ? (const unsigned char*)&all.ring[0] : at + sizeof(typename Shared::Stage); };
    const T zero = narrow<T>(A(0));
    A sum = 0;                                    // LOCAL: dt summed over the chunk
    if (!FILLED && tid < 2) sh.infinite[tid] = 0;
    auto lay = [&](int buf, int live, auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        Two<A> dt[kOwnPairs], x[kOwnPairs];
#pragma unroll
        for (int i = 0; i < kOwnPairs; ++i) {
            const int k = 2 * i + 1 < kOwn ? 2 * i + 1 : 2 * i;
            dt[i] = {widen(*(const T*)(lay_at + S * Shared::kRow + own_at[2 * i])), widen(*(const T*)(lay_at + S * Shared::kRow + own_at[k]))};
            x[i] = {widen(*(const T*)(lay_at + own_at[2 * i])), widen(*(const T*)(lay_at + own_at[k]))};
            dt[i] = add(dt[i], both(bias));
        }
        if (a.softplus) {
#pragma unroll
            for (int i = 0; i < kOwnPairs; ++i) dt[i] = softplus(dt[i]);
        }
        if (!FILLED) {
            // dt x shows an infinite dt too, as an infinity or NaN.  Noted for good: states stay infinite
            bool all = true;
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
                if (row + i * kRows < live) all = all && fabs(i & 1 ? dt[i / 2].y * x[i / 2].y : dt[i / 2].x * x[i / 2].x) < (A)INFINITY;
            if (on && !all) sh.infinite[buf] = 1;
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int s = row + i * kRows;
            A v = i & 1 ? dt[i / 2].y : dt[i / 2].x, w = v * (i & 1 ? x[i / 2].y : x[i / 2].x);
            if (!kWhole && s >= live) v = w = 0;      // what lies there is left over
            if (kRows * kOwn > S && s >= S) break;
            *(Two<A>*)&sh.step[buf][slot][s][0] = {v, w};
            if (LOCAL) sum += v;
        }
#pragma unroll
        for (int i = 0; i < kOwnB; ++i) {
            const int e = tid + i * kHelpers;
            if (S * kStates % kHelpers && e >= S * kStates) break;
            const int s = e / kStates, n = e % kStates;
            const int p = n / (2 * L), l = n % (2 * L) / 2, j = (s & 1) * 2 + (n & 1);
            constexpr int W = 16 / (int)sizeof(T);
            sh.bc[buf][s / 2][p][j / W][l][j % W] = n < a.n ? *(const T*)(lay_at + own_b[i]) : zero;
            if (!LOCAL) sh.bc[buf][s / 2][p][(4 + j) / W][l][(4 + j) % W] = n < a.n ? *(const T*)(lay_at + S * Shared::kRowB + own_b[i]) : zero;
        }
        next_stage(lay_at);
    };
    T* ys = (T*)a.y + base + (int64_t)row * a.d + slot;
    const int64_t stride = (int64_t)kRows * a.d, tile_stride = (int64_t)S * a.d;
    auto finish = [&](int buf, int live, auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        Two<A> y[kOwnPairs];
#pragma unroll
        for (int i = 0; i < kOwnPairs; ++i) {
            const int k = 2 * i + 1 < kOwn ? 2 * i + 1 : 2 * i, s0 = min(row + 2 * i * kRows, S - 1), s1 = min(row + k * kRows, S - 1);
            y[i] = {lanes_sum<L / 2>(sh.y[buf][s0], slot), lanes_sum<L / 2>(sh.y[buf][s1], slot)};
        }
        if (a.D) {
#pragma unroll
            for (int i = 0; i < kOwnPairs; ++i) {
                const int k = 2 * i + 1 < kOwn ? 2 * i + 1 : 2 * i;
                y[i] = fma(both(skip), {widen(*(const T*)(finish_at + own_at[2 * i])), widen(*(const T*)(finish_at + own_at[k]))}, y[i]);
            }
        }
        if (a.z) {
#pragma unroll
            for (int i = 0; i < kOwnPairs; ++i) {
                const int k = 2 * i + 1 < kOwn ? 2 * i + 1 : 2 * i;
                const unsigned char* const z = finish_at + 2 * S * Shared::kRow;
                y[i] = mul(y[i], gate(Two<A>{widen(*(const T*)(z + own_at[2 * i])), widen(*(const T*)(z + own_at[k]))}));
            }
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (on && (kRows * kOwn == S && kWhole ? true : row + i * kRows < live)) ys[i * stride] = narrow<T>(i & 1 ? y[i / 2].y : y[i / 2].x);
        ys += tile_stride;
        next_stage(finish_at);
    };
    auto lay_tile = [&](int tile) {
        if (tile < tiles - 1 || last == S) lay(tile & 1, S, std::true_type());
        else lay(tile & 1, last, std::false_type());
    };
    auto finish_tile = [&](int tile) {
        if (tile < tiles - 1 || last == S) finish(tile & 1, S, std::true_type());
        else finish(tile & 1, last, std::false_type());
    };
    for (int i = 0; i < kAhead; ++i) request();
    arrived();
    asm volatile("bar.sync 1, %0;" ::"n"(kHelpers) : "memory");     // tiles 0 and 1 are there for every helper
    if (tiles > 0) lay_tile(0);
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
        // tile i is walked: request i + kAhead, into the place of i - 2; finish i - 1, lay i + 1
        request();
        if (!LOCAL && i > 0) finish_tile(i - 1);
        if (i + 1 < tiles) lay_tile(i + 1);
        arrived();           // tile i + 2, which the next turn lays down
        __syncthreads();
    }
    if (LOCAL) {
        // dt of a channel was summed by up to kRows helpers: add them up in their order
        A* const part = (A*)&sh.step;
        part[tid] = row < S ? sum : A(0);
        __syncthreads();
        if (tid < channels) {
            A s = 0;
            for (int i = tid; i < kHelpers; i += kChannels) s += part[i];
            ck.sums[(b * ck.count + blockIdx.y) * a.d + c0 + tid] = s;
        }
        return;
    }
    if (tiles > 0) finish_tile(tiles - 1);
    // rows behind the end of the sequence
    const int64_t behind = max(end, t0);
    for (int64_t e = tid; e < (stop - behind) * kChannels; e += kHelpers) {
        const int cc = (int)(e % kChannels);
        if (cc < channels) ((T*)a.y)[(b * a.t + behind + e / kChannels) * a.d + c0 + cc] = zero;
    }
}

// ---- single tokens ------------------------------------------------------------------------------------
//
// Bound by the states, which are read and written once: a lane has V neighbouring states of a channel
// (16 bytes where n allows), `lanes` lanes the channel.  An inactive sequence's states are copied.
// 128 sequences of 4096 x 16 in 16 bits: 72 MB in 18.6 us, 3.9 TB/s (floor 11 us); latency behind the loads
// of four sequences at once is what is left.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) scan_token_kernel(SelectiveScanArgs a, int lanes) {
    using A = typename Acc<T>::type;
    const int lane = threadIdx.x & (lanes - 1);
    const int64_t c = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / lanes;
    const bool on = c < a.d;
    const int64_t bn = (int64_t)a.groups * a.n, g = on ? c / (a.d / a.groups) * a.n : 0;
    const A bias = on && a.delta_bias ? ((const A*)a.delta_bias)[c] : A(0), skip = on && a.D ? ((const A*)a.D)[c] : A(0);
    for (int64_t b = blockIdx.y; b < a.b; b += gridDim.y) {
        const bool live = on && !(a.lengths && a.lengths[b] < 1);
        const int64_t at = b * a.d + c;
        A x = 0, dt = 0, out = 1, y = 0;
        if (live) {
            x = widen(((const T*)a.x)[at]);
            dt = widen(((const T*)a.delta)[at]) + bias;
            if (a.z) out = gate(widen(((const T*)a.z)[at]));
            if (a.softplus) dt = softplus(dt);
        }
        for (int n = lane * V; on && n < a.n; n += lanes * V) {
            Pack<A, V> h;
#pragma unroll
            for (int j = 0; j < V; ++j) h.v[j] = 0;
            if (a.state) h = *(const Pack<A, V>*)((const A*)a.state + at * a.n + n);
            if (live) {
                const Pack<A, V> w = *(const Pack<A, V>*)((const A*)a.A + c * a.n + n);
                const Pack<T, V> bb = *(const Pack<T, V>*)((const T*)a.B + b * bn + g + n), cc = *(const Pack<T, V>*)((const T*)a.C + b * bn + g + n);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    h.v[j] = decay_of(dt, w.v[j] * decay_scale<A>()) * h.v[j] + dt * x * widen(bb.v[j]);
                    y += widen(cc.v[j]) * h.v[j];
                }
            }
            *(Pack<A, V>*)((A*)a.new_state + at * a.n + n) = h;
        }
        for (int o = lanes / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
        if (on && lane == 0) ((T*)a.y)[at] = narrow<T>(live ? (a.D ? y + skip * x : y) * out : A(0));
    }
}

// Runs of sequences, four at a time, with four or more lanes a channel that have all of its states:
// lane k of a channel computes dt, D x and the gate of sequence k alone, hands dt and dt x to the others,
// and ends with the sum of that sequence.  Addresses are stepped from sequence to sequence.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 8 ? 2 : 4) scan_tokens_kernel(SelectiveScanArgs a, int lanes, int run) {
    using A = typename Acc<T>::type;
    const int lane = threadIdx.x & (lanes - 1), head = (threadIdx.x & 31) - lane, mine = lane & 3, n = lane * V;
    const int64_t c = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / lanes;
    const bool on = c < a.d, mid = on && n < a.n;
    const int64_t bn = (int64_t)a.groups * a.n, dn = a.d * a.n;
    const int64_t b0 = (int64_t)blockIdx.y * run, b1 = min(b0 + run, a.b);
    const A bias = on && a.delta_bias ? ((const A*)a.delta_bias)[c] : A(0), skip = on && a.D ? ((const A*)a.D)[c] : A(0);
    Pack<A, V> w;
#pragma unroll
    for (int j = 0; j < V; ++j) w.v[j] = mid ? ((const A*)a.A)[c * a.n + n + j] * decay_scale<A>() : A(0);
    const int64_t first = mid ? b0 * dn + c * a.n + n : 0;
    const A* hs = (const A*)a.state + first;
    A* hn = (A*)a.new_state + first;
    const int64_t first_b = mid ? b0 * bn + c / (a.d / a.groups) * a.n + n : 0;
    const T *bs = (const T*)a.B + first_b, *cs = (const T*)a.C + first_b;
    int64_t at = (b0 + mine) * a.d + (on ? c : 0);
    for (int64_t b = b0; b < b1; b += 4, at += 4 * a.d) {
        const int here = (int)min(b1 - b, (int64_t)4);
        Pack<A, V> h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) h[k].v[j] = 0;
            if (mid && k < here && a.state) h[k] = *(const Pack<A, V>*)hs;
            hs += dn;
        }
        const bool live = on && mine < here && !(a.lengths && a.lengths[b + mine] < 1);
        A x = 0, dt = 0, z = 0, y[4] = {0, 0, 0, 0};
        if (live) {
            x = widen(((const T*)a.x)[at]);
            dt = widen(((const T*)a.delta)[at]) + bias;
            if (a.z) z = widen(((const T*)a.z)[at]);
            if (a.softplus) dt = softplus(dt);
        }
        const A dtx = dt * x;
        const unsigned lives = __ballot_sync(0xffffffffu, live) >> head;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const A dtk = __shfl_sync(0xffffffffu, dt, head + k), dtxk = __shfl_sync(0xffffffffu, dtx, head + k);
            if (mid && lives >> k & 1) {
                const Pack<T, V> bb = *(const Pack<T, V>*)bs, cc = *(const Pack<T, V>*)cs;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    h[k].v[j] = decay_of(dtk, w.v[j]) * h[k].v[j] + dtxk * widen(bb.v[j]);
                    y[k] += widen(cc.v[j]) * h[k].v[j];
                }
            }
            if (mid && k < here) *(Pack<A, V>*)hn = h[k];
            hn += dn;
            bs += bn;
            cs += bn;
        }
        // lanes at distance 2, then 1 exchange halves of the sequences; further lanes add theirs
        const bool up2 = lane & 2, up1 = lane & 1;
        const A s0 = (up2 ? y[2] : y[0]) + __shfl_xor_sync(0xffffffffu, up2 ? y[0] : y[2], 2);
        const A s1 = (up2 ? y[3] : y[1]) + __shfl_xor_sync(0xffffffffu, up2 ? y[1] : y[3], 2);
        A s = (up1 ? s1 : s0) + __shfl_xor_sync(0xffffffffu, up1 ? s0 : s1, 1);
        for (int o = 4; o < lanes; o *= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (on && mine < here && lane < 4) {
            if (a.D) s += skip * x;
            if (a.z) s *= gate(z);
            ((T*)a.y)[at] = narrow<T>(live ? s : A(0));
        }
    }
}

template <typename T, int V>
cudaError_t token(const SelectiveScanArgs& a, int lanes, int sm_count, cudaStream_t s) {
    const int64_t across = (a.d * lanes + kThreads - 1) / kThreads;
    if (across >= (1LL << 31)) return cudaErrorInvalidValue;
    // runs of up to 16 sequences, as long as three blocks for every SM are left; else one by one
    // (128 sequences of 4096 x 16: 39.0 us one by one; in runs of 4, 8, 16, 32: 20.5, 18.8, 18.6, 39 us)
    int64_t run = 16;
    while (run > 4 && across * ((a.b + run - 1) / run) < 3 * sm_count) run /= 2;
    const int64_t runs = (a.b + run - 1) / run;
    if (a.b >= 4 && lanes >= 4 && lanes * V >= a.n && across * runs >= 2 * sm_count && runs <= 65535)
        scan_tokens_kernel<T, V><<<dim3((unsigned)across, (unsigned)runs), kThreads, 0, s>>>(a, lanes, (int)run);
    else
        scan_token_kernel<T, V><<<dim3((unsigned)across, (unsigned)std::min<int64_t>(a.b, 65535)), kThreads, 0, s>>>(a, lanes);
    return cudaGetLastError();
}

template <typename T>
cudaError_t token(const SelectiveScanArgs& a, int sm_count, cudaStream_t s) {
    using A = typename Acc<T>::type;
    const int wide = sizeof(A) == 8 ? 2 : 4;
    const int v = a.n % wide == 0 ? wide : a.n % 2 == 0 ? 2 : 1;
    int lanes = 1;
    while (lanes < 32 && lanes * v < a.n) lanes *= 2;
    if (v == 4) return token<T, 4>(a, lanes, sm_count, s);
    return v == 2 ? token<T, 2>(a, lanes, sm_count, s) : token<T, 1>(a, lanes, sm_count, s);
}

// ---- launches -------------------------------------------------------------------------------------------

int lanes_for(int n) { return n <= 8 ? 4 : n <= 64 ? 8 : n <= 128 ? 16 : 32; }

int64_t channel_blocks(const SelectiveScanArgs& a) {
    const int64_t channels = kThreads / lanes_for(a.n);
    return a.groups * ((a.d / a.groups + channels - 1) / channels);
}

constexpr int kBorder = 32;     // chunks begin at multiples of every tile's steps

// Chunks of the time axis: none while the channels' blocks give half of the SMs one each, since
// chunks compute every exponential twice; else as many as make two blocks an SM, of at least 64 steps.
template <typename A>
ScanChunks<A> chunks_for(const SelectiveScanArgs& a, int sm_count) {
    ScanChunks<A> ck;
    ck.length = std::max<int64_t>((a.t + kBorder - 1) / kBorder, 1) * kBorder;
    const int64_t blocks = channel_blocks(a) * a.b;
    if (2 * blocks >= sm_count || a.t < 128) return ck;
    const int64_t want = std::min<int64_t>(2 * sm_count / blocks, a.t / 64);
    ck.length = ((a.t + want - 1) / want + kBorder - 1) / kBorder * kBorder;
    ck.count = (int)((a.t + ck.length - 1) / ck.length);
    return ck;
}

template <typename T, int L, int N, int S, bool LOCAL, bool FILLED>
cudaError_t scan_pass(const SelectiveScanArgs& a, const ScanChunks<typename Acc<T>::type>& ck, int64_t blocks, int count, int piece, cudaStream_t s) {
    constexpr size_t bytes = sizeof(ScanShared<T, L, N, S, LOCAL>);
    const auto kernel = scan_kernel<T, L, N, S, LOCAL, FILLED>;
    if (bytes > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return e;
    }
    kernel<<<dim3((unsigned)(blocks * a.b), count), kThreads + kHelpers, bytes, s>>>(a, ck, (int)blocks, piece);
    return cudaGetLastError();
}

template <typename T, int L, int N>
cudaError_t prompt(const SelectiveScanArgs& a, int sm_count, cudaStream_t s) {
    using A = typename Acc<T>::type;
    // tiles as long as shared memory allows, twice where two blocks can share an SM
    constexpr int S = sizeof(T) == 2 && N == 2 ? 32 : sizeof(T) == 8 && L > 8 ? 8 : 16;
    const int64_t rows = a.d / a.groups * (int64_t)sizeof(T), rows_b = a.n * (int64_t)sizeof(T);
    const int piece = rows % 16 == 0 && rows_b % 16 == 0 ? 16 : sizeof(T) == 8 ? 8 : 4;
    ScanChunks<A> ck = chunks_for<A>(a, sm_count);
    const int64_t blocks = channel_blocks(a);
    if (blocks * a.b >= (1LL << 31)) return cudaErrorInvalidValue;
    if (ck.count > 1) {
        ck.local = (A*)a.workspace;
        ck.sums = ck.local + a.b * ck.count * a.d * a.n;
        // the last chunk's states are never entered from
        const cudaError_t e = scan_pass<T, L, N, S, true, true>(a, ck, blocks, ck.count - 1, piece, s);
        if (e != cudaSuccess) return e;
    }
    if (a.n == L * N) return scan_pass<T, L, N, S, false, true>(a, ck, blocks, ck.count, piece, s);
    return scan_pass<T, L, N, S, false, false>(a, ck, blocks, ck.count, piece, s);
}

template <typename T>
cudaError_t scan(const SelectiveScanArgs& a, int sm_count, cudaStream_t s) {
    if (a.t == 1) return token<T>(a, sm_count, s);
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
