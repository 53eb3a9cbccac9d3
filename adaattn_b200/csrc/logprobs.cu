// Log probabilities of given tokens, with entropy and top alternatives, and
// their gradient.
//
// For a row z of V logits, m = max z, s = sum exp(z_i - m), p_i = exp(z_i - m) / s:
//   lse = m + log s          log p_t = (z_t - m) - log s
//   H   = log s - sum exp(z_i - m) (z_i - m) / s
// A logit of -inf has p = 0 and adds nothing; a row of nothing else, or one
// with NaN or +inf, gives NaN (lse: -inf for the row of -inf). Gradient, for
// upstream g of log p_t, H and lse:
//   dz_i = p_i (g_lse - g_lp - g_H (log p_i + H)) + g_lp [i = t].
//
// One pass over the logits: every thread keeps a running maximum, sum and
// weighted sum (fp32, base 2, two of each in packed pairs), joined at the end.
// A row is shared by a cluster of CTAs when there are few rows; its parts are
// joined through distributed shared memory, no workspace.
//
// HBM reads of V elements bound it, if the instructions per element are few:
// at 6.5 TB/s an SM takes 11.7 16-bit elements a cycle, of 128 instruction
// lanes and 16 exponentials. Unpacking (1), clamping and the maximum on packed
// pairs (1/2 each), argument, sum and weighted sum as packed fp32 pairs (1/2
// each) and the exponential make 4.5; with moves, addresses and each row's end
// the counters show 10.8, and 16384 rows of 50257 bf16 logits take 300 us (5.5
// TB/s; fp32 473 us, 7.0 TB/s), 385 us with 5 and 437 us with 20 alternatives.
// The gradient runs at 6.5 TB/s of reads and writes. Logits are clamped from below (-2^100;
// fp16: its lowest value) so that -inf stays out of the weighted sum; a row
// whose maximum is beyond 2^15 in size is done again by the plain formulas (16384
// such rows 742 us instead of 303).
//
// Top k (k <= 64): candidates are 64-bit keys, the value's order above the
// inverted column, so all keys differ and equal values rank by lowest index.
// While the row is read, a thread only keeps the maxima of its two best rounds,
// which they were, and the third largest maximum. The k-th largest of 128
// thread pairs' maxima bounds the k-th best logit from below, and what reaches
// it lies with the few threads (about k) whose maximum does: each reads those
// rounds again (L2), and the rare thread with a third round at the bound has
// all its rounds read by its warp. The logits
// at or above the bound are sorted. A row with more of them than fit (masked or
// constant rows) takes radix passes over all its keys instead.
#include <cooperative_groups.h>

#include "ada_common.cuh"
#include "ada_internal.h"

namespace ada {
namespace {

namespace cg = cooperative_groups;

constexpr int kT = 256;             // threads
constexpr int kWarps = kT / 32;
constexpr int kPer = 16;            // elements per thread and round
constexpr int kRound = kT * kPer;
constexpr int kMaxTop = 64;
constexpr int kCand = 2304;         // candidates: 32 k of a sorted row and some
constexpr int kGroups = kT / 2;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Key of a logit: larger for larger values, then for lower columns; NaN above all.
__device__ __forceinline__ uint64_t key_of(float x, int col) {
    const uint32_t b = __float_as_uint(x + 0.f);  // -0 ranks as 0
    const uint32_t o = isnan(x) ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (static_cast<uint64_t>(o) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(col));
}
// Its value (0 for -0).
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ int column_of(uint64_t key) {
    return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}

// ---- reading a row ---------------------------------------------------------------
//
// Columns are counted from the 32-byte boundary at or before the row's start,
// so vector loads are aligned whatever the row's address: column c = e - shift.
// Vectors that reach past either end of the row are read element by element;
// what is outside counts as -inf.
template <int DT>
struct Reader {
    static constexpr int EB = DT == ADA_F32 ? 4 : 2;
    static constexpr int EPV = 32 / EB;         // elements per vector
    static constexpr int NV = kPer / EPV;       // vectors per thread and round
    static constexpr uint32_t kNegInf = DT == ADA_F32 ? 0xFF800000u : DT == ADA_BF16 ? 0xFF80FF80u : 0xFC00FC00u;
    const uint8_t* mine;  // this thread's first vector
    int c0, V;            // its column
    int shift;

    __device__ Reader(const void* row, int v) : V(v) {
        const uint64_t a = reinterpret_cast<uint64_t>(row);
        shift = static_cast<int>(a & 31u) / EB;
        mine = reinterpret_cast<const uint8_t*>(a & ~uint64_t(31)) + threadIdx.x * 32;
        c0 = static_cast<int>(threadIdx.x) * EPV - shift;
    }
    __device__ int rounds() const { return (V + shift + kRound - 1) / kRound; }
    // Whether this thread's warp has columns in a round.
    __device__ bool any(int round) const {
        return round * kRound + static_cast<int>(threadIdx.x & ~31u) * EPV - shift < V;
    }
    // First column of vector j of this thread in a round.
    __device__ int column(int round, int j) const { return round * kRound + j * kT * EPV + c0; }
    // The vector that begins at column c.
    __device__ void vector(int c, uint32_t* w) const {
        const uint8_t* p = mine + static_cast<int64_t>(c - c0) * EB;
        if (c >= 0 && c <= V - EPV) {
            asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(p));
        } else if (c >= V || c + EPV <= 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = kNegInf;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (DT == ADA_F32) {
                    w[i] = (c + i >= 0 && c + i < V) ? reinterpret_cast<const uint32_t*>(p)[i] : kNegInf;
                } else {
                    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
                    const uint32_t lo = (c + 2 * i >= 0 && c + 2 * i < V) ? h[2 * i] : kNegInf & 0xFFFFu;
                    const uint32_t hi = (c + 2 * i + 1 >= 0 && c + 2 * i + 1 < V) ? h[2 * i + 1] : kNegInf & 0xFFFFu;
                    w[i] = lo | (hi << 16);
                }
            }
        }
    }
    __device__ void load(int round, uint32_t (&w)[NV * 8]) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) vector(column(round, j), w + 8 * j);
    }
    template <int WORDS, int N>
    __device__ static void unpack(const uint32_t (&w)[WORDS], float (&x)[N]) {
        if constexpr (DT == ADA_F32) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                if constexpr (DT == ADA_BF16) {
                    x[2 * i] = __uint_as_float(w[i] << 16);
                    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                } else {
                    unpack_f16x2(w[i], x[2 * i], x[2 * i + 1]);
                }
            }
        }
    }
};

// ---- running sums ------------------------------------------------------------------

// Packed pairs of 16-bit elements: maximum that keeps NaN.
template <int DT>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (DT == ADA_BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <int DT>
__device__ __forceinline__ float lowest_kept() {
    return DT == ADA_F16 ? -65504.f : -1.2676506e30f;  // fp16's lowest value, -2^100
}
// A row maximum far enough from 0 (NaN too) that the row takes the plain
// formulas. The one-pass sums stand for exponents of x - M: M's rounding, up to
// 2^-25 |M|, is in all of them until the end takes it out. Up to 2^15 that is at
// most 2^-9 of an exponent; at 5e9 it passed 126 and the sums over- or
// underflowed. It also keeps m so far above the clamp that what is clamped adds 0.
constexpr float kFar = 32768.f;
__device__ __forceinline__ bool ends_of_range(float m) { return !(fabsf(m) <= kFar); }
template <int DT>
__device__ __forceinline__ void unpack_pair(uint32_t w, float& lo, float& hi) {
    if constexpr (DT == ADA_BF16) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xFFFF0000u);
    } else {
        unpack_f16x2(w, lo, hi);
    }
}

// With x_i = z_i log2 e and M = m log2 e rounded: s = sum 2^(x_i - M), t = sum (x_i - M) 2^(x_i - M).
struct Sums {
    float m, s, t;
};

// What a change of the maximum from a to b adds to the exponents: the difference
// of the two M, each rounded as the sums' own was. As one fused multiply-add it
// would leave a's rounding in, 2^-24 |M| for every join, even where a equals b
// (logits around 10^4 lost 2e-3 of their log probabilities so).
__device__ __forceinline__ float exponent_shift(float a, float b) {
    return __fsub_rn(__fmul_rn(a, kLog2e), __fmul_rn(b, kLog2e));
}

__device__ __forceinline__ void shift_sums(float d, float& s, float& t) {
    if (s == 0.f) return;
    const float w = exp2f(d);
    t = w == 0.f ? 0.f : w * fmaf(s, d, t);
    s *= w;
}
// The sums of the first n lanes of a warp (n a power of two), in every one of them.
__device__ __forceinline__ Sums join_warp(Sums a, int n) {
    float m = a.m;
    for (int o = n / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    shift_sums(exponent_shift(a.m, m), a.s, a.t);
    for (int o = n / 2; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
    }
    a.m = m;
    return a;
}

// A thread's sums in two halves.
struct PairSums {
    float m;
    uint64_t s, t;
};

// One round's elements; returns their maximum (clamped).
template <int DT>
__device__ __forceinline__ float add_round(PairSums& a, const uint32_t (&w)[Reader<DT>::NV * 8]) {
    uint32_t v[Reader<DT>::NV * 8];
    float top;
    if constexpr (DT == ADA_F32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(max_nan(__uint_as_float(w[i]), lowest_kept<DT>()));
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            q[i] = max_nan(max_nan(__uint_as_float(v[i]), __uint_as_float(v[i + 4])),
                           max_nan(__uint_as_float(v[i + 8]), __uint_as_float(v[i + 12])));
        top = max_nan(max_nan(q[0], q[1]), max_nan(q[2], q[3]));
    } else {
        constexpr uint32_t kClamp = DT == ADA_BF16 ? 0xF180F180u : 0xFBFFFBFFu;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = max2_nan<DT>(w[i], kClamp);
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = max2_nan<DT>(v[i], v[i + 4]);
        q[0] = max2_nan<DT>(max2_nan<DT>(q[0], q[1]), max2_nan<DT>(q[2], q[3]));
        float lo, hi;
        unpack_pair<DT>(q[0], lo, hi);
        top = max_nan(lo, hi);
    }
    if (!(top <= a.m)) {  // NaN too
        const float d = exponent_shift(a.m, top);
        float s0, s1, t0, t1;
        f2_unpack(a.s, s0, s1);
        f2_unpack(a.t, t0, t1);
        shift_sums(d, s0, t0);
        shift_sums(d, s1, t1);
        a.s = f2_pack(s0, s1);
        a.t = f2_pack(t0, t1);
        a.m = top;
    }
    const uint64_t l2 = f2_splat(kLog2e), m2 = f2_splat(-(a.m * kLog2e));
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) {
        uint64_t x;
        if constexpr (DT == ADA_F32) {
            x = f2_pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
        } else {
            float lo, hi;
            unpack_pair<DT>(v[i], lo, hi);
            x = f2_pack(lo, hi);
        }
        const uint64_t d = f2_fma(x, l2, m2);
        float d0, d1;
        f2_unpack(d, d0, d1);
        const uint64_t e = f2_pack(fast_exp2(d0), fast_exp2(d1));
        a.s = f2_add(a.s, e);
        a.t = f2_fma(e, d, a.t);
    }
    return top;
}

// A row whose maximum is far from 0, by the whole block: m, and s and t of x_i - m itself.
template <int DT>
__device__ Sums plain_sums(const Reader<DT>& R, Sums* s_warp) {
    Sums a{-INFINITY, 0.f, 0.f};
    for (int pass = 0; pass < 2; ++pass) {
        const float ref = a.m == -INFINITY ? 0.f : a.m;
        for (int r = 0; r < R.rounds(); ++r) {
            uint32_t w[Reader<DT>::NV * 8];
            float x[kPer];
            R.load(r, w);
            Reader<DT>::unpack(w, x);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (pass == 0) {
                    a.m = max_nan(a.m, x[i]);
                } else {
                    const float d = max_nan((x[i] - ref) * kLog2e, -1e30f);
                    const float e = exp2f(d);
                    a.s += e;
                    a.t = fmaf(e, d, a.t);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            a.m = max_nan(a.m, __shfl_xor_sync(0xffffffffu, a.m, o));
            a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
            a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
        }
        if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = a;
        __syncthreads();
        for (int i = 0; i < kWarps; ++i) a.m = max_nan(a.m, s_warp[i].m);
    }
    a.s = a.t = 0.f;
    for (int i = 0; i < kWarps; ++i) {
        a.s += s_warp[i].s;
        a.t += s_warp[i].t;
    }
    return a;
}

// ---- top k ---------------------------------------------------------------------------

struct TopState {
    uint64_t cand[kCand];
    uint64_t best[8 * kMaxTop];    // the row's best, then those of the cluster's other parts
    uint64_t sorted[kMaxTop];
    float seen[kGroups];           // largest logit of a pair of threads
    int count, n_best;
    uint32_t hist[256];
    uint32_t digit, below;
};

// Of a thread's rounds: the three largest maxima and the rounds of the first
// two. A NaN gives way to the next round's maximum and steps down a place; it
// stays among the three, as `third` keeps NaN, so top and second together show it.
struct Seen {
    float top, second, third;
    int round, round2;
    __device__ __forceinline__ void add(float x, int r) {
        const bool first = !(x <= top), next = !(x <= second);  // NaN too
        third = max_nan(third, next ? second : x);
        second = first ? top : next ? x : second;
        round2 = first ? round : next ? r : round2;
        top = first ? x : top;
        round = first ? r : round;
    }
};

// Order of a value as an unsigned number (NaN above all).
__device__ __forceinline__ uint32_t order_of(float x) { return static_cast<uint32_t>(key_of(x, 0) >> 32); }

// A lower bound of the k-th best logit, as an order; 0 where that is not above
// the clamp: the k-th largest of the maxima of 32 groups of threads (k <= 24;
// sorted across the lanes) or of 128 pairs (to the first 16 bits of its order,
// a bit at a time). The k-th largest of n groups' maxima has about
// n log(n / (n - k)) logits above it.
template <int DT>
__device__ uint32_t find_bound(const TopState& S, int k) {
    const int lane = threadIdx.x & 31;
    uint32_t v[kGroups / 32], found = 0;
#pragma unroll
    for (int i = 0; i < kGroups / 32; ++i) v[i] = order_of(S.seen[i * 32 + lane]);
    if (k <= 24) {
        uint32_t x = max(max(v[0], v[1]), max(v[2], v[3]));
#pragma unroll
        for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
            for (int o = n >> 1; o > 0; o >>= 1) {
                const uint32_t y = __shfl_xor_sync(0xffffffffu, x, o);
                const bool down = (lane & n) == 0 || n == 32;  // this run is sorted downwards
                x = (((lane & o) == 0) == down) ? max(x, y) : min(x, y);
            }
        found = __shfl_sync(0xffffffffu, x, k - 1);
    } else {
#pragma unroll 1
        for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1) {
            const uint32_t c = found | bit;
            int n = 0;
#pragma unroll
            for (int i = 0; i < kGroups / 32; ++i) n += __popc(__ballot_sync(0xffffffffu, v[i] >= c));
            if (n >= k) found = c;
        }
    }
    return found <= order_of(lowest_kept<DT>()) ? 0u : found;
}

// The k best keys of the first n of best[] (n <= 512), in order, to sorted[].
__device__ void sort_best(TopState& S, int n, int k) {
    for (int i = threadIdx.x; i < n; i += kT) {
        const uint64_t mine = S.best[i];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) r += S.best[j] > mine;
        if (r < k) S.sorted[r] = mine;
    }
    __syncthreads();
}

// Adds one to the digit's bin for every lane that takes part; lanes that share
// the first one's digit (all of them in a constant row) add up first.
__device__ __forceinline__ void count_digit(TopState& S, bool on, uint32_t digit) {
    const uint32_t active = __ballot_sync(0xffffffffu, on);
    if (active == 0) return;
    const int first = __ffs(active) - 1;
    const uint32_t shared = __shfl_sync(0xffffffffu, digit, first);  // every lane takes part in the exchange
    const bool same = on && digit == shared;
    const uint32_t together = __ballot_sync(0xffffffffu, same);
    if (same) {
        if (static_cast<int>(threadIdx.x & 31) == first) atomicAdd(&S.hist[digit], static_cast<uint32_t>(__popc(together)));
    } else if (on) {
        atomicAdd(&S.hist[digit], 1u);
    }
}

// The k-th largest of a set of keys, a byte at a time; each(f) calls f(key, on)
// for all of them, whole warps at a time. 0 when there are fewer than k.
template <class Each>
__device__ uint64_t select_key(TopState& S, int k, const Each& each) {
    uint64_t prefix = 0, mask = 0;
    int want = k;
    for (int b = 56; b >= 0; b -= 8) {
        __syncthreads();
        S.hist[threadIdx.x] = 0;
        __syncthreads();
        each([&](uint64_t key, bool on) {
            count_digit(S, on && (key & mask) == prefix, static_cast<uint32_t>(key >> b) & 255u);
        });
        __syncthreads();
        if (threadIdx.x == 0) {
            int d = 255, before = 0;
            while (d > 0 && before + static_cast<int>(S.hist[d]) < want) before += static_cast<int>(S.hist[d--]);
            S.digit = static_cast<uint32_t>(d);
            S.below = static_cast<uint32_t>(before);
        }
        __syncthreads();
        prefix |= static_cast<uint64_t>(S.digit) << b;
        mask |= uint64_t(255) << b;
        want -= static_cast<int>(S.below);
    }
    return prefix;
}

// The k best keys of this block's rounds of the row (all, when it has fewer),
// in order, to sorted[].
template <int DT>
__device__ void best_keys(TopState& S, int k, const Seen& mine, const Reader<DT>& R, int rank, int parts) {
    constexpr int EPV = Reader<DT>::EPV, NV = Reader<DT>::NV;
    const int lane = threadIdx.x & 31;
    const float pair = max_nan(mine.top, __shfl_xor_sync(0xffffffffu, mine.top, 1));
    if ((lane & 1) == 0) S.seen[threadIdx.x >> 1] = pair;
    if (threadIdx.x == 0) S.count = S.n_best = 0;
    __syncthreads();
    const uint32_t bound = find_bound<DT>(S, k);
    const int rounds = R.rounds();
    const int vectors = rank < rounds ? ((rounds - rank + parts - 1) / parts) * NV : 0;  // of each thread
    if (bound != 0) {
        // A warp takes its threads at the bound four at a time: half of the lanes
        // read the elements of the best round, the others those of the second.
        const int half = lane >> 4, e = lane & 15;
        const int at = (e / EPV) * kT * EPV + e % EPV - lane * EPV + R.c0;
        uint32_t todo = __ballot_sync(0xffffffffu, order_of(max_nan(mine.top, mine.second)) >= bound);
        const uint32_t more = __ballot_sync(0xffffffffu, order_of(mine.second) >= bound);
        while (todo != 0) {
            float x[4];
            int c[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                c[u] = -1;
                x[u] = -INFINITY;
                if (todo == 0) continue;
                const int who = __ffs(todo) - 1;
                todo &= todo - 1;
                const int r1 = __shfl_sync(0xffffffffu, mine.round, who), r2 = __shfl_sync(0xffffffffu, mine.round2, who);
                if (half == 0 || ((more >> who) & 1u)) c[u] = (half == 0 ? r1 : r2) * kRound + who * EPV + at;
                if (c[u] >= 0 && c[u] < R.V) x[u] = load_as_f32(R.mine, c[u] - R.c0, DT);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool ok = c[u] >= 0 && c[u] < R.V && order_of(x[u]) >= bound;
                const uint32_t oks = __ballot_sync(0xffffffffu, ok);
                if (oks == 0) continue;
                int base = 0;
                if (lane == 0) base = atomicAdd(&S.count, __popc(oks));
                base = __shfl_sync(0xffffffffu, base, 0) + __popc(oks & ((1u << lane) - 1u));
                if (ok && base < kCand) S.cand[base] = key_of(x[u], c[u]);
            }
        }
        // further rounds of a thread, a lane for each vector
        for (uint32_t rare = __ballot_sync(0xffffffffu, order_of(mine.third) >= bound); rare != 0; rare &= rare - 1) {
            const int who = __ffs(rare) - 1;
            const int done = __shfl_sync(0xffffffffu, mine.round, who);
            const int done2 = __shfl_sync(0xffffffffu, mine.round2, who);
            for (int v = lane; v < vectors; v += 32) {
                const int round = rank + (v / NV) * parts;
                if (round == done || round == done2) continue;
                const int col = R.column(round, v % NV) + (who - lane) * EPV;
                uint32_t w[8];
                float x[EPV];
                R.vector(col, w);
                Reader<DT>::unpack(w, x);
#pragma unroll
                for (int i = 0; i < EPV; ++i) {
                    if (col + i < 0 || col + i >= R.V || order_of(x[i]) < bound) continue;
                    const int slot = atomicAdd(&S.count, 1);
                    if (slot < kCand) S.cand[slot] = key_of(x[i], col + i);
                }
            }
            __syncwarp();
        }
    }
    __syncthreads();
    const int n = S.count;
    if (bound == 0 || n > kCand) {  // too many equal logits, or too few above the clamp: all keys of the rounds
        auto each = [&](auto&& f) {
            for (int r = rank; r < rounds; r += parts) {
                uint32_t w[NV * 8];
                float x[kPer];
                R.load(r, w);
                Reader<DT>::unpack(w, x);
#pragma unroll 4
                for (int i = 0; i < kPer; ++i) {
                    const int c = R.column(r, i / EPV) + i % EPV;
                    f(key_of(x[i], c), c >= 0 && c < R.V);
                }
            }
        };
        const uint64_t from = select_key(S, k, each);
        each([&](uint64_t key, bool on) {
            if (on && key >= from) S.best[atomicAdd(&S.n_best, 1)] = key;
        });
    } else {
        uint64_t from = 0;
        if (n > 8 * kMaxTop) {
            from = select_key(S, k, [&](auto&& f) {
                for (int i = threadIdx.x; i - lane < n; i += kT) f(i < n ? S.cand[i] : 0, i < n);
            });
        }
        for (int i = threadIdx.x; i < n; i += kT)
            if (S.cand[i] >= from) S.best[atomicAdd(&S.n_best, 1)] = S.cand[i];
    }
    __syncthreads();
    const int have = S.n_best;
    if (static_cast<int>(threadIdx.x) >= have && static_cast<int>(threadIdx.x) < k) S.sorted[threadIdx.x] = 0;  // below any key
    sort_best(S, have, k);
}

// ---- forward -------------------------------------------------------------------------

template <int DT, bool TOP>
__global__ void __launch_bounds__(kT, DT == ADA_F32 ? 0 : TOP ? 6 : 8) token_logprobs_kernel(const __grid_constant__ LogprobLaunch L) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Sums s_warp[kWarps];
    __shared__ Sums s_part;
    TopState& S = *reinterpret_cast<TopState*>(smem);
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank()), parts = L.cluster;
    const int64_t row = blockIdx.x / parts;
    const int64_t off = (row / L.R) * L.s0 + (row % L.R) * L.s1;
    constexpr int EB = Reader<DT>::EB;
    const uint8_t* zr = static_cast<const uint8_t*>(L.logits) + off * EB;
    const Reader<DT> R(zr, L.V);
    const int k = TOP ? L.top : 0;
    // the given token's logit is on its way while the row is read
    float zt = 0.f;
    int token = 0;  // 1: ignored, 2: outside the vocabulary
    if (rank == 0 && threadIdx.x == 0) {
        const int64_t t = L.tok64 ? static_cast<const int64_t*>(L.tokens)[row] : static_cast<const int32_t*>(L.tokens)[row];
        token = t == L.ignore ? 1 : (t < 0 || t >= L.V) ? 2 : 0;
        if (token == 0) zt = load_as_f32(zr, t, DT);
    }
    PairSums sums{-INFINITY, f2_splat(0.f), f2_splat(0.f)};
    Seen seen{-INFINITY, -INFINITY, -INFINITY, 0, 0};
    const int rounds = R.rounds();
    uint32_t w[Reader<DT>::NV * 8], next[Reader<DT>::NV * 8];
    if (rank < rounds) R.load(rank, w);
#pragma unroll 2
    for (int r = rank; r < rounds; r += parts) {
        if (r + parts < rounds) R.load(r + parts, next);
        if (R.any(r)) {
            const float top = add_round<DT>(sums, w);
            if (TOP) seen.add(top, r);
        }
#pragma unroll
        for (int j = 0; j < Reader<DT>::NV * 8; ++j) w[j] = next[j];
    }
    Sums a;
    {
        float s0, s1, t0, t1;
        f2_unpack(sums.s, s0, s1);
        f2_unpack(sums.t, t0, t1);
        a = join_warp(Sums{sums.m, s0 + s1, t0 + t1}, 32);
    }
    if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = a;
    __syncthreads();
    if (threadIdx.x < 32) {
        a = join_warp(threadIdx.x < kWarps ? s_warp[threadIdx.x] : Sums{-INFINITY, 0.f, 0.f}, kWarps);
        if (threadIdx.x == 0) s_part = a;
    }
    if constexpr (TOP) best_keys<DT>(S, k, seen, R, rank, parts);
    if (parts > 1) {
        cluster.sync();
        if (rank == 0) {
            if (threadIdx.x < 32) {
                a = join_warp(threadIdx.x < parts ? *cluster.map_shared_rank(&s_part, threadIdx.x)
                                                  : Sums{-INFINITY, 0.f, 0.f}, 8);
                __syncwarp();
                if (threadIdx.x == 0) s_part = a;
            }
            if constexpr (TOP) {
                for (int i = threadIdx.x; i < parts * k; i += kT)
                    S.best[i] = cluster.map_shared_rank(&S, i / k)->sorted[i % k];
                __syncthreads();
                sort_best(S, parts * k, k);
            }
        }
        cluster.sync();  // the parts stay until they are read
        if (rank != 0) return;
    }
    __syncthreads();
    a = s_part;
    if (!ends_of_range(a.m) && threadIdx.x >= (TOP ? kMaxTop : 32)) return;
    // ls = log sum exp(z_i - m), mean = sum p_i (z_i - m), in base 2 first
    float ls, mean;
    if (ends_of_range(a.m)) {
        a = plain_sums<DT>(R, s_warp);
        ls = logf(a.s);
        mean = a.t / a.s * kLn2;
    } else {
        const float r = fmaf(a.m, kLog2e, -(a.m * kLog2e));  // what M's rounding left out
        ls = (log2f(a.s) - r) * kLn2;
        mean = (a.t / a.s - r) * kLn2;
    }
    if (threadIdx.x == 0) {
        float lp = token == 0 ? (zt - a.m) - ls : 0.f;
        if (token == 2) {
            lp = __int_as_float(0x7FFFFFFF);
            record_error(L.status, ADA_ERR_INVALID);
        }
        L.logprobs[row] = lp;
        L.entropy[row] = ls - mean;
        L.lse[row] = a.m + ls;
        if (L.stats != nullptr) {
            L.stats[2 * row] = a.m;
            L.stats[2 * row + 1] = ls;
        }
    }
    if constexpr (TOP) {
        for (int i = threadIdx.x; i < k; i += kT) {
            const int c = column_of(S.sorted[i]);
            L.top_tokens[row * k + i] = c;
            L.top_logprobs[row * k + i] = (value_of(S.sorted[i]) - a.m) - ls;
        }
    }
}

// ---- backward ------------------------------------------------------------------------

// Block (row, segment): rounds segment, segment + segments, ... of the row.
template <int DT>
__global__ void __launch_bounds__(kT) token_logprobs_bwd_kernel(const __grid_constant__ LogprobLaunch L) {
    constexpr int EB = Reader<DT>::EB, EPV = Reader<DT>::EPV, NV = Reader<DT>::NV;
    const int64_t row = blockIdx.x / L.segments;
    const int seg = static_cast<int>(blockIdx.x % L.segments);
    const int64_t a = row / L.R, b = row % L.R;
    const Reader<DT> R(static_cast<const uint8_t*>(L.logits) + (a * L.s0 + b * L.s1) * EB, L.V);
    uint8_t* gr = static_cast<uint8_t*>(L.grad) + (a * L.gs0 + b * L.gs1) * EB;
    const bool aligned = (reinterpret_cast<uint64_t>(gr) & 31u) / EB == static_cast<uint64_t>(R.shift);
    const float m = L.stats[2 * row], ls = L.stats[2 * row + 1];
    const int64_t t = L.tok64 ? static_cast<const int64_t*>(L.tokens)[row] : static_cast<const int32_t*>(L.tokens)[row];
    float g_lp = (L.g_logprobs != nullptr && t != L.ignore) ? L.g_logprobs[row] : 0.f;
    if (t != L.ignore && (t < 0 || t >= L.V)) g_lp = __int_as_float(0x7FFFFFFF);  // as its log probability
    const float g_h = L.g_entropy != nullptr ? L.g_entropy[row] : 0.f;
    const float g_lse = L.g_lse != nullptr ? L.g_lse[row] : 0.f;
    const float c0 = g_lse - g_lp - g_h * L.entropy[row];
    const int rounds = R.rounds();
    // log2 p = (x - M) + shift with M as the forward's; rows near the ends of the range take the plain difference
    const bool plain = ends_of_range(m);
    const float M = plain ? 0.f : m * kLog2e;
    const float shift = plain ? 0.f : -fmaf(ls, kLog2e, fmaf(m, kLog2e, -M));
    const uint64_t l2 = f2_splat(kLog2e), m2 = f2_splat(-M), sh2 = f2_splat(shift);
    const uint64_t c2 = f2_splat(c0), gh2 = f2_splat(-g_h * kLn2);
    for (int r = seg; r < rounds; r += L.segments) {
        if (!R.any(r)) break;
        uint32_t w[NV * 8];
        float x[kPer];
        R.load(r, w);
        Reader<DT>::unpack(w, x);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = R.column(r, j);
            float g[EPV];
#pragma unroll
            for (int i = 0; i < EPV; i += 2) {
                float d0, d1;
                if (plain) {
                    d0 = ((x[j * EPV + i] - m) - ls) * kLog2e;
                    d1 = ((x[j * EPV + i + 1] - m) - ls) * kLog2e;
                } else {
                    f2_unpack(f2_add(f2_fma(f2_pack(x[j * EPV + i], x[j * EPV + i + 1]), l2, m2), sh2), d0, d1);
                }
                // p is 0 from -150 on: the bound keeps -inf out of the product
                d0 = max_nan(d0, -1000.f);
                d1 = max_nan(d1, -1000.f);
                const uint64_t e = f2_pack(fast_exp2(d0), fast_exp2(d1));
                f2_unpack(f2_mul(e, f2_fma(gh2, f2_pack(d0, d1), c2)), g[i], g[i + 1]);
            }
            if (t >= c && t < c + EPV) {
#pragma unroll
                for (int i = 0; i < EPV; ++i)
                    if (c + i == t) g[i] += g_lp;
            }
            uint32_t u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (DT == ADA_F32) u[i] = __float_as_uint(g[i]);
                else if constexpr (DT == ADA_BF16) u[i] = pack_bf16x2(g[2 * i], g[2 * i + 1]);
                else u[i] = pack_f16x2(g[2 * i], g[2 * i + 1]);
            }
            if (aligned && c >= 0 && c + EPV <= L.V) {
                st_global_v8(gr + static_cast<int64_t>(c) * EB, u);
            } else {
#pragma unroll
                for (int i = 0; i < EPV; ++i) {
                    if (c + i < 0 || c + i >= L.V) continue;
                    if constexpr (DT == ADA_F32) reinterpret_cast<uint32_t*>(gr)[c + i] = u[i];
                    else reinterpret_cast<uint16_t*>(gr)[c + i] = static_cast<uint16_t>(u[i / 2] >> (16 * (i & 1)));
                }
            }
        }
    }
}

template <int DT, bool TOP>
int launch_fwd(const LogprobLaunch& L, cudaStream_t stream) {
    const size_t smem = TOP ? sizeof(TopState) : 0;
    auto kernel = token_logprobs_kernel<DT, TOP>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
        return ADA_ERR_LAUNCH;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(L.rows * L.cluster));
    cfg.blockDim = dim3(kT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(L.cluster);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, L) == cudaSuccess ? ADA_OK : ADA_ERR_LAUNCH;
}

template <int DT>
int launch_fwd_dt(const LogprobLaunch& L, cudaStream_t stream) {
    return L.top > 0 ? launch_fwd<DT, true>(L, stream) : launch_fwd<DT, false>(L, stream);
}

}  // namespace

int launch_token_logprobs(const LogprobLaunch& L, cudaStream_t stream) {
    switch (L.dtype) {
        case ADA_F32: return launch_fwd_dt<ADA_F32>(L, stream);
        case ADA_F16: return launch_fwd_dt<ADA_F16>(L, stream);
        case ADA_BF16: return launch_fwd_dt<ADA_BF16>(L, stream);
        default: return ADA_ERR_DTYPE;
    }
}

int launch_token_logprobs_bwd(const LogprobLaunch& L, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(L.rows * L.segments);
    switch (L.dtype) {
        case ADA_F32: token_logprobs_bwd_kernel<ADA_F32><<<grid, kT, 0, stream>>>(L); break;
        case ADA_F16: token_logprobs_bwd_kernel<ADA_F16><<<grid, kT, 0, stream>>>(L); break;
        case ADA_BF16: token_logprobs_bwd_kernel<ADA_BF16><<<grid, kT, 0, stream>>>(L); break;
        default: return ADA_ERR_DTYPE;
    }
    return cudaGetLastError() == cudaSuccess ? ADA_OK : ADA_ERR_LAUNCH;
}

}  // namespace ada
