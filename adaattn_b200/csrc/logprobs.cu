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
// weighted sum (fp32, base 2), joined at the end, so HBM reads of V elements
// bound it (each costs about six instructions, near half the issue rate at
// full bandwidth). A row is shared by a cluster of CTAs when there are few
// rows; its parts are joined through distributed shared memory, no workspace.
//
// Top k (k <= 64): candidates are 64-bit keys, the value's order above the
// inverted column, so all keys differ and equal values rank by lowest index.
// 128 thread pairs keep the maximum of what they saw; the k-th largest of
// those bounds the k-th best logit from below, and only logits at or above
// that bound enter the candidate list (a few k per row). The bound is renewed
// at rounds 0, 1, 3, 7, ... The list is cut to its k best keys by radix
// selection when it fills, whatever the order of the logits.
#include <cooperative_groups.h>

#include "ada_common.cuh"
#include "ada_internal.h"

namespace ada {
namespace {

namespace cg = cooperative_groups;

constexpr int kT = 256;             // threads
constexpr int kPer = 16;            // elements per thread and round
constexpr int kRound = kT * kPer;
constexpr int kCap = 5120;          // candidates: kRound more than the cut's mark
constexpr int kMark = kCap - kRound;
constexpr int kGroups = kT / 2;
constexpr int kMaxTop = 64;
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
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ int column_of(uint64_t key) {
    return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}

// ---- reading a row ---------------------------------------------------------------
//
// Columns are counted from the 16-byte boundary at or before the row's start,
// so vector loads are aligned whatever the row's address: column c = e - shift.
// Vectors that reach past either end of the row are read element by element.
template <int DT>
struct Reader {
    static constexpr int EB = DT == ADA_F32 ? 4 : 2;
    static constexpr int EPV = 16 / EB;         // elements per vector
    static constexpr int NV = kPer / EPV;       // vectors per thread and round
    const uint8_t* base;  // the boundary
    int shift, V;

    __device__ Reader(const void* row, int v) : V(v) {
        const uint64_t a = reinterpret_cast<uint64_t>(row);
        base = reinterpret_cast<const uint8_t*>(a & ~uint64_t(15));
        shift = static_cast<int>(a & 15u) / EB;
    }
    __device__ int rounds() const { return (V + shift + kRound - 1) / kRound; }
    // First column of vector j of this thread in a round.
    __device__ int column(int round, int j) const {
        return ((round * NV + j) * kT + static_cast<int>(threadIdx.x)) * EPV - shift;
    }
    __device__ void load(int round, uint4 (&w)[NV]) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = column(round, j);
            const uint8_t* p = base + static_cast<int64_t>(c + shift) * EB;
            if (c >= 0 && c + EPV <= V) {
                w[j] = __ldcs(reinterpret_cast<const uint4*>(p));
            } else {
                uint32_t u[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (DT == ADA_F32) {
                        u[i] = (c + i >= 0 && c + i < V) ? reinterpret_cast<const uint32_t*>(p)[i] : 0xFF800000u;
                    } else {
                        constexpr uint32_t kNegInf = DT == ADA_BF16 ? 0xFF80u : 0xFC00u;
                        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
                        const uint32_t lo = (c + 2 * i >= 0 && c + 2 * i < V) ? h[2 * i] : kNegInf;
                        const uint32_t hi = (c + 2 * i + 1 >= 0 && c + 2 * i + 1 < V) ? h[2 * i + 1] : kNegInf;
                        u[i] = lo | (hi << 16);
                    }
                }
                w[j] = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
    }
    __device__ static void unpack(const uint4 (&w)[NV], float (&x)[kPer]) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const uint32_t u[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (DT == ADA_F32) {
                    x[4 * j + i] = __uint_as_float(u[i]);
                } else if constexpr (DT == ADA_BF16) {
                    x[8 * j + 2 * i] = __uint_as_float(u[i] << 16);
                    x[8 * j + 2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
                } else {
                    unpack_f16x2(u[i], x[8 * j + 2 * i], x[8 * j + 2 * i + 1]);
                }
            }
        }
    }
};

// ---- running sums ------------------------------------------------------------------

struct Sums {
    float m, s, t;  // maximum; sum of 2^x and of x 2^x with x = (z - m) log2 e
};

// Changes the maximum to m (at least s.m).
__device__ __forceinline__ void shift_to(Sums& a, float m) {
    if (a.s != 0.f) {
        const float d = (a.m - m) * kLog2e;
        const float w = exp2f(d);
        a.t = w == 0.f ? 0.f : w * fmaf(a.s, d, a.t);
        a.s *= w;
    }
    a.m = m;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
    const float m = max_nan(a.m, b.m);
    shift_to(a, m);
    shift_to(b, m);
    return Sums{m, a.s + b.s, a.t + b.t};
}

__device__ __forceinline__ void add_elements(Sums& a, const float (&x)[kPer], float top) {
    if (!(top <= a.m)) shift_to(a, top);  // NaN too
    const float ref = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        // -inf (and what is as far below) counts as -1e30: its power is 0 and so is the product
        const float d = max_nan((x[i] - ref) * kLog2e, -1e30f);
        const float e = fast_exp2(d);
        a.s += e;
        a.t = fmaf(e, d, a.t);
    }
}

// ---- top k ---------------------------------------------------------------------------

struct TopState {
    uint64_t cand[kCap];
    uint64_t best[kMaxTop];
    uint64_t group[kGroups];
    uint64_t bound;   // candidates are keys above it
    int count, n_best;
    uint32_t hist[256];
    uint32_t digit, below;
};

// The k best of the first n candidates to best[] (unordered); n > k. Radix
// selection of the k-th largest key, a byte at a time; all keys differ.
__device__ void cut(TopState& S, int n, int k) {
    uint64_t prefix = 0, mask = 0;
    int want = k;
    for (int b = 56; b >= 0; b -= 8) {
        S.hist[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kT)
            if ((S.cand[i] & mask) == prefix) atomicAdd(&S.hist[(S.cand[i] >> b) & 255u], 1u);
        __syncthreads();
        if (threadIdx.x < 32) {  // lane l: digits 255 - 8 l downwards
            uint32_t c[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                c[i] = S.hist[255 - 8 * threadIdx.x - i];
                sum += c[i];
            }
            uint32_t scan = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, scan, o);
                if (threadIdx.x >= o) scan += up;
            }
            uint32_t before = scan - sum;
            if (before < want && scan >= want) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (before < want && before + c[i] >= want) {
                        S.digit = 255 - 8 * threadIdx.x - i;
                        S.below = before;
                        break;
                    }
                    before += c[i];
                }
            }
        }
        __syncthreads();
        prefix |= static_cast<uint64_t>(S.digit) << b;
        mask |= uint64_t(255) << b;
        want -= static_cast<int>(S.below);
    }
    if (threadIdx.x == 0) S.n_best = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kT)
        if (S.cand[i] >= prefix) S.best[atomicAdd(&S.n_best, 1)] = S.cand[i];
    __syncthreads();
    if (threadIdx.x == 0 && prefix > S.bound + 1) S.bound = prefix - 1;
}

// The k best candidates, in order, to best[0 .. n_best).
__device__ void rank_best(TopState& S, int k) {
    int n = S.count;
    if (n > 512) {
        cut(S, n, k);
        n = k;
        for (int i = threadIdx.x; i < n; i += kT) S.cand[i] = S.best[i];
        __syncthreads();
    }
    for (int i = threadIdx.x; i < n; i += kT) {
        const uint64_t mine = S.cand[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += S.cand[j] > mine;
        if (r < k) S.best[r] = mine;
    }
    if (threadIdx.x == 0) S.n_best = min(n, k);
    __syncthreads();
}

// One round of logits. `seen`: the largest logit this thread has met.
template <int DT>
__device__ __forceinline__ void top_round(TopState& S, int k, const float (&x)[kPer], float top, float& seen, int turn,
                                          const Reader<DT>& R, int round) {
    seen = max_nan(seen, top);
    if ((turn & (turn + 1)) == 0) {  // 0, 1, 3, 7, ...
        const float other = __shfl_xor_sync(0xffffffffu, seen, 1);
        // one key per pair: the value alone decides, pairs of one value count by their number
        const uint64_t g = key_of(max_nan(seen, other), threadIdx.x >> 1);
        if ((threadIdx.x & 1) == 0) S.group[threadIdx.x >> 1] = g;
        __syncthreads();
        if (threadIdx.x < kGroups) {
            const uint64_t mine = S.group[threadIdx.x];
            int r = 0;
#pragma unroll 8
            for (int j = 0; j < kGroups; ++j) r += S.group[j] > mine;
            if (r == k - 1) {
                const uint64_t bound = (mine >> 32) << 32;  // every column of that value passes
                if (bound != 0 && bound - 1 > S.bound && value_of(mine) != -INFINITY) S.bound = bound - 1;
            }
        }
        __syncthreads();
    }
    const uint64_t bound = S.bound;
    const uint32_t hi = static_cast<uint32_t>((bound + 1) >> 32);
    const float low = hi == 0 ? -INFINITY : value_of(static_cast<uint64_t>(hi) << 32);
    if (!(top < low)) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            constexpr int EPV = Reader<DT>::EPV;
            if (x[i] < low) continue;
            const int c = R.column(round, i / EPV) + i % EPV;
            if (c < 0 || c >= R.V) continue;
            const uint64_t key = key_of(x[i], c);
            if (key > bound) S.cand[atomicAdd(&S.count, 1)] = key;
        }
    }
    __syncthreads();
    const int n = S.count;
    __syncthreads();
    if (n > kMark) {
        cut(S, n, k);
        for (int i = threadIdx.x; i < k; i += kT) S.cand[i] = S.best[i];
        if (threadIdx.x == 0) S.count = k;
        __syncthreads();
    }
}

// ---- forward -------------------------------------------------------------------------

template <int DT, bool TOP>
__global__ void __launch_bounds__(kT) token_logprobs_kernel(const __grid_constant__ LogprobLaunch L) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Sums s_warp[kT / 32];
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
    if (TOP && threadIdx.x == 0) {
        S.bound = 0;
        S.count = 0;
        S.n_best = 0;
    }
    if (TOP) __syncthreads();
    Sums a{-INFINITY, 0.f, 0.f};
    float seen = -INFINITY;
    const int rounds = R.rounds();
    uint4 w[Reader<DT>::NV];
    if (rank < rounds) R.load(rank, w);
    int turn = 0;
    for (int r = rank; r < rounds; r += parts, ++turn) {
        float x[kPer];
        Reader<DT>::unpack(w, x);
        if (r + parts < rounds) R.load(r + parts, w);
        float top = x[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i) top = max_nan(top, x[i]);
        add_elements(a, x, top);
        if constexpr (TOP) top_round<DT>(S, k, x, top, seen, turn, R, r);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
        a = join(a, b);
    }
    if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kT / 32; ++i) a = join(a, s_warp[i]);
        s_part = a;
    }
    if (TOP) rank_best(S, k);
    if (parts > 1) {
        cluster.sync();
        if (rank == 0) {
            if (threadIdx.x == 0) {
                for (int i = 1; i < parts; ++i) a = join(a, *cluster.map_shared_rank(&s_part, i));
                s_part = a;
            }
            if (TOP) {
                int n = 0;
                for (int i = 0; i < parts; ++i) {
                    const TopState* T = cluster.map_shared_rank(&S, i);
                    const int m = T->n_best;
                    for (int j = threadIdx.x; j < m; j += kT) S.cand[n + j] = T->best[j];
                    n += m;
                }
                __syncthreads();
                if (threadIdx.x == 0) S.count = n;
                __syncthreads();
                rank_best(S, k);
            }
        }
        cluster.sync();  // the parts stay until they are read
        if (rank != 0) return;
    }
    __syncthreads();
    a = s_part;
    const float ls = logf(a.s);
    if (threadIdx.x == 0) {
        const int64_t t = L.tok64 ? static_cast<const int64_t*>(L.tokens)[row] : static_cast<const int32_t*>(L.tokens)[row];
        float lp = 0.f;
        if (t != L.ignore) {
            if (t >= 0 && t < L.V) {
                lp = (load_as_f32(zr, t, DT) - a.m) - ls;
            } else {
                lp = __int_as_float(0x7FFFFFFF);
                record_error(L.status, ADA_ERR_INVALID);
            }
        }
        L.logprobs[row] = lp;
        L.entropy[row] = ls - a.t / a.s * kLn2;
        L.lse[row] = a.m + ls;
        L.stats[2 * row] = a.m;
        L.stats[2 * row + 1] = ls;
    }
    if constexpr (TOP) {
        for (int i = threadIdx.x; i < k; i += kT) {
            const int c = column_of(S.best[i]);
            L.top_tokens[row * k + i] = c;
            L.top_logprobs[row * k + i] = (load_as_f32(zr, c, DT) - a.m) - ls;
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
    const bool aligned = (reinterpret_cast<uint64_t>(gr) & 15u) / EB == static_cast<uint64_t>(R.shift);
    const float m = L.stats[2 * row], ls = L.stats[2 * row + 1];
    const int64_t t = L.tok64 ? static_cast<const int64_t*>(L.tokens)[row] : static_cast<const int32_t*>(L.tokens)[row];
    float g_lp = (L.g_logprobs != nullptr && t != L.ignore) ? L.g_logprobs[row] : 0.f;
    if (t != L.ignore && (t < 0 || t >= L.V)) g_lp = __int_as_float(0x7FFFFFFF);  // as its log probability
    const float g_h = L.g_entropy != nullptr ? L.g_entropy[row] : 0.f;
    const float g_lse = L.g_lse != nullptr ? L.g_lse[row] : 0.f;
    const float c0 = g_lse - g_lp - g_h * L.entropy[row];
    const int rounds = R.rounds();
    for (int r = seg; r < rounds; r += L.segments) {
        uint4 w[NV];
        float x[kPer];
        R.load(r, w);
        Reader<DT>::unpack(w, x);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = R.column(r, j);
            float g[EPV];
#pragma unroll
            for (int i = 0; i < EPV; ++i) {
                const float logp = (x[j * EPV + i] - m) - ls;
                const float p = exp2f(logp * kLog2e);
                g[i] = p == 0.f ? 0.f * c0 : p * fmaf(-g_h, logp, c0);
                if (c + i == t) g[i] += g_lp;
            }
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (DT == ADA_F32) u[i] = __float_as_uint(g[i]);
                else if constexpr (DT == ADA_BF16) u[i] = pack_bf16x2(g[2 * i], g[2 * i + 1]);
                else u[i] = pack_f16x2(g[2 * i], g[2 * i + 1]);
            }
            if (aligned && c >= 0 && c + EPV <= L.V) {
                __stcs(reinterpret_cast<uint4*>(gr + static_cast<int64_t>(c) * EB), make_uint4(u[0], u[1], u[2], u[3]));
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
