// Attention of one new token per sequence over a paged key-value cache.
//
// For sequence b (table row r), query head h of key/value head g = h / G:
//   s_j = scale * ks_g * (q_h . k_j) + add_j      over visible keys j < len_b
//   o_h = vs_g * sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j
// (ks, vs: the scales of an 8-bit cache; add: a float key mask). A key hidden
// by a bool mask or by -inf takes no part, whatever its page holds (the
// CUDA-core kernel does not read it, the other one puts zeros in its values'
// place); a sequence with no visible key gives zeros and lse = -inf.
//
// Each key and value is read once per block of up to 8 query heads and costs 4
// multiply-adds per head and element: the cache's bytes bound the operator.
// So the work is split evenly over the cache, not over sequences: the tiles of
// 32 keys of all (sequence, head block) units stand in one line, CTA c takes
// the c-th equal piece of it and each of its warps an equal piece of that. A
// unit begins with kLead empty places, which stand for what a warp spends to
// start and finish one (without them a warp with eight two-tile units ran four
// times as long as the others). A unit that lies in one warp's piece is
// finished there. Pieces of a unit that
// spans warps are joined in shared memory (each with its running maximum m,
// sum l and unnormalised accumulator), pieces that span CTAs are joined by a
// second kernel. The split depends on the lengths alone, so results repeat.
#include "ada_common.cuh"
#include "ada_internal.h"

namespace ada {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = kPagedTile, kLead = kPagedLead;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// ---- the line of tiles -------------------------------------------------------

// Table row of batch entry b (-1: outside the table).
__device__ __forceinline__ int64_t table_row(const PagedAttnLaunch& L, int b) {
    const int64_t r = L.seqs != nullptr ? L.seqs[b] : b;
    return (r >= 0 && r < L.S) ? r : -1;
}

// Keys of batch entry b; a row or length outside the table is recorded and cut.
__device__ __forceinline__ int seq_length(const PagedAttnLaunch& L, int b) {
    const int64_t r = table_row(L, b);
    if (r < 0) {
        record_error(L.status, ADA_ERR_INVALID);
        return 0;
    }
    const int n = L.lens[r];
    const int64_t most = L.W * L.page;
    if (n < 0 || n > most) {
        record_error(L.status, ADA_ERR_INVALID);
        return n < 0 ? 0 : static_cast<int>(most);
    }
    return n;
}

// pref[b] = places per unit of the sequences before b, pref[B] = of all (every thread of the block calls it).
__device__ void tile_prefix(const PagedAttnLaunch& L, int* pref, int* warp_sums) {
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
    const int per = (L.B + nt - 1) / nt;
    const int b0 = min(tid * per, L.B), b1 = min(b0 + per, L.B);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
        const int tiles = static_cast<int>((static_cast<uint32_t>(seq_length(L, b)) + (kTile - 1)) / kTile);  // (up to 2^31 - 1 keys)
        const int n = tiles > 0 ? tiles + kLead : 0;
        pref[b] = n;
        sum += n;
    }
    int scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += up;
    }
    if (lane == 31) warp_sums[warp] = scan;
    __syncthreads();
    int before = scan - sum;
    for (int w = 0; w < warp; ++w) before += warp_sums[w];
    for (int b = b0; b < b1; ++b) {
        const int n = pref[b];
        pref[b] = before;
        before += n;
    }
    if (b1 == L.B && b0 < b1) pref[L.B] = before;
    __syncthreads();
}

// A unit: one sequence's keys for one block of query heads of one key/value head.
struct Unit {
    int b, u;
    int64_t t0, t1;  // its tiles on the line
};

// The unit whose tiles or leading places hold place t.
__device__ __forceinline__ Unit unit_at(const PagedAttnLaunch& L, const int* pref, int64_t t) {
    const int q = static_cast<int>(t / L.U);
    int lo = 0, hi = L.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pref[mid] <= q) lo = mid;
        else hi = mid - 1;
    }
    Unit x;
    x.b = lo;
    const int64_t first = static_cast<int64_t>(pref[lo]) * L.U;
    const int n = pref[lo + 1] - pref[lo];
    x.u = static_cast<int>((t - first) / n);
    x.t0 = first + static_cast<int64_t>(x.u) * n + kLead;
    x.t1 = x.t0 + n - kLead;
    return x;
}

// The unit after x; t0 past the line's end when there is none.
__device__ __forceinline__ Unit unit_after(const PagedAttnLaunch& L, const int* pref, Unit x) {
    const int64_t n = x.t1 - x.t0;
    x.t0 = x.t1 + kLead;
    x.t1 = x.t0 + n;
    if (++x.u < L.U) return x;
    x.u = 0;
    do ++x.b;
    while (x.b < L.B && pref[x.b + 1] == pref[x.b]);
    if (x.b < L.B) x.t1 = x.t0 + (pref[x.b + 1] - pref[x.b] - kLead);
    return x;
}

// The CTAs that take part and the piece of CTA c: [c T / n, (c + 1) T / n).
__device__ __forceinline__ int64_t pieces(int64_t T, int64_t most) { return T < most ? T : most; }
__device__ __forceinline__ int64_t piece_start(int64_t c, int64_t T, int64_t n) { return c * T / n; }
// The piece that holds place t.
__device__ __forceinline__ int64_t piece_of(int64_t t, int64_t T, int64_t n) { return ((t + 1) * n - 1) / T; }

// ---- element access ----------------------------------------------------------

// Four elements from column c of a row; VEC: rows aligned to 4 elements and D a multiple of 4.
template <int DT, bool VEC>
__device__ __forceinline__ float4 load4(const void* base, int64_t row, int c, int D) {
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c >= D) return f;
    if constexpr (VEC) {
        if constexpr (DT == ADA_F32) {
            f = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + row + c);
        } else if constexpr (DT == ADA_E4M3) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(base) + row + c);
            const __half2 a(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xFFFFu), __NV_E4M3));
            const __half2 b(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3));
            const float2 x = __half22float2(a), y = __half22float2(b);
            f = make_float4(x.x, x.y, y.x, y.y);
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + row + c);
            if constexpr (DT == ADA_BF16) {
                f = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u),
                                __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u));
            } else {
                unpack_f16x2(w.x, f.x, f.y);
                unpack_f16x2(w.y, f.z, f.w);
            }
        }
    } else {
        float e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (c + i >= D) break;
            if constexpr (DT == ADA_E4M3) {
                const __half h(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(base)[row + c + i], __NV_E4M3));
                e[i] = __half2float(h);
            } else {
                e[i] = load_as_f32(base, row + c + i, DT);
            }
        }
        f = make_float4(e[0], e[1], e[2], e[3]);
    }
    return f;
}

// Writes the finished head: acc / l (0 where no key was visible) and its log-sum-exp.
__device__ __forceinline__ void store_out(const PagedAttnLaunch& L, int b, int h, int d, float x) {
    store_from_f32(L.out, b * L.os[0] + h * L.os[1] + d, L.q_dtype, x);
}
__device__ __forceinline__ float value_scale(const PagedAttnLaunch& L, int g) {
    return L.v_scale != nullptr ? L.v_scale[g] : 1.f;
}

// ---- joining pieces ----------------------------------------------------------

// What a warp left of a unit that its piece holds only in part: slot 0 of a
// unit that began before the piece, slot 1 of one that goes on after it.
struct Left {
    int valid, b, u;
    int64_t t0, t1;
};

// Accumulators [GB][DP] and (m, l) [GB][2] of the block's warps and slots.
struct Join {
    float* acc[2];   // of warp 0, by slot
    int stride[2];   // floats from one warp's to the next one's
    float* ml;       // [warps][2][GB][2]
    Left* left;      // [warps][2]
    __device__ float* part(int warp, int slot) const { return acc[slot] + warp * stride[slot]; }
};

// Joins the pieces that the block's warps left. A unit inside the block's own
// piece [a, z) is finished; another goes to the workspace, slot 0 / 1 as above.
template <int WARPS, int GB, int DP>
__device__ void join_block(const PagedAttnLaunch& L, const Join& J, int64_t a, int64_t z) {
    constexpr int NE = 2 * WARPS;
    int e = 0;
    while (e < NE) {
        if (!J.left[e].valid) {
            ++e;
            continue;
        }
        const Left x = J.left[e];
        int end = e + 1;
        while (end < NE && (!J.left[end].valid || J.left[end].t0 == x.t0)) ++end;
        const int g = x.u / L.HB, h0 = g * L.G + (x.u % L.HB) * GB;
        const int heads = min(GB, (g + 1) * L.G - h0);
        const bool whole = x.t0 >= a && x.t1 <= z;
        const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (x.t0 < a ? 0 : 1);
        for (int i = threadIdx.x; i < heads * DP; i += WARPS * 32) {
            const int h = i / DP, d = i - h * DP;
            float m = -INFINITY;
            for (int k = e; k < end; ++k)
                if (J.left[k].valid) m = fmaxf(m, J.ml[(k * GB + h) * 2]);
            const float ref = m == -INFINITY ? 0.f : m;
            float l = 0.f, acc = 0.f;
            for (int k = e; k < end; ++k) {
                if (!J.left[k].valid) continue;
                const float w = exp2f((J.ml[(k * GB + h) * 2] - ref) * kLog2e);
                l += w * J.ml[(k * GB + h) * 2 + 1];
                acc += w * J.part(k >> 1, k & 1)[h * DP + d];
            }
            if (whole) {
                if (d < L.D) store_out(L, x.b, h0 + h, d, l == 0.f ? 0.f : acc / l * value_scale(L, g));
                if (d == 0 && L.lse != nullptr) L.lse[static_cast<int64_t>(x.b) * L.H + h0 + h] = m + logf(l);
            } else {
                if (d < L.D) L.part_acc[(slot * GB + h) * L.D + d] = acc;
                if (d == 0) {
                    L.part_ml[(slot * GB + h) * 2] = m;
                    L.part_ml[(slot * GB + h) * 2 + 1] = l;
                }
            }
        }
        e = end;
    }
}

// The outputs of sequences without keys, shared out over the grid.
__device__ void write_empty(const PagedAttnLaunch& L, const int* pref) {
    for (int b = blockIdx.x; b < L.B; b += gridDim.x) {
        if (pref[b + 1] != pref[b]) continue;
        for (int i = threadIdx.x; i < L.H * L.D; i += blockDim.x) store_out(L, b, i / L.D, i % L.D, 0.f);
        if (L.lse != nullptr)
            for (int h = threadIdx.x; h < L.H; h += blockDim.x) L.lse[static_cast<int64_t>(b) * L.H + h] = -INFINITY;
    }
}

// Joins what CTAs left of a unit that spans several: block (c, h) serves head
// h of the unit that goes on from CTA c's piece into the next one, when it
// began in c's. Its partial sums are one per CTA: c's in slot 1, the others'
// in slot 0. The weights of up to 512 parts are worked out side by side.
constexpr int kJoinThreads = 128;
constexpr int kMaxParts = 512;

__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedAttnLaunch L) {
    __shared__ float s_w[kMaxParts];
    __shared__ float s_red[2][kJoinThreads / 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t T = static_cast<int64_t>(L.pref[L.B]) * L.U;
    const int64_t nc = pieces(T, L.n_cta);
    const int64_t c0 = blockIdx.x;
    const int h = blockIdx.y, tid = threadIdx.x;
    if (c0 + 1 >= nc) return;
    const int64_t edge = piece_start(c0 + 1, T, nc);
    const Unit x = unit_at(L, L.pref, edge);
    if (x.t0 >= edge || piece_of(x.t0, T, nc) != c0) return;
    const int g = x.u / L.HB, h0 = g * L.G + (x.u % L.HB) * L.GB;
    if (h >= min(L.GB, (g + 1) * L.G - h0)) return;
    const int n = static_cast<int>(piece_of(x.t1 - 1, T, nc) - c0 + 1);
    auto slot = [&](int i) { return (c0 + i) * 2 + (i == 0 ? 1 : 0); };
    float m = -INFINITY;
    for (int i = tid; i < n; i += kJoinThreads) m = fmaxf(m, L.part_ml[(slot(i) * L.GB + h) * 2]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) s_red[0][tid >> 5] = m;
    __syncthreads();
    for (int w = 0; w < kJoinThreads / 32; ++w) m = fmaxf(m, s_red[0][w]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int i = tid; i < n; i += kJoinThreads) {
        const float w = exp2f((L.part_ml[(slot(i) * L.GB + h) * 2] - ref) * kLog2e);
        s_w[i] = w;
        l += w * L.part_ml[(slot(i) * L.GB + h) * 2 + 1];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if ((tid & 31) == 0) s_red[1][tid >> 5] = l;
    __syncthreads();
    l = 0.f;
    for (int w = 0; w < kJoinThreads / 32; ++w) l += s_red[1][w];
    if (tid == 0 && L.lse != nullptr) L.lse[static_cast<int64_t>(x.b) * L.H + h0 + h] = m + logf(l);
    if (tid >= L.D) return;
    float acc = 0.f;
#pragma unroll 8
    for (int i = 0; i < n; ++i) acc = fmaf(s_w[i], L.part_acc[(slot(i) * L.GB + h) * L.D + tid], acc);
    store_out(L, x.b, h0 + h, tid, l == 0.f ? 0.f : acc / l * value_scale(L, g));
}

// ---- CUDA-core kernel: every type, head dim and layout ------------------------
//
// LPK lanes share a key, four elements each, so a warp holds 32 / LPK keys at
// a time. A lane's partial products for GB heads are summed over its LPK
// lanes by halving exchanges that leave head (lane mod GB) with each lane:
// GB - 1 + log2(LPK / GB) shuffles for GB sums instead of GB log2(LPK).
// About 90 instructions per key of 8 heads, and its loads go through registers.
// 16 sequences of 8192 keys, 32/8 heads: fp32 heads of 128 297 us (3.6 TB/s),
// bf16 heads of 80 and 96 600 us (0.6 TB/s), of 32 172 us (0.8), E4M3 heads of
// 80 533 us (0.3), bf16 heads of 128 in pages of 5 598 us (0.9). So it serves
// what the tensor-core kernel does not take (fp32, other head dims, unaligned
// rows and pages that are no multiple of 8).
template <int GB, int LPK>
__device__ __forceinline__ float sum_heads(float (&x)[GB], int lane) {
    int width = LPK;
#pragma unroll
    for (int n = GB; n > 1; n >>= 1) {
        width = n >> 1;
        const bool up = (lane & width) != 0;
#pragma unroll
        for (int i = 0; i < n / 2; ++i) {
            const float give = up ? x[i] : x[i + n / 2];
            const float keep = up ? x[i + n / 2] : x[i];
            x[i] = keep + __shfl_xor_sync(0xffffffffu, give, width);
        }
    }
    float r = x[0];
#pragma unroll
    for (int o = GB; o < LPK; o <<= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    return r;
}

template <int DT, int GB, int LPK, bool VEC>
__global__ void __launch_bounds__(kThreads) paged_simt_kernel(const __grid_constant__ PagedAttnLaunch L) {
    constexpr int DP = LPK * 4, KP = 32 / LPK, STEPS = LPK < 4 ? LPK : 4;  // keys per chunk: STEPS * KP
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Left s_left[2 * kWarps];
    __shared__ int s_sums[kWarps];
    Join J;
    J.acc[0] = reinterpret_cast<float*>(smem);
    J.acc[1] = J.acc[0] + GB * DP;
    J.stride[0] = J.stride[1] = 2 * GB * DP;
    J.ml = J.acc[0] + 2 * kWarps * GB * DP;
    J.left = s_left;
    int* pref = reinterpret_cast<int*>(J.ml + 2 * kWarps * GB * 2);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x < 2 * kWarps) s_left[threadIdx.x].valid = 0;
    tile_prefix(L, pref, s_sums);
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= L.B; b += kThreads) L.pref[b] = pref[b];
    write_empty(L, pref);
    const int64_t T = static_cast<int64_t>(pref[L.B]) * L.U;
    const int64_t nc = pieces(T, L.n_cta);
    if (static_cast<int64_t>(blockIdx.x) >= nc) return;
    const int64_t ca = piece_start(blockIdx.x, T, nc), cz = piece_start(blockIdx.x + 1, T, nc);
    int64_t t = ca + (cz - ca) * warp / kWarps;
    const int64_t a = t, z = ca + (cz - ca) * (warp + 1) / kWarps;
    const int kg = lane / LPK, c0 = (lane & (LPK - 1)) * 4;
    for (Unit x = t < z ? unit_at(L, pref, t) : Unit{0, 0, z, z}; x.t0 < z; x = unit_after(L, pref, x)) {
        if (t < x.t0) t = x.t0;
        const int64_t tz = x.t1 < z ? x.t1 : z;
        const int g = x.u / L.HB, h0 = g * L.G + (x.u % L.HB) * GB;
        const int heads = min(GB, (g + 1) * L.G - h0);
        const int64_t row = table_row(L, x.b);
        const int len = seq_length(L, x.b);
        float4 q[GB], acc[GB];
        const float qs = L.scale * (L.k_scale != nullptr ? L.k_scale[g] : 1.f);
#pragma unroll
        for (int h = 0; h < GB; ++h) {
            acc[h] = make_float4(0.f, 0.f, 0.f, 0.f);
            float e[4] = {0.f, 0.f, 0.f, 0.f};
            if (h < heads)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c0 + i < L.D)
                        e[i] = qs * load_as_f32(L.q, x.b * L.qs[0] + (h0 + h) * L.qs[1] + c0 + i, L.q_dtype);
            q[h] = make_float4(e[0], e[1], e[2], e[3]);
        }
        float m = -INFINITY, l = 0.f;  // of head lane mod GB
        for (; t < tz; ++t) {
            // lane i looks key i of the tile up
            const int key = static_cast<int>(t - x.t0) * kTile + lane;
            int page = -1, off = 0;
            float add = 0.f;
            if (key < len) {
                page = L.table[row * L.table_ld + key / L.page];
                off = key % L.page;
                if (page < 0 || page >= L.P) {
                    record_error(L.status, ADA_ERR_INVALID);
                    page = -1;
                } else if (L.mask.data != nullptr && key < L.mask_len) {
                    const float mv = load_as_f32(L.mask.data, x.b * L.mask.s[0] + key * L.mask.s[1], L.mask.dtype);
                    if (L.mask.dtype == ADA_BOOL ? mv == 0.f : mv == -INFINITY) page = -1;
                    else if (L.mask.dtype != ADA_BOOL) add = mv;
                }
            }
#pragma unroll 1
            for (int chunk = 0; chunk < LPK; chunk += STEPS) {
                if (static_cast<int>(t - x.t0) * kTile + chunk * KP >= len) break;
                float4 kx[STEPS], vx[STEPS];
                bool on[STEPS];
                float av[STEPS];
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const int src = (chunk + i) * KP + kg;
                    const int64_t pg = __shfl_sync(0xffffffffu, page, src);
                    const int64_t po = __shfl_sync(0xffffffffu, off, src);
                    av[i] = __shfl_sync(0xffffffffu, add, src);
                    on[i] = pg >= 0;
                    kx[i] = vx[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (on[i]) {
                        kx[i] = load4<DT, VEC>(L.k, pg * L.ks[0] + g * L.ks[1] + po * L.ks[2], c0, L.D);
                        vx[i] = load4<DT, VEC>(L.v, pg * L.vs[0] + g * L.vs[1] + po * L.vs[2], c0, L.D);
                    }
                }
                float s[STEPS], top = -INFINITY;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    float part[GB];
#pragma unroll
                    for (int h = 0; h < GB; ++h)
                        part[h] = fmaf(q[h].x, kx[i].x, fmaf(q[h].y, kx[i].y, fmaf(q[h].z, kx[i].z, q[h].w * kx[i].w)));
                    const float dot = sum_heads<GB, LPK>(part, lane);
                    s[i] = on[i] ? dot + av[i] : -INFINITY;
                    top = fmaxf(top, s[i]);
                }
#pragma unroll
                for (int o = LPK; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float m_new = fmaxf(m, top);
                const float ref = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = exp2f((m - ref) * kLog2e);
                m = m_new;
                l *= alpha;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    s[i] = on[i] ? exp2f((s[i] - ref) * kLog2e) : 0.f;
                    l += s[i];
                }
#pragma unroll
                for (int h = 0; h < GB; ++h) {
                    const int from = kg * LPK + h;
                    const float al = __shfl_sync(0xffffffffu, alpha, from);
                    float4 o = make_float4(acc[h].x * al, acc[h].y * al, acc[h].z * al, acc[h].w * al);
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) {
                        const float p = __shfl_sync(0xffffffffu, s[i], from);
                        o.x = fmaf(p, vx[i].x, o.x);
                        o.y = fmaf(p, vx[i].y, o.y);
                        o.z = fmaf(p, vx[i].z, o.z);
                        o.w = fmaf(p, vx[i].w, o.w);
                    }
                    acc[h] = o;
                }
            }
        }
        // sum over the warp's key groups
#pragma unroll
        for (int o = LPK; o < 32; o <<= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
            for (int h = 0; h < GB; ++h) {
                acc[h].x += __shfl_xor_sync(0xffffffffu, acc[h].x, o);
                acc[h].y += __shfl_xor_sync(0xffffffffu, acc[h].y, o);
                acc[h].z += __shfl_xor_sync(0xffffffffu, acc[h].z, o);
                acc[h].w += __shfl_xor_sync(0xffffffffu, acc[h].w, o);
            }
        }
        const bool whole = x.t0 >= a && x.t1 <= z;
        const int side = x.t0 < a ? 0 : 1, slot = warp * 2 + side;
        const float vs = value_scale(L, g);
#pragma unroll
        for (int h = 0; h < GB; ++h) {
            const float lh = __shfl_sync(0xffffffffu, l, h), mh = __shfl_sync(0xffffffffu, m, h);
            if (h >= heads) continue;
            const float o[4] = {acc[h].x, acc[h].y, acc[h].z, acc[h].w};
            if (whole) {
                if (kg == 0)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (c0 + i < L.D) store_out(L, x.b, h0 + h, c0 + i, lh == 0.f ? 0.f : o[i] / lh * vs);
                if (lane == 0 && L.lse != nullptr) L.lse[static_cast<int64_t>(x.b) * L.H + h0 + h] = mh + logf(lh);
            } else {
                if (kg == 0) *reinterpret_cast<float4*>(J.part(warp, side) + h * DP + c0) = acc[h];
                if (lane == 0) {
                    J.ml[(slot * GB + h) * 2] = mh;
                    J.ml[(slot * GB + h) * 2 + 1] = lh;
                }
            }
        }
        if (!whole && lane == 0) s_left[slot] = Left{1, x.b, x.u, x.t0, x.t1};
        __syncwarp();
    }
    __syncthreads();
    join_block<kWarps, GB, DP>(L, J, ca, cz);
}

template <int DT, int GB, int LPK, bool VEC>
int launch_simt(const PagedAttnLaunch& L, cudaStream_t stream) {
    const size_t smem = (2 * kWarps * GB * (LPK * 4 + 2) + L.B + 1) * sizeof(float);
    if (cudaFuncSetAttribute(paged_simt_kernel<DT, GB, LPK, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem)) != cudaSuccess)
        return ADA_ERR_LAUNCH;
    paged_simt_kernel<DT, GB, LPK, VEC><<<static_cast<unsigned>(L.n_cta), kThreads, smem, stream>>>(L);
    return cudaGetLastError() == cudaSuccess ? ADA_OK : ADA_ERR_LAUNCH;
}

template <int DT, int GB>
int launch_simt_dt(const PagedAttnLaunch& L, cudaStream_t stream) {
    if (!L.vec) return L.D <= 32 ? launch_simt<DT, GB, 8, false>(L, stream) : launch_simt<DT, GB, 32, false>(L, stream);
    if (L.D <= 32) return launch_simt<DT, GB, 8, true>(L, stream);
    if (L.D <= 64) return launch_simt<DT, GB, 16, true>(L, stream);
    return launch_simt<DT, GB, 32, true>(L, stream);
}

template <int DT>
int launch_simt_gb(const PagedAttnLaunch& L, cudaStream_t stream) {
    switch (L.GB) {
        case 1: return launch_simt_dt<DT, 1>(L, stream);
        case 2: return launch_simt_dt<DT, 2>(L, stream);
        case 4: return launch_simt_dt<DT, 4>(L, stream);
        default: return launch_simt_dt<DT, 8>(L, stream);
    }
}


// ---- tensor-core kernel: 16-bit and 8-bit pages, head dims 64 and 128 ----------
//
// Query heads of a group are few (8, or 16 with NT = 2), so they take the
// narrow side of the warp-level products: S^T = K q^T is 16 keys x 8 heads and
// O^T += V^T P^T is 16 elements x 8 heads per instruction (m16n8k16), where
// padding the heads to a 128-row tile would leave most of it empty. Scores
// come out with a key per row; an 8 x 8 transpose in registers (movmatrix)
// turns P into the next product's operand. P enters as two 16-bit parts
// hi + lo: 16 bits of it for bf16, 22 for fp16. fp16 ends at 2^-24, so there p
// carries a factor 2^15 (p <= 2^15 fits) until the sums leave the warp, and what
// is lost of a p is at most 2^-40 of the largest: without it a tail 17 below an
// attention sink's score, whose own value is near 0, came out as nothing.
// 8-bit pages become fp16 operands in registers: E4M3 values are fp16
// values, q is scaled into fp16's range by a power of two per head (elements
// below 2^-14 of the head's largest lose bits to fp16's end). The order
// of elements within a head is free as long as K and q agree on it, and V's
// with the output, so 4 consecutive bytes of a row serve two k positions.
//
// Every warp runs alone: it requests its own tiles by TMA, STAGES ahead (also
// across units), into its own ring, and no barrier is shared between warps
// until the join at the end. One CTA per SM with the stages that fit beside the
// join: 192 KB of tiles in flight, 128 KB for 8-bit heads of 128 and for wide
// groups of heads of 128 (their third stage misses the space by little).
// Measured: 131071 keys of 8 heads of 128 in fp16 (537 MB) 102 us a call, 5.3 TB/s
// (82 us at the copy rate); 64 sequences up to 16384 keys in E4M3 (1.07 GB)
// 190 us, 5.7 TB/s; the CUDA-core kernel above took 541 us and 2.02 ms. Shorter
// units cost more each: 1000 sequences of 160 keys, 32/8 heads of 128, 178 us in
// bf16 (3.7 TB/s) and 121 us in E4M3 (2.7); 128 heads over 8, 16 sequences of 8192
// keys, 160 us (3.4 TB/s) and 121 us (2.2) where 32 over 8 take 125 and 78.
template <int KIND, int D, int NT>  // KIND: 0 bf16, 1 fp16, 2 E4M3
struct TcCfg {
    static constexpr int EB = KIND == 2 ? 1 : 2;
    static constexpr int RB = D * EB < 128 ? D * EB : 128;   // bytes of a box row, and of its swizzle
    static constexpr int NBOX = D * EB / RB;
    static constexpr int HALF = kTile * D * EB;              // K or V bytes of a tile
    static constexpr int TILE = 2 * HALF;
    static constexpr int WARPS = TILE >= 16384 ? 4 : 8;      // (8-bit heads of 128: 10, with the same 2 stages, 3 % slower)
    static constexpr int STAGES = TILE >= 8192 ? 3 : 6;      // at most; fewer when the rest needs the space
    static constexpr int GB = 8 * NT;
    static constexpr int PART = GB * D;                      // floats a warp leaves per slot
    // the exponent that p carries on its way through fp16 operands
    static constexpr float LIFT = KIND == 0 ? 0.f : 15.f;
    static constexpr float DROP = KIND == 0 ? 1.f : 1.f / 32768.f;
    // beside the ring: slot 0 of the join (slot 1 lies in the drained ring) and (m, l)
    static constexpr int BESIDE = WARPS * (PART * 4 + 2 * GB * 2 * 4);
};

template <int KIND>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (KIND == 0)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Four E4M3 bytes as two fp16 pairs.
__device__ __forceinline__ void e4m3_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
}
// p as a 16-bit pair hi + lo of the operand type.
template <int KIND>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    if constexpr (KIND == 0) {
        hi = pack_bf16x2(x, y);
        lo = pack_bf16x2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xFFFF0000u));
    } else {
        hi = pack_f16x2(x, y);
        float a, b;
        unpack_f16x2(hi, a, b);
        lo = pack_f16x2(x - a, y - b);
    }
}

template <int KIND, int D, int NT>
__global__ void __launch_bounds__(TcCfg<KIND, D, NT>::WARPS * 32, 1)
    paged_tc_kernel(const __grid_constant__ PagedAttnLaunch L) {
    using C = TcCfg<KIND, D, NT>;
    constexpr int EB = C::EB, RB = C::RB, W = C::WARPS, SMAX = C::STAGES, GB = C::GB;
    const int S = L.stages, ring_bytes = S * C::TILE;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ Left s_left[2 * W];
    __shared__ int s_sums[W];
    __shared__ __align__(8) uint64_t s_full[W * SMAX];
    __shared__ uint32_t s_ok[W * SMAX];
    __shared__ int s_abort;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint8_t* ring = smem + warp * ring_bytes;
    Join J;
    J.acc[0] = reinterpret_cast<float*>(smem + W * ring_bytes);
    J.stride[0] = C::PART;
    J.acc[1] = reinterpret_cast<float*>(smem);
    J.stride[1] = ring_bytes / 4;
    J.ml = J.acc[0] + W * C::PART;
    J.left = s_left;
    int* pref = reinterpret_cast<int*>(J.ml + W * 2 * GB * 2);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x < 2 * W) s_left[threadIdx.x].valid = 0;
    if (threadIdx.x == 0) s_abort = 0;
    if (lane == 0)
        for (int i = 0; i < S; ++i) mbar_init(smem_u32(&s_full[warp * SMAX + i]), 1);
    fence_mbar_init();
    tile_prefix(L, pref, s_sums);
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= L.B; b += W * 32) L.pref[b] = pref[b];
    write_empty(L, pref);
    const int64_t T = static_cast<int64_t>(pref[L.B]) * L.U;
    const int64_t nc = pieces(T, L.n_cta);
    if (static_cast<int64_t>(blockIdx.x) >= nc) return;
    const int64_t ca = piece_start(blockIdx.x, T, nc), cz = piece_start(blockIdx.x + 1, T, nc);
    const int64_t a = ca + (cz - ca) * warp / W, z = ca + (cz - ca) * (warp + 1) / W;

    // launch fields that the loop uses (barrier asm would have them reloaded)
    const uint32_t page = static_cast<uint32_t>(L.page), page_inv = L.page_inv;
    auto page_of = [&](int key) {  // key / page: the estimate is at most one too large
        const uint32_t q = page_inv == 0 ? static_cast<uint32_t>(key) : __umulhi(static_cast<uint32_t>(key), page_inv);
        return q - (q * page > static_cast<uint32_t>(key) ? 1u : 0u);
    };
    const int CK = L.chunk, G = L.G, HB = L.HB, mask_len = static_cast<int>(L.mask_len);
    const int64_t P = L.P, table_ld = L.table_ld;
    const int32_t* table = L.table;
    const void* mask = L.mask.data;
    const int mask_type = L.mask.dtype;
    unsigned int* status = L.status;
    const uint64_t limit = L.timeout_ns;
    const uint32_t bar0 = smem_u32(&s_full[warp * SMAX]), ring0 = smem_u32(ring);
    volatile int* abort_flag = &s_abort;

    // ---- requests: lane i issues box i of a tile (chunk, K or V, half of the row)
    const int nch = kTile / CK;
    const int my_chunk = lane % nch, my_v = (lane / nch) & 1, my_box = lane / (2 * nch);
    const bool issues = my_box < C::NBOX;
    int64_t pt = a, prow = 0;
    Unit px{};
    int asked = 0, used = 0;  // tiles
    int plen = 0, pid = -1, pg = 0;
    auto look_up = [&]() {  // unit of tile pt and this lane's page of it
        pid = -1;
        if (pt == px.t1) {
            const int b = px.b;
            px = unit_after(L, pref, px);
            pt = px.t0;
            if (pt < z && px.b != b) {
                prow = table_row(L, px.b);
                plen = seq_length(L, px.b);
            }
            pg = px.u / HB;
        }
        if (pt >= z) return;
        const int key = static_cast<int>(pt - px.t0) * kTile + my_chunk * CK;
        if (issues && key < plen) pid = table[prow * table_ld + page_of(key)];
    };
    auto request = [&](int slot) {
        const int key = static_cast<int>(pt - px.t0) * kTile + my_chunk * CK;
        bool ok = issues && key < plen;
        if (ok && (pid < 0 || pid >= P)) {
            record_error(status, ADA_ERR_INVALID);
            ok = false;
        }
        const uint32_t who = __ballot_sync(0xffffffffu, ok);
        const uint32_t bar = bar0 + slot * 8;
        if (lane == 0) {
            s_ok[warp * SMAX + slot] = who;  // lanes 0 .. nch - 1 are the chunks
            mbar_arrive_expect_tx(bar, __popc(who) * CK * RB);
        }
        __syncwarp();
        if (ok)
            tma_load_4d(ring0 + slot * C::TILE + my_v * C::HALF + my_box * (kTile * RB) + my_chunk * CK * RB,
                        my_v ? &L.tv : &L.tk, bar, my_box * (RB / EB), key - static_cast<int>(page_of(key) * page), pg, pid);
        ++pt;
        ++asked;
        look_up();
    };
    if (a < z) {
        px = unit_at(L, pref, a);
        pt = px.t0 > a ? px.t0 : a;
        prow = table_row(L, px.b);
        plen = seq_length(L, px.b);
        pg = px.u / HB;
        look_up();
    }
    for (int i = 0; i < S && pt < z; ++i) request(i);

    // ---- this lane's part of every fragment: keys / elements g and g + 8, heads 2 t and 2 t + 1
    const int fg = lane >> 2, ft = lane & 3;
    // ldmatrix row addresses: K rows (lane & 15), 16-byte column lane >> 4; V rows and columns as the kind needs
    const int l7 = lane & 7;
    auto swz = [](int row, int col) { return RB == 128 ? (col ^ (row & 7)) : (col ^ ((row >> 1) & 3)); };
    const uint32_t k_row = static_cast<uint32_t>((lane & 15) * RB);
    const int k_col = lane >> 4;
    const int v_key = KIND == 2 ? (lane & 15) : ((lane >> 4) * 8 + l7);
    const int v_col = KIND == 2 ? (lane >> 4) : ((lane >> 3) & 1);

    // Scores are in base 2 unless a float mask is added to them (its lowest
    // values times log2 e would be infinite).
    const bool biased = mask != nullptr && mask_type != ADA_BOOL;
    const float unit = biased ? kLog2e : 1.f;

    int64_t t = a;
    int slot = 0;             // the ring's slot of tile t and the parity of its barrier
    uint32_t parity = 0;
    bool alive = true;
    auto next = [&]() {
        __syncwarp();  // the slot is read
        ++used;
        if (pt < z) request(slot);
        if (++slot == S) {
            slot = 0;
            parity ^= 1u;
        }
    };
    Unit x{-1, 0, z, z};
    if (a < z) x = unit_at(L, pref, a);
    int len = 0;
    for (int len_of = -1; x.t0 < z; x = unit_after(L, pref, x)) {
        if (t < x.t0) t = x.t0;
        const int64_t tz = x.t1 < z ? x.t1 : z;
        const int g = x.u / HB, h0 = g * G + (x.u % HB) * GB;
        const int heads = min(GB, (g + 1) * G - h0);
        if (x.b != len_of) {
            len = seq_length(L, x.b);
            len_of = x.b;
        }
        const float vs = value_scale(L, g);
        const int64_t mrow = x.b * L.mask.s[0], mcol = L.mask.s[1];
        // q^T: element pairs of head fg (of each tile of 8 heads)
        uint32_t qf[D / 16][NT][2];
        float qs[NT][2];
        {
            const float base = L.scale * (L.k_scale != nullptr ? L.k_scale[g] : 1.f) * (biased ? 1.f : kLog2e);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const bool on = n * 8 + fg < heads;
                const uint32_t* qr = reinterpret_cast<const uint32_t*>(
                    static_cast<const uint16_t*>(L.q) + x.b * L.qs[0] + (h0 + n * 8 + fg) * L.qs[1]);
                if constexpr (KIND != 2) {
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) {
                        qf[s][n][0] = on ? qr[s * 8 + ft] : 0u;
                        qf[s][n][1] = on ? qr[s * 8 + ft + 4] : 0u;
                    }
                    qs[n][0] = qs[n][1] = base;
                } else {
                    float top = 0.f;
                    const bool half = L.q_dtype == ADA_F16;
                    auto pair = [&](uint32_t w, float& lo, float& hi) {
                        if (half) {
                            unpack_f16x2(w, lo, hi);
                        } else {
                            lo = __uint_as_float(w << 16);
                            hi = __uint_as_float(w & 0xFFFF0000u);
                        }
                    };
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            qf[s][n][i] = on ? qr[s * 8 + 2 * ft + i] : 0u;
                            float lo, hi;
                            pair(qf[s][n][i], lo, hi);
                            top = fmaxf(top, fmaxf(fabsf(lo), fabsf(hi)));
                        }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    // 2^-e with max |q| 2^-e in [1, 2); none for 0, infinity and what 2^-e does not fit
                    const uint32_t e = (__float_as_uint(top) >> 23) & 0xFFu;
                    const bool fits = e >= 1 && e <= 253;
                    const float down = fits ? __uint_as_float((254u - e) << 23) : 1.f;
                    const float up = fits ? __uint_as_float(e << 23) : 1.f;
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float lo, hi;
                            pair(qf[s][n][i], lo, hi);
                            qf[s][n][i] = pack_f16x2(lo * down, hi * down);
                        }
                    qs[n][0] = base * __shfl_sync(0xffffffffu, up, 8 * ft);
                    qs[n][1] = base * __shfl_sync(0xffffffffu, up, 8 * ft + 4);
                }
            }
        }
        float o[D / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
        }
        for (; t < tz; ++t) {
            const int key0 = static_cast<int>(t - x.t0) * kTile;
            // lane i: key i's mask
            bool open = key0 + lane < len;
            float add = 0.f;
            if (mask != nullptr && open && key0 + lane < mask_len) {
                const float mv = load_as_f32(mask, mrow + (key0 + lane) * mcol, mask_type);
                if (mask_type == ADA_BOOL) {
                    open = mv != 0.f;
                } else {
                    open = mv != -INFINITY;
                    add = open ? mv : 0.f;
                }
            }
            if (!mbar_wait_warp(bar0 + slot * 8, parity, abort_flag, limit, status)) {
                alive = false;
                break;
            }
            open = open && ((s_ok[warp * SMAX + slot] >> (lane / CK)) & 1u);
            const uint32_t vis = __ballot_sync(0xffffffffu, open);
            if (vis == 0u) {  // nothing to see in this tile
                next();
                continue;
            }
            const uint32_t kb = ring0 + slot * C::TILE, vb = kb + C::HALF;
            // S^T = K q^T
            float c[2][NT][4];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[r][n][e] = 0.f;
            if constexpr (KIND != 2) {
#pragma unroll
                for (int s = 0; s < D / 16; ++s)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        uint32_t f[4];
                        const int col = (s & 3) * 2 + k_col;
                        ldsm4(f, kb + (s >> 2) * (kTile * RB) + r * 16 * RB + k_row + swz(lane & 15, col) * 16);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_16816<KIND>(c[r][n], f, qf[s][n][0], qf[s][n][1]);
                    }
            } else {
#pragma unroll
                for (int s = 0; s < D / 32; ++s)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        uint32_t w[4], f0[4], f1[4];
                        ldsm4(w, kb + r * 16 * RB + k_row + swz(lane & 15, 2 * s + k_col) * 16);
                        e4m3_to_f16(w[0], f0[0], f0[2]);
                        e4m3_to_f16(w[1], f0[1], f0[3]);
                        e4m3_to_f16(w[2], f1[0], f1[2]);
                        e4m3_to_f16(w[3], f1[1], f1[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma_16816<KIND>(c[r][n], f0, qf[2 * s][n][0], qf[2 * s][n][1]);
                            mma_16816<KIND>(c[r][n], f1, qf[2 * s + 1][n][0], qf[2 * s + 1][n][1]);
                        }
                    }
            }
            // scores, their maximum over the tile, probabilities
            if (vis == 0xffffffffu && !biased) {
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[r][n][e] *= qs[n][e & 1];
            } else {
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int key = r * 16 + j * 8 + fg;
                        const float av = __shfl_sync(0xffffffffu, add, key);
                        const bool on = (vis >> key) & 1u;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                c[r][n][2 * j + e] = on ? fmaf(c[r][n][2 * j + e], qs[n][e], av) : -INFINITY;
                    }
                // a hidden key's values are zeroed, whatever they hold: half a warp per row
                for (uint32_t hidden = ~vis; hidden != 0; hidden &= hidden - 1) {
                    const int key = __ffs(hidden) - 1;
#pragma unroll
                    for (int x4 = 0; x4 < C::NBOX; ++x4)
                        if (lane < RB / 4)
                            *reinterpret_cast<uint32_t*>(ring + slot * C::TILE + C::HALF + x4 * (kTile * RB) + key * RB +
                                                         lane * 4) = 0u;
                }
                fence_proxy_async_smem();  // before the slot's next tile arrives
                __syncwarp();
            }
            bool moved = false;
            uint32_t ph[2][NT][2], pl[2][NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float ref[2], alpha[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = max3f(max3f(c[0][n][e], c[0][n][2 + e], c[1][n][e]), c[1][n][2 + e], -INFINITY);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float mn = fmaxf(m[n][e], top);
                    ref[e] = mn == -INFINITY ? 0.f : mn;
                    moved = moved || mn != m[n][e];
                    alpha[e] = fast_exp2((m[n][e] - ref[e]) * unit);
                    m[n][e] = mn;
                    l[n][e] *= alpha[e];
                }
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float p0 = fast_exp2(fmaf(c[r][n][2 * j] - ref[0], unit, C::LIFT));
                        const float p1 = fast_exp2(fmaf(c[r][n][2 * j + 1] - ref[1], unit, C::LIFT));
                        l[n][0] += p0;
                        l[n][1] += p1;
                        uint32_t hi, lo;
                        split2<KIND>(p0, p1, hi, lo);
                        ph[r][n][j] = transpose8x8(hi);
                        pl[r][n][j] = transpose8x8(lo);
                    }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        o[i][n][0] *= alpha[0];
                        o[i][n][1] *= alpha[1];
                        o[i][n][2] *= alpha[0];
                        o[i][n][3] *= alpha[1];
                    }
                }
                moved = false;
            }
            // O^T += V^T P^T
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                auto product = [&](int i, uint32_t (&f)[4]) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_16816<KIND>(o[i][n], f, ph[r][n][0], ph[r][n][1]);
                        mma_16816<KIND>(o[i][n], f, pl[r][n][0], pl[r][n][1]);
                    }
                };
                if constexpr (KIND != 2) {
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        uint32_t f[4];
                        const int col = (i & 3) * 2 + v_col;
                        ldsm4_t(f, vb + (i >> 2) * (kTile * RB) + (r * 16 + v_key) * RB + swz(v_key, col) * 16);
                        product(i, f);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        uint32_t w[4], f0[4], f1[4];
                        ldsm4_t(w, vb + (r * 16 + v_key) * RB + swz(v_key, 2 * i + v_col) * 16);
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = __byte_perm(w[e], 0, 0x3120);
                        e4m3_to_f16(w[0], f0[0], f0[1]);
                        e4m3_to_f16(w[1], f0[2], f0[3]);
                        e4m3_to_f16(w[2], f1[0], f1[1]);
                        e4m3_to_f16(w[3], f1[2], f1[3]);
                        product(2 * i, f0);
                        product(2 * i + 1, f1);
                    }
                }
            }
            next();
        }
        if (!alive) break;
        const bool whole = x.t0 >= a && x.t1 <= z;
        const int side = x.t0 < a ? 0 : 1, left = warp * 2 + side;
        float* part = J.part(warp, side);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[n][e];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                sum *= C::DROP;
                const int h = n * 8 + 2 * ft + e;
                if (h >= heads) continue;
                const float inv = whole ? (sum == 0.f ? 0.f : vs / sum) : 1.f;
                const float mn = biased ? m[n][e] : m[n][e] * kLn2;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int d = KIND == 2 ? i * 16 + 2 * fg + j : i * 16 + fg + 8 * j;
                        const float v = sum == 0.f ? 0.f : o[i][n][2 * j + e] * C::DROP * inv;
                        if (whole) store_out(L, x.b, h0 + h, d, v);
                        else part[h * D + d] = v;
                    }
                if (fg == 0) {
                    if (whole) {
                        if (L.lse != nullptr) L.lse[static_cast<int64_t>(x.b) * L.H + h0 + h] = mn + logf(sum);
                    } else {
                        J.ml[(left * GB + h) * 2] = mn;
                        J.ml[(left * GB + h) * 2 + 1] = sum;
                    }
                }
            }
        if (!whole && lane == 0) s_left[left] = Left{1, x.b, x.u, x.t0, x.t1};
        __syncwarp();
    }
    if (!alive) {  // a wait ran out (recorded): the tiles still requested are awaited, then the block gives up
        for (; asked > used; ++used) {
            const uint64_t t0 = globaltimer_ns();
            while (!mbar_try_wait(bar0 + slot * 8, parity) && globaltimer_ns() - t0 < limit) {}
            if (++slot == S) {
                slot = 0;
                parity ^= 1u;
            }
        }
    }
    __syncthreads();
    if (s_abort) return;
    join_block<W, GB, D>(L, J, ca, cz);
}

template <int KIND, int D, int NT>
int launch_tc(const PagedAttnLaunch& launch, cudaStream_t stream) {
    using C = TcCfg<KIND, D, NT>;
    constexpr int kSpace = 227 * 1024 - 2048 - 1024;  // less the static shared memory and the alignment
    PagedAttnLaunch L = launch;
    const int beside = C::BESIDE + (L.B + 1) * 4;
    L.stages = (kSpace - beside) / (C::WARPS * C::TILE);
    if (L.stages > C::STAGES) L.stages = C::STAGES;
    const size_t smem = static_cast<size_t>(L.stages) * C::WARPS * C::TILE + beside + 1024;
    if (cudaFuncSetAttribute(paged_tc_kernel<KIND, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem)) != cudaSuccess)
        return ADA_ERR_LAUNCH;
    paged_tc_kernel<KIND, D, NT><<<static_cast<unsigned>(L.n_cta), C::WARPS * 32, smem, stream>>>(L);
    return cudaGetLastError() == cudaSuccess ? ADA_OK : ADA_ERR_LAUNCH;
}

template <int KIND>
int launch_tc_kind(const PagedAttnLaunch& L, cudaStream_t stream) {
    if (L.D == 64) return L.GB == 8 ? launch_tc<KIND, 64, 1>(L, stream) : launch_tc<KIND, 64, 2>(L, stream);
    return L.GB == 8 ? launch_tc<KIND, 128, 1>(L, stream) : launch_tc<KIND, 128, 2>(L, stream);
}

}  // namespace

int launch_paged_attn(const PagedAttnLaunch& L, cudaStream_t stream) {
    int rc;
    switch (L.kv_dtype) {
        case ADA_F32: rc = launch_simt_gb<ADA_F32>(L, stream); break;
        case ADA_F16: rc = L.tc ? launch_tc_kind<1>(L, stream) : launch_simt_gb<ADA_F16>(L, stream); break;
        case ADA_BF16: rc = L.tc ? launch_tc_kind<0>(L, stream) : launch_simt_gb<ADA_BF16>(L, stream); break;
        case ADA_E4M3: rc = L.tc ? launch_tc_kind<2>(L, stream) : launch_simt_gb<ADA_E4M3>(L, stream); break;
        default: return ADA_ERR_DTYPE;
    }
    if (rc || L.n_cta < 2) return rc;
    // The join starts while the last pieces run and waits for them on the device.
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(L.n_cta - 1), static_cast<unsigned>(L.GB < L.G ? L.GB : L.G));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_join_kernel, L) == cudaSuccess ? ADA_OK : ADA_ERR_LAUNCH;
}

}  // namespace ada
