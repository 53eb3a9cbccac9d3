// Attention of one new token per sequence over a paged key-value cache.
//
// For sequence b (table row r), query head h of key/value head g = h / G:
//   s_j = scale * ks_g * (q_h . k_j) + add_j      over visible keys j < len_b
//   o_h = vs_g * sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j
// (ks, vs: the scales of an 8-bit cache; add: a float key mask). A key hidden
// by a bool mask or by -inf is never read, so what its page holds does not
// matter; a sequence with no visible key gives zeros and lse = -inf.
//
// Each key and value is read once per block of up to 8 query heads and costs 4
// multiply-adds per head and element: the cache's bytes bound the operator.
// So the work is split evenly over the cache, not over sequences: the tiles of
// 32 keys of all (sequence, head block) units stand in one line, CTA c takes
// the c-th equal piece of it and each of its warps an equal piece of that. A
// unit that lies in one warp's piece is finished there. Pieces of a unit that
// spans warps are joined in shared memory (each with its running maximum m,
// sum l and unnormalised accumulator), pieces that span CTAs are joined by a
// second kernel. The split depends on the lengths alone, so results repeat.
#include "ada_common.cuh"
#include "ada_internal.h"

namespace ada {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;       // keys per tile
constexpr float kLog2e = 1.4426950408889634f;

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

// pref[b] = tiles of the sequences before b, pref[B] = all (every thread of the block calls it).
__device__ void tile_prefix(const PagedAttnLaunch& L, int* pref, int* warp_sums) {
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
    const int per = (L.B + nt - 1) / nt;
    const int b0 = min(tid * per, L.B), b1 = min(b0 + per, L.B);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
        const int n = (seq_length(L, b) + kTile - 1) / kTile;
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
    x.t0 = first + static_cast<int64_t>(x.u) * n;
    x.t1 = x.t0 + n;
    return x;
}

// The CTAs that take part and the piece of CTA c: [c T / n, (c + 1) T / n).
__device__ __forceinline__ int64_t pieces(int64_t T, int64_t most) { return T < most ? T : most; }
__device__ __forceinline__ int64_t piece_start(int64_t c, int64_t T, int64_t n) { return c * T / n; }
// The piece that holds tile t.
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

struct Join {
    float* acc;   // [kWarps][2][GB][DP]
    float* ml;    // [kWarps][2][GB][2]
    Left* left;   // [kWarps][2]
};

// Joins the pieces that the block's warps left. A unit inside the block's own
// piece [a, z) is finished; another goes to the workspace, slot 0 / 1 as above.
template <int GB, int DP>
__device__ void join_block(const PagedAttnLaunch& L, const Join& J, int64_t a, int64_t z) {
    constexpr int NE = 2 * kWarps;
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
        for (int i = threadIdx.x; i < heads * DP; i += kThreads) {
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
                acc += w * J.acc[(k * GB + h) * DP + d];
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

// Joins what CTAs left of each unit that spans several, and writes the units of empty sequences.
__global__ void __launch_bounds__(kThreads) paged_join_kernel(const __grid_constant__ PagedAttnLaunch L) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t unit = blockIdx.x;
    const int b = static_cast<int>(unit / L.U), u = static_cast<int>(unit % L.U);
    const int g = u / L.HB, h0 = g * L.G + (u % L.HB) * L.GB;
    const int heads = min(L.GB, (g + 1) * L.G - h0);
    const int first = L.pref[b], n = L.pref[b + 1] - first;
    if (n == 0) {
        for (int i = threadIdx.x; i < heads * L.D; i += kThreads) store_out(L, b, h0 + i / L.D, i % L.D, 0.f);
        if (L.lse != nullptr && threadIdx.x < heads) L.lse[static_cast<int64_t>(b) * L.H + h0 + threadIdx.x] = -INFINITY;
        return;
    }
    const int64_t T = static_cast<int64_t>(L.pref[L.B]) * L.U;
    const int64_t nc = pieces(T, L.n_cta);
    const int64_t t0 = static_cast<int64_t>(first) * L.U + static_cast<int64_t>(u) * n;
    const int64_t c0 = piece_of(t0, T, nc), c1 = piece_of(t0 + n - 1, T, nc);
    if (c0 == c1) return;
    const int64_t slot0 = c0 * 2 + 1;  // the unit begins in c0's piece; later CTAs begin inside the unit: slot 0
    for (int i = threadIdx.x; i < heads * L.D; i += kThreads) {
        const int h = i / L.D, d = i - h * L.D;
        float m = -INFINITY;
        for (int64_t c = c0; c <= c1; ++c) {
            const int64_t s = c == c0 ? slot0 : c * 2;
            m = fmaxf(m, L.part_ml[(s * L.GB + h) * 2]);
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float l = 0.f, acc = 0.f;
#pragma unroll 4
        for (int64_t c = c0; c <= c1; ++c) {
            const int64_t s = c == c0 ? slot0 : c * 2;
            const float w = exp2f((L.part_ml[(s * L.GB + h) * 2] - ref) * kLog2e);
            l += w * L.part_ml[(s * L.GB + h) * 2 + 1];
            acc += w * L.part_acc[(s * L.GB + h) * L.D + d];
        }
        store_out(L, b, h0 + h, d, l == 0.f ? 0.f : acc / l * value_scale(L, g));
        if (d == 0 && L.lse != nullptr) L.lse[static_cast<int64_t>(b) * L.H + h0 + h] = m + logf(l);
    }
}

// ---- CUDA-core kernel: every type, head dim and layout ------------------------
//
// LPK lanes share a key, four elements each, so a warp holds 32 / LPK keys at
// a time. A lane's partial products for GB heads are summed over its LPK
// lanes by halving exchanges that leave head (lane mod GB) with each lane:
// GB - 1 + log2(LPK / GB) shuffles for GB sums instead of GB log2(LPK).
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
    J.acc = reinterpret_cast<float*>(smem);
    J.ml = J.acc + 2 * kWarps * GB * DP;
    J.left = s_left;
    int* pref = reinterpret_cast<int*>(J.ml + 2 * kWarps * GB * 2);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x < 2 * kWarps) s_left[threadIdx.x].valid = 0;
    tile_prefix(L, pref, s_sums);
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= L.B; b += kThreads) L.pref[b] = pref[b];
    const int64_t T = static_cast<int64_t>(pref[L.B]) * L.U;
    const int64_t nc = pieces(T, L.n_cta);
    if (static_cast<int64_t>(blockIdx.x) >= nc) return;
    const int64_t ca = piece_start(blockIdx.x, T, nc), cz = piece_start(blockIdx.x + 1, T, nc);
    int64_t t = ca + (cz - ca) * warp / kWarps;
    const int64_t a = t, z = ca + (cz - ca) * (warp + 1) / kWarps;
    const int kg = lane / LPK, c0 = (lane & (LPK - 1)) * 4;
    while (t < z) {
        const Unit x = unit_at(L, pref, t);
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
        const int slot = warp * 2 + (x.t0 < a ? 0 : 1);
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
                if (kg == 0) *reinterpret_cast<float4*>(J.acc + (slot * GB + h) * DP + c0) = acc[h];
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
    join_block<GB, DP>(L, J, ca, cz);
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

}  // namespace

int launch_paged_attn(const PagedAttnLaunch& L, cudaStream_t stream) {
    int rc;
    switch (L.kv_dtype) {
        case ADA_F32: rc = launch_simt_gb<ADA_F32>(L, stream); break;
        case ADA_F16: rc = launch_simt_gb<ADA_F16>(L, stream); break;
        case ADA_BF16: rc = launch_simt_gb<ADA_BF16>(L, stream); break;
        case ADA_E4M3: rc = launch_simt_gb<ADA_E4M3>(L, stream); break;
        default: return ADA_ERR_DTYPE;
    }
    if (rc) return rc;
    // The join starts while the last pieces run and waits for them on the device.
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(L.B) * L.U));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_join_kernel, L) == cudaSuccess ? ADA_OK : ADA_ERR_LAUNCH;
}

}  // namespace ada
