// The paged key-value cache: appending new keys and values, and the page
// operations (reserve, fork, copy, free, compact).
//
// Pages live in one pool. A sequence s holds the pages table[s][0 .. held),
// held = ceil(lens[s] / page); refs[p] counts the sequences that hold page p
// and a page with refs[p] = 0 is free. All of it is device memory and every
// operation is a few launches on the caller's stream: a decoding loop neither
// waits for the host nor leaves a captured graph to allocate. Free pages are
// handed out lowest first, to the sequences of a call in their order, so the
// outcome depends on the arguments alone (integer atomics commute).
//
// What bounds them: append, copy and compact move bytes (HBM); fork, free and
// the allocation touch a few kilobytes (latency: a launch and some dependent
// loads). Measured: prompts up to 4096 tokens into an 8-bit cache 28 us (3.6
// TB/s), 8 prompts of 4096 tokens of 8 heads of 128 bf16 to bf16 51 us (5.2 TB/s),
// heads of 33, element by element, 61 us (1.1 TB/s), copies of 16 sequences (1.1 GB moved) 194 us (5.7 TB/s), two compactions
// of 2.4 GB with their accounting 436 us (5.5 TB/s), a fork, a reserve with
// copies on write and a free of 32 branches 22 us.
#include "ada_common.cuh"
#include "ada_internal.h"

namespace ada {
namespace {

// ---- append --------------------------------------------------------------------

constexpr int kAppendThreads = 256;
constexpr int kAppendUnroll = 2;

// x / s rounded once, for several x: the three-instruction quotient, and the
// plain one for all of them where that leaves the finite numbers (infinities,
// NaN, scales whose reciprocal is none). Checked one by one, the test cost more
// than the quotients: the 8-bit prompt append took 49 us instead of 28.
__device__ __noinline__ float plain_quotient(float x, float s) { return x / s; }
template <int N>
__device__ __forceinline__ void quotients(const float (&x)[N], float s, float inv, float (&q)[N]) {
    float none = 0.f;  // NaN when some q is not finite
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = div_by(x[i], s, inv);
        none = fmaf(q[i], 0.f, none);
    }
    if (none != 0.f) {
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = plain_quotient(x[i], s);
    }
}

// Eight values (or one, VEC = false) of new key/value data on their way to a
// page: copied when the types agree, otherwise divided by the head's scale and
// rounded once to E4M3 (saturating at 448).
template <int SRC, int DST, bool VEC>
struct AppendItem {
    static constexpr int EB = SRC == ADA_F32 ? 4 : 2;
    uint4 w[VEC ? EB / 2 : 1];
    __device__ __forceinline__ void load(const void* src, int64_t at) {
        const uint8_t* a = static_cast<const uint8_t*>(src) + at * EB;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < EB / 2; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(a) + i);
        } else if constexpr (EB == 4) {
            w[0].x = *reinterpret_cast<const uint32_t*>(a);
        } else {
            w[0].x = *reinterpret_cast<const uint16_t*>(a);
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (SRC == ADA_F32) {
            const uint4& v = w[i / 4];
            return __uint_as_float(i % 4 == 0 ? v.x : i % 4 == 1 ? v.y : i % 4 == 2 ? v.z : v.w);
        } else {
            const uint32_t u = i / 2 == 0 ? w[0].x : i / 2 == 1 ? w[0].y : i / 2 == 2 ? w[0].z : w[0].w;
            if constexpr (SRC == ADA_BF16) return __uint_as_float(i % 2 ? u & 0xFFFF0000u : u << 16);
            float lo, hi;
            unpack_f16x2(u, lo, hi);
            return i % 2 ? hi : lo;
        }
    }
    __device__ __forceinline__ void store(void* dst, int64_t at, float s, float inv) const {
        if constexpr (DST != ADA_E4M3) {
            uint8_t* b = static_cast<uint8_t*>(dst) + at * EB;
            if constexpr (VEC) {
#pragma unroll
                for (int i = 0; i < EB / 2; ++i) reinterpret_cast<uint4*>(b)[i] = w[i];
            } else if constexpr (EB == 4) {
                *reinterpret_cast<uint32_t*>(b) = w[0].x;
            } else {
                *reinterpret_cast<uint16_t*>(b) = static_cast<uint16_t>(w[0].x);
            }
        } else if constexpr (VEC) {
            float x[8], v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = value(i);
            quotients(x, s, inv, v);
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(dst) + at) =
                make_uint2(pack_e4m3x4(v[0], v[1], v[2], v[3]), pack_e4m3x4(v[4], v[5], v[6], v[7]));
        } else {
            const float x[1] = {value(0)};
            float v[1];
            quotients(x, s, inv, v);
            static_cast<uint8_t*>(dst)[at] = static_cast<uint8_t>(pack_e4m3x4(v[0], 0.f, 0.f, 0.f) & 0xFFu);
        }
    }
};

// Block (b, chunk): a chunk of sequence b's tokens x heads x elements, of both tensors.
template <int SRC, int DST, bool VEC>
__global__ void __launch_bounds__(kAppendThreads, 4) paged_append_kernel(const __grid_constant__ AppendLaunch L) {
    constexpr int E = VEC ? 8 : 1;
    const int64_t b = blockIdx.x / L.chunks, chunk = blockIdx.x % L.chunks;
    const int64_t r = L.seqs != nullptr ? L.seqs[b] : b;
    bool bad = r < 0 || r >= L.S;
    if (L.seqs != nullptr) {  // a sequence named twice is written by its first row only
        bool twice = false;
        for (int64_t j = threadIdx.x; j < b; j += kAppendThreads) twice |= L.seqs[j] == r;
        bad = __syncthreads_or(twice) || bad;
    }
    int64_t len = 0, n = 0;
    if (!bad) {
        len = L.lens[r];
        n = L.new_tokens != nullptr ? L.new_tokens[b] : L.N;
        bad = n < 0 || n > L.N || len < n || len > L.W * L.page || (L.prompts != 0 && n > 0 && len != n);
    }
    if (bad) {
        if (threadIdx.x == 0) record_error(L.status, ADA_ERR_INVALID);
        return;
    }
    // A thread keeps its place in a token (head and elements) and walks over the
    // tokens, two at a time with all their loads under way: one at a time, the
    // chain table -> data -> store held a prompt's append at 1.9 TB/s.
    const int per = L.D / E, in_token = static_cast<int>(L.Hkv) * per;  // items of a row, of a token
    const int tokens = in_token < kAppendThreads ? kAppendThreads / in_token : 1;  // of a block at a time
    const int lead = static_cast<int>(threadIdx.x) / in_token;
    const int32_t* row = L.table + r * L.table_ld;
    const int first = static_cast<int>(len - n);
    const unsigned page = static_cast<unsigned>(L.page);
    for (int e = static_cast<int>(threadIdx.x) - lead * in_token; lead < tokens && e < in_token;
         e += tokens == 1 ? kAppendThreads : in_token) {
        const int h = e / per, d = (e - h * per) * E;
        const float ks = L.k_scale != nullptr ? L.k_scale[h] : 1.f, vs = L.v_scale != nullptr ? L.v_scale[h] : 1.f;
        const float ki = 1.f / ks, vi = 1.f / vs;
        const int64_t k0 = b * L.ks[0] + h * L.ks[1] + d, v0 = b * L.vs[0] + h * L.vs[1] + d;
        const int64_t kp0 = h * L.kps[1] + d, vp0 = h * L.vps[1] + d;
        const int64_t step = static_cast<int64_t>(L.chunks) * tokens;
        for (int64_t t = chunk * tokens + lead; t < n; t += kAppendUnroll * step) {
            AppendItem<SRC, DST, VEC> ki4[kAppendUnroll], vi4[kAppendUnroll];
            int64_t p[kAppendUnroll];
            unsigned off[kAppendUnroll];
#pragma unroll
            for (int u = 0; u < kAppendUnroll; ++u) {
                p[u] = -1;
                if (t + u * step >= n) continue;
                const unsigned pos = static_cast<unsigned>(first) + static_cast<unsigned>(t + u * step);
                const unsigned in_row = pos / page;
                off[u] = pos - in_row * page;
                p[u] = row[in_row];
                if (p[u] < 0 || p[u] >= L.P) {
                    record_error(L.status, ADA_ERR_INVALID);
                    p[u] = -1;
                }
                ki4[u].load(L.k, k0 + (t + u * step) * L.ks[2]);
                vi4[u].load(L.v, v0 + (t + u * step) * L.vs[2]);
            }
#pragma unroll
            for (int u = 0; u < kAppendUnroll; ++u) {
                if (p[u] < 0) continue;
                ki4[u].store(L.k_pages, kp0 + p[u] * L.kps[0] + off[u] * L.kps[2], ks, ki);
                vi4[u].store(L.v_pages, vp0 + p[u] * L.vps[0] + off[u] * L.vps[2], vs, vi);
            }
        }
    }
}

template <int SRC, int DST>
int launch_append_dt(const AppendLaunch& L, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(L.B * L.chunks);
    if (L.vec) paged_append_kernel<SRC, DST, true><<<grid, kAppendThreads, 0, stream>>>(L);
    else paged_append_kernel<SRC, DST, false><<<grid, kAppendThreads, 0, stream>>>(L);
    return cudaGetLastError() == cudaSuccess ? ADA_OK : ADA_ERR_LAUNCH;
}

// ---- page accounting -------------------------------------------------------------

constexpr int kPageThreads = 256;
constexpr int kAllocThreads = 1024;

// Pages that sequence s holds (a length outside the table is recorded and cut).
__device__ __forceinline__ int64_t held_pages(const PagesLaunch& L, int64_t s) {
    int64_t n = L.lens[s];
    const int64_t most = L.W * L.page;
    if (n < 0 || n > most) {
        record_error(L.status, ADA_ERR_INVALID);
        n = n < 0 ? 0 : most;
    }
    return (n + L.page - 1) / L.page;
}

__device__ __forceinline__ bool page_ok(const PagesLaunch& L, int64_t p) {
    if (p >= 0 && p < L.P) return true;
    record_error(L.status, ADA_ERR_INVALID);
    return false;
}

// Whether pair i (src[i] -> dst[i]) takes part: both in range, the destination
// no source of the call, and named by no earlier pair. Block-uniform.
__device__ bool pair_counts(const PagesLaunch& L, int64_t i) {
    const int64_t s = L.src[i], d = L.dst[i];
    bool bad = s < 0 || s >= L.S || d < 0 || d >= L.S;
    for (int64_t j = threadIdx.x; j < L.n; j += blockDim.x) bad |= L.src[j] == d || (j < i && L.dst[j] == d);
    bad = __syncthreads_or(bad);
    if (bad && threadIdx.x == 0) record_error(L.status, ADA_ERR_INVALID);
    return !bad;
}

// free: block i gives up the pages of sequence seqs[i]; fork: block i makes
// dst[i] hold src[i]'s pages instead of its own.
template <bool FORK>
__global__ void __launch_bounds__(kPageThreads) pages_share_kernel(const __grid_constant__ PagesLaunch L) {
    const int64_t i = blockIdx.x;
    const int64_t d = L.dst[i];
    if constexpr (FORK) {
        if (!pair_counts(L, i)) return;
    } else {
        bool skip = d < 0 || d >= L.S;
        if (skip && threadIdx.x == 0) record_error(L.status, ADA_ERR_INVALID);
        for (int64_t j = threadIdx.x; j < i; j += kPageThreads) skip |= L.dst[j] == d;  // freed already
        if (__syncthreads_or(skip)) return;
    }
    const int64_t old = held_pages(L, d);
    const int64_t s = FORK ? L.src[i] : 0;
    const int64_t now = FORK ? held_pages(L, s) : 0;
    __syncthreads();  // every thread has read the lengths
    int32_t* drow = L.table + d * L.table_ld;
    for (int64_t j = threadIdx.x; j < old || j < now; j += kPageThreads) {
        if (j < old) {
            const int64_t p = drow[j];
            if (page_ok(L, p)) atomicSub(L.refs + p, 1);
        }
        int32_t q = -1;
        if (FORK && j < now) {
            q = L.table[s * L.table_ld + j];
            if (page_ok(L, q)) atomicAdd(L.refs + q, 1);
        }
        drow[j] = q;
    }
    if (threadIdx.x == 0) L.lens[d] = FORK ? L.lens[s] : 0;
}

// Exclusive prefix sum over the block (1024 threads) and the block's total.
__device__ int block_scan(int x, int* total, int* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int scan = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += up;
    }
    __syncthreads();  // the sums of the call before are read
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    const int w = sums[lane];  // 32 warps
    int ws = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, ws, o);
        if (lane >= o) ws += up;
    }
    *total = __shfl_sync(0xffffffffu, ws, 31);
    return __shfl_sync(0xffffffffu, ws - w, warp) + scan - x;
}

// Allocation, one block. reserve: sequence src[i] grows by extra[i] tokens; it
// needs the pages past those it holds, and a copy of its last page when that
// page is part full and others hold it too. Of the call's sequences that share
// such a page the last one keeps it, if the call covers all its holders and
// every other one got its copy. copy: dst[i] gives its pages up and gets as
// many fresh ones as src[i] holds. Sequence i is served when it needs no page
// or when the needs up to and including its own fit the free pages; another is
// left as it was (reserve) or empty (copy). The pages to copy go to L.pairs.
constexpr int kCopies = 1 << 30, kKeeps = 1 << 29, kNeed = kKeeps - 1;  // flags beside a need
static_assert(kNeed == kMaxNeed, "a need with its flags");

template <bool COPY>
__global__ void __launch_bounds__(kAllocThreads) pages_alloc_kernel(const __grid_constant__ PagesLaunch L) {
    __shared__ int s_sums[32];
    __shared__ int s_npairs;
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid == 0) s_npairs = 0;
    // The last page of sequence s, whose tokens end inside it.
    auto tail_of = [&](int64_t s) -> int64_t { return L.table[s * L.table_ld + L.lens[s] / L.page]; };
    // 1. which entries count: the first to name its (destination) sequence
    for (int64_t i = tid; i < L.n; i += kAllocThreads) {
        const int64_t s = L.src[i], d = COPY ? L.dst[i] : s;
        if (d >= 0 && d < L.S) L.claim[d] = 0x7FFFFFFF;
        if (COPY && s >= 0 && s < L.S) L.claim[s] = 0x7FFFFFFF;
    }
    __syncthreads();
    for (int64_t i = tid; i < L.n; i += kAllocThreads) {
        const int64_t s = L.src[i], d = COPY ? L.dst[i] : s;
        if (d >= 0 && d < L.S) atomicMin(L.claim + d, static_cast<int>(i));
        if (COPY && s >= 0 && s < L.S) atomicMin(L.claim + s, -1);  // a source is no destination
    }
    __syncthreads();
    // 2. what each needs (-1: does not count)
    for (int64_t i = tid; i < L.n; i += kAllocThreads) {
        const int64_t s = L.src[i], d = COPY ? L.dst[i] : s;
        int need = -1;
        if (s >= 0 && s < L.S && d >= 0 && d < L.S && L.claim[d] == static_cast<int>(i)) {
            if constexpr (COPY) {
                need = static_cast<int>(held_pages(L, s));
            } else {
                const int64_t len = L.lens[s], add = L.extra[i];
                if (len >= 0 && add >= 0 && len + add <= L.W * L.page) {
                    need = static_cast<int>((len + add + L.page - 1) / L.page - (len + L.page - 1) / L.page);
                    if (add > 0 && len % L.page != 0) {
                        const int64_t tail = tail_of(s);
                        if (!page_ok(L, tail)) {
                            need = -1;
                        } else if (L.refs[tail] > 1) {
                            L.sharers[tail] = 0;
                            L.last[tail] = -1;
                            L.copied[tail] = 0;
                            need |= kCopies;
                        }
                    }
                }
            }
        }
        if (need < 0) record_error(L.status, ADA_ERR_INVALID);
        L.need[i] = need;
    }
    __syncthreads();
    if constexpr (COPY) {
        // the destinations' own pages, a warp per pair
        for (int64_t i = tid >> 5; i < L.n; i += kAllocThreads / 32) {
            if (L.need[i] < 0) continue;
            const int64_t d = L.dst[i], old = held_pages(L, d);
            for (int64_t j = lane; j < old; j += 32) {
                const int64_t p = L.table[d * L.table_ld + j];
                if (page_ok(L, p)) atomicSub(L.refs + p, 1);
                L.table[d * L.table_ld + j] = -1;
            }
            __syncwarp();
            if (lane == 0) L.lens[d] = 0;
        }
    } else {
        for (int64_t i = tid; i < L.n; i += kAllocThreads) {
            if (L.need[i] < 0 || !(L.need[i] & kCopies)) continue;
            const int64_t tail = tail_of(L.src[i]);
            atomicAdd(L.sharers + tail, 1);
            atomicMax(L.last + tail, static_cast<int>(i));
        }
    }
    __syncthreads();
    // 3. where each one's pages begin among the free ones
    int wanted = 0;
    for (int64_t i0 = 0; i0 < L.n; i0 += kAllocThreads) {
        const int64_t i = i0 + tid;
        int need = 0;
        if (i < L.n && L.need[i] >= 0) {
            need = L.need[i] & kNeed;
            if (!COPY && (L.need[i] & kCopies)) {
                const int64_t tail = tail_of(L.src[i]);
                const bool keeps = L.sharers[tail] == L.refs[tail] && L.last[tail] == static_cast<int>(i);
                need += keeps ? 0 : 1;
                L.need[i] = need | (keeps ? kKeeps : kCopies);
            }
        }
        int total;
        const int at = block_scan(need, &total, s_sums);
        if (i < L.n) L.first[i] = wanted + at;
        wanted += total;
    }
    __syncthreads();
    // 4. the lowest free pages, as many as are wanted
    int found = 0;
    for (int64_t p0 = 0; p0 < L.P && found < wanted; p0 += 4 * kAllocThreads) {
        int open[4], mine = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t p = p0 + 4 * tid + k;
            open[k] = p < L.P && L.refs[p] <= 0;
            mine += open[k];
        }
        int total;
        int at = found + block_scan(mine, &total, s_sums);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (open[k]) {
                if (at < wanted) L.free_list[at] = static_cast<int>(p0 + 4 * tid + k);
                ++at;
            }
        found += total;
    }
    __syncthreads();
    // 5. the sharers that get their copy are counted
    if constexpr (!COPY) {
        for (int64_t i = tid; i < L.n; i += kAllocThreads)
            if (L.need[i] >= 0 && (L.need[i] & kCopies) && L.first[i] + (L.need[i] & kNeed) <= found)
                atomicAdd(L.copied + tail_of(L.src[i]), 1);
        __syncthreads();
    }
    // 6. hand out, a warp per sequence
    for (int64_t i = tid >> 5; i < L.n; i += kAllocThreads / 32) {
        const int flags = L.need[i];
        if (flags < 0) {
            if (lane == 0) L.granted[i] = 0;
            continue;
        }
        const int64_t s = L.src[i];
        int need = flags & kNeed, at = L.first[i];
        bool served = need == 0 || at + need <= found;
        if constexpr (COPY) {
            const int64_t d = L.dst[i];
            for (int j = lane; served && j < need; j += 32) {
                const int to = L.free_list[at + j], from = L.table[s * L.table_ld + j];
                L.table[d * L.table_ld + j] = to;
                L.refs[to] = 1;
                if (page_ok(L, from)) {
                    const int k = atomicAdd(&s_npairs, 1);
                    L.pairs[2 * k] = from;
                    L.pairs[2 * k + 1] = to;
                }
            }
            if (lane == 0) {
                const int64_t most = L.W * L.page, len = L.lens[s];
                const int n = served ? static_cast<int>(len < 0 ? 0 : (len > most ? most : len)) : 0;
                L.lens[d] = n;
                L.granted[i] = n;
            }
        } else {
            const int64_t len = L.lens[s], held = (len + L.page - 1) / L.page;
            const int64_t tail = (flags & (kCopies | kKeeps)) ? tail_of(s) : -1;
            if (flags & kKeeps) served = served && L.copied[tail] == L.sharers[tail] - 1;
            __syncwarp();
            if (served && (flags & kCopies)) {
                if (lane == 0) {
                    const int to = L.free_list[at];
                    L.table[s * L.table_ld + len / L.page] = to;
                    L.refs[to] = 1;
                    atomicSub(L.refs + tail, 1);
                    const int k = atomicAdd(&s_npairs, 1);
                    L.pairs[2 * k] = static_cast<int>(tail);
                    L.pairs[2 * k + 1] = to;
                }
                ++at;
                --need;
            }
            for (int j = lane; served && j < need; j += 32) {
                const int to = L.free_list[at + j];
                L.table[s * L.table_ld + held + j] = to;
                L.refs[to] = 1;
            }
            if (lane == 0) {
                L.granted[i] = served ? L.extra[i] : 0;
                if (served) L.lens[s] = static_cast<int>(len) + L.extra[i];
            }
        }
    }
    __syncthreads();
    if (tid == 0) *L.n_pairs = s_npairs;
}

// compact, one block: with n live pages, the live pages from n on (ascending)
// move into the free pages below n (ascending); to[p] is where such a page went.
__global__ void __launch_bounds__(kAllocThreads) pages_compact_kernel(const __grid_constant__ PagesLaunch L) {
    __shared__ int s_sums[32];
    const int tid = threadIdx.x;
    int live = 0;
    for (int64_t p = tid; p < L.P; p += kAllocThreads) live += L.refs[p] > 0;
    int n;
    block_scan(live, &n, s_sums);
    int holes = 0, high = 0;
    for (int64_t p0 = 0; p0 < L.P; p0 += 4 * kAllocThreads) {
        int kind[4], nh = 0, nm = 0;  // 1: hole below n, 2: live from n on
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t p = p0 + 4 * tid + k;
            const bool used = p < L.P && L.refs[p] > 0;
            kind[k] = (p < n && !used) ? 1 : (p >= n && used) ? 2 : 0;
            if (p >= n && p < L.P && !used) L.to[p] = static_cast<int>(p);
            nh += kind[k] == 1;
            nm += kind[k] == 2;
        }
        int th, tm;
        int ah = holes + block_scan(nh, &th, s_sums), am = high + block_scan(nm, &tm, s_sums);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int p = static_cast<int>(p0 + 4 * tid + k);
            if (kind[k] == 1) L.pairs[2 * ah++ + 1] = p;
            if (kind[k] == 2) L.pairs[2 * am++] = p;
        }
        holes += th;
        high += tm;
    }
    __syncthreads();
    for (int k = tid; k < high; k += kAllocThreads) {
        const int from = L.pairs[2 * k], to = L.pairs[2 * k + 1];
        L.to[from] = to;
        L.refs[to] = L.refs[from];
        L.refs[from] = 0;
    }
    if (tid == 0) {
        *L.n_pairs = high;
        *L.granted = n;
    }
}

// ---- moving page data --------------------------------------------------------------

constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 8;

// Copies the pages of the list in every plane, a block per piece of a page;
// after a compaction the table's entries follow their pages as well. The list
// and its length are in device memory. No page is both read and written.
template <typename V, bool REMAP>
__global__ void __launch_bounds__(kMoveThreads) pages_move_kernel(const __grid_constant__ PagesLaunch L) {
    constexpr int64_t kPiece = static_cast<int64_t>(kMoveThreads) * kMoveUnroll;  // vectors
    const int64_t vecs = L.page_bytes / static_cast<int64_t>(sizeof(V));
    const int64_t pieces = (vecs + kPiece - 1) / kPiece;
    const int64_t items = static_cast<int64_t>(*L.n_pairs) * L.planes * pieces;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const int64_t piece = it % pieces, rest = it / pieces;
        const int64_t plane = rest % L.planes, k = rest / L.planes;
        uint8_t* base = static_cast<uint8_t*>(L.data) + plane * L.plane_bytes;
        const V* a = reinterpret_cast<const V*>(base + L.pairs[2 * k] * L.page_stride);
        V* b = reinterpret_cast<V*>(base + L.pairs[2 * k + 1] * L.page_stride);
        const int64_t v0 = piece * kPiece + threadIdx.x;
        V r[kMoveUnroll];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u)
            if (v0 + u * kMoveThreads < vecs) r[u] = a[v0 + u * kMoveThreads];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u)
            if (v0 + u * kMoveThreads < vecs) b[v0 + u * kMoveThreads] = r[u];
    }
    if constexpr (REMAP) {
        const int n = *L.granted;  // live pages: an entry from n on has moved
        for (int64_t s = blockIdx.x; s < L.S; s += gridDim.x) {
            const int64_t held = held_pages(L, s);
            for (int64_t j = threadIdx.x; j < held; j += kMoveThreads) {
                const int64_t p = L.table[s * L.table_ld + j];
                if (page_ok(L, p) && p >= n) L.table[s * L.table_ld + j] = L.to[p];
            }
        }
    }
}

template <bool REMAP>
int launch_move(const PagesLaunch& L, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(L.move_blocks);
    if (L.vec == 16) pages_move_kernel<uint4, REMAP><<<grid, kMoveThreads, 0, stream>>>(L);
    else if (L.vec == 4) pages_move_kernel<uint32_t, REMAP><<<grid, kMoveThreads, 0, stream>>>(L);
    else if (L.vec == 2) pages_move_kernel<uint16_t, REMAP><<<grid, kMoveThreads, 0, stream>>>(L);
    else pages_move_kernel<uint8_t, REMAP><<<grid, kMoveThreads, 0, stream>>>(L);
    return cudaGetLastError() == cudaSuccess ? ADA_OK : ADA_ERR_LAUNCH;
}

}  // namespace

int launch_paged_append(const AppendLaunch& L, cudaStream_t stream) {
    if (L.dst_dtype == ADA_E4M3) {
        switch (L.src_dtype) {
            case ADA_F32: return launch_append_dt<ADA_F32, ADA_E4M3>(L, stream);
            case ADA_F16: return launch_append_dt<ADA_F16, ADA_E4M3>(L, stream);
            case ADA_BF16: return launch_append_dt<ADA_BF16, ADA_E4M3>(L, stream);
            default: return ADA_ERR_DTYPE;
        }
    }
    // one type on both sides: the bytes move
    if (L.src_dtype == ADA_F32) return launch_append_dt<ADA_F32, ADA_F32>(L, stream);
    return launch_append_dt<ADA_BF16, ADA_BF16>(L, stream);
}

int launch_pages_share(const PagesLaunch& L, bool fork, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(L.n);
    if (fork) pages_share_kernel<true><<<grid, kPageThreads, 0, stream>>>(L);
    else pages_share_kernel<false><<<grid, kPageThreads, 0, stream>>>(L);
    return cudaGetLastError() == cudaSuccess ? ADA_OK : ADA_ERR_LAUNCH;
}

int launch_pages_alloc(const PagesLaunch& L, bool copy, cudaStream_t stream) {
    if (copy) pages_alloc_kernel<true><<<1, kAllocThreads, 0, stream>>>(L);
    else pages_alloc_kernel<false><<<1, kAllocThreads, 0, stream>>>(L);
    if (cudaGetLastError() != cudaSuccess) return ADA_ERR_LAUNCH;
    return launch_move<false>(L, stream);
}

int launch_pages_compact(const PagesLaunch& L, cudaStream_t stream) {
    pages_compact_kernel<<<1, kAllocThreads, 0, stream>>>(L);
    if (cudaGetLastError() != cudaSuccess) return ADA_ERR_LAUNCH;
    return launch_move<true>(L, stream);
}

}  // namespace ada
