// C entry points of the serving operators (include/adaattn_b200.h): attention
// over a paged key-value cache, the append, the page operations and token log
// probabilities. Argument checks, workspace carving and launch descriptions;
// no device memory is allocated here and nothing synchronises.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "ada_common.cuh"
#include "ada_internal.h"

namespace ada {
namespace {

int fail(int code, const char* fmt, ...) {
    char msg[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    return record_last_error(code, msg);
}

constexpr int64_t kMaxInt = 0x7FFFFFFF;

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
bool is_float(int dtype) { return dtype == ADA_F32 || dtype == ADA_F16 || dtype == ADA_BF16; }
int elt_bytes(int dtype) { return dtype == ADA_F32 ? 4 : dtype == ADA_E4M3 ? 1 : 2; }
// An optional tensor is omitted when it is null or describes elements at null; one without elements is given.
bool given(const AdaTensor* t) {
    if (t == nullptr || t->data != nullptr) return t != nullptr;
    for (int i = 0; i < t->ndim && i < 4; ++i)
        if (t->shape[i] == 0) return true;
    return false;
}

// SMs of the current device (asked for once per device).
int sm_count(int* n) {
    static std::mutex mu;
    static int known[64] = {0};
    int dev;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(ADA_ERR_DEVICE, "cudaGetDevice failed");
    std::lock_guard<std::mutex> lock(mu);
    if (known[dev] == 0 && cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return fail(ADA_ERR_DEVICE, "the SM count of device %d is unavailable", dev);
    *n = known[dev];
    return ADA_OK;
}

// A tensor of `ndim` dimensions with a unit innermost stride; data may be null only when it is empty.
int check_view(const AdaTensor* t, const char* name, int ndim) {
    if (t == nullptr) return fail(ADA_ERR_INVALID, "%s is null", name);
    if (t->ndim != ndim) return fail(ADA_ERR_SHAPE, "%s must be %d-D, got %d-D", name, ndim, t->ndim);
    int64_t n = 1;
    for (int i = 0; i < ndim; ++i) {
        if (t->shape[i] < 0) return fail(ADA_ERR_SHAPE, "%s has a negative extent", name);
        n *= t->shape[i];
    }
    if (n > 0 && t->data == nullptr) return fail(ADA_ERR_INVALID, "%s is null", name);
    if (t->shape[ndim - 1] > 1 && t->stride[ndim - 1] != 1)
        return fail(ADA_ERR_LAYOUT, "%s needs a unit innermost stride", name);
    return ADA_OK;
}

int check_ints(const AdaTensor* t, const char* name, int64_t n) {
    int rc = check_view(t, name, 1);
    if (rc) return rc;
    if (t->dtype != ADA_I32) return fail(ADA_ERR_DTYPE, "%s must be int32", name);
    if (n >= 0 && t->shape[0] != n)
        return fail(ADA_ERR_SHAPE, "%s must have %lld elements, got %lld", name, (long long)n, (long long)t->shape[0]);
    return ADA_OK;
}

// page_table [S, W] and seq_lens [S].
int check_table(const AdaTensor* table, const AdaTensor* lens) {
    int rc = check_view(table, "page_table", 2);
    if (rc) return rc;
    if (table->dtype != ADA_I32) return fail(ADA_ERR_DTYPE, "page_table must be int32");
    if (table->shape[0] > kMaxInt || table->shape[1] > kMaxInt)
        return fail(ADA_ERR_UNSUPPORTED, "page_table extents must be below 2^31");
    return check_ints(lens, "seq_lens", table->shape[0]);
}

// A tensor that is written must hold each element once: along the dimensions
// in the order of their strides, each step goes past all that is inside it.
int check_apart(const AdaTensor* t, const char* name) {
    int order[4], n = 0;
    for (int i = 0; i < t->ndim; ++i) {
        if (t->shape[i] == 0) return ADA_OK;
        if (t->shape[i] > 1) order[n++] = i;
    }
    auto step = [&](int i) { return t->stride[i] < 0 ? -t->stride[i] : t->stride[i]; };
    std::sort(order, order + n, [&](int a, int b) { return step(a) < step(b); });
    int64_t span = 1;
    for (int i = 0; i < n; ++i) {
        if (step(order[i]) < span) return fail(ADA_ERR_LAYOUT, "%s overlaps itself", name);
        span += (t->shape[order[i]] - 1) * step(order[i]);
    }
    return ADA_OK;
}

int64_t row_stride(const AdaTensor* t, int i) { return t->shape[i] > 1 ? t->stride[i] : 0; }

// Every row of a view starts on an `align`-byte boundary.
bool rows_aligned(const AdaTensor* t, int eb, int align) {
    if (reinterpret_cast<uintptr_t>(t->data) % align) return false;
    for (int i = 0; i + 1 < t->ndim; ++i)
        if (t->shape[i] > 1 && (t->stride[i] * eb) % align) return false;
    return true;
}

// k_pages and v_pages [P, Hkv, page, D] of one type.
int check_pages(const AdaTensor* k, const AdaTensor* v, int64_t D) {
    int rc;
    if ((rc = check_view(k, "k_pages", 4)) || (rc = check_view(v, "v_pages", 4))) return rc;
    if (k->dtype != v->dtype) return fail(ADA_ERR_DTYPE, "k_pages and v_pages must share one dtype");
    if (!is_float(k->dtype) && k->dtype != ADA_E4M3) return fail(ADA_ERR_DTYPE, "pages must be fp32, fp16, bf16 or E4M3");
    for (int i = 0; i < 4; ++i)
        if (k->shape[i] != v->shape[i]) return fail(ADA_ERR_SHAPE, "k_pages and v_pages differ in extent %d", i);
    if (k->shape[3] != D) return fail(ADA_ERR_SHAPE, "pages hold heads of %lld elements, not %lld", (long long)k->shape[3], (long long)D);
    if (D < 1 || D > 128) return fail(ADA_ERR_UNSUPPORTED, "head dim %lld outside [1, 128]", (long long)D);
    if (k->shape[2] < 1 || k->shape[2] > 65536)
        return fail(ADA_ERR_UNSUPPORTED, "page size %lld outside [1, 65536]", (long long)k->shape[2]);
    if (k->shape[1] < 1) return fail(ADA_ERR_SHAPE, "pages need at least one key/value head");
    if (k->shape[0] > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "at most 2^31 - 1 pages");
    return ADA_OK;
}

int check_width(const AdaTensor* table, int64_t page) {
    if (table->shape[1] * page > kMaxInt)
        return fail(ADA_ERR_UNSUPPORTED, "page_table covers 2^31 or more tokens per sequence");
    return ADA_OK;
}

int check_scales(const AdaTensor* s, const char* name, int64_t heads, int kv_dtype) {
    if (!given(s)) return ADA_OK;
    if (kv_dtype != ADA_E4M3) return fail(ADA_ERR_UNSUPPORTED, "%s goes with E4M3 pages only", name);
    if (s->dtype != ADA_F32) return fail(ADA_ERR_DTYPE, "%s must be float32", name);
    if (s->ndim != 1 || s->shape[0] != heads || (heads > 1 && s->stride[0] != 1))
        return fail(ADA_ERR_SHAPE, "%s must be a contiguous [%lld] vector", name, (long long)heads);
    return ADA_OK;
}

// ---- attention -------------------------------------------------------------------

constexpr int64_t kMaxBatch = 4096;  // the tile prefix is kept in shared memory
constexpr int kMaxCtas = 2 * 148;    // pieces that the workspace is sized for

// Query heads per block: the tensor-core kernel takes 8 or 16 (its products'
// narrow side), the CUDA-core kernel up to 8.
int heads_per_block(int64_t g, bool tc) { return tc ? (g <= 8 ? 8 : 16) : g <= 1 ? 1 : g <= 2 ? 2 : g <= 4 ? 4 : 8; }

// A tensor map over pages [P, Hkv, page, D] (innermost first: D, page, Hkv, P)
// with boxes of `rows` keys x up to 128 bytes, swizzled over that width.
int pages_map(CUtensorMap* map, const AdaTensor* t, int rows) {
    PFN_cuTensorMapEncodeTiled_v12000 enc;
    int rc = tensor_map_encoder(&enc);
    if (rc) return rc;
    const int eb = elt_bytes(t->dtype);
    const int64_t row = t->shape[3] * eb;
    cuuint64_t dims[4], strides[3];
    int64_t dense = row;
    for (int i = 0; i < 4; ++i) dims[i] = static_cast<cuuint64_t>(t->shape[3 - i]);
    for (int i = 0; i < 3; ++i) {
        strides[i] = static_cast<cuuint64_t>(t->shape[2 - i] > 1 ? t->stride[2 - i] * eb : dense);
        dense = static_cast<int64_t>(strides[i]) * t->shape[2 - i];
    }
    cuuint32_t box[4] = {static_cast<cuuint32_t>(std::min<int64_t>(row, 128) / eb), static_cast<cuuint32_t>(rows), 1, 1};
    cuuint32_t es[4] = {1, 1, 1, 1};
    const CUtensorMapDataType dt = t->dtype == ADA_F16    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                   : t->dtype == ADA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const CUresult r = enc(map, dt, 4, t->data, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           row >= 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(ADA_ERR_LAYOUT, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return ADA_OK;
}

// Whether TMA can read the pages: rows on 16-byte boundaries, positive strides below 2^40 bytes.
bool tma_pages(const AdaTensor* t, int eb) {
    if (!rows_aligned(t, eb, 16) || t->shape[0] < 1) return false;
    for (int i = 0; i < 3; ++i)
        if (t->shape[i] > 1 && (t->stride[i] <= 0 || t->stride[i] * eb >= (int64_t(1) << 40))) return false;
    return true;
}

// ---- page operations ---------------------------------------------------------------

struct PagesSpace {
    size_t pairs, free_list, to, sharers, last, copied, claim, need, first, total;
};
PagesSpace pages_space(int64_t P, int64_t S, int64_t n) {
    PagesSpace w;
    size_t at = 256;  // the pair count
    auto take = [&](int64_t ints) {
        const size_t here = at;
        at += align256(static_cast<size_t>(ints) * 4);
        return here;
    };
    w.pairs = take(2 * P);
    w.free_list = take(P);
    w.to = take(P);
    w.sharers = take(P);
    w.last = take(P);
    w.copied = take(P);
    w.claim = take(S);
    w.need = take(n);
    w.first = take(n);
    w.total = at;
    return w;
}

int pages_table(const AdaTensor* table, const AdaTensor* lens, const AdaTensor* refs, int64_t page, PagesLaunch* L) {
    int rc;
    if ((rc = check_table(table, lens)) || (rc = check_ints(refs, "ref_counts", -1))) return rc;
    if (page < 1 || page > 65536) return fail(ADA_ERR_UNSUPPORTED, "page size %lld outside [1, 65536]", (long long)page);
    if ((rc = check_width(table, page))) return rc;
    if (refs->shape[0] > (int64_t(1) << 30)) return fail(ADA_ERR_UNSUPPORTED, "at most 2^30 pages");
    // the pages that a call can need are counted in 32 bits
    if (table->shape[0] * (table->shape[1] + 1) > kMaxInt)
        return fail(ADA_ERR_UNSUPPORTED, "page_table has 2^31 or more entries");
    // and a sequence's share the word with two flags (kNeed)
    if (table->shape[1] >= kMaxNeed)
        return fail(ADA_ERR_UNSUPPORTED, "at most 2^29 - 2 page_table entries per sequence");
    if (table->shape[0] > 1 && table->stride[0] < table->shape[1])
        return fail(ADA_ERR_LAYOUT, "the rows of page_table overlap");
    *L = PagesLaunch{};
    L->table = static_cast<int32_t*>(table->data);
    L->lens = static_cast<int32_t*>(lens->data);
    L->refs = static_cast<int32_t*>(refs->data);
    L->S = table->shape[0];
    L->W = table->shape[1];
    L->P = refs->shape[0];
    L->table_ld = row_stride(table, 0);
    L->page = page;
    return ADA_OK;
}

// `pages` [planes, P, ...] (page blocks contiguous) and the workspace.
int pages_data(const AdaTensor* pages, void* workspace, size_t bytes, PagesLaunch* L) {
    int rc = check_view(pages, "pages", 3);
    if (rc) return rc;
    if (!is_float(pages->dtype) && pages->dtype != ADA_E4M3) return fail(ADA_ERR_DTYPE, "pages must be fp32, fp16, bf16 or E4M3");
    if (pages->shape[1] != L->P) return fail(ADA_ERR_SHAPE, "pages and ref_counts differ in their page count");
    const int eb = elt_bytes(pages->dtype);
    L->data = pages->data;
    L->planes = pages->shape[0];
    L->page_bytes = pages->shape[2] * eb;
    L->page_stride = row_stride(pages, 1) * eb;
    L->plane_bytes = row_stride(pages, 0) * eb;
    if (pages->shape[1] > 1 && pages->stride[1] < pages->shape[2]) return fail(ADA_ERR_LAYOUT, "pages overlap");
    if (pages->shape[0] > 1 && pages->stride[0] < pages->shape[2]) return fail(ADA_ERR_LAYOUT, "planes overlap");
    if (pages->shape[0] > 1 && pages->shape[1] > 1) {  // one of the two lies inside the other's stride
        const int in = pages->stride[0] < pages->stride[1] ? 0 : 1;
        if (pages->stride[1 - in] < pages->stride[in] * pages->shape[in]) return fail(ADA_ERR_LAYOUT, "pages and planes overlap");
    }
    const uint64_t all = reinterpret_cast<uint64_t>(pages->data) | static_cast<uint64_t>(L->page_bytes) |
                         static_cast<uint64_t>(L->page_stride) | static_cast<uint64_t>(L->plane_bytes);
    L->vec = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
    const PagesSpace w = pages_space(L->P, L->S, L->n);
    if (workspace == nullptr || bytes < w.total) return fail(ADA_ERR_WORKSPACE, "page workspace too small");
    uint8_t* base = static_cast<uint8_t*>(workspace);
    auto at = [&](size_t o) { return reinterpret_cast<int32_t*>(base + o); };
    L->n_pairs = at(0);
    L->pairs = at(w.pairs);
    L->free_list = at(w.free_list);
    L->to = at(w.to);
    L->sharers = at(w.sharers);
    L->last = at(w.last);
    L->copied = at(w.copied);
    L->claim = at(w.claim);
    L->need = at(w.need);
    L->first = at(w.first);
    int sms;
    if ((rc = device_status_word(&L->status)) || (rc = sm_count(&sms))) return rc;
    // Enough blocks to fill the GPU; fewer when the pool itself holds fewer pieces.
    const int64_t per_piece = int64_t(2048) * L->vec;
    const int64_t most = std::max<int64_t>(1, L->P) * std::max<int64_t>(1, L->planes) *
                         std::max<int64_t>(1, (L->page_bytes + per_piece - 1) / per_piece);
    L->move_blocks = static_cast<int>(std::min<int64_t>(most, int64_t(sms) * 8));
    return ADA_OK;
}

int check_row_tokens(const AdaTensor* tokens, int64_t rows, LogprobLaunch* L) {
    int rc = check_view(tokens, "tokens", 1);
    if (rc) return rc;
    if (tokens->dtype != ADA_I64 && tokens->dtype != ADA_I32) return fail(ADA_ERR_DTYPE, "tokens must be int64 or int32");
    if (tokens->shape[0] != rows) return fail(ADA_ERR_SHAPE, "tokens must have one entry per row of logits");
    L->tokens = tokens->data;
    L->tok64 = tokens->dtype == ADA_I64;
    return ADA_OK;
}

// logits [A, R, V].
int logits_setup(const AdaTensor* logits, LogprobLaunch* L) {
    int rc = check_view(logits, "logits", 3);
    if (rc) return rc;
    if (!is_float(logits->dtype)) return fail(ADA_ERR_DTYPE, "logits must be fp32, fp16 or bf16");
    const int64_t V = logits->shape[2];
    if (V < 1 || V > (int64_t(1) << 30)) return fail(ADA_ERR_UNSUPPORTED, "vocabulary %lld outside [1, 2^30]", (long long)V);
    if (reinterpret_cast<uintptr_t>(logits->data) % elt_bytes(logits->dtype))
        return fail(ADA_ERR_LAYOUT, "logits are not aligned to their elements");
    *L = LogprobLaunch{};
    L->logits = logits->data;
    L->dtype = logits->dtype;
    L->R = std::max<int64_t>(1, logits->shape[1]);
    L->rows = logits->shape[0] * logits->shape[1];
    L->s0 = row_stride(logits, 0);
    L->s1 = row_stride(logits, 1);
    L->V = static_cast<int>(V);
    return ADA_OK;
}

}  // namespace
}  // namespace ada

using namespace ada;

extern "C" {

size_t ada_paged_attn_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim) {
    if (batch < 0 || batch > kMaxBatch || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || head_dim > 128)
        return 0;
    const size_t gb = static_cast<size_t>(heads_per_block(heads / kv_heads, true));
    return align256(static_cast<size_t>(batch + 1) * 4) + align256(kMaxCtas * 2 * gb * 2 * 4) +
           align256(kMaxCtas * 2 * gb * static_cast<size_t>(head_dim) * 4);
}

int ada_paged_attn(const AdaTensor* q, const AdaTensor* k_pages, const AdaTensor* v_pages, const AdaTensor* page_table,
                   const AdaTensor* seq_lens, const AdaTensor* seqs, const AdaTensor* key_mask, const AdaTensor* k_scale,
                   const AdaTensor* v_scale, float scale, AdaTensor* out, float* lse, void* workspace,
                   size_t workspace_bytes, void* stream) {
    int rc;
    if ((rc = check_view(q, "q", 3)) || (rc = check_view(out, "out", 3))) return rc;
    if (!is_float(q->dtype)) return fail(ADA_ERR_DTYPE, "q must be fp32, fp16 or bf16");
    if (out->dtype != q->dtype) return fail(ADA_ERR_DTYPE, "out must have q's dtype");
    const int64_t B = q->shape[0], H = q->shape[1], D = q->shape[2];
    for (int i = 0; i < 3; ++i)
        if (out->shape[i] != q->shape[i]) return fail(ADA_ERR_SHAPE, "out and q differ in extent %d", i);
    if ((rc = check_pages(k_pages, v_pages, D)) || (rc = check_table(page_table, seq_lens))) return rc;
    if (k_pages->dtype != ADA_E4M3 && k_pages->dtype != q->dtype)
        return fail(ADA_ERR_DTYPE, "q and the pages must share one dtype (or the pages be E4M3)");
    const int64_t Hkv = k_pages->shape[1], page = k_pages->shape[2];
    if ((rc = check_width(page_table, page))) return rc;
    if (H < 1 || H % Hkv) return fail(ADA_ERR_SHAPE, "%lld query heads do not divide over %lld key/value heads", (long long)H, (long long)Hkv);
    if (B > kMaxBatch) return fail(ADA_ERR_UNSUPPORTED, "at most %lld sequences per call", (long long)kMaxBatch);
    // the places of all sequences are counted in 32 bits
    if (B * ((page_table->shape[1] * page + kPagedTile - 1) / kPagedTile + kPagedLead) > kMaxInt)
        return fail(ADA_ERR_UNSUPPORTED, "the tables of %lld sequences cover 2^36 keys or more", (long long)B);
    const bool picked = given(seqs);
    if (picked && (rc = check_ints(seqs, "seqs", B))) return rc;
    if (!picked && page_table->shape[0] != B)
        return fail(ADA_ERR_SHAPE, "page_table must have one row per sequence of q");
    if ((rc = check_scales(k_scale, "k_scale", Hkv, k_pages->dtype)) || (rc = check_scales(v_scale, "v_scale", Hkv, k_pages->dtype)))
        return rc;
    if (given(key_mask)) {
        if (key_mask->ndim != 2 || (key_mask->shape[0] != B && key_mask->shape[0] != 1))
            return fail(ADA_ERR_SHAPE, "key_mask must be [B, L]");
        if (key_mask->dtype != ADA_BOOL && !is_float(key_mask->dtype)) return fail(ADA_ERR_DTYPE, "key_mask must be bool or floating point");
    }
    if ((rc = check_apart(out, "out"))) return rc;
    if (B == 0) return ADA_OK;
    if (out->data == q->data) return fail(ADA_ERR_LAYOUT, "out shares q's memory");
    if (workspace == nullptr || workspace_bytes < ada_paged_attn_workspace_bytes(B, H, Hkv, D))
        return fail(ADA_ERR_WORKSPACE, "paged attention workspace too small");
    unsigned int* st;
    int sms;
    if ((rc = device_status_word(&st)) || (rc = sm_count(&sms))) return rc;
    PagedAttnLaunch L{};
    L.q = q->data;
    L.k = k_pages->data;
    L.v = v_pages->data;
    L.q_dtype = q->dtype;
    L.kv_dtype = k_pages->dtype;
    for (int i = 0; i < 2; ++i) {
        L.qs[i] = row_stride(q, i);
        L.os[i] = row_stride(out, i);
    }
    for (int i = 0; i < 3; ++i) {
        L.ks[i] = row_stride(k_pages, i);
        L.vs[i] = row_stride(v_pages, i);
    }
    const int eb = elt_bytes(k_pages->dtype);
    L.vec = D % 4 == 0 && rows_aligned(k_pages, eb, 4 * eb) && rows_aligned(v_pages, eb, 4 * eb);
    L.table = static_cast<const int32_t*>(page_table->data);
    L.lens = static_cast<const int32_t*>(seq_lens->data);
    L.seqs = picked ? static_cast<const int32_t*>(seqs->data) : nullptr;
    L.S = page_table->shape[0];
    L.W = page_table->shape[1];
    L.table_ld = row_stride(page_table, 0);
    L.P = k_pages->shape[0];
    L.page = static_cast<int>(page);
    L.page_inv = page == 1 ? 0u : static_cast<uint32_t>(((uint64_t(1) << 32) + page - 1) / page);
    if (given(key_mask)) {
        L.mask.data = key_mask->data;
        L.mask.dtype = key_mask->dtype;
        L.mask.s[0] = row_stride(key_mask, 0);
        L.mask.s[1] = row_stride(key_mask, 1);
        L.mask_len = std::min(key_mask->shape[1], kMaxInt);  // (no sequence is longer)
    }
    L.k_scale = given(k_scale) ? static_cast<const float*>(k_scale->data) : nullptr;
    L.v_scale = given(v_scale) ? static_cast<const float*>(v_scale->data) : nullptr;
    L.scale = scale;
    L.B = static_cast<int>(B);
    L.H = static_cast<int>(H);
    L.D = static_cast<int>(D);
    L.G = static_cast<int>(H / Hkv);
    // The tensor-core kernel serves 16- and 8-bit pages that TMA can read with
    // heads of 64 or 128 and a page of a multiple of 8 keys (a swizzle's rows).
    L.tc = k_pages->dtype != ADA_F32 && q->dtype != ADA_F32 && (D == 64 || D == 128) && page % 8 == 0 &&
           tma_pages(k_pages, eb) && tma_pages(v_pages, eb) && rows_aligned(q, 2, 4);
    if (L.tc) {
        L.chunk = static_cast<int>(std::min<int64_t>(32, page & -page));
        if ((rc = pages_map(&L.tk, k_pages, L.chunk)) || (rc = pages_map(&L.tv, v_pages, L.chunk))) return rc;
    }
    L.GB = heads_per_block(L.G, L.tc != 0);
    L.HB = (L.G + L.GB - 1) / L.GB;
    L.U = Hkv * L.HB;
    if (B * L.U > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many heads");
    L.out = out->data;
    L.lse = lse;
    L.n_cta = std::min(kMaxCtas, L.tc ? sms : 2 * sms);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    L.pref = reinterpret_cast<int*>(ws);
    ws += align256(static_cast<size_t>(B + 1) * 4);
    L.part_ml = reinterpret_cast<float*>(ws);
    ws += align256(kMaxCtas * 2 * static_cast<size_t>(L.GB) * 2 * 4);
    L.part_acc = reinterpret_cast<float*>(ws);
    L.status = st;
    L.timeout_ns = default_wait_timeout_ns();
    rc = launch_paged_attn(L, static_cast<cudaStream_t>(stream));
    return rc ? fail(rc, "paged attention launch failed: %s", cudaGetErrorString(cudaGetLastError())) : ADA_OK;
}

namespace {
int append(const AdaTensor* k, const AdaTensor* v, AdaTensor* k_pages, AdaTensor* v_pages, const AdaTensor* page_table,
           const AdaTensor* seq_lens, const AdaTensor* new_tokens, const AdaTensor* seqs, const AdaTensor* k_scale,
           const AdaTensor* v_scale, bool prompts, void* stream) {
    int rc;
    if ((rc = check_view(k, "k", 4)) || (rc = check_view(v, "v", 4))) return rc;
    if (!is_float(k->dtype)) return fail(ADA_ERR_DTYPE, "k must be fp32, fp16 or bf16");
    if (v->dtype != k->dtype) return fail(ADA_ERR_DTYPE, "k and v must share one dtype");
    for (int i = 0; i < 4; ++i)
        if (k->shape[i] != v->shape[i]) return fail(ADA_ERR_SHAPE, "k and v differ in extent %d", i);
    const int64_t B = k->shape[0], Hkv = k->shape[1], N = k->shape[2], D = k->shape[3];
    if ((rc = check_pages(k_pages, v_pages, D)) || (rc = check_table(page_table, seq_lens))) return rc;
    if (k_pages->shape[1] != Hkv) return fail(ADA_ERR_SHAPE, "k and the pages differ in their heads");
    if (k_pages->dtype != ADA_E4M3 && k_pages->dtype != k->dtype)
        return fail(ADA_ERR_DTYPE, "k and the pages must share one dtype (or the pages be E4M3)");
    const int64_t page = k_pages->shape[2];
    if ((rc = check_width(page_table, page))) return rc;
    const bool picked = given(seqs);
    if (picked && (rc = check_ints(seqs, "seqs", B))) return rc;
    if (!picked && page_table->shape[0] != B)
        return fail(ADA_ERR_SHAPE, "page_table must have one row per sequence of k");
    if (given(new_tokens) && (rc = check_ints(new_tokens, "new_tokens", B))) return rc;
    if ((rc = check_scales(k_scale, "k_scale", Hkv, k_pages->dtype)) || (rc = check_scales(v_scale, "v_scale", Hkv, k_pages->dtype)))
        return rc;
    if ((rc = check_apart(k_pages, "k_pages")) || (rc = check_apart(v_pages, "v_pages"))) return rc;
    if (B == 0 || N == 0) return ADA_OK;
    if (N > kMaxInt || B > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many tokens");
    unsigned int* st;
    int sms;
    if ((rc = device_status_word(&st)) || (rc = sm_count(&sms))) return rc;
    AppendLaunch L{};
    L.k = k->data;
    L.v = v->data;
    L.k_pages = k_pages->data;
    L.v_pages = v_pages->data;
    L.src_dtype = k->dtype;
    L.dst_dtype = k_pages->dtype;
    for (int i = 0; i < 3; ++i) {
        L.ks[i] = row_stride(k, i);
        L.vs[i] = row_stride(v, i);
        L.kps[i] = row_stride(k_pages, i);
        L.vps[i] = row_stride(v_pages, i);
    }
    const int se = elt_bytes(k->dtype), de = elt_bytes(k_pages->dtype);
    const int da = de == 1 ? 8 : 16;
    L.vec = D % 8 == 0 && rows_aligned(k, se, 16) && rows_aligned(v, se, 16) && rows_aligned(k_pages, de, da) &&
            rows_aligned(v_pages, de, da);
    L.table = static_cast<const int32_t*>(page_table->data);
    L.lens = static_cast<const int32_t*>(seq_lens->data);
    L.new_tokens = given(new_tokens) ? static_cast<const int32_t*>(new_tokens->data) : nullptr;
    L.seqs = picked ? static_cast<const int32_t*>(seqs->data) : nullptr;
    L.S = page_table->shape[0];
    L.W = page_table->shape[1];
    L.table_ld = row_stride(page_table, 0);
    L.P = k_pages->shape[0];
    L.B = B;
    L.N = N;
    L.Hkv = Hkv;
    L.page = static_cast<int>(page);
    L.D = static_cast<int>(D);
    L.k_scale = given(k_scale) ? static_cast<const float*>(k_scale->data) : nullptr;
    L.v_scale = given(v_scale) ? static_cast<const float*>(v_scale->data) : nullptr;
    L.status = st;
    // Blocks of 256 items (of whole tokens), and no more than fill the GPU twice.
    const int64_t in_token = Hkv * (L.vec ? D / 8 : D);
    if (in_token > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many heads");
    const int64_t at_once = in_token < 256 ? 256 / in_token : 1;
    const int64_t most = std::max<int64_t>(1, int64_t(sms) * 16 / B);
    L.chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((N + at_once - 1) / at_once, most)));
    if (B * L.chunks > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many sequences");
    L.prompts = prompts;
    rc = launch_paged_append(L, static_cast<cudaStream_t>(stream));
    return rc ? fail(rc, "append launch failed: %s", cudaGetErrorString(cudaGetLastError())) : ADA_OK;
}
}  // namespace

int ada_paged_append(const AdaTensor* k, const AdaTensor* v, AdaTensor* k_pages, AdaTensor* v_pages,
                     const AdaTensor* page_table, const AdaTensor* seq_lens, const AdaTensor* new_tokens,
                     const AdaTensor* seqs, const AdaTensor* k_scale, const AdaTensor* v_scale, void* stream) {
    return append(k, v, k_pages, v_pages, page_table, seq_lens, new_tokens, seqs, k_scale, v_scale, false, stream);
}

int ada_paged_append_prompts(const AdaTensor* k, const AdaTensor* v, AdaTensor* k_pages, AdaTensor* v_pages,
                             const AdaTensor* page_table, const AdaTensor* seq_lens, const AdaTensor* new_tokens,
                             const AdaTensor* seqs, const AdaTensor* k_scale, const AdaTensor* v_scale, void* stream) {
    return append(k, v, k_pages, v_pages, page_table, seq_lens, new_tokens, seqs, k_scale, v_scale, true, stream);
}

size_t ada_pages_workspace_bytes(int64_t num_pages, int64_t num_sequences, int64_t n) {
    if (num_pages < 0 || num_sequences < 0 || n < 0) return 0;
    return pages_space(num_pages, num_sequences, n).total;
}

int ada_pages_free(AdaTensor* page_table, AdaTensor* seq_lens, AdaTensor* ref_counts, int64_t page_size,
                   const AdaTensor* seqs, void* stream) {
    PagesLaunch L;
    int rc = pages_table(page_table, seq_lens, ref_counts, page_size, &L);
    if (rc || (rc = check_ints(seqs, "seqs", -1))) return rc;
    L.n = seqs->shape[0];
    if (L.n == 0) return ADA_OK;
    if (L.n > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many sequences");
    if ((rc = device_status_word(&L.status))) return rc;
    L.dst = static_cast<const int32_t*>(seqs->data);
    rc = launch_pages_share(L, false, static_cast<cudaStream_t>(stream));
    return rc ? fail(rc, "free launch failed: %s", cudaGetErrorString(cudaGetLastError())) : ADA_OK;
}

int ada_pages_fork(AdaTensor* page_table, AdaTensor* seq_lens, AdaTensor* ref_counts, int64_t page_size,
                   const AdaTensor* src, const AdaTensor* dst, void* stream) {
    PagesLaunch L;
    int rc = pages_table(page_table, seq_lens, ref_counts, page_size, &L);
    if (rc || (rc = check_ints(src, "src", -1)) || (rc = check_ints(dst, "dst", src->shape[0]))) return rc;
    L.n = src->shape[0];
    if (L.n == 0) return ADA_OK;
    if (L.n > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many sequences");
    if ((rc = device_status_word(&L.status))) return rc;
    L.src = static_cast<const int32_t*>(src->data);
    L.dst = static_cast<const int32_t*>(dst->data);
    rc = launch_pages_share(L, true, static_cast<cudaStream_t>(stream));
    return rc ? fail(rc, "fork launch failed: %s", cudaGetErrorString(cudaGetLastError())) : ADA_OK;
}

int ada_pages_reserve(const AdaTensor* pages, AdaTensor* page_table, AdaTensor* seq_lens, AdaTensor* ref_counts,
                      int64_t page_size, const AdaTensor* seqs, const AdaTensor* new_tokens, AdaTensor* granted,
                      void* workspace, size_t workspace_bytes, void* stream) {
    PagesLaunch L;
    int rc = pages_table(page_table, seq_lens, ref_counts, page_size, &L);
    if (rc || (rc = check_ints(seqs, "seqs", -1)) || (rc = check_ints(new_tokens, "new_tokens", seqs->shape[0])) ||
        (rc = check_ints(granted, "granted", seqs->shape[0])))
        return rc;
    L.n = seqs->shape[0];
    if (L.n > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many sequences");
    if ((rc = pages_data(pages, workspace, workspace_bytes, &L))) return rc;
    if (L.n == 0) return ADA_OK;
    L.src = static_cast<const int32_t*>(seqs->data);
    L.extra = static_cast<const int32_t*>(new_tokens->data);
    L.granted = static_cast<int32_t*>(granted->data);
    rc = launch_pages_alloc(L, false, static_cast<cudaStream_t>(stream));
    return rc ? fail(rc, "reserve launch failed: %s", cudaGetErrorString(cudaGetLastError())) : ADA_OK;
}

int ada_pages_copy(AdaTensor* pages, AdaTensor* page_table, AdaTensor* seq_lens, AdaTensor* ref_counts,
                   int64_t page_size, const AdaTensor* src, const AdaTensor* dst, AdaTensor* granted, void* workspace,
                   size_t workspace_bytes, void* stream) {
    PagesLaunch L;
    int rc = pages_table(page_table, seq_lens, ref_counts, page_size, &L);
    if (rc || (rc = check_ints(src, "src", -1)) || (rc = check_ints(dst, "dst", src->shape[0])) ||
        (rc = check_ints(granted, "granted", src->shape[0])))
        return rc;
    L.n = src->shape[0];
    if (L.n > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many sequences");
    if ((rc = pages_data(pages, workspace, workspace_bytes, &L))) return rc;
    if (L.n == 0) return ADA_OK;
    L.src = static_cast<const int32_t*>(src->data);
    L.dst = static_cast<const int32_t*>(dst->data);
    L.granted = static_cast<int32_t*>(granted->data);
    rc = launch_pages_alloc(L, true, static_cast<cudaStream_t>(stream));
    return rc ? fail(rc, "copy launch failed: %s", cudaGetErrorString(cudaGetLastError())) : ADA_OK;
}

int ada_pages_compact(AdaTensor* pages, AdaTensor* page_table, AdaTensor* seq_lens, AdaTensor* ref_counts,
                      int64_t page_size, AdaTensor* live, void* workspace, size_t workspace_bytes, void* stream) {
    PagesLaunch L;
    int rc = pages_table(page_table, seq_lens, ref_counts, page_size, &L);
    if (rc || (rc = check_ints(live, "live", 1))) return rc;
    L.n = 0;
    if ((rc = pages_data(pages, workspace, workspace_bytes, &L))) return rc;
    L.granted = static_cast<int32_t*>(live->data);
    rc = launch_pages_compact(L, static_cast<cudaStream_t>(stream));
    return rc ? fail(rc, "compact launch failed: %s", cudaGetErrorString(cudaGetLastError())) : ADA_OK;
}

int ada_token_logprobs(const AdaTensor* logits, const AdaTensor* tokens, int64_t ignore_index, int32_t top_k,
                       float* logprobs, float* entropy, float* lse, float* stats, float* top_logprobs,
                       int64_t* top_tokens, void* stream) {
    LogprobLaunch L;
    int rc = logits_setup(logits, &L);
    if (rc || (rc = check_row_tokens(tokens, L.rows, &L))) return rc;
    if (top_k < 0 || top_k > 64) return fail(ADA_ERR_UNSUPPORTED, "top_k %d outside [0, 64]", top_k);
    if (top_k > L.V) return fail(ADA_ERR_SHAPE, "top_k %d exceeds the vocabulary", top_k);
    if (L.rows == 0) return ADA_OK;
    if (logprobs == nullptr || entropy == nullptr || lse == nullptr ||
        (top_k > 0 && (top_logprobs == nullptr || top_tokens == nullptr)))
        return fail(ADA_ERR_INVALID, "null output");
    L.ignore = ignore_index;
    L.top = top_k;
    L.logprobs = logprobs;
    L.entropy = entropy;
    L.lse = lse;
    L.stats = stats;
    L.top_logprobs = top_logprobs;
    L.top_tokens = top_tokens;
    if (L.rows * 8 > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many rows");
    int sms;
    if ((rc = device_status_word(&L.status)) || (rc = sm_count(&sms))) return rc;
    // Few rows: a cluster of up to 8 CTAs per row, while the CTAs are at most
    // two per SM and each still has a round of 4096 logits.
    L.cluster = 1;
    const int64_t rounds = (L.V + 4095) / 4096;
    while (L.cluster < 8 && L.rows * L.cluster * 2 <= 2 * sms && L.cluster * 2 <= rounds) L.cluster *= 2;
    rc = launch_token_logprobs(L, static_cast<cudaStream_t>(stream));
    return rc ? fail(rc, "token log-probability launch failed: %s", cudaGetErrorString(cudaGetLastError())) : ADA_OK;
}

int ada_token_logprobs_bwd(const AdaTensor* logits, const AdaTensor* tokens, int64_t ignore_index, const float* stats,
                           const float* entropy, const float* g_logprobs, const float* g_entropy, const float* g_lse,
                           AdaTensor* grad, void* stream) {
    LogprobLaunch L;
    int rc = logits_setup(logits, &L);
    if (rc || (rc = check_row_tokens(tokens, L.rows, &L)) || (rc = check_view(grad, "grad", 3))) return rc;
    if (grad->dtype != logits->dtype) return fail(ADA_ERR_DTYPE, "grad must have the logits' dtype");
    for (int i = 0; i < 3; ++i)
        if (grad->shape[i] != logits->shape[i]) return fail(ADA_ERR_SHAPE, "grad and logits differ in extent %d", i);
    if ((rc = check_apart(grad, "grad"))) return rc;
    if (L.rows == 0) return ADA_OK;
    if (stats == nullptr || entropy == nullptr) return fail(ADA_ERR_INVALID, "null argument");
    L.ignore = ignore_index;
    L.stats = const_cast<float*>(stats);
    L.entropy = const_cast<float*>(entropy);
    L.g_logprobs = g_logprobs;
    L.g_entropy = g_entropy;
    L.g_lse = g_lse;
    L.grad = grad->data;
    L.gs0 = row_stride(grad, 0);
    L.gs1 = row_stride(grad, 1);
    if (L.rows * 8 > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many rows");
    int sms;
    if ((rc = device_status_word(&L.status)) || (rc = sm_count(&sms))) return rc;
    // Blocks to fill the GPU eight deep, of at least a round of 4096 logits each.
    const int64_t rounds = (L.V + 4095) / 4096;
    L.segments = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rounds, (int64_t(sms) * 8 + L.rows - 1) / L.rows)));
    if (L.rows * L.segments > kMaxInt) return fail(ADA_ERR_UNSUPPORTED, "too many rows");
    rc = launch_token_logprobs_bwd(L, static_cast<cudaStream_t>(stream));
    return rc ? fail(rc, "token log-probability gradient launch failed: %s", cudaGetErrorString(cudaGetLastError())) : ADA_OK;
}

}  // extern "C"
