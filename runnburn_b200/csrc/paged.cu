// Operators of a paged key-value cache (declarations: include/rnb_b200.h): checks of arguments and launches.
#include <cuda.h>

#include <algorithm>

#include "launch_k.hpp"
#include "paged.cuh"
#include "paged_decode.cuh"
#include "paged_prefill.cuh"

namespace rnb {

// The library's device for the length of a call, whatever device the caller has current.
struct PkCall {
    std::lock_guard<std::mutex> g;
    State &st;
    int before = -1, rc;
    PkCall() : g(state_mutex()), st(state()) { rc = enter(); }
    ~PkCall() {
        if (before >= 0 && before != st.device) cudaSetDevice(before);
    }
    int enter() {
        RNB_CU(cudaGetDevice(&before));
        RNB_TRY(st.open());
        if (before != st.device) RNB_CU(cudaSetDevice(st.device));
        return RNB_B200_OK;
    }
};

static int pk_bad(const char *what) { return fail(RNB_B200_VALIDATION_FAILED, "paged cache: %s", what); }

struct PkStep {
    uint64_t stride, n;
};
// Steps from the smallest to the largest: each at least what the ones below it span, so that no two rows of `dim` elements overlap.  A stride that is
// never stepped (one head) may be anything.
static bool pk_steps_apart(PkStep *steps, int n, uint64_t dim) {
    std::sort(steps, steps + n, [](const PkStep &a, const PkStep &b) { return a.stride < b.stride; });
    unsigned __int128 span = dim;
    for (int i = 0; i < n; i++) {
        if (steps[i].n == 1) continue;
        if (steps[i].stride < span) return false;
        span += (unsigned __int128)steps[i].stride * (steps[i].n - 1);
    }
    return true;
}
// Whether two pools of such steps, in ascending order, share elements when they begin d elements apart: some difference of two rows is d to within a row.
// From the largest step down, what is left of d has to be below one step: the ones below do not span more.
static bool pk_pools_meet(const PkStep *steps, int n, uint64_t dim, int64_t d) {
    if (n == 0) return d < (int64_t)dim && -d < (int64_t)dim;
    const PkStep &s = steps[n - 1];
    if (s.n == 1) return pk_pools_meet(steps, n - 1, dim, d);
    const int64_t stride = (int64_t)s.stride, most = (int64_t)s.n - 1, low = d / stride - (d % stride < 0 ? 1 : 0);
    for (int64_t i = low; i <= low + 1; i++)
        if (i >= -most && i <= most && pk_pools_meet(steps, n - 1, dim, d - i * stride)) return true;
    return false;
}
// For calls that write: layers of a pool, and keys and values, must not share elements.
static int pk_check_written(const rnb_b200_paged_cache *c, size_t n_layers, uint64_t layer_stride) {
    const uint64_t dim = (uint64_t)c->head_dim;
    PkStep steps[4] = {{c->page_stride, (uint64_t)c->n_pages}, {c->pos_stride, (uint64_t)c->page_size}, {c->head_stride, (uint64_t)c->kv_heads}, {layer_stride, (uint64_t)n_layers}};
    if (!pk_steps_apart(steps, 4, dim)) return pk_bad("layers overlap: a stride is smaller than what lies below it");
    if (pk_pools_meet(steps, 4, dim, ((int64_t)(uintptr_t)c->v - (int64_t)(uintptr_t)c->k) / 2)) return pk_bad("keys and values overlap");
    return RNB_B200_OK;
}

static int pk_check_cache(const rnb_b200_paged_cache *c, PkCache *out) {
    if (!c || !c->k || !c->v) return fail(RNB_B200_VALIDATION_FAILED, "null pointer argument");
    if (c->type != RNB_B200_TYPE_F16 && c->type != RNB_B200_TYPE_BF16) return fail(RNB_B200_UNSUPPORTED, "paged cache: type must be F16 or BF16, got %u", c->type);
    if (c->head_dim < 8 || c->head_dim > 512 || c->head_dim % 8) return fail(RNB_B200_VALIDATION_FAILED, "paged cache: head_dim must be a multiple of 8 up to 512, got %d", c->head_dim);
    if (c->kv_heads < 1 || c->kv_heads > 65535) return fail(RNB_B200_VALIDATION_FAILED, "paged cache: kv_heads must be in 1..65535, got %d", c->kv_heads);
    if (c->page_size < 8 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return fail(RNB_B200_VALIDATION_FAILED, "paged cache: page_size must be a power of two from 8 to 256, got %d", c->page_size);
    if (c->n_pages < 1) return fail(RNB_B200_VALIDATION_FAILED, "paged cache: n_pages must be at least 1, got %d", c->n_pages);
    PkStep steps[3] = {{c->page_stride, (uint64_t)c->n_pages}, {c->pos_stride, (uint64_t)c->page_size}, {c->head_stride, (uint64_t)c->kv_heads}};
    for (const PkStep &s : steps)
        if (s.n > 1 && (s.stride % 8 || s.stride > (uint64_t)1 << 38)) return pk_bad("strides must be multiples of 8 elements, at most 2^38");
    if (!pk_steps_apart(steps, 3, (uint64_t)c->head_dim)) return pk_bad("rows overlap: a stride is smaller than what lies below it");
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15u) return pk_bad("k and v must be 16-byte aligned");
    int shift = 0;
    while ((1 << shift) < c->page_size) shift++;
    *out = {(uint16_t *)c->k, (uint16_t *)c->v, c->page_stride, c->pos_stride, c->head_stride, c->n_pages, shift, c->kv_heads, c->head_dim};
    return RNB_B200_OK;
}
static int pk_check_batch(const rnb_b200_paged_batch *b, PkBatch *out) {
    if (!b) return fail(RNB_B200_VALIDATION_FAILED, "null pointer argument");
    if (b->n_seq < 0 || b->n_tokens < 0) return pk_bad("n_seq and n_tokens must not be negative");
    if (!b->q_start && b->n_tokens != b->n_seq) return fail(RNB_B200_VALIDATION_FAILED, "paged cache: one token per sequence without q_start, got %d tokens of %d sequences", b->n_tokens, b->n_seq);
    if (b->n_seq > 0 && (!b->table || !b->kv_len)) return fail(RNB_B200_VALIDATION_FAILED, "null pointer argument");
    if (b->max_pages < 1 || b->table_stride < b->max_pages) return pk_bad("max_pages must be at least 1 and table_stride at least max_pages");
    if (((uintptr_t)b->table | (uintptr_t)b->kv_len | (uintptr_t)b->q_start) & 3u) return pk_bad("table, kv_len and q_start must be 4-byte aligned");
    *out = {b->table, b->kv_len, b->q_start, b->table_stride, b->max_pages, b->n_seq, b->n_tokens};
    return RNB_B200_OK;
}

// ---- append and copy ----------------------------------------------------------------------------------
static int pk_append(const rnb_b200_paged_cache *cache, const rnb_b200_paged_batch *batch, uint32_t src_type, const void *k_new, const void *v_new, size_t src_stride,
                     cudaStream_t s) {
    PkCache c{};
    PkBatch b{};
    RNB_TRY(pk_check_cache(cache, &c));
    RNB_TRY(pk_check_batch(batch, &b));
    if (src_type != RNB_B200_TYPE_F32 && src_type != cache->type) return fail(RNB_B200_UNSUPPORTED, "paged cache: rows must be F32 or of the cache's type, got type %u", src_type);
    if (b.n_tokens == 0 || b.n_seq == 0) return RNB_B200_OK;
    if (!k_new || !v_new) return fail(RNB_B200_VALIDATION_FAILED, "null pointer argument");
    if (((uintptr_t)k_new | (uintptr_t)v_new) & 15u || src_stride % 8) return pk_bad("rows must be 16-byte aligned and src_stride a multiple of 8");
    if (b.n_tokens > 1 && src_stride < (size_t)c.kv_heads * c.head_dim) return pk_bad("src_stride is smaller than a token's rows");
    RNB_TRY(pk_check_written(cache, 1, 0));
    PkCall call;
    RNB_TRY(call.rc);
    const dim3 grid((unsigned)b.n_tokens), block((unsigned)std::min(256, (c.kv_heads * c.head_dim / 8 + 31) / 32 * 32));
    int *err = call.st.dev_error;
    if (cache->type == RNB_B200_TYPE_F16) {
        if (src_type == RNB_B200_TYPE_F32) RNB_CU(launch_k(paged_append_kernel<float, F16>, grid, block, 0, s, c, b, (const float *)k_new, (const float *)v_new, src_stride, err));
        else RNB_CU(launch_k(paged_append_kernel<F16, F16>, grid, block, 0, s, c, b, (const F16 *)k_new, (const F16 *)v_new, src_stride, err));
    } else {
        if (src_type == RNB_B200_TYPE_F32) RNB_CU(launch_k(paged_append_kernel<float, Bf16>, grid, block, 0, s, c, b, (const float *)k_new, (const float *)v_new, src_stride, err));
        else RNB_CU(launch_k(paged_append_kernel<Bf16, Bf16>, grid, block, 0, s, c, b, (const Bf16 *)k_new, (const Bf16 *)v_new, src_stride, err));
    }
    return RNB_B200_OK;
}

template <int N>
static int pk_copy_some(const PkCache &c, size_t n_layers, uint64_t layer_stride, const int32_t *src, const int32_t *dst, const int32_t *rows, size_t n, cudaStream_t s) {
    PkPairs<N> pairs;
    pairs.n = (int)n;
    for (size_t i = 0; i < n; i++) {
        pairs.src[i] = src[i];
        pairs.dst[i] = dst[i];
        pairs.rows[i] = rows ? rows[i] : 1 << c.page_shift;
    }
    const int chunks = (c.kv_heads * c.head_dim / 8) << c.page_shift;
    const dim3 grid((unsigned)n, (unsigned)std::min(64, (chunks + 1023) / 1024), (unsigned)(2 * n_layers));
    RNB_CU(launch_k(paged_copy_kernel<N>, grid, dim3(256), 0, s, c, layer_stride, pairs));
    return RNB_B200_OK;
}
static int pk_copy(const rnb_b200_paged_cache *cache, size_t n_layers, uint64_t layer_stride, const int32_t *src, const int32_t *dst, const int32_t *rows, size_t n,
                   cudaStream_t s) {
    PkCache c{};
    RNB_TRY(pk_check_cache(cache, &c));
    if (n_layers < 1 || n_layers > 32767) return fail(RNB_B200_VALIDATION_FAILED, "paged cache: n_layers must be in 1..32767, got %zu", n_layers);
    if (layer_stride % 8 || layer_stride > (uint64_t)1 << 38 || (n_layers > 1 && layer_stride < (uint64_t)c.head_dim))
        return pk_bad("layer_stride must be a multiple of 8 below 2^38 and at least head_dim");
    if (n == 0) return RNB_B200_OK;
    if (!src || !dst) return fail(RNB_B200_VALIDATION_FAILED, "null pointer argument");
    if (n > (size_t)c.n_pages) return pk_bad("more copies than pages");
    std::vector<uint8_t> role(c.n_pages, 0);   // 1: read, 2: written
    for (size_t i = 0; i < n; i++) {
        if (src[i] < 0 || src[i] >= c.n_pages || dst[i] < 0 || dst[i] >= c.n_pages)
            return fail(RNB_B200_VALIDATION_FAILED, "paged cache: copy %zu is of page %d to page %d, the pool has %d", i, src[i], dst[i], c.n_pages);
        if (rows && (rows[i] < 0 || rows[i] > 1 << c.page_shift))
            return fail(RNB_B200_VALIDATION_FAILED, "paged cache: copy %zu is of %d positions, a page has %d", i, rows[i], 1 << c.page_shift);
        if (role[src[i]] & 2 || role[dst[i]] || src[i] == dst[i])
            return fail(RNB_B200_VALIDATION_FAILED, "paged cache: copy %zu (page %d to page %d): a page is written twice, or read and written", i, src[i], dst[i]);
        role[src[i]] = 1;
        role[dst[i]] = 2;
    }
    RNB_TRY(pk_check_written(cache, n_layers, layer_stride));
    PkCall call;
    RNB_TRY(call.rc);
    for (size_t at = 0; at < n;) {
        const size_t left = n - at, m = left > 64 ? std::min<size_t>(left, 2048) : left;
        if (m > 64) RNB_TRY(pk_copy_some<2048>(c, n_layers, layer_stride, src + at, dst + at, rows ? rows + at : nullptr, m, s));
        else RNB_TRY(pk_copy_some<64>(c, n_layers, layer_stride, src + at, dst + at, rows ? rows + at : nullptr, m, s));
        at += m;
    }
    return RNB_B200_OK;
}

// ---- attention ------------------------------------------------------------------------------------------
struct PkAttention {   // a checked call
    PkCache c{};
    PkBatch b{};
    uint32_t q_type, c_type;
    const void *q;
    size_t q_stride, out_stride;
    int heads, window, sinks;
    float scale;
    void *out, *workspace;
    float *lse;
};
// the mark and the counters, and two records for every CTA of the decode kernel; the prompts' kernel joins in shared memory
constexpr int PK_MAX_SMS = 148;
constexpr size_t PK_WORKSPACE_BYTES = PD_WS_RECORDS + (size_t)PK_MAX_SMS * 2 * std::max({PdShape<64, 1>::PER_SM * PdShape<64, 1>::RECORD, PdShape<64, 2>::PER_SM * PdShape<64, 2>::RECORD,
                                                                                         PdShape<128, 1>::PER_SM * PdShape<128, 1>::RECORD, PdShape<128, 2>::PER_SM * PdShape<128, 2>::RECORD});
static_assert(PD_WS_RECORDS % 256 == 0, "records are read by 16 bytes");

// Whether two matrices share bytes: their ranges do, unless their rows lie beside each other in rows of one length.  strides in elements.
static bool pk_rows_meet(const void *x, size_t x_stride, const void *y, size_t y_stride, size_t row, size_t rows, size_t element) {
    const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
    const size_t xs = x_stride * element, ys = y_stride * element;
    if (a + (rows - 1) * xs + row <= b || b + (rows - 1) * ys + row <= a) return false;
    if (xs != ys || rows == 1) return true;
    const size_t d = a > b ? (a - b) % xs : (b - a) % xs;
    return d < row || xs - d < row;
}

static int pk_check_attention(const rnb_b200_paged_cache *cache, const rnb_b200_paged_batch *batch, uint32_t q_type, const void *q, size_t q_stride, size_t num_heads,
                              float scale, int32_t window, int32_t sinks, void *workspace, size_t workspace_bytes, void *out, size_t out_stride, float *lse, PkAttention *a) {
    RNB_TRY(pk_check_cache(cache, &a->c));
    RNB_TRY(pk_check_batch(batch, &a->b));
    if (cache->head_dim != 64 && cache->head_dim != 128) return fail(RNB_B200_UNSUPPORTED, "paged attention: head_dim must be 64 or 128, got %d", cache->head_dim);
    if (num_heads == 0 || num_heads > 65535 || num_heads % (size_t)cache->kv_heads != 0)
        return fail(RNB_B200_VALIDATION_FAILED, "attention: num_heads(%zu) must be a multiple of num_kv_heads(%d)", num_heads, cache->kv_heads);
    if (!(q_type == cache->type || (q_type == RNB_B200_TYPE_F32 && cache->type == RNB_B200_TYPE_F16)))
        return fail(RNB_B200_UNSUPPORTED, "paged attention: queries must be F32 on an F16 cache or of the cache's type, got type %u on %u", q_type, cache->type);
    if (window < 0 || sinks < 0) return fail(RNB_B200_VALIDATION_FAILED, "paged attention: window and sinks must not be negative, got %d and %d", window, sinks);
    const float to_log2 = scale * 1.4426950408889634f;
    if (!(to_log2 - to_log2 == 0.f)) return fail(RNB_B200_VALIDATION_FAILED, "paged attention: scale must be finite, and so must scale * log2(e)");
    if (!workspace || ((uintptr_t)workspace & 255u) || workspace_bytes < PK_WORKSPACE_BYTES)
        return fail(RNB_B200_VALIDATION_FAILED, "paged attention: the workspace must be 256-byte aligned and hold %zu bytes, got %zu", PK_WORKSPACE_BYTES, workspace_bytes);
    if (a->b.n_tokens > 0 && (!q || !out)) return fail(RNB_B200_VALIDATION_FAILED, "null pointer argument");
    if (((uintptr_t)q | (uintptr_t)out) & 15u || q_stride % 8 || out_stride % 8 || ((uintptr_t)lse & 3u))
        return fail(RNB_B200_VALIDATION_FAILED, "paged attention: q and out must be 16-byte aligned with strides that are multiples of 8, lse 4-byte aligned");
    if (a->b.n_tokens > 1 && (q_stride < num_heads * cache->head_dim || out_stride < num_heads * cache->head_dim))
        return fail(RNB_B200_VALIDATION_FAILED, "paged attention: q_stride and out_stride must be at least num_heads * head_dim");
    if (a->b.n_tokens > 0 && pk_rows_meet(q, q_stride, out, out_stride, num_heads * cache->head_dim * (q_type == RNB_B200_TYPE_F32 ? 4 : 2), (size_t)a->b.n_tokens, q_type == RNB_B200_TYPE_F32 ? 4 : 2))
        return fail(RNB_B200_VALIDATION_FAILED, "paged attention: q and out must not overlap");
    a->q_type = q_type;
    a->c_type = cache->type;
    a->q = q;
    a->q_stride = q_stride;
    a->out_stride = out_stride;
    a->heads = (int)num_heads;
    a->window = window;
    a->sinks = window ? sinks : 0;
    a->scale = scale;
    a->out = out;
    a->workspace = workspace;
    a->lse = lse;
    return RNB_B200_OK;
}

static int pk_encode_tiled(PkTensorMap *out, void *base, uint32_t type, uint32_t rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box, const char *what) {
    static_assert(sizeof(PkTensorMap) == sizeof(CUtensorMap) && alignof(PkTensorMap) >= alignof(CUtensorMap), "descriptor size");
    typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                    const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeTiled encode = nullptr;   // under the library's lock
    if (!encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        RNB_CU(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
        if (q != cudaDriverEntryPointSuccess || !fn) return fail(RNB_B200_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
        encode = reinterpret_cast<EncodeTiled>(fn);
    }
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    const CUresult r = encode(reinterpret_cast<CUtensorMap *>(out), type == RNB_B200_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, base, dims,
                              strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(RNB_B200_CUDA_ERROR, "cuTensorMapEncodeTiled(%s) failed with driver code %d", what, (int)r);
    return RNB_B200_OK;
}
// keys: positions of a box; parts: 64-element parts of a row in it
static int pk_encode(PkTensorMap *out, void *base, const PkAttention &a, int keys, int parts) {
    const PkCache &c = a.c;
    auto step = [](uint64_t stride, uint64_t n) { return (cuuint64_t)(n > 1 ? stride * 2 : 128); };   // of one entry only: never stepped
    const cuuint64_t page = (cuuint64_t)1 << c.page_shift;
    const cuuint64_t dims[5] = {64, page, (cuuint64_t)c.head_dim / 64, (cuuint64_t)c.kv_heads, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[4] = {step(c.pos_stride, page), 128, step(c.head_stride, c.kv_heads), step(c.page_stride, c.n_pages)};
    const cuuint32_t box[5] = {64, (cuuint32_t)std::min<cuuint64_t>(page, keys), (cuuint32_t)parts, 1, 1};
    return pk_encode_tiled(out, base, a.c_type, 5, dims, strides, box, "pages");
}

template <class Q, class C, int D, int HT>
static int pk_decode_launch(const PkAttention &a, cudaStream_t s, State &st) {
    using S = PdShape<D, HT>;
    static bool ready = false;   // under the library's lock; one device
    if (!ready) RNB_CU(cudaFuncSetAttribute(paged_decode_kernel<Q, C, D, HT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM));
    ready = true;
    PdParams P{};
    P.q = a.q;
    P.q_stride = a.q_stride;
    P.out_stride = a.out_stride;
    P.heads = a.heads;
    P.group = a.heads / a.c.kv_heads;
    P.splits = (P.group + 8 * HT - 1) / (8 * HT);
    P.window = a.window;
    P.sinks = a.sinks;
    P.scale_log2 = a.scale * 1.4426950408889634f;
    P.out = a.out;
    P.lse = a.lse;
    P.workspace = (uint8_t *)a.workspace;
    P.err = st.dev_error;
    // tiles are counted in 31 bits: of a sequence at most what its table holds, or its window and sinks with the tiles that they begin in
    const uint64_t held = (((uint64_t)a.b.max_pages << a.c.page_shift) + PD_TILE - 1) / PD_TILE, seen = ((uint64_t)a.window + a.sinks) / PD_TILE + 4;
    if ((uint64_t)a.b.n_seq * (a.window ? std::min(held, seen) : held) * P.splits * a.c.kv_heads > 0x7fffffffu)
        return fail(RNB_B200_UNSUPPORTED, "paged attention: %d sequences with tables of %d pages are more than a launch can have", a.b.n_seq, a.b.max_pages);
    const int grid = std::min(st.sm_count, PK_MAX_SMS) * S::PER_SM;
    static_assert(PK_MAX_SMS * S::PER_SM <= PD_MAX_GRID && PK_MAX_SMS * S::PER_SM * 2 * S::RECORD <= PK_WORKSPACE_BYTES - PD_WS_RECORDS, "records");
    PkMaps maps;
    RNB_TRY(pk_encode(&maps.k, a.c.k, a, PD_TILE, D / 64));
    RNB_TRY(pk_encode(&maps.v, a.c.v, a, PD_TILE, D / 64));
    RNB_CU(launch_k(paged_decode_kernel<Q, C, D, HT>, dim3((unsigned)grid), dim3(S::THREADS), S::SMEM, s, a.c, a.b, P, maps));
    return RNB_B200_OK;
}
// Up to eight query heads per key head: four warps; more: eight warps, 16 heads at a time.
template <class Q, class C>
static int pk_decode(const PkAttention &a, cudaStream_t s, State &st) {
    const bool many = a.heads / a.c.kv_heads > 8;
    if (a.c.head_dim == 64) return many ? pk_decode_launch<Q, C, 64, 2>(a, s, st) : pk_decode_launch<Q, C, 64, 1>(a, s, st);
    return many ? pk_decode_launch<Q, C, 128, 2>(a, s, st) : pk_decode_launch<Q, C, 128, 1>(a, s, st);
}
template <class Q, class C, int D>
static int pk_prefill(const PkAttention &a, cudaStream_t s, State &st) {
    using S = PpShape<Q, D>;
    static bool ready = false;
    if (!ready) RNB_CU(cudaFuncSetAttribute(paged_prefill_kernel<Q, C, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM));
    ready = true;
    PpParams P{};
    P.q = a.q;
    P.q_stride = a.q_stride;
    P.out_stride = a.out_stride;
    P.heads = a.heads;
    P.group = a.heads / a.c.kv_heads;
    P.blocks = (P.group + 127) / 128;
    P.per_block = (P.group + P.blocks - 1) / P.blocks;
    P.queries = 128 / P.per_block;
    P.window = a.window;
    P.sinks = a.sinks;
    P.scale = a.scale;
    P.out = a.out;
    P.lse = a.lse;
    P.err = st.dev_error;
    P.by_vh = pp_by((uint32_t)(a.c.kv_heads * P.blocks));
    P.by_rows = pp_by((uint32_t)(S::BLOCKS * P.queries));
    P.by_heads = (65536 + P.per_block - 1) / P.per_block;
    PpMaps maps{};
    RNB_TRY(pk_encode(&maps.k, a.c.k, a, PP_KEYS, 1));
    RNB_TRY(pk_encode(&maps.v, a.c.v, a, PP_KEYS, 1));
    if (sizeof(Q) == 2) {
        const cuuint64_t dims[4] = {64, (cuuint64_t)a.heads, (cuuint64_t)a.b.n_tokens, D / 64}, strides[3] = {D * 2, (cuuint64_t)(a.b.n_tokens > 1 ? a.q_stride * 2 : 128), 128};
        const cuuint32_t box[4] = {64, (cuuint32_t)P.per_block, (cuuint32_t)P.queries, 1};
        RNB_TRY(pk_encode_tiled(&maps.q, const_cast<void *>(a.q), a.c_type, 4, dims, strides, box, "queries"));
    }
    // Pairs of row blocks: the starts are on the device, so there is one more per sequence than the tokens could need.
    const size_t pairs = std::min<size_t>((size_t)a.b.n_tokens, (size_t)a.b.n_tokens / (S::BLOCKS * P.queries) + (size_t)a.b.n_seq) * a.c.kv_heads * P.blocks;
    if (pairs > 0x7fffffffu) return fail(RNB_B200_UNSUPPORTED, "paged attention: %zu blocks of rows are more than a launch can have", pairs);
    // How many tiles there are is taken from the table's width, since the lengths are on the device: a table that is wider than its sequences need (a captured
    // step's) is shared out as if they were as long (four prompts of 200 tokens, f32: 44.5 us with a table of 131072 positions, 20.9 with one that fits).
    // Keys are shared out where the launch leaves most of the chip idle, down to one tile of what a pair could see for each: a join costs less than a tile
    // (33 tokens of f32 behind 300 positions: 11.3 us, without 16.5).
    long long tiles = (((long long)a.b.max_pages << a.c.page_shift) + PP_KEYS - 1) / PP_KEYS;
    if (a.window) tiles = std::min(tiles, ((long long)a.window + a.sinks + S::BLOCKS * P.queries) / PP_KEYS + 3);
    unsigned ranks = 1;
    while (ranks < PP_MAX_CLUSTER && pairs * ranks * 2 <= (size_t)std::min(st.sm_count, PK_MAX_SMS) && tiles > (long long)ranks) ranks *= 2;
    // Several sequences are seldom of one length, and the longest decides: where it takes longer than all SMs need for halves of everything, lengths spread
    // evenly from nothing on and a CTA costing FIXED tiles' time beside its tiles, two share (3 sequences of up to 512 tokens behind up to 6000, 32 heads on 8:
    // 70 us, without 92; 10 of up to 100: 55, without 83; 9 of up to 512, which the rule leaves alone: 145, without 118.  Four alike of 200: 106, without 98).
    constexpr long long FIXED = 6;
    if (ranks == 1 && a.b.n_seq > 2 && (long long)pairs * (tiles + 4 * FIXED) * 10 < 17 * (tiles + FIXED) * std::min(st.sm_count, PK_MAX_SMS)) ranks = 2;
    if (ranks == 1) RNB_CU(launch_k(paged_prefill_kernel<Q, C, D>, dim3((unsigned)pairs), dim3(PP_THREADS), S::SMEM, s, a.c, a.b, P, maps));
    else RNB_CU(launch_k_cluster(paged_prefill_kernel<Q, C, D>, dim3((unsigned)pairs * ranks), dim3(PP_THREADS), S::SMEM, s, dim3(ranks), a.c, a.b, P, maps));
    return RNB_B200_OK;
}
template <class Q, class C>
static int pk_attention_of(const PkAttention &a, cudaStream_t s, State &st) {
    if (!a.b.q_start) return pk_decode<Q, C>(a, s, st);
    return a.c.head_dim == 64 ? pk_prefill<Q, C, 64>(a, s, st) : pk_prefill<Q, C, 128>(a, s, st);
}
static int pk_attention(const PkAttention &a, cudaStream_t s) {
    if (a.b.n_tokens == 0 || a.b.n_seq == 0) return RNB_B200_OK;
    PkCall call;
    RNB_TRY(call.rc);
    if (a.q_type == RNB_B200_TYPE_F32) return pk_attention_of<float, F16>(a, s, call.st);
    return a.q_type == RNB_B200_TYPE_F16 ? pk_attention_of<F16, F16>(a, s, call.st) : pk_attention_of<Bf16, Bf16>(a, s, call.st);
}

// Nothing is thrown through the C entries.
template <class F>
static int pk_guarded(F &&f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return fail(RNB_B200_OUT_OF_MEMORY, "paged cache: out of host memory");
    }
}

}  // namespace rnb

using namespace rnb;

extern "C" {

int rnb_b200_dev_paged_kv_append(const rnb_b200_paged_cache *cache, const rnb_b200_paged_batch *batch, uint32_t src_type, const void *k_new, const void *v_new,
                                 size_t src_stride, void *stream) {
    return pk_append(cache, batch, src_type, k_new, v_new, src_stride, (cudaStream_t)stream);
}
int rnb_b200_dev_paged_kv_copy(const rnb_b200_paged_cache *cache, size_t n_layers, uint64_t layer_stride, const int32_t *src, const int32_t *dst, const int32_t *rows,
                               size_t n_pages, void *stream) {
    return pk_guarded([&] { return pk_copy(cache, n_layers, layer_stride, src, dst, rows, n_pages, (cudaStream_t)stream); });
}
size_t rnb_b200_paged_workspace_bytes(void) { return PK_WORKSPACE_BYTES; }
int rnb_b200_paged_workspace_init(void *workspace, size_t workspace_bytes, void *stream) {
    if (!workspace || ((uintptr_t)workspace & 255u) || workspace_bytes < PK_WORKSPACE_BYTES)
        return fail(RNB_B200_VALIDATION_FAILED, "paged attention: the workspace must be 256-byte aligned and hold %zu bytes, got %zu", PK_WORKSPACE_BYTES, workspace_bytes);
    PkCall call;
    RNB_TRY(call.rc);
    RNB_CU(cudaMemsetAsync((uint8_t *)workspace + PD_WS_HEAD, 0, PD_WS_RECORDS - PD_WS_HEAD, (cudaStream_t)stream));
    RNB_CU(cudaMemsetAsync(workspace, (int)(PD_WS_MARK & 0xffu), PD_WS_HEAD, (cudaStream_t)stream));
    return RNB_B200_OK;
}
int rnb_b200_dev_attention_decode_paged(const rnb_b200_paged_cache *cache, const rnb_b200_paged_batch *batch, uint32_t q_type, const void *q, size_t q_stride,
                                        size_t num_heads, float scale, int32_t window, int32_t sinks, void *workspace, size_t workspace_bytes, void *out,
                                        size_t out_stride, float *lse, void *stream) {
    PkAttention a{};
    RNB_TRY(pk_check_attention(cache, batch, q_type, q, q_stride, num_heads, scale, window, sinks, workspace, workspace_bytes, out, out_stride, lse, &a));
    if (a.b.q_start) return fail(RNB_B200_VALIDATION_FAILED, "paged decode attention takes one token per sequence: q_start must be null");
    return pk_attention(a, (cudaStream_t)stream);
}
int rnb_b200_dev_attention_prefill_paged(const rnb_b200_paged_cache *cache, const rnb_b200_paged_batch *batch, uint32_t q_type, const void *q, size_t q_stride,
                                         size_t num_heads, float scale, int32_t window, int32_t sinks, void *workspace, size_t workspace_bytes, void *out,
                                         size_t out_stride, float *lse, void *stream) {
    PkAttention a{};
    RNB_TRY(pk_check_attention(cache, batch, q_type, q, q_stride, num_heads, scale, window, sinks, workspace, workspace_bytes, out, out_stride, lse, &a));
    return pk_attention(a, (cudaStream_t)stream);
}

}  // extern "C"
