// A key-value cache in pages: what its kernels share, and the kernels that write it.
//
// A pool holds pages of 2^page_shift positions; a table per sequence names the page of every 2^page_shift positions.  Tables, lengths
// and starts lie on the device and are checked here: what points outside raises DEV_ERR_BAD_PAGE and is left out.
#pragma once
#include "common.cuh"
#include "mma_types.cuh"

namespace rnb {

struct PkCache {
    uint16_t *k, *v;
    uint64_t page_stride, pos_stride, head_stride;   // elements
    int n_pages, page_shift, kv_heads, head_dim;
};
struct PkBatch {
    const int *table, *kv_len, *q_start;   // q_start null: row i is the one token of sequence i
    int table_stride, max_pages, n_seq, n_tokens;
};

#ifdef __CUDACC__
// Positions of a sequence, within what its table can hold, and so far below 2^31 that the end of a tile or page behind the last one is a position too.
constexpr int PK_MAX_POSITIONS = 0x7fffff00;
__device__ __forceinline__ int pk_length(const PkBatch &b, int page_shift, int seq, int *err) {
    const int n = b.kv_len[seq];
    const long long most = min((long long)b.max_pages << page_shift, (long long)PK_MAX_POSITIONS);
    if (n < 0 || n > most) {
        atomicExch(err, DEV_ERR_BAD_PAGE);
        return n < 0 ? 0 : (int)most;
    }
    return n;
}
struct PkRow {
    int seq, pos;   // sequence (-1: a row of padding) and position in it (below 0: nothing is seen)
};
// The sequence and position of a row of the token matrices.
__device__ __forceinline__ PkRow pk_row(const PkBatch &b, int page_shift, int row, int *err) {
    if (!b.q_start) return {row, pk_length(b, page_shift, row, err) - 1};
    int lo = 0, hi = b.n_seq;   // the last sequence that starts at or before the row, and has tokens
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (b.q_start[mid + 1] <= row) lo = mid + 1;
        else hi = mid;
    }
    if (lo == b.n_seq) return {-1, -1};
    const int start = b.q_start[lo], end = b.q_start[lo + 1];
    if (row < start || row >= end) return {-1, -1};   // starts out of order
    return {lo, pk_length(b, page_shift, lo, err) - (end - row)};
}
// Some threads of a launch look through the starts: from 0, not descending, within the token matrices.
__device__ __forceinline__ void pk_check_starts(const PkBatch &b, int thread, int threads, int *err) {
    if (!b.q_start) return;
    for (int i = thread; i <= b.n_seq; i += threads) {
        const int x = b.q_start[i];
        if (i == 0 ? x != 0 : x < b.q_start[i - 1]) atomicExch(err, DEV_ERR_BAD_PAGE);
        if (i == b.n_seq && x > b.n_tokens) atomicExch(err, DEV_ERR_BAD_PAGE);
    }
}
// The page of a position, or -1 where the table's entry is none.
__device__ __forceinline__ int pk_page(const PkBatch &b, const PkCache &c, int seq, int pos, int *err) {
    const int page = b.table[(size_t)seq * b.table_stride + (pos >> c.page_shift)];
    if ((unsigned)page < (unsigned)c.n_pages) return page;
    atomicExch(err, DEV_ERR_BAD_PAGE);
    return -1;
}

// Powers of two for a row of f32 queries that enters products as two f16 terms: `down` brings its largest absolute value to 2^14 .. 2^15, the top of f16, and
// `up` is its reciprocal.  Of an element 2^-k times as large the second term's step, 2^-24 at least, is 2^(k - 38) of it: 22 bits are kept up to k = 17, 19 up
// to k = 20.  (With the largest brought to one, rows with one element 10^4 times the others, where the keys have nothing, came out 6e-4 off; now 7.5e-7, as other rows.)
// `up` and `down` stay normal numbers: rows below 2^-112 are brought up by 2^126.
__device__ __forceinline__ void pk_factor(float most, float &down, float &up) {
    constexpr uint32_t TOP = 14, BIAS = 127;
    const uint32_t e = min(max(__float_as_uint(most) >> 23 & 0xffu, TOP + 1), 2 * BIAS);
    up = __uint_as_float((e - TOP) << 23);
    down = __uint_as_float((2 * BIAS + TOP - e) << 23);
}

// ---- append -----------------------------------------------------------------------------------------
// Rows of the call's tokens, rounded to the cache's type (to nearest, ties to even: the caches' one rounding), eight elements of K
// and of V a thread, a block per token: whatever the lengths, one pass finds the token's place.  Bound by HBM where there are tokens enough (4 prompts
// of up to 3000 tokens, 8 heads of 128, f32 to f16: 13.9 us, 5.3 TB/s), by the launch for a token or a few of each sequence (64: 5.7 us, two microseconds of it
// the way to the place: starts or row, length, table entry).
template <class Src, class Dst>
__device__ __forceinline__ uint4 pk_eight(const Src *p) {
    if constexpr (sizeof(Src) == 2) {
        return *reinterpret_cast<const uint4 *>(p);
    } else {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
        return make_uint4(pk_pack<Dst>(a.x, a.y), pk_pack<Dst>(a.z, a.w), pk_pack<Dst>(b.x, b.y), pk_pack<Dst>(b.z, b.w));
    }
}
template <class Src, class Dst>
RNB_GLOBAL void paged_append_kernel(PkCache c, PkBatch b, const Src *k_new, const Src *v_new, size_t src_stride, int *err) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x;
    if (row == 0) pk_check_starts(b, threadIdx.x, blockDim.x, err);
    const PkRow at = pk_row(b, c.page_shift, row, err);
    if (at.seq < 0) return;
    if (at.pos < 0) {   // more tokens than positions
        if (threadIdx.x == 0) atomicExch(err, DEV_ERR_BAD_PAGE);
        return;
    }
    const int page = pk_page(b, c, at.seq, at.pos, err);
    if (page < 0) return;
    const size_t dst = (size_t)page * c.page_stride + (size_t)(at.pos & ((1 << c.page_shift) - 1)) * c.pos_stride;
    const int per_head = c.head_dim / 8, n = c.kv_heads * per_head;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const size_t from = (size_t)row * src_stride + (size_t)i * 8, to = dst + (size_t)(i / per_head) * c.head_stride + (size_t)(i % per_head) * 8;
        const uint4 x = pk_eight<Src, Dst>(k_new + from), y = pk_eight<Src, Dst>(v_new + from);
        *reinterpret_cast<uint4 *>(c.k + to) = x;
        *reinterpret_cast<uint4 *>(c.v + to) = y;
    }
}

// ---- copies of pages ----------------------------------------------------------------------------------
// The list travels as a kernel parameter: nothing to upload, and a captured call keeps it.  16 bytes a thread at a time, K and V of every layer side by
// side in the grid; HBM-bound (500 pages of 64 positions, 8 heads of 128, in 4 layers: 165 us, 6.3 TB/s of reads and writes together) or, for few
// pages, bound by the launch (8 pages of 16 positions in 32 layers: 7.9 us).
template <int N>
struct PkPairs {
    int n;
    int src[N], dst[N], rows[N];
};
template <int N>
RNB_GLOBAL void paged_copy_kernel(PkCache c, uint64_t layer_stride, const __grid_constant__ PkPairs<N> pairs) {
    pdl_launch_dependents();
    pdl_wait();
    const int i = blockIdx.x, per_head = c.head_dim / 8, per_row = c.kv_heads * per_head, n = pairs.rows[i] * per_row;
    uint16_t *const pool = (blockIdx.z & 1 ? c.v : c.k) + (size_t)(blockIdx.z >> 1) * layer_stride;
    const uint16_t *const src = pool + (size_t)pairs.src[i] * c.page_stride;
    uint16_t *const dst = pool + (size_t)pairs.dst[i] * c.page_stride;
    for (int e = blockIdx.y * blockDim.x + threadIdx.x; e < n; e += gridDim.y * blockDim.x) {
        const int r = e / per_row, x = e % per_row;
        const size_t at = (size_t)r * c.pos_stride + (size_t)(x / per_head) * c.head_stride + (size_t)(x % per_head) * 8;
        *reinterpret_cast<uint4 *>(dst + at) = *reinterpret_cast<const uint4 *>(src + at);
    }
}
#endif  // __CUDACC__

}  // namespace rnb
