// Causal attention of prompts over a paged cache on the 5th-generation tensor cores.
//
// A CTA owns blocks of 128 (query, head) rows of one key head - a block is 128 / group consecutive queries of a sequence times the group's heads - and
// walks the keys that some of its queries sees in tiles of 128.  A row is a tensor-memory lane; its threads, of as many warps, take a part of a tile's
// keys each and tell each other their maxima.  One thread issues the products: scores from queries and keys in shared memory, then
// probabilities from tensor memory times values.  One warp copies K0 V0 K1 V1 ... into a ring, a box per page and 64 dims, its lanes following
// the table; another sets values that nobody sees to zero.
//
// 16-bit queries: two blocks, which use a tile while it is in shared memory, two threads a row.  One block's softmax runs under the other's
// products.  Tensor memory holds two outputs and probabilities, and scores of one block at a time: as soon as they are read it is the other's turn.
// What sets the pace is this turn: 1650 cycles from one block's reading to the other's (the exponentials take 1024 of a block's tile, its products 1100).
// (5 prompts of up to 512 tokens behind up to 6000, 32 heads on 8: 93 us.  Of 92, with one meeting a tile of a row's warps less: with columns of its own for each
// block's scores, in which its probabilities come, so that the next scores wait for their product: 117; the same in steps of 64 keys, two of them in flight: 146.)
// Queries are exact; probabilities are rounded once to the cache's type, half a step of the output's own rounding (against 64 bits 1.9e-3 with bf16 and 2.7e-4
// with f16, where rounded outputs alone give 1.6e-3 and 2.0e-4; in two terms every product of theirs would be made twice).  The sum that divides the output is of
// the probabilities as they were, since the logarithm of the sum keeps f32 accuracy: keys that all score alike are off by their common rounding.
//
// f32 queries: one block, four threads a row.  Queries enter as f16 "hi" + remainder "lo" (scaled by a power of two per row into f16's range), and so do the
// probabilities: every product is made twice and keeps 22 bits, so the products set the pace.  Three tiles' scores are under way, and probabilities take their place.
// The tensor cores cut sums off at every step, which adds up over long rows: outputs are taken out of tensor memory every FLUSH tiles and summed in f32
// registers, behind the next probabilities, while the last product is still under way (2048 tokens, 32 heads on 8: 80.5 us; error against 64 bits 6.2e-7, at
// 60000 positions 9.4e-7; summed in tensor memory throughout 1.6e-6 and more).
//
// Probabilities are scaled by 2^BIAS so that small ones keep their bits, and the output is scaled only when a row's maximum has grown by more than 2^GROWTH.
// Few rows behind many keys: a cluster of up to eight CTAs shares the keys, and joins maxima, sums and outputs over distributed shared memory.
#pragma once
#include "paged_attention_plain.cuh"
#include "paged_decode.cuh"
#include "prefill_attention_tiled.cuh"

namespace rnb {

constexpr int PP_KEYS = 128;
constexpr int PP_SOFTMAX_WARPS = 16, PP_THREADS = PP_SOFTMAX_WARPS * 32 + 128;   // the last warp is there for the register split, which goes by four warps
constexpr int PP_SOFTMAX_REGS = 104, PP_OTHER_REGS = 64;
static_assert(PP_SOFTMAX_WARPS * 32 * PP_SOFTMAX_REGS + 128 * PP_OTHER_REGS <= PP_THREADS * 96, "what the block is launched with");
constexpr float PP_BIAS = 8.f, PP_GROWTH = 7.f;   // log2; together below f16's 2^16
constexpr int PP_FLUSH = 2;                       // 3: 2 us less of 80 and errors of 7.6e-7 and 1.2e-6, in sums that are too small
constexpr int PP_MAX_CLUSTER = 8;
constexpr uint32_t PP_PANEL = 128 * 128;          // 128 rows of 64 elements, 128-byte swizzle

template <class Q, int D>
struct PpShape {
    static constexpr int TERMS = sizeof(Q) == 4 ? 2 : 1, PANELS = D / 64;
    static constexpr int BLOCKS = TERMS == 2 ? 1 : 2, ROWS = 128 * BLOCKS, WAYS = PP_SOFTMAX_WARPS / (4 * BLOCKS);   // threads of a row
    static constexpr uint32_t Q_BYTES = BLOCKS * TERMS * PANELS * PP_PANEL, TILE_BYTES = PANELS * PP_PANEL;
    // tensor memory.  One block: scores of three tiles, in whose place their probabilities come, and the output.  Two: outputs, scores of one of them, probabilities
    static constexpr bool TURNS = BLOCKS == 2;
    static constexpr int BUFFERS = TURNS ? 1 : 3;
    static __device__ __forceinline__ uint32_t scores_at(int t) { return TURNS ? 2 * D : (uint32_t)(t % BUFFERS) * 128u; }
    static __device__ __forceinline__ uint32_t probabilities_at(int x, int t) { return TURNS ? 2 * D + 128 + (uint32_t)x * 64u : scores_at(t); }
    static constexpr uint32_t outputs_at(int x) { return TURNS ? (uint32_t)(x * D) : 384u; }
    static_assert(TURNS ? 2 * D + 256 <= 512 : 384 + D <= 512, "tensor memory");
    static constexpr int SLOTS = (int)((224 * 1024 - Q_BYTES) / TILE_BYTES) < 8 ? (int)((224 * 1024 - Q_BYTES) / TILE_BYTES) : 8;
    static constexpr size_t TAIL = 512 + 512 * 4;                                     // barriers; what the threads of a row tell each other
    static constexpr size_t JOIN = ROWS * (D + 4) * 4 + ROWS * 8 + ROWS * PP_MAX_CLUSTER * 4 + ROWS * 8;   // outputs; maximum, sum; weights; joined
    static constexpr size_t RING = Q_BYTES + (size_t)SLOTS * TILE_BYTES;
    static constexpr size_t SMEM = (RING > JOIN ? RING : JOIN) + TAIL;
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct PpMaps {
    PkTensorMap k, v;
    PkTensorMap q;   // 16-bit queries [token][head][64-element part]: boxes of a row block, 64 dims
};
struct PpParams {
    const void *q;
    size_t q_stride, out_stride;
    int heads, group, blocks, per_block, queries, window, sinks;   // blocks of per_block heads per key head; queries of a row block
    uint32_t by_heads;   // 2^16 / per_block, rounded up: row / per_block = row * by_heads >> 16
    // 2^64 / d, rounded up (d = 1: 0), for d = key heads * blocks and the queries of a CTA: x / d = x * by >> 64 for all 32-bit x.  (A division by what
    // is only known now takes a CTA 100 to 200 cycles, and there were six on the way to its first tile.)
    uint64_t by_vh, by_rows;
    float scale;
    void *out;
    float *lse;
    int *err;
};

#ifdef __CUDACC__
__device__ __forceinline__ float2 pp_ld_remote2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 pp_ld_remote4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void pp_tmem_st(uint32_t taddr, const uint32_t (&v)[32]) { pat_tmem_st32(taddr, v); }
__device__ __forceinline__ void pp_tmem_st(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
// 16, 32 or 64 columns of this thread's lane
__device__ __forceinline__ void pp_tmem_ld(uint32_t taddr, uint32_t (&v)[64]) { pat_tmem_ld64(taddr, v); }
__device__ __forceinline__ void pp_tmem_ld(uint32_t taddr, uint32_t (&v)[32]) { pg_tmem_ld32(taddr, v); }
__device__ __forceinline__ void pp_tmem_ld(uint32_t taddr, uint32_t (&v)[16]) { ps_tmem_ld<16>(taddr, v); }
template <int N>
__device__ __forceinline__ void pp_registers(bool more) {
    if (more) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// (x, y) in two terms by cutting x and y to the first one's bits: f16 has ten behind the point, bf16 seven
template <class T>
__device__ __forceinline__ void pp_cut(float x, float y, uint32_t &hi, uint32_t &lo) {
    constexpr uint32_t MASK = std::is_same<T, F16>::value ? 0xffffe000u : 0xffff0000u;
    const float a = __uint_as_float(__float_as_uint(x) & MASK), b = __uint_as_float(__float_as_uint(y) & MASK);
    hi = pk_pack<T>(a, b);
    lo = pk_pack<T>(x - a, y - b);
}
__device__ __forceinline__ void pp_tma_4d(uint32_t dst, const PkTensorMap *map, int head, int token, int part, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(0), "r"(head), "r"(token), "r"(part), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void pp_prefetch_map(const PkTensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ float2 pp_mul2(float x, float y, uint64_t m) {
    float2 r;
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%2, %3};\n\tmul.rn.f32x2 t, t, %4;\n\tmov.b64 {%0, %1}, t;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(x), "f"(y), "l"(m));
    return r;
}
// check += {x, y} * 0: zeros stay zeros (of any sign) while both are finite
__device__ __forceinline__ void pp_check2(uint64_t &check, float x, float y) {
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tfma.rn.f32x2 %0, t, %3, %0;\n\t}" : "+l"(check) : "f"(x), "f"(y), "l"(0ull));
}
// V as the second operand: dims contiguous, 8 keys x 64 dims are 1024 bytes, the other 64 dims are a panel further
__device__ __forceinline__ uint64_t pp_v_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | ((uint64_t)(PP_PANEL >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// D = f32, A and B of the cache's type, M = 128
template <class C>
constexpr uint32_t pp_idesc(int n, bool b_mn_major) {
    return (1u << 4) | (std::is_same<C, Bf16>::value ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__host__ __device__ inline uint64_t pp_by(uint32_t d) { return d == 1 ? 0 : ~0ull / d + 1; }
__device__ __forceinline__ unsigned pp_over(unsigned x, uint64_t by) { return by ? (unsigned)__umul64hi(x, by) : x; }
// The tiles of PP_KEYS keys that queries see who see 0 .. sink - 1 and from .. len - 1.
struct PpSeen {
    int len, from, sink, lead, skip, tiles;
    __device__ __forceinline__ int start(int i) const { return PP_KEYS * (i < lead ? i : i + skip); }
    __device__ __forceinline__ bool ragged(int k0) const { return k0 + PP_KEYS > len || (k0 < from && k0 + PP_KEYS > sink); }   // not all of its keys are seen
};

template <class Q, class C, int D>
RNB_GLOBAL void __launch_bounds__(PP_THREADS, 1)
paged_prefill_kernel(PkCache c, PkBatch b, PpParams P, const __grid_constant__ PpMaps maps) {
    using S = PpShape<Q, D>;
    extern __shared__ __align__(1024) uint8_t pp_smem[];
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint64_t *const bars = reinterpret_cast<uint64_t *>(pp_smem + S::SMEM - S::TAIL);
    uint64_t *const full = bars, *const empty = bars + 8, *const q_full = bars + 16, *const s_full = bars + 18, *const p_full = bars + 21, *const pv_done = bars + 24, *const s_free = bars + 27, *const cleared = bars + 44;   // s_full, p_full, pv_done: per block, or per buffer of one
    volatile uint32_t *const tmem_slot = reinterpret_cast<volatile uint32_t *>(bars + 28);
    volatile int *const failed = reinterpret_cast<volatile int *>(bars + 29);
    volatile int *const found = reinterpret_cast<volatile int *>(bars + 30);   // sequence, first query, queries of the sequence, first row of its tokens, its positions
    unsigned *const todo = reinterpret_cast<unsigned *>(bars + 34);   // rows of each warp to be done again
    float *const told = reinterpret_cast<float *>(pp_smem + S::SMEM - S::TAIL + 512);   // [block][way][row]
    uint32_t rank, ranks;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    if (tid == PP_THREADS - 1) {   // (the first box of a launch waits for its map otherwise)
        pp_prefetch_map(&maps.k);
        pp_prefetch_map(&maps.v);
        if (S::TERMS == 1) pp_prefetch_map(&maps.q);
    }
    if (tid == 0) {
        for (int s = 0; s < S::SLOTS; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; i++) mbar_init(&q_full[i], S::TERMS == 2 ? PP_SOFTMAX_WARPS : 1);
        for (int i = 0; i < 3; i++) {
            mbar_init(&pv_done[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4 * S::WAYS);
        }
        mbar_init(s_free, 4 * S::WAYS);
        for (int i = 0; i < 8; i++) mbar_init(&cleared[i], 1);
        mbar_fence_init();
        *failed = (smem_u32(pp_smem) & 1023u) != 0;
        for (int i = 0; i < PP_SOFTMAX_WARPS; i++) todo[i] = 0;
    }
    pdl_wait();   // tensor memory too is asked for when no earlier launch can still hold it
    const int to_ranks = 31 - __clz((int)ranks);   // a power of two
    const int VH = c.kv_heads * P.blocks, item = (int)(blockIdx.x >> to_ranks), turn = (int)pp_over((unsigned)item, P.by_vh), vh = item - turn * VH;
    const int head = P.blocks == 1 ? vh : vh / P.blocks, head0 = (vh - head * P.blocks) * P.per_block;
    // rows of a block: (query, head) = (row / per_block, row % per_block), by multiplication, exact for rows below 128; the last of several head blocks may have fewer heads
    const int heads_here = min(P.per_block, P.group - head0);
    auto query_of = [&](int row) { return (int)((uint32_t)row * P.by_heads >> 16); };
    if (warp == 0) {
        // which queries: the launch's CTAs' worth of row blocks are numbered through from the last to the first, long rows before short ones
        struct Span {
            int start, n, len;
        };
        auto span = [&](int s) {   // a sequence's tokens; starts out of order are cut to the matrices
            Span v{0, 0, 0};
            if (s >= b.n_seq) return v;
            const int from = b.q_start[s], to = b.q_start[s + 1];
            v.len = pk_length(b, c.page_shift, s, P.err);
            v.start = min(max(from, 0), b.n_tokens);
            v.n = max(0, min(to, b.n_tokens) - v.start);
            return v;
        };
        auto pairs_of = [&](const Span &v) { return (int)pp_over((unsigned)(v.n + S::BLOCKS * P.queries - 1), P.by_rows); };
        const Span first32 = span(lane);
        int total = pairs_of(first32);
        for (int s = lane + 32; s < b.n_seq; s += 32) total += pairs_of(span(s));
        total = __reduce_add_sync(0xffffffffu, total);
        const int want = total - 1 - turn;
        if (lane == 0) found[0] = -1;
        __syncwarp();
        int before = 0;
        for (int s0 = 0; s0 < b.n_seq && want >= 0; s0 += 32) {
            const Span v = s0 == 0 ? first32 : span(s0 + lane);
            const int pairs = pairs_of(v);
            int up = pairs;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, up, o);
                if (lane >= o) up += y;
            }
            const unsigned behind = __ballot_sync(0xffffffffu, before + up > want);
            if (behind) {
                const int i = want - before - (up - pairs);
                if (lane == __ffs(behind) - 1 && i >= 0 && i < pairs) {   // (starts out of order may add up to more than 31 bits: then there is no such place)
                    found[0] = s0 + lane;
                    found[1] = i * S::BLOCKS * P.queries;
                    found[2] = v.n;
                    found[3] = v.start;
                    found[4] = v.len;
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, up, 31);
        }
    }
    if (warp == PP_SOFTMAX_WARPS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t *>(tmem_slot))), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pg_fence_before();
    __syncthreads();
    pg_fence_after();
    const uint32_t tmem = *tmem_slot;
    // The barriers of block x's tile t.  With several buffers nobody is more than their number of tiles ahead, so each has its own: a phase of one barrier for
    // all would be taken for the one two tiles on.
    auto passed = [&](uint64_t *bar, int x, int t) {
        return S::TURNS ? mbar_wait_bounded(&bar[x], (uint32_t)(t & 1)) : mbar_wait_bounded(&bar[t % S::BUFFERS], (uint32_t)(t / S::BUFFERS) & 1u);
    };
    auto of_tile = [&](uint64_t *bar, int x, int t) { return &bar[S::TURNS ? x : t % S::BUFFERS]; };
    const int seq = found[0];
    const int first = seq < 0 ? 0 : found[1], n_new = seq < 0 ? 0 : found[2], token0 = seq < 0 ? 0 : found[3], shift = seq < 0 ? 0 : found[4] - n_new;
    bool ok = *failed == 0;
    // block x holds queries first + x * queries ..; query i sits at position shift + i
    const int live_a = seq >= 0 ? min(P.queries, n_new - first) : 0, live_b = S::BLOCKS == 2 && seq >= 0 ? max(0, min(P.queries, n_new - first - P.queries)) : 0;
    PpSeen seen;
    seen.len = max(0, shift + first + live_a + live_b);
    seen.from = P.window && shift + first >= P.window ? shift + first - P.window + 1 : 0;   // (positions may be below 0, and a window up to 2^31 - 1)
    seen.sink = min(P.sinks, seen.from);
    seen.lead = min((seen.sink + PP_KEYS - 1) / PP_KEYS, seen.from / PP_KEYS);
    seen.skip = seen.from / PP_KEYS - seen.lead;
    seen.tiles = max(0, (seen.len + PP_KEYS - 1) / PP_KEYS - seen.skip);
    // this CTA's share of the tiles, and of these the ones that block a sees some of (block b is behind it and sees something of all)
    const int per = (seen.tiles + (int)ranks - 1) >> to_ranks, t0 = min(seen.tiles, per * (int)rank), n_tiles = min(per, seen.tiles - t0);
    const int tiles_a = max(0, (shift + first + live_a + PP_KEYS - 1) / PP_KEYS - (shift + first + live_a > 0 ? seen.skip : 0));
    const int n_a = live_b > 0 ? min(max(tiles_a - t0, 0), n_tiles) : n_tiles, n_b = live_b > 0 ? n_tiles : 0;

    // (one instruction for all warps of a warpgroup)
    if (warp < PP_SOFTMAX_WARPS) pp_registers<PP_SOFTMAX_REGS>(true);
    else pp_registers<PP_OTHER_REGS>(false);
    if (warp < PP_SOFTMAX_WARPS) {
        // a row's threads: lane `lane` of the warps (x, way, w), which take KEYS of a tile's keys and DIMS of the output's dims each
        constexpr int KEYS = PP_KEYS / S::WAYS, DIMS = D / S::WAYS;
        const int x = warp / (4 * S::WAYS), way = (warp >> 2) % S::WAYS, w = warp & 3, mine = x ? n_b : n_a, live = x ? live_b : live_a, q0 = first + x * P.queries;
        auto meet = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + x * 4 + w), "n"(32 * S::WAYS) : "memory"); };   // a row's warps
        uint8_t *const q_smem = pp_smem + (uint32_t)(x * S::TERMS * S::PANELS) * PP_PANEL;   // this block's
        if constexpr (S::TERMS == 2) {
            // ---- f32 queries in two terms: a warp takes its share of the rows, all under way ----
            constexpr int LANES = D / 4, ROWS = 32 / LANES, LOADS = 32 / S::WAYS / ROWS < 1 ? 1 : 32 / S::WAYS / ROWS;   // lanes of a row, rows of a load
            const int d0 = lane % LANES * 4, row0 = (way * 4 + w) * (32 / S::WAYS);
            const float *const q = reinterpret_cast<const float *>(P.q) + (size_t)(token0 + q0) * P.q_stride + (size_t)(head * P.group + head0) * D + d0;
            if (mine > 0) {
                float4 raw[LOADS];
#pragma unroll
                for (int j = 0; j < LOADS; j++) {
                    const int row = row0 + j * ROWS + lane / LANES, ql = query_of(row), h = row - ql * P.per_block;
                    raw[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (ql < live && h < heads_here) raw[j] = *reinterpret_cast<const float4 *>(q + (size_t)ql * P.q_stride + (size_t)h * D);
                }
                uint8_t *const to = q_smem + (uint32_t)(d0 / 64) * PP_PANEL + (uint32_t)(row0 + lane / LANES) * 128u + (uint32_t)(d0 & 7) * 2u;
#pragma unroll
                for (int j = 0; j < LOADS; j++) {
                    const float4 v = raw[j];
                    float most = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
                    if constexpr (LANES == 32) {
                        most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));   // of values that are not negative, as whole numbers
                    } else {
#pragma unroll
                        for (int o = LANES / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    }
                    float down, up;
                    pk_factor(most, down, up);
                    if (lane % LANES < S::WAYS) told[lane % LANES * 128 + row0 + j * ROWS + lane / LANES] = up;   // to all threads of the row
                    uint2 hi, lo;
                    pp_cut<C>(v.x * down, v.y * down, hi.x, lo.x);
                    pp_cut<C>(v.z * down, v.w * down, hi.y, lo.y);
                    uint8_t *const at = to + j * ROWS * 128 + (((d0 % 64 / 8) ^ ((j * ROWS + lane / LANES) & 7)) << 4);
                    *reinterpret_cast<uint2 *>(at) = hi;
                    *reinterpret_cast<uint2 *>(at + S::PANELS * PP_PANEL) = lo;
                }
            }
            pg_proxy_fence();
            __syncwarp();
            if (lane == 0) pg_arrive(&q_full[x]);
        }
        // ---- softmax: this thread's row ----
        const int r = w * 32 + lane, ql = query_of(r);
        const bool alive = ql < live && r - ql * P.per_block < heads_here;
        const int pos = shift + q0 + min(ql, max(live - 1, 0));                       // dead rows see what the last one sees, and are not stored
        const int pos0 = shift + q0, pos1 = shift + q0 + live - 1;                    // the block's positions
        const uint32_t lanes = (uint32_t)(w * 32) << 16, t_o = tmem + S::outputs_at(x) + (uint32_t)(way * DIMS) + lanes;
        const float turned = P.scale > 0.f ? 1.f : P.scale == 0.f ? 0.f : -1.f;   // maxima are of unscaled scores: they need a positive scale
        float sl2 = (P.scale == 0.f ? 1.f : fabsf(P.scale)) * 1.4426950408889634f;   // to log2 units
        float *const say = told + (x * S::WAYS + way) * 128 + r;
        auto heard = [&](int i) { return told[(x * S::WAYS + i) * 128 + r]; };
        const size_t row = (size_t)(token0 + q0 + min(ql, max(live - 1, 0)));
        const int q_head = head * P.group + head0 + r - ql * P.per_block;
        Q *const out0 = reinterpret_cast<Q *>(P.out) + (size_t)(token0 + q0) * P.out_stride + (size_t)(head * P.group + head0) * D;   // the block's first row
        float m_ref = -INFINITY, l_run = 0.f, m_sums = -INFINITY;
        float sums[S::TERMS == 2 ? DIMS : 1];   // f32 sums of the outputs up to the last flush, in units of 2^m_sums
#pragma unroll
        for (int i = 0; i < (int)(sizeof(sums) / 4); i++) sums[i] = 0.f;
        // the output in tensor memory, in units of 2^m, joins the sums (nothing seen yet: of no weight)
        auto collect = [&](float m) {
            if constexpr (S::TERMS == 2) {
                const float old = exp2f(m_sums - (m == -INFINITY ? 0.f : m));
                uint32_t v[DIMS];
                pp_tmem_ld(t_o, v);
#pragma unroll
                for (int i = 0; i < DIMS; i++) sums[i] = fmaf(sums[i], old, __uint_as_float(v[i]));
                m_sums = m;
            }
        };
        for (int t = 0; t < mine; t++) {
            ok = ok && __all_sync(0xffffffffu, passed(s_full, x, t));
            if (!ok) {   // a row's warps meet in every tile, whatever has failed
                meet();
                meet();
                continue;
            }
            pg_fence_after();
            uint32_t s[KEYS];
            pp_tmem_ld(tmem + S::scores_at(t) + lanes + (uint32_t)(way * KEYS), s);
            if constexpr (S::TURNS) {   // the other block's turn
                pg_fence_before();
                __syncwarp();
                if (lane == 0) pg_arrive(s_free);
            }
            if (S::TERMS == 2 && t == 0) sl2 *= *say;   // the row's factor, from before the scores' product
            if (turned != 1.f) {
#pragma unroll
                for (int i = 0; i < KEYS; i++) s[i] = __float_as_uint(__uint_as_float(s[i]) * turned);
            }
            const int k0 = seen.start(t0 + t) + way * KEYS;
            if (!(k0 + KEYS - 1 <= pos0 && (P.window == 0 || pos1 - k0 < P.window || k0 + KEYS <= P.sinks))) {
                // keys a .. z of these, and those before the end of the sinks
                const int z = pos - k0, a = P.window && z >= P.window ? z - P.window + 1 : 0, k = P.sinks - k0;
                auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };   // bits 0 .. n - 1
#pragma unroll
                for (int j = 0; j < KEYS / 32; j++) {
                    const uint32_t keep = below(z + 1 - 32 * j) & (~below(a - 32 * j) | below(k - 32 * j));
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (!(keep & (1u << i))) s[32 * j + i] = 0xff800000u;   // -inf
                }
            }
            float mxs[4];
#pragma unroll
            for (int j = 0; j < 4; j++) mxs[j] = __uint_as_float(s[j]);
#pragma unroll
            for (int i = 4; i < KEYS; i++) mxs[i & 3] = fmaxf(mxs[i & 3], __uint_as_float(s[i]));
            // The row's maximum, once all its threads have read the last tile's: no barrier of the products holds a warp back until then.  (f32 2048 tokens 80.6 us, 16-bit
            // 5 x 512 93.3; with this meeting ahead of the wait for the scores 82.6 and 94.4, with a barrier that the readers arrive at 83.5 and 101.9.)  When all
            // have their scores, probabilities may take the scores' place.
            meet();
            *say = fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3]));
            pg_fence_before();
            meet();
            pg_fence_after();
            float top = heard(0);
#pragma unroll
            for (int i = 1; i < S::WAYS; i++) top = fmaxf(top, heard(i));
            const float mx = top * sl2;
            // the product before this one is through, the output stands
            bool waited = t == 0;
            auto through = [&]() {
                if (!waited) ok = ok && __all_sync(0xffffffffu, passed(pv_done, x, t - 1));
                waited = true;
                pg_fence_after();
            };
            const bool flush = S::TERMS == 2 && t > 0 && t % PP_FLUSH == 0;   // the next product starts from zero
            const float m_before = m_ref;
            float corr = 1.f;
            if (mx > m_ref + PP_GROWTH || m_ref == -INFINITY) {
                const float m_new = fmaxf(mx, m_ref);
                corr = exp2f(m_ref - (m_new == -INFINITY ? 0.f : m_new));
                m_ref = m_new;
            }
            const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
            if (t > 0 && !flush && __any_sync(0xffffffffu, corr != 1.f)) {
                through();
                constexpr int SOME = DIMS < 32 ? DIMS : 32;
#pragma unroll 1
                for (int k = 0; k < DIMS; k += SOME) {
                    uint32_t v[SOME];
                    pp_tmem_ld(t_o + (uint32_t)k, v);
#pragma unroll
                    for (int i = 0; i < SOME; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * corr);
                    pp_tmem_st(t_o + (uint32_t)k, v);
                }
            }
            __syncwarp();
            const uint64_t sl22 = pg_pair_f32(sl2, sl2), nm2 = pg_pair_f32(PP_BIAS - m_use, PP_BIAS - m_use);
            uint64_t sum[2] = {0, 0};
            uint32_t hi[KEYS / 2], lo[KEYS / 2];   // columns of a term
#pragma unroll
            for (int i = 0; i < KEYS / 2; i++) {
                const float2 y = pat_fma2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]), sl22, nm2);
                const float p0 = pat_exp2(y.x), p1 = pat_exp2(y.y);
                pat_add2(sum[i & 1], p0, p1);
                if constexpr (S::TERMS == 2) pp_cut<C>(p0, p1, hi[i], lo[i]);
                else hi[i] = pk_pack<C>(p0, p1);
            }
            if (S::TURNS) through();   // (a buffer's own product was through before its scores came)
            if (ok) {
                const uint32_t to = tmem + S::probabilities_at(x, t) + lanes + (uint32_t)(way * (KEYS / 2));
                pp_tmem_st(to, hi);
                if constexpr (S::TERMS == 2) pp_tmem_st(to + 64u, lo);
            }
            if (flush) {   // (as late as the product allows, which is under way until now)
                through();
                collect(m_before);
            }
            if (ok) {
                pat_tmem_st_wait();
                pg_fence_before();
                __syncwarp();
                if (lane == 0) pg_arrive(of_tile(p_full, x, t));
            }
            l_run = fmaf(l_run, corr, pat_total(sum[0], sum[1]));
        }
        if (ok && mine > 0) ok = __all_sync(0xffffffffu, passed(pv_done, x, mine - 1));
        pg_fence_after();
        // ---- the row's end ----
        meet();
        *say = l_run;
        meet();
        l_run = heard(0);
#pragma unroll
        for (int i = 1; i < S::WAYS; i++) l_run += heard(i);
        const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
        if (S::TERMS == 2 && mine > 0 && ok) collect(m_ref);
        constexpr int SOME = DIMS < 32 ? DIMS : 32;
        auto output = [&](int k, float (&o)[SOME]) {   // unscaled, dims SOME * k .. of this thread's
            if constexpr (S::TERMS == 2) {
                static_assert(S::TERMS == 1 || DIMS == SOME, "all of them");
#pragma unroll
                for (int i = 0; i < SOME; i++) o[i] = sums[i];
            } else if (mine > 0 && ok) {
                uint32_t v[SOME];
                pp_tmem_ld(t_o + (uint32_t)(k * SOME), v);
#pragma unroll
                for (int i = 0; i < SOME; i++) o[i] = __uint_as_float(v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < SOME; i++) o[i] = 0.f;
            }
        };
        auto store4 = [](Q *to, float a, float b2, float c2, float d) {
            if constexpr (sizeof(Q) == 4) *reinterpret_cast<float4 *>(to) = make_float4(a, b2, c2, d);
            else *reinterpret_cast<uint2 *>(to) = make_uint2(pk_pack<Q>(a, b2), pk_pack<Q>(c2, d));
        };
        if (ranks == 1) {
            // BYTES of this thread's part of every row at a time through shared memory, where the queries were, so that a few lanes store a row's
            constexpr int BYTES = DIMS * (int)sizeof(Q) < 128 ? DIMS * (int)sizeof(Q) : 128, COLS = BYTES / (int)sizeof(Q), LANES = BYTES / 16;
            uint8_t *const box = q_smem + (way * 4 + w) * (S::TERMS * S::PANELS * PP_PANEL / (4 * S::WAYS));
            static_assert(32 * BYTES <= S::TERMS * S::PANELS * PP_PANEL / (4 * S::WAYS), "a box per warp");
            const float inv = l_run > 0.f ? 1.f / l_run : l_run != l_run ? l_run : 0.f;
            const uint64_t inv2 = pg_pair_f32(inv, inv);
            uint64_t check = 0;   // stays zero while all are finite
#pragma unroll 1
            for (int k = 0; k < DIMS / COLS; k++) {
                __syncwarp();   // a row's sums are read by now, and what was stored out of the box
#pragma unroll
                for (int j = 0; j < COLS / SOME; j++) {
                    float o[SOME];
                    output(k * (COLS / SOME) + j, o);
#pragma unroll
                    for (int i = 0; i < SOME; i += 16 / (int)sizeof(Q)) {
                        uint32_t v[4];
#pragma unroll
                        for (int e = 0; e < 16 / (int)sizeof(Q); e += 2) {
                            const float2 y = pp_mul2(o[i + e], o[i + e + 1], inv2);
                            pp_check2(check, y.x, y.y);
                            if constexpr (sizeof(Q) == 4) {
                                v[e] = __float_as_uint(y.x);
                                v[e + 1] = __float_as_uint(y.y);
                            } else {
                                v[e / 2] = pk_pack<Q>(y.x, y.y);
                            }
                        }
                        const int ch = (j * SOME + i) * (int)sizeof(Q) / 16;
                        *reinterpret_cast<uint4 *>(box + lane * BYTES + ((ch ^ (lane & (LANES - 1))) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < LANES; i++) {
                    const int rr = (32 / LANES) * i + lane / LANES, ch = lane % LANES, R = w * 32 + rr, rq = query_of(R), h = R - rq * P.per_block;
                    const uint4 y = *reinterpret_cast<const uint4 *>(box + rr * BYTES + ((ch ^ (rr & (LANES - 1))) << 4));
                    if (rq < live && h < heads_here && ok)
                        *reinterpret_cast<uint4 *>(out0 + (size_t)rq * P.out_stride + (size_t)h * D + way * DIMS + k * COLS + ch * (16 / (int)sizeof(Q))) = y;
                }
            }
            const bool strange = alive && ok && !((uint32_t)check << 1 == 0 && (uint32_t)(check >> 32) << 1 == 0);
            if (alive && ok && way == 0 && P.lse) P.lse[row * P.heads + q_head] = l_run > 0.f ? (m_use - PP_BIAS + log2f(l_run)) * 0.6931471805599453f : l_run != l_run ? l_run : -INFINITY;
            if (strange) atomicOr(&todo[x * 4 + w], 1u << lane);
            __syncwarp();
            meet();
        } else {
            // ---- a cluster's shares: outputs, maxima and sums in shared memory, where the tiles were ----
            if (!ok) *failed = 1;
            asm volatile("bar.sync 9, %0;" ::"n"(32 * PP_SOFTMAX_WARPS) : "memory");   // both blocks' products are through (each block's warps have waited for its own)
            float *const o_all = reinterpret_cast<float *>(pp_smem), *const ml = o_all + S::ROWS * (D + 4);
#pragma unroll 1
            for (int k = 0; k < DIMS / SOME; k++) {
                float o[SOME];
                output(k, o);
#pragma unroll
                for (int i = 0; i < SOME; i += 4) *reinterpret_cast<float4 *>(o_all + (x * 128 + r) * (D + 4) + way * DIMS + k * SOME + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
            if (way == 0) *reinterpret_cast<float2 *>(ml + 2 * (x * 128 + r)) = make_float2(m_ref, ok ? l_run : 0.f);
            __syncwarp();
            ps_cluster_sync();
            // this CTA joins rows [rank * n, (rank + 1) * n)
            const int n = S::ROWS / (int)ranks;
            float *const weights = ml + 2 * S::ROWS, *const joined = weights + S::ROWS * PP_MAX_CLUSTER;
            const uint32_t o_addr = smem_u32(o_all), ml_addr = smem_u32(ml);
            if (tid < n) {
                const int R = (int)rank * n + tid;
                float2 y[PP_MAX_CLUSTER];
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int p = 0; p < PP_MAX_CLUSTER; p++) y[p] = pp_ld_remote2(ps_map(ml_addr + 8u * (uint32_t)R, p & ((int)ranks - 1)));   // (read twice: of no weight)
#pragma unroll
                for (int p = 0; p < PP_MAX_CLUSTER; p++) M = fmaxf(M, y[p].x);
#pragma unroll
                for (int p = 0; p < PP_MAX_CLUSTER; p++) {
                    const float wgt = exp2f(y[p].x - (M == -INFINITY ? 0.f : M));
                    weights[tid * PP_MAX_CLUSTER + p] = wgt;
                    if (p < (int)ranks) L += wgt * y[p].y;
                }
                *reinterpret_cast<float2 *>(joined + 2 * tid) = make_float2(M == -INFINITY ? 0.f : M, L);
            }
            asm volatile("bar.sync 9, %0;" ::"n"(32 * PP_SOFTMAX_WARPS) : "memory");
            const bool good = *failed == 0;
            // a warp per row, and as many rows at a time that eight parts are asked for before the first is used
            auto join = [&](auto parts) {
                constexpr int PARTS = decltype(parts)::value, AT_ONCE = PP_MAX_CLUSTER / PARTS;
                for (int e0 = warp; e0 < n; e0 += AT_ONCE * PP_SOFTMAX_WARPS) {
                    float4 a[AT_ONCE][PARTS];
                    auto is_live = [&](int e) {
                        const int R = (int)rank * n + e, rr = R & 127, rq = query_of(rr);
                        return e < n && rq < (R >> 7 ? live_b : live_a) && rr - rq * P.per_block < heads_here && good;
                    };
#pragma unroll
                    for (int j = 0; j < AT_ONCE; j++) {
                        const int e = e0 + j * PP_SOFTMAX_WARPS;
                        if (lane < D / 4 && is_live(e))
#pragma unroll
                            for (int p = 0; p < PARTS; p++) a[j][p] = pp_ld_remote4(ps_map(o_addr + (uint32_t)(((int)rank * n + e) * (D + 4) + lane * 4) * 4u, p));
                    }
#pragma unroll
                    for (int j = 0; j < AT_ONCE; j++) {
                        const int e = e0 + j * PP_SOFTMAX_WARPS;
                        if (!is_live(e)) continue;
                        const int R = (int)rank * n + e, bx = R >> 7, rr = R & 127, rq = query_of(rr);
                        const float2 ML = *reinterpret_cast<const float2 *>(joined + 2 * e);
                        const float inv = ML.y > 0.f ? 1.f / ML.y : ML.y != ML.y ? ML.y : 0.f;
                        const size_t token = (size_t)(token0 + first + bx * P.queries + rq);
                        const int h = head * P.group + head0 + rr - rq * P.per_block;
                        bool strange = false;
                        if (lane < D / 4) {
                            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                            for (int p = 0; p < PARTS; p++) {
                                const float wgt = weights[e * PP_MAX_CLUSTER + p];
                                v = make_float4(fmaf(wgt, a[j][p].x, v.x), fmaf(wgt, a[j][p].y, v.y), fmaf(wgt, a[j][p].z, v.z), fmaf(wgt, a[j][p].w, v.w));
                            }
                            v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                            strange = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, v.w * 0.f))) != 0.f;
                            store4(reinterpret_cast<Q *>(P.out) + token * P.out_stride + (size_t)h * D + lane * 4, v.x, v.y, v.z, v.w);
                        }
                        if (lane == 0 && P.lse) P.lse[token * P.heads + h] = ML.y > 0.f ? (ML.x - PP_BIAS + log2f(ML.y)) * 0.6931471805599453f : ML.y != ML.y ? ML.y : -INFINITY;
                        if (__any_sync(0xffffffffu, strange) && lane == 0) atomicOr(&todo[warp], 1u << (e / PP_SOFTMAX_WARPS));
                    }
                }
            };
            if (ranks == 2) join(std::integral_constant<int, 2>());
            else if (ranks == 4) join(std::integral_constant<int, 4>());
            else join(std::integral_constant<int, 8>());
            __syncwarp();
            ps_cluster_sync();
        }
        // ---- rows that came out infinite or undefined, one by one ----
        const int step = ranks == 1 ? 1 : PP_SOFTMAX_WARPS, row0 = ranks == 1 ? x * 128 + w * 32 : (int)rank * (S::ROWS / (int)ranks) + warp;
        for (unsigned left = ranks > 1 ? todo[warp] : way == 0 ? todo[x * 4 + w] : 0; left; left &= left - 1) {
            const int R = row0 + (__ffs(left) - 1) * step, bx = R >> 7, rq = query_of(R & 127), h = head * P.group + head0 + (R & 127) - rq * P.per_block;
            const size_t token = (size_t)(token0 + first + bx * P.queries + rq);
            pk_plain_row<Q, C, D>(c, b, reinterpret_cast<const Q *>(P.q) + token * P.q_stride + (size_t)h * D, seq, shift + first + bx * P.queries + rq, head, P.scale, P.window,
                                  P.sinks, reinterpret_cast<Q *>(P.out) + token * P.out_stride + (size_t)h * D, P.lse ? P.lse + token * P.heads + h : nullptr, P.err);
        }
    } else if (warp == PP_SOFTMAX_WARPS) {
        // ---- products: K of tile t is item 2t of the ring, V item 2t + 1.  One thread waits and issues (votes of a warp around every wait took 100 to 200
        // cycles each, in which the tensor cores had nothing to do) ----
        if (pg_elect()) {
            const uint32_t base = smem_u32(pp_smem), ring = base + S::Q_BYTES;
            const int last = n_b > 0 ? 1 : 0;   // the block that uses a tile last
            uint32_t turns = 0;                 // scores issued
            auto arrived = [&](int i) { return mbar_wait_bounded(&full[i % S::SLOTS], (uint32_t)(i / S::SLOTS) & 1u); };
            auto scores = [&](int x, int t) {
                // their columns are free: the other block has read its scores, or the probabilities in them have been multiplied (nothing but its end orders a
                // product behind one that reads what it overwrites)
                ok = arrived(2 * t) && (S::TURNS ? turns == 0 || mbar_wait_bounded(s_free, (turns - 1) & 1u)
                                                 : t < S::BUFFERS || passed(pv_done, x, t - S::BUFFERS));
                turns++;
                if (!ok) return;
                pg_fence_after();
                const int slot = 2 * t % S::SLOTS;
                const uint32_t kt = ring + (uint32_t)slot * S::TILE_BYTES;
#pragma unroll
                for (int term = S::TERMS - 1; term >= 0; term--)   // remainders first: the accumulator cuts off what it adds, and adds less often to full sums
#pragma unroll
                    for (int p = 0; p < S::PANELS; p++) {
                        const uint64_t dq = pg_smem_desc(base + (uint32_t)((x * S::TERMS + term) * S::PANELS + p) * PP_PANEL), dk = pg_smem_desc(kt + (uint32_t)p * PP_PANEL);
#pragma unroll
                        for (int k = 0; k < 4; k++) ps_mma(tmem + S::scores_at(t), dq + 2u * k, dk + 2u * k, pp_idesc<C>(128, false), (S::TERMS - 1 - term) | p | k);
                    }
                pg_commit(of_tile(s_full, x, t));
                if (x == last) pg_commit(&empty[slot]);
            };
            auto outputs = [&](int x, int t, int slot) {
                ok = passed(p_full, x, t);
                if (!ok) return;
                pg_fence_after();
                const uint64_t dv = pp_v_desc(ring + (uint32_t)slot * S::TILE_BYTES);
                const uint32_t tp = tmem + S::probabilities_at(x, t), to = tmem + S::outputs_at(x);
                const uint32_t more = t > 0 && !(S::TERMS == 2 && t % PP_FLUSH == 0);
#pragma unroll
                for (int k = 0; k < PP_KEYS / 16; k++) {   // 16 keys: 2048 bytes of a panel of V, eight columns of probabilities
                    pat_mma_ta(to, tp + 8u * k, dv + (uint64_t)(k * (2048 >> 4)), pp_idesc<C>(D, true), more | (uint32_t)(k != 0));
                    if constexpr (S::TERMS == 2) pat_mma_ta(to, tp + 64u + 8u * k, dv + (uint64_t)(k * (2048 >> 4)), pp_idesc<C>(D, true), 1u);
                }
                pg_commit(of_tile(pv_done, x, t));
                if (x == last) pg_commit(&empty[slot]);
            };
            constexpr int AHEAD = S::BLOCKS == 2 ? 1 : S::BUFFERS - 1;   // tiles whose scores are under way before a product of probabilities
            for (int x = 0; x < S::BLOCKS && ok; x++) {
                if ((x ? n_b : n_a) == 0) continue;
                ok = mbar_wait_bounded(&q_full[x], 0u);
                for (int t = 0; t < AHEAD && t < (x ? n_b : n_a) && ok; t++) scores(x, t);
            }
            for (int t = 0; t < n_tiles && ok; t++) {
                const int slot = (2 * t + 1) % S::SLOTS;
                for (int x = 0; x < S::BLOCKS && ok; x++) {
                    const int mine = x ? n_b : n_a;
                    if (S::TURNS && t + AHEAD < mine) scores(x, t + AHEAD);
                    if (ok && t < mine) {
                        if (x == 0 || n_a <= t) ok = mbar_wait_bounded(&cleared[t & 7], (uint32_t)(t >> 3) & 1u) && arrived(2 * t + 1);
                        if (ok) outputs(x, t, slot);
                    }
                    // (behind the product: a flush waits for that one)
                    if (!S::TURNS && ok && t + AHEAD < mine) scores(x, t + AHEAD);
                }
            }
        }
        __syncwarp();
    } else if (warp == PP_SOFTMAX_WARPS + 2) {
        // ---- values that nobody sees become zeros: whatever they were, zero times it has to be zero.  (Every tile passes here: its product
        // waits for this warp, so that it never falls behind the ring, and the ring keeps it less than eight tiles ahead) ----
        for (int t = 0; t < n_tiles && ok; t++) {
            const int k0 = seen.start(t0 + t), slot = (2 * t + 1) % S::SLOTS;
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[slot], (uint32_t)((2 * t + 1) / S::SLOTS) & 1u));
            if (!ok) break;
            auto clear = [&](int lo, int hi) {
                for (int e = max(lo, 0) * 8 + lane; e < min(hi, PP_KEYS) * 8; e += 32)
#pragma unroll
                    for (int p = 0; p < S::PANELS; p++)
                        *reinterpret_cast<uint4 *>(pp_smem + S::Q_BYTES + (uint32_t)slot * S::TILE_BYTES + (uint32_t)p * PP_PANEL + (uint32_t)e * 16u) = make_uint4(0, 0, 0, 0);
            };
            if (seen.ragged(k0)) {
                clear(seen.len - k0, PP_KEYS);
                clear(seen.sink - k0, seen.from - k0);
                pg_proxy_fence();
            }
            __syncwarp();
            if (lane == 0) pg_arrive(&cleared[t & 7]);
        }
    } else if (warp == PP_SOFTMAX_WARPS + 1) {
        // ---- copies: lane i has box i / PANELS of a tile, 64 dims of it ----
        const int box = min(1 << c.page_shift, PP_KEYS), blk = lane / S::PANELS * box, part = lane % S::PANELS;
        const uint32_t dst = smem_u32(pp_smem) + S::Q_BYTES + (uint32_t)part * PP_PANEL + (uint32_t)blk * 128u;
        auto look_up = [&](int t, int &pos, bool &live) {
            pos = seen.start(t0 + t) + blk;
            live = blk < PP_KEYS && pos < seen.len && (pos + box > seen.from || pos < seen.sink);
            return live ? b.table[(size_t)seq * b.table_stride + (pos >> c.page_shift)] : 0;
        };
        uint32_t it = 0;
        int pos = 0, page = 0;
        bool live = false;
        if (n_tiles > 0) page = look_up(0, pos, live);
        if constexpr (S::TERMS == 1) {   // 16-bit queries are copied as they are, with those of sequences behind this one where a block has room
            for (int x = 0; x < 2; x++)
                if ((x ? n_b : n_a) > 0) {
                    if (lane == 0) mbar_arrive_expect_tx(&q_full[x], (uint32_t)(S::PANELS * P.queries * P.per_block) * 128u);
                    __syncwarp();
                    if (lane < S::PANELS)
                        pp_tma_4d(smem_u32(pp_smem) + (uint32_t)(x * S::PANELS + lane) * PP_PANEL, &maps.q, head * P.group + head0, token0 + first + x * P.queries, lane, &q_full[x]);
                }
        }
        for (int t = 0; t < n_tiles && ok; t++) {
            if (live && (unsigned)page >= (unsigned)c.n_pages) {
                atomicExch(P.err, DEV_ERR_BAD_PAGE);
                live = false;
            }
            const bool now = live;
            const int at_pos = pos & ((1 << c.page_shift) - 1), at_page = page;
            if (t + 1 < n_tiles) page = look_up(t + 1, pos, live);
            const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, now)) * (uint32_t)box * 128u;
            for (int v = 0; v < 2; v++) {
                const uint32_t slot = it % S::SLOTS;
                ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(&empty[slot], ((it / S::SLOTS) & 1u) ^ 1u));
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&full[slot], bytes);
                __syncwarp();
                if (now) pk_tma_5d(dst + slot * S::TILE_BYTES, v ? &maps.v : &maps.k, at_pos, part, head, at_page, &full[slot]);
                it++;
            }
        }
        if constexpr (S::TERMS == 1)
            for (int x = 0; x < 2; x++)
                if ((x ? n_b : n_a) > 0) mbar_wait_bounded(&q_full[x], 0u);
        pg_drain(full, it, S::SLOTS);
    } else if (blockIdx.x == 0) {
        pk_check_starts(b, lane, 32, P.err);
    }
    __syncwarp();
    if (warp >= PP_SOFTMAX_WARPS && ranks > 1) {
        ps_cluster_sync();
        ps_cluster_sync();
    }
    if (!ok) *failed = 1;
    __syncwarp();
    pg_fence_before();
    __syncthreads();
    if (warp == PP_SOFTMAX_WARPS) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        if (lane == 0 && *failed) atomicExch(P.err, DEV_ERR_MBAR_TIMEOUT);
    }
}
#endif  // __CUDACC__

}  // namespace rnb
