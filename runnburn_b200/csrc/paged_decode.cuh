// Attention of one new token per sequence over a paged cache: one pass over the visible positions with a running maximum and sum.
//
// The work is a list of tiles of 64 positions, (sequence, key head, tile) with the tiles fastest, that the launch cuts into equal
// runs, one per CTA: lengths may differ as they like, and one long sequence uses the whole chip.  Every CTA finds its run by a scan over the lengths.
// A (sequence, key head) that lies within one run is finished there; of one that is cut, each CTA leaves (maximum, sum, output) in the
// workspace, and the CTA that arrives last joins them in the order of the runs, so the result does not depend on who was last.
//
// In a CTA four warps share a tile, 16 positions each, with a softmax of their own that is joined at the end of a segment; eight query heads
// are the rows of the products (HT = 2: eight warps for up to 16 heads).  Rows 0-7 hold the queries rounded to the cache's type and rows 8-15 what the
// rounding left, so one product gives both and their sum keeps f32 queries at 22 bits; the same with the probabilities.  Queries are scaled
// by a power of two per head into the range of f16, probabilities by 2^BIAS, so that small ones keep their bits.  Products start from zero and are
// added to the f32 sums in registers: long sums in the tensor cores' accumulators would be cut off at each step.
//
// A warp of its own brings K and V tiles in by tiled copies, a box per page (or 64 positions of a larger one), its lanes following the table
// one tile ahead; a ring of barriers lets every warp go at its own pace.  Boxes that hold nothing visible are not fetched.  Where a tile
// has rows that are not visible, their scores are left out and their values set to zero, so what lies there never enters a product.
#pragma once
#include "paged.cuh"

namespace rnb {

constexpr int PD_TILE = 64;
constexpr float PD_BIAS = 12.f;
// The shortest run, in tiles: a join reads one of n parts after the other, a tile takes about as long as the reading of 16, so runs of sqrt(tiles) / 4 are best
// where there are CTAs enough.  32 heads on 8 key heads, 128 dims: 300 positions 7.0 us, 600 8.1, 1000 8.7 (with runs of four tiles 10.6, 10.5, 9.9);
// 32768 positions of one key head 19.8 us (with the shortest that give all CTAs work 35.5).
constexpr float PD_RUN = 0.25f;
// Where the longest sequence has up to so many tiles, the shortest run is as long as it: sequences of one length are then not cut at all (180 positions: 6.4 us,
// cut 6.9; 250: 7.2, cut 7.0).  Of unlike ones some still are, at the ends of equal runs.
constexpr int PD_WHOLE = 3;
constexpr size_t PD_WS_HEAD = 256;                      // a mark that the workspace has been initialised
constexpr int PD_MAX_GRID = 1024;                       // runs of a launch
constexpr size_t PD_WS_RECORDS = PD_WS_HEAD + PD_MAX_GRID * sizeof(unsigned);
constexpr unsigned PD_WS_MARK = 0x5a5a5a5au;

template <int D, int HT>
struct PdShape {
    static constexpr int WORKERS = 128 * HT, THREADS = WORKERS + 64;
    static constexpr int STAGES = D == 128 ? (HT == 1 ? 3 : 5) : 4;
    static constexpr int PER_SM = HT == 1 ? (D == 128 ? 2 : 3) : (D == 128 ? 1 : 2);
    static constexpr int ROW = D + 4;                                                    // floats between the heads of a partial output
    static constexpr uint32_t TILE_BYTES = PD_TILE * D * 2;
    static constexpr size_t MERGE = sizeof(float) * HT * 4 * 8 * ROW;                    // outputs of the warps; weights of the parts in a join
    static constexpr int WEIGHTS = 256;                                                  // parts whose weights a join has at hand
    static constexpr size_t SMEM = STAGES * 2 * TILE_BYTES + MERGE + sizeof(float) * HT * 8 * 10 + 192;
    static_assert(WEIGHTS * 8 * HT * sizeof(float) <= MERGE, "they lie where the outputs were");
    static_assert(PER_SM * (SMEM + 1024) <= 228 * 1024, "shared memory");
    static constexpr size_t RECORD = sizeof(float) * HT * 8 * (D + 4);                   // per head: maximum, sum, two unused, output
};

struct PdParams {
    const void *q;
    size_t q_stride, out_stride;
    int heads, group, splits, window, sinks;   // splits: CTAs' worth of heads per key head
    float scale_log2;
    void *out;
    float *lse;
    uint8_t *workspace;
    int *err;
};

// Pools as tensors of [page][head][64-element part of a row][position][64]: a box is up to 64 positions of a page with all parts of their rows, each part
// in the 128-byte swizzle.
struct alignas(64) PkTensorMap {
    unsigned long long opaque[16];
};
struct PkMaps {
    PkTensorMap k, v;
};

#ifdef __CUDACC__
__device__ __forceinline__ void pk_tma_5d(uint32_t dst, const PkTensorMap *map, int pos, int part, int head, int page, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
                 ::"r"(dst), "l"(map), "r"(0), "r"(pos), "r"(part), "r"(head), "r"(page), "r"(smem_u32(bar))
                 : "memory");
}
// One more arrival at a counter: what the CTA wrote before the barrier ahead of this is visible to whoever reads the count afterwards.
__device__ __forceinline__ unsigned pk_arrive_gpu(unsigned *count) {
    unsigned before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
    return before;
}
// the workers of a CTA, without its copying warp
template <int N>
__device__ __forceinline__ void pk_sync_some() {
    asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float pd_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The tiles of a query that sees positions 0 .. sink - 1 and from .. len - 1.
struct PdSeen {
    int len, from, sink, lead, skip;   // tile i starts at position 64 (i < lead ? i : i + skip)
    int tiles;
};
__device__ __forceinline__ PdSeen pd_seen(int len, int window, int sinks) {
    PdSeen s;
    s.len = len;
    s.from = window && len > window ? len - window : 0;
    s.sink = min(sinks, s.from);
    s.lead = min((s.sink + PD_TILE - 1) / PD_TILE, s.from / PD_TILE);
    s.skip = s.from / PD_TILE - s.lead;
    s.tiles = max(1, (len + PD_TILE - 1) / PD_TILE - s.skip);   // an empty one too: its output is written
    return s;
}

template <class Q, class C, int D, int HT>
RNB_GLOBAL void __launch_bounds__(PdShape<D, HT>::THREADS, PdShape<D, HT>::PER_SM)
paged_decode_kernel(PkCache c, PkBatch b, PdParams P, const __grid_constant__ PkMaps maps) {
    using S = PdShape<D, HT>;
    constexpr int KS = D / 16;
    extern __shared__ __align__(1024) uint8_t pd_smem[];
    float *const merge = reinterpret_cast<float *>(pd_smem + S::STAGES * 2 * S::TILE_BYTES);
    float *const ml = reinterpret_cast<float *>(pd_smem + S::SMEM - 192 - sizeof(float) * HT * 8 * 10);   // [head][m of 4 warps, l of 4 warps, M, L]
    uint64_t *const full = reinterpret_cast<uint64_t *>(pd_smem + S::SMEM - 192), *const empty = full + S::STAGES;
    volatile int *const note = reinterpret_cast<volatile int *>(full + 2 * S::STAGES);   // [1]: something gave up; [2] .. [7]: the run
    volatile int *const jobs = note + 8;   // two cut segments: sequence, head block, first CTA, parts (0: none), whether this CTA came last
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 4 * HT);
        }
        mbar_fence_init();
        jobs[3] = jobs[8] = jobs[4] = jobs[9] = 0;
        note[1] = (smem_u32(pd_smem) & 1023u) != 0;   // a wait gave up (or the swizzle would not hold): no more waits, the results are void
    }
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, w4 = warp & 3, ht = warp >> 2;
    const int VH = c.kv_heads * P.splits;

    // ---- this CTA's run: units [begin, end) of VH * (tiles of all sequences) ----
    volatile int *const found = note + 2;
    if (warp == 0) {
        const unsigned mark = lane == 0 ? ld_l2(reinterpret_cast<const uint32_t *>(P.workspace)) : 0;
        auto tiles_of = [&](int r) { return r < b.n_seq ? pd_seen(pk_length(b, c.page_shift, r, P.err), P.window, P.sinks).tiles : 0; };
        const int len32 = lane < b.n_seq ? pk_length(b, c.page_shift, lane, P.err) : 0, first32 = lane < b.n_seq ? pd_seen(len32, P.window, P.sinks).tiles : 0;
        int sum = first32, most = first32;
        for (int r = lane + 32; r < b.n_seq; r += 32) {
            const int n = tiles_of(r);
            sum += n;
            most = max(most, n);
        }
        const unsigned units = (unsigned)__reduce_add_sync(0xffffffffu, sum) * VH;   // (the host has seen to it that this fits)
        const int longest = __reduce_max_sync(0xffffffffu, most);
        const unsigned per = max((units + gridDim.x - 1) / gridDim.x, longest <= PD_WHOLE ? (unsigned)longest : (unsigned)(sqrtf((float)longest) * PD_RUN + 1.f)), begin = per * blockIdx.x;
        if (begin < units) {   // the sequence that unit `begin` lies in
            unsigned before = 0;
            for (int r0 = 0;; r0 += 32) {
                const unsigned n = r0 == 0 ? first32 : tiles_of(r0 + lane);
                unsigned up = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned x = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += x;
                }
                const unsigned behind = __ballot_sync(0xffffffffu, (before + up) * VH > begin);
                if (behind) {
                    const int l = __ffs(behind) - 1;
                    if (lane == l) {
                        const unsigned rest = begin - (before + up - n) * VH;
                        found[2] = r0 + l;
                        found[3] = (int)(rest / n);
                        found[4] = (int)(rest % n);
                        found[5] = r0 == 0 ? len32 : pk_length(b, c.page_shift, r0 + lane, P.err);
                    }
                    break;
                }
                before += __shfl_sync(0xffffffffu, up, 31);
            }
        }
        if (lane == 0) {
            if (mark != PD_WS_MARK) atomicExch(P.err, DEV_ERR_BAD_WORKSPACE);
            found[0] = mark == PD_WS_MARK && begin < units ? (int)min(per, units - begin) : 0;
            found[1] = (int)per;
        }
    }
    __syncthreads();
    const int n_units = found[0], per = found[1], begin = per * (int)blockIdx.x;
    struct Walk {
        int row, vh, i;
        PdSeen s;
    } at;
    if (n_units == 0) return;
    at.row = found[2];
    at.vh = found[3];
    at.i = found[4];
    at.s = pd_seen(found[5], P.window, P.sinks);
    auto advance = [&](Walk &w) {
        if (++w.i < w.s.tiles) return;
        w.i = 0;
        if (++w.vh < VH) return;
        w.vh = 0;
        if (++w.row < b.n_seq) w.s = pd_seen(pk_length(b, c.page_shift, w.row, P.err), P.window, P.sinks);
    };
    auto start = [](const Walk &w) { return PD_TILE * (w.i < w.s.lead ? w.i : w.i + w.s.skip); };

    auto visible = [](const PdSeen &s, int pos) { return pos < s.len && (pos >= s.from || pos < s.sink); };
    const int box = min(1 << c.page_shift, PD_TILE);   // positions of a box

    if (warp == 4 * HT) {
        // ---- copies: lane i has box i / 2 of a tile, keys or values ----
        const int mine = (lane >> 1) * box;
        const PkTensorMap *const map = lane & 1 ? &maps.v : &maps.k;
        const uint32_t dst = smem_u32(pd_smem) + (lane & 1) * S::TILE_BYTES + mine * (D * 2);
        bool ok = note[1] == 0;
        int u = 0, stage = 0;
        uint32_t phase = 1;   // of the empty barriers: a fresh one counts as passed
        auto look_up = [&](int &pos, bool &live) {   // the page of this lane's box of tile `at`
            pos = start(at) + mine;
            live = mine < PD_TILE && pos < at.s.len && (pos + box > at.s.from || pos < at.s.sink);
            return live ? b.table[(size_t)at.row * b.table_stride + (pos >> c.page_shift)] : 0;
        };
        int pos, vh = at.vh;
        bool live;
        int page = look_up(pos, live);
        for (; u < n_units && ok; u++) {
            if (live && (unsigned)page >= (unsigned)c.n_pages) {
                atomicExch(P.err, DEV_ERR_BAD_PAGE);
                live = false;
            }
            const bool now = live;
            const int at_pos = pos & ((1 << c.page_shift) - 1), at_page = page, at_head = vh / P.splits;
            if (u + 1 < n_units) {
                advance(at);
                vh = at.vh;
                page = look_up(pos, live);
            }
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[stage], phase));
            if (!ok) break;
            const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, now)) * (uint32_t)box * (D * 2);
            if (lane == 0) mbar_arrive_expect_tx(&full[stage], bytes);
            __syncwarp();
            if (now) pk_tma_5d(dst + stage * 2 * S::TILE_BYTES, map, at_pos, 0, at_head, at_page, &full[stage]);
            if (++stage == S::STAGES) stage = 0, phase ^= 1;
        }
        if (!ok && lane == 0) {
            note[1] = 1;
            atomicExch(P.err, DEV_ERR_MBAR_TIMEOUT);
        }
        // no copy is under way when the CTA ends: the last STAGES tiles have been waited for by the workers, or are here
        for (int i = 0; i < S::STAGES && u > 0; i++, u--) {
            if (--stage < 0) stage = S::STAGES - 1, phase ^= 1;
            mbar_wait_bounded(&full[stage], phase ^ 1);
        }
        return;
    }

    // A warp that tells of cut segments: the workers' records have to be visible before the count, and behind loads that wait for the memory that took up to
    // 10000 cycles, in which the workers go on.
    if (warp == 4 * HT + 1) {
        for (int k = 0; k < 2; k++) {
            asm volatile("bar.sync %0, %1;" ::"r"(2 + k), "n"(S::WORKERS + 32) : "memory");
            if (lane == 0 && jobs[5 * k + 3]) {
                unsigned *const count = reinterpret_cast<unsigned *>(P.workspace + PD_WS_HEAD) + jobs[5 * k + 2];
                const bool last = pk_arrive_gpu(count) == (unsigned)jobs[5 * k + 3] - 1;   // all workers' records before it, the others' behind it
                if (last) *count = 0;   // for the next launch
                jobs[5 * k + 4] = last;
            }
            __syncwarp();
        }
        asm volatile("bar.sync 4, %0;" ::"n"(S::WORKERS + 32) : "memory");
        return;
    }

    // ---- products ----
    const int head = lane >> 2, quad = lane & 3;   // of the rows and columns that this thread holds
    uint32_t qa[KS][4];
    float o[KS * 2][2], m = -INFINITY, l = 0.f, to_log2 = 0.f;
    // a row's place in a tile: boxes one after the other, in a box the parts of 64 elements, rows of 128 bytes
    auto place = [&](uint32_t r) { return (r & ~(uint32_t)(box - 1)) * (D * 2) + (r & (uint32_t)(box - 1)) * 128u; };
    const uint32_t part = (uint32_t)box * 128u;
    const uint32_t k_row = 16 * w4 + (lane & 7) + ((lane >> 4) << 3), v_row = 16 * w4 + (lane & 7) + (((lane >> 3) & 1) << 3);
    const uint32_t k_base = smem_u32(pd_smem) + place(k_row), v_base = smem_u32(pd_smem) + S::TILE_BYTES + place(v_row);
    const uint32_t k_x = k_row & 7, v_x = v_row & 7, k_c = (lane >> 3) & 1, v_c = lane >> 4;
    uint32_t phase = 0;
    bool ok = note[1] == 0;
    auto heads_of = [&](int vh) { return min(8 * HT, P.group - (vh % P.splits) * (8 * HT)); };
    auto put = [&](int row, int vh, int h, int d, float4 v, float M, float L) {   // four dims of an output
        const float inv = L > 0.f ? 1.f / L : L != L ? L : 0.f;
        const int q_head = (vh / P.splits) * P.group + (vh % P.splits) * (8 * HT) + h;
        Q *const out = reinterpret_cast<Q *>(P.out) + (size_t)row * P.out_stride + (size_t)q_head * D + d;
        if constexpr (sizeof(Q) == 4) *reinterpret_cast<float4 *>(out) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        else *reinterpret_cast<uint2 *>(out) = make_uint2(pk_pack<Q>(v.x * inv, v.y * inv), pk_pack<Q>(v.z * inv, v.w * inv));
        if (d == 0 && P.lse) P.lse[(size_t)row * P.heads + q_head] = L > 0.f ? (M - PD_BIAS + log2f(L)) * 0.6931471805599453f : L != L ? L : -INFINITY;
    };
    bool fresh = true, first_segment = true;   // a segment begins
    int unit = begin, first_tile = at.i;
    int stage = 0;
    for (int u = 0; u < n_units; u++, unit++) {
        const int group0 = (at.vh % P.splits) * (8 * HT) + ht * 8, mine = group0 + head, q_head = (at.vh / P.splits) * P.group + mine;
        if (fresh) {
            fresh = false;
            first_tile = at.i;
            float2 x[KS][2];
            float most = 0.f;
            const Q *const q = reinterpret_cast<const Q *>(P.q) + (size_t)at.row * P.q_stride + (size_t)q_head * D + quad * 2;
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    x[k][h] = make_float2(0.f, 0.f);
                    if (mine < P.group) {
                        if constexpr (sizeof(Q) == 4) {
                            x[k][h] = *reinterpret_cast<const float2 *>(q + k * 16 + h * 8);
                            most = fmaxf(most, fmaxf(fabsf(x[k][h].x), fabsf(x[k][h].y)));
                        } else {
                            qa[k][2 * h] = *reinterpret_cast<const uint32_t *>(q + k * 16 + h * 8);
                        }
                    } else {
                        qa[k][2 * h] = 0;
                    }
                    qa[k][2 * h + 1] = 0;
                }
            to_log2 = P.scale_log2;
            if constexpr (sizeof(Q) == 4) {
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                float down, up;
                pk_factor(most, down, up);
                to_log2 = P.scale_log2 * up;
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int h = 0; h < 2; h++) pk_split<C>(x[k][h].x * down, x[k][h].y * down, qa[k][2 * h], qa[k][2 * h + 1]);
            }
#pragma unroll
            for (int n = 0; n < KS * 2; n++) o[n][0] = o[n][1] = 0.f;
            m = -INFINITY;
            l = 0.f;
        }
        const int p0 = start(at) + 16 * w4;
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[stage], phase));
        if (!ok && lane == 0) {
            note[1] = 1;
            atomicExch(P.err, DEV_ERR_MBAR_TIMEOUT);
        }
        if (p0 < at.s.len && (p0 + 15 >= at.s.from || p0 < at.s.sink)) {
            float s0[2][4] = {}, s1[2][4] = {};   // even and odd steps: shorter chains
            const uint32_t kt = k_base + stage * 2 * S::TILE_BYTES, vt = v_base + stage * 2 * S::TILE_BYTES;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                uint32_t r[4];
                pk_ldmatrix(r, kt + (k >> 2) * part + (((2 * (k & 3) + k_c) ^ k_x) << 4));
                pk_mma<C>(s0[k & 1], qa[k], r[0], r[1]);
                pk_mma<C>(s1[k & 1], qa[k], r[2], r[3]);
            }
            // an infinite value is one already in the first term; its product with the remainder says nothing
            auto both = [](float hi, float lo) { return fabsf(hi) < INFINITY ? hi + lo : hi; };
            float t[4] = {both(s0[0][0] + s0[1][0], s0[0][2] + s0[1][2]), both(s0[0][1] + s0[1][1], s0[0][3] + s0[1][3]), both(s1[0][0] + s1[1][0], s1[0][2] + s1[1][2]),
                          both(s1[0][1] + s1[1][1], s1[0][3] + s1[1][3])};
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                t[i] = visible(at.s, p0 + quad * 2 + (i & 1) + (i >> 1) * 8) ? t[i] * to_log2 : -INFINITY;
                mx = fmaxf(mx, t[i]);
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m, mx), ref = m_new == -INFINITY ? 0.f : m_new, corr = pd_exp2(m - ref);
            m = m_new;
#pragma unroll
            for (int i = 0; i < 4; i++) t[i] = pd_exp2(t[i] - ref + PD_BIAS);
            l = l * corr + ((t[0] + t[1]) + (t[2] + t[3]));
            if (p0 + 15 >= at.s.len || (p0 < at.s.from && p0 + 15 >= at.s.sink)) {
                // values that are not visible become zeros: whatever they were, zero times it has to be zero
                const uint4 zero = make_uint4(0, 0, 0, 0);
                for (int e = lane; e < 16 * (D / 8); e += 32) {
                    const uint32_t r = 16 * w4 + e / (D / 8), ch = e % (D / 8);
                    if (!visible(at.s, start(at) + (int)r))
                        *reinterpret_cast<uint4 *>(pd_smem + stage * 2 * S::TILE_BYTES + S::TILE_BYTES + place(r) + (ch >> 3) * part + (ch & 7) * 16) = zero;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the next copy to the same place
                __syncwarp();
            }
            uint32_t pa[4];
            pk_split<C>(t[0], t[1], pa[0], pa[1]);
            pk_split<C>(t[2], t[3], pa[2], pa[3]);
#pragma unroll
            for (int d = 0; d < KS; d++) {
                uint32_t r[4];
                pk_ldmatrix_trans(r, vt + (d >> 2) * part + (((2 * (d & 3) + v_c) ^ v_x) << 4));
                float x0[4] = {}, x1[4] = {};
                pk_mma<C>(x0, pa, r[0], r[1]);
                pk_mma<C>(x1, pa, r[2], r[3]);
                o[2 * d][0] = fmaf(o[2 * d][0], corr, both(x0[0], x0[2]));
                o[2 * d][1] = fmaf(o[2 * d][1], corr, both(x0[1], x0[3]));
                o[2 * d + 1][0] = fmaf(o[2 * d + 1][0], corr, both(x1[0], x1[2]));
                o[2 * d + 1][1] = fmaf(o[2 * d + 1][1], corr, both(x1[1], x1[3]));
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
        if (++stage == S::STAGES) stage = 0, phase ^= 1;
        const bool ends = at.i == at.s.tiles - 1;
        if (ends || u == n_units - 1) {
            // ---- the segment's end: the four warps' parts of each head ----
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            float *const of_head = ml + (ht * 8 + head) * 10;
            if (quad == 0) {
                of_head[w4] = m;
                of_head[4 + w4] = l;
            }
            pk_sync_some<S::WORKERS>();
            const float M = fmaxf(fmaxf(of_head[0], of_head[1]), fmaxf(of_head[2], of_head[3])), ref = M == -INFINITY ? 0.f : M;
            const float weight = pd_exp2(m - ref);
            float *const mine_o = merge + ((ht * 4 + w4) * 8 + head) * S::ROW + quad * 2;
#pragma unroll
            for (int n = 0; n < KS * 2; n++) *reinterpret_cast<float2 *>(mine_o + n * 8) = make_float2(o[n][0] * weight, o[n][1] * weight);
            if (w4 == 0 && quad == 0) {
                float L = 0.f;
#pragma unroll
                for (int w = 0; w < 4; w++) L += of_head[4 + w] * pd_exp2(of_head[w] - ref);
                of_head[8] = M;
                of_head[9] = L;
            }
            pk_sync_some<S::WORKERS>();
            const bool whole = ends && first_tile == 0;
            // the CTAs that share the segment, and this one's record: the first of its two where the segment began before it
            const int seg = unit - at.i, cta0 = seg / per, parts = (seg + at.s.tiles - 1) / per - cta0 + 1;
            float *const record = reinterpret_cast<float *>(P.workspace + PD_WS_RECORDS + (size_t)(2 * blockIdx.x + (first_tile == 0 ? 1 : 0)) * S::RECORD);
            const int heads_here = heads_of(at.vh);
            for (int e = tid; e < heads_here * (D / 4); e += S::WORKERS) {
                const int h = e / (D / 4), d = e % (D / 4) * 4;
                const float *const from = merge + ((h >> 3) * 32 + (h & 7)) * S::ROW + d;
                float4 v = *reinterpret_cast<const float4 *>(from);
#pragma unroll
                for (int w = 1; w < 4; w++) {
                    const float4 x = *reinterpret_cast<const float4 *>(from + w * 8 * S::ROW);
                    v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
                }
                const float M_h = ml[h * 10 + 8], L_h = ml[h * 10 + 9];
                if (whole) {
                    put(at.row, at.vh, h, d, v, M_h, L_h);
                } else {
                    float *const r = record + h * (D + 4);
                    if (d == 0) *reinterpret_cast<float2 *>(r) = make_float2(M_h, L_h);
                    *reinterpret_cast<float4 *>(r + 4 + d) = v;
                }
            }
            if (!whole && tid == 0) {
                volatile int *const job = jobs + (first_tile == 0 ? 5 : 0);
                job[0] = at.row, job[1] = at.vh, job[2] = cta0, job[3] = parts;
            }
            if (first_segment) asm volatile("bar.arrive 2, %0;" ::"n"(S::WORKERS + 32) : "memory");
            if (u == n_units - 1) asm volatile("bar.arrive 3, %0;" ::"n"(S::WORKERS + 32) : "memory");
            first_segment = false;
            fresh = true;
        }
        advance(at);
    }
    asm volatile("bar.sync 4, %0;" ::"n"(S::WORKERS + 32) : "memory");   // the counts are in
    for (int k = 0; k < 2; k++) {
        volatile const int *const job = jobs + 5 * k;
        if (!job[4]) continue;
        const int row = job[0], vh = job[1], cta0 = job[2], parts = job[3], heads_here = heads_of(vh);
        pk_sync_some<S::WORKERS>();   // the weights' place and the maxima are free
        // ---- join: part p is of CTA cta0 + p, its second record for p = 0 and its first one after that ----
        const float *const base = reinterpret_cast<const float *>(P.workspace + PD_WS_RECORDS);
        auto part = [&](int p, int h) { return base + ((size_t)2 * (cta0 + p) + (p == 0 ? 1 : 0)) * (S::RECORD / 4) + h * (D + 4); };
        // outputs of the first parts are asked for before their weights are known
        constexpr int AHEAD = 8;
        float4 x[AHEAD];
        auto ask = [&](int e, int p0) {
#pragma unroll
            for (int i = 0; i < AHEAD; i++)
                if (p0 + i < parts && e < heads_here * (D / 4)) x[i] = ld_l2(reinterpret_cast<const float4 *>(part(p0 + i, e / (D / 4)) + 4 + e % (D / 4) * 4));
        };
        ask(tid, 0);
        for (int h = warp; h < heads_here; h += S::WORKERS / 32) {
            float M_h = -INFINITY, L_h = 0.f;
            for (int p0 = lane; p0 < parts; p0 += 128) {
                float2 y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = p0 + 32 * i < parts ? ld_l2(reinterpret_cast<const float2 *>(part(p0 + 32 * i, h))) : make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (p0 + 32 * i < min(parts, S::WEIGHTS)) merge[(p0 + 32 * i) * (8 * HT) + h] = y[i].x;
                    const float top = fmaxf(M_h, y[i].x), ref = top == -INFINITY ? 0.f : top;
                    L_h = L_h * pd_exp2(M_h - ref) + y[i].y * pd_exp2(y[i].x - ref);
                    M_h = top;
                }
            }
            const float M_all = warp_max(M_h), ref_h = M_all == -INFINITY ? 0.f : M_all;
            L_h = warp_sum(L_h * pd_exp2(M_h - ref_h));
            for (int p = lane; p < min(parts, S::WEIGHTS); p += 32) merge[p * (8 * HT) + h] = pd_exp2(merge[p * (8 * HT) + h] - ref_h);
            if (lane == 0) {
                ml[h * 10 + 8] = M_all;
                ml[h * 10 + 9] = L_h;
            }
        }
        pk_sync_some<S::WORKERS>();
        for (int e = tid; e < heads_here * (D / 4); e += S::WORKERS) {
            const int h = e / (D / 4), d = e % (D / 4) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            const float top = ml[h * 10 + 8], ref = top == -INFINITY ? 0.f : top;
            for (int p0 = 0; p0 < parts; p0 += AHEAD) {
                if (p0 > 0 || e != tid) ask(e, p0);
#pragma unroll
                for (int i = 0; i < AHEAD; i++)
                    if (p0 + i < parts) {
                        const float w = p0 < S::WEIGHTS ? merge[(p0 + i) * (8 * HT) + h] : pd_exp2(ld_l2(part(p0 + i, h)) - ref);
                        v = make_float4(fmaf(w, x[i].x, v.x), fmaf(w, x[i].y, v.y), fmaf(w, x[i].z, v.z), fmaf(w, x[i].w, v.w));
                    }
            }
            put(row, vh, h, d, v, top, ml[h * 10 + 9]);
        }
    }
}
#endif  // __CUDACC__

}  // namespace rnb
