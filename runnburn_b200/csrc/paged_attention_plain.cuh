// Attention over a paged cache, the plain form: a warp per (token, query head) walks the visible positions one by one with a running
// maximum and sum, eight-byte loads, sums in f32.
#pragma once
#include "paged.cuh"

namespace rnb {

template <class Q, class C, int D>
RNB_GLOBAL void paged_attention_plain_kernel(PkCache c, PkBatch b, const Q *q, size_t q_stride, int heads, float scale, int window, int sinks, Q *out, size_t out_stride,
                                             float *lse, int *err) {
    constexpr int PER = D / 32;   // dims of a lane
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == 0) pk_check_starts(b, err);
    const int lane = threadIdx.x & 31;
    const size_t item = (size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int row = (int)(item / heads), head = (int)(item % heads);
    if (row >= b.n_tokens) return;
    const PkRow at = pk_row(b, c.page_shift, row, err);
    if (at.seq < 0) return;
    float x[PER], o[PER] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < PER; i++) x[i] = pk_value<Q>(q[(size_t)row * q_stride + (size_t)head * D + lane * PER + i]);
    const int from = window ? max(0, at.pos - window + 1) : 0, group = heads / c.kv_heads;
    for (int j = min(sinks, from) > 0 ? 0 : from; j <= at.pos; j++) {
        if (j < from && j >= sinks) j = from;
        const int page = pk_page(b, c, at.seq, j, err);
        if (page < 0) continue;
        const size_t e = (size_t)page * c.page_stride + (size_t)(j & ((1 << c.page_shift) - 1)) * c.pos_stride + (size_t)(head / group) * c.head_stride + lane * PER;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < PER; i++) s += x[i] * pk_value<C>(reinterpret_cast<const C *>(c.k)[e + i]);
        s = warp_sum(s) * scale;
        const float m_new = fmaxf(m, s), corr = m_new == -INFINITY ? 1.f : expf(m - m_new), p = m_new == -INFINITY ? 0.f : expf(s - m_new);
        m = m_new;
        l = l * corr + p;
#pragma unroll
        for (int i = 0; i < PER; i++) o[i] = o[i] * corr + p * pk_value<C>(reinterpret_cast<const C *>(c.v)[e + i]);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) out[(size_t)row * out_stride + (size_t)head * D + lane * PER + i] = pk_rounded<Q>(l == 0.f ? 0.f : o[i] / l);
    if (lse && lane == 0) lse[(size_t)row * heads + head] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace rnb
