// A row of attention over a paged cache in the plain way: a warp walks the visible positions one by one with a running maximum and sum in f32.
// The tensor-core kernel of prompts takes it for rows whose outputs come out infinite or undefined: a value that is not finite,
// times a probability of zero or the remainder of one, says nothing about rows that do not see it.
#pragma once
#include "paged.cuh"

namespace rnb {

#ifdef __CUDACC__
// q, out: the row's D elements; position `pos` of sequence `seq`, key head `head`; lse may be null.
template <class Q, class C, int D>
__device__ __forceinline__ void pk_plain_row(const PkCache &c, const PkBatch &b, const Q *q, int seq, int pos, int head, float scale, int window, int sinks, Q *out, float *lse,
                                                 int *err) {
    constexpr int PER = D / 32;   // dims of a lane
    const int lane = threadIdx.x & 31;
    float x[PER], o[PER] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < PER; i++) x[i] = pk_value<Q>(q[lane * PER + i]);
    const int from = window ? max(0, pos - window + 1) : 0;
#pragma unroll 1
    for (int j = min(sinks, from) > 0 ? 0 : from; j <= pos; j++) {
        if (j < from && j >= sinks) j = from;
        const int page = pk_page(b, c, seq, j, err);
        if (page < 0) continue;
        const size_t e = (size_t)page * c.page_stride + (size_t)(j & ((1 << c.page_shift) - 1)) * c.pos_stride + (size_t)head * c.head_stride + lane * PER;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < PER; i++) s += x[i] * pk_value<C>(reinterpret_cast<const C *>(c.k)[e + i]);
        s = warp_sum(s) * scale;
        const float m_new = fmaxf(m, s), corr = m_new == -INFINITY ? 1.f : expf(m - m_new), p = s != s ? s : m_new == -INFINITY ? 0.f : expf(s - m_new);
        m = m_new;
        l = l * corr + p;
#pragma unroll
        for (int i = 0; i < PER; i++) o[i] = o[i] * corr + p * pk_value<C>(reinterpret_cast<const C *>(c.v)[e + i]);
        if (l != l) break;   // an undefined score, or an infinite one: so is the whole row
    }
#pragma unroll
    for (int i = 0; i < PER; i++) out[lane * PER + i] = pk_rounded<Q>(l == 0.f ? 0.f : o[i] / l);
    if (lse && lane == 0) *lse = l == 0.f ? -INFINITY : m + logf(l);
}
#endif  // __CUDACC__

}  // namespace rnb
