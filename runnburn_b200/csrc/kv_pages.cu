// Book-keeping of a paged key-value cache (declarations: include/rnb_b200.h).  Host only: the pages of every sequence,
// how many sequences hold each page, and the free ones.
#include <algorithm>
#include <functional>
#include <memory>
#include <new>

#include "state.hpp"

using namespace rnb;

struct rnb_b200_kv_pages {
    struct Seq {
        bool used = false;
        int32_t len = 0;
        int32_t window = 0, sinks = 0;   // of the last release
        std::vector<int32_t> pages;      // -1: released
    };
    mutable std::mutex mutex;
    int32_t n_pages, page_size;
    std::vector<int32_t> holders;   // sequences that hold a page
    std::vector<int32_t> free_heap; // smallest first
    std::vector<Seq> seqs;

    Seq *find(int32_t s) { return s >= 0 && (size_t)s < seqs.size() && seqs[s].used ? &seqs[s] : nullptr; }
    // The heap has room for every page from the start, so giving one back cannot fail.
    void give(int32_t page) {
        if (page < 0 || --holders[page] > 0) return;
        free_heap.push_back(page);
        std::push_heap(free_heap.begin(), free_heap.end(), std::greater<int32_t>());
    }
    int32_t take() {
        std::pop_heap(free_heap.begin(), free_heap.end(), std::greater<int32_t>());
        const int32_t page = free_heap.back();
        free_heap.pop_back();
        holders[page] = 1;
        return page;
    }
    int32_t place(Seq &&s) {   // of a new sequence: the lowest free number
        s.used = true;
        for (size_t i = 0; i < seqs.size(); i++)
            if (!seqs[i].used) {
                seqs[i] = std::move(s);
                return (int32_t)i;
            }
        seqs.push_back(std::move(s));
        return (int32_t)seqs.size() - 1;
    }
};

namespace {
// std::bad_alloc becomes a status: nothing is thrown through the C entries
template <class F>
int guarded(F &&f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return fail(RNB_B200_OUT_OF_MEMORY, "KV pages: out of host memory");
    }
}
int no_seq(int32_t seq) { return fail(RNB_B200_VALIDATION_FAILED, "KV pages: no sequence %d", seq); }
int null_arg() { return fail(RNB_B200_VALIDATION_FAILED, "null pointer argument"); }
}  // namespace

extern "C" {

int rnb_b200_kv_pages_create(int32_t n_pages, int32_t page_size, rnb_b200_kv_pages **out) {
    if (!out) return null_arg();
    if (n_pages < 1) return fail(RNB_B200_VALIDATION_FAILED, "KV pages: n_pages must be at least 1, got %d", n_pages);
    if (page_size < 8 || page_size > 256 || (page_size & (page_size - 1)))
        return fail(RNB_B200_VALIDATION_FAILED, "KV pages: page_size must be a power of two from 8 to 256, got %d", page_size);
    return guarded([&] {
        std::unique_ptr<rnb_b200_kv_pages> p(new rnb_b200_kv_pages);
        p->n_pages = n_pages;
        p->page_size = page_size;
        p->holders.assign(n_pages, 0);
        p->free_heap.resize(n_pages);
        for (int32_t i = 0; i < n_pages; i++) p->free_heap[i] = i;   // ascending is a heap
        *out = p.release();
        return RNB_B200_OK;
    });
}
void rnb_b200_kv_pages_destroy(rnb_b200_kv_pages *p) { delete p; }

int rnb_b200_kv_pages_get_info(const rnb_b200_kv_pages *p, rnb_b200_kv_pages_info *out) {
    if (!p || !out) return null_arg();
    std::lock_guard<std::mutex> g(p->mutex);
    out->n_pages = p->n_pages;
    out->page_size = p->page_size;
    out->free_pages = (int32_t)p->free_heap.size();
    out->n_seqs = (int32_t)std::count_if(p->seqs.begin(), p->seqs.end(), [](const rnb_b200_kv_pages::Seq &s) { return s.used; });
    return RNB_B200_OK;
}

int rnb_b200_kv_pages_new(rnb_b200_kv_pages *p, int32_t *seq_out) {
    if (!p || !seq_out) return null_arg();
    return guarded([&] {
        std::lock_guard<std::mutex> g(p->mutex);
        *seq_out = p->place({});
        return RNB_B200_OK;
    });
}

int rnb_b200_kv_pages_extend(rnb_b200_kv_pages *p, int32_t seq, int32_t n_new, int32_t *n_copies, int32_t *src, int32_t *dst, int32_t *rows) {
    if (!p || !n_copies || !src || !dst || !rows) return null_arg();
    return guarded([&] {
        std::lock_guard<std::mutex> g(p->mutex);
        rnb_b200_kv_pages::Seq *s = p->find(seq);
        if (!s) return no_seq(seq);
        if (n_new < 0 || n_new > INT32_MAX - s->len) return fail(RNB_B200_VALIDATION_FAILED, "KV pages: cannot add %d positions to %d", n_new, s->len);
        const size_t want = (size_t)(((int64_t)s->len + n_new + p->page_size - 1) / p->page_size), have = s->pages.size();
        const int32_t part = s->len % p->page_size, last = have ? s->pages[have - 1] : -1;
        const bool parted = n_new > 0 && part && p->holders[last] > 1;
        const size_t need = want - have + (parted ? 1 : 0);
        if (need > p->free_heap.size())
            return fail(RNB_B200_OUT_OF_MEMORY, "KV pages: %zu pages needed, %zu free", need, p->free_heap.size());
        s->pages.reserve(want);
        *n_copies = 0;
        if (parted) {
            *n_copies = 1;
            *src = last;
            *dst = s->pages[have - 1] = p->take();
            *rows = part;
            p->give(last);
        }
        while (s->pages.size() < want) s->pages.push_back(p->take());
        s->len += n_new;
        return RNB_B200_OK;
    });
}

int rnb_b200_kv_pages_fork(rnb_b200_kv_pages *p, int32_t seq, int32_t *seq_out) {
    if (!p || !seq_out) return null_arg();
    return guarded([&] {
        std::lock_guard<std::mutex> g(p->mutex);
        const rnb_b200_kv_pages::Seq *s = p->find(seq);
        if (!s) return no_seq(seq);
        rnb_b200_kv_pages::Seq copy = *s;
        const std::vector<int32_t> pages = copy.pages;
        *seq_out = p->place(std::move(copy));
        for (int32_t page : pages)
            if (page >= 0) p->holders[page]++;
        return RNB_B200_OK;
    });
}

int rnb_b200_kv_pages_truncate(rnb_b200_kv_pages *p, int32_t seq, int32_t len) {
    if (!p) return null_arg();
    std::lock_guard<std::mutex> g(p->mutex);
    rnb_b200_kv_pages::Seq *s = p->find(seq);
    if (!s) return no_seq(seq);
    if (len < 0 || len > s->len) return fail(RNB_B200_VALIDATION_FAILED, "KV pages: cannot keep %d of %d positions", len, s->len);
    const size_t keep = (size_t)((len + (int64_t)p->page_size - 1) / p->page_size);
    if (len % p->page_size && s->pages[keep - 1] < 0) return fail(RNB_B200_VALIDATION_FAILED, "KV pages: position %d lies in a released page", len - 1);
    for (size_t i = 0; i < keep; i++) {   // the window comes back with the positions
        const int64_t from = (int64_t)i * p->page_size, last = std::min<int64_t>(from + p->page_size, len) - 1;
        if (s->pages[i] < 0 && (last > (int64_t)len - s->window || from < s->sinks))
            return fail(RNB_B200_VALIDATION_FAILED, "KV pages: a token at position %d sees position %lld (window %d, %d sinks), which lies in a released page", len,
                        (long long)(from < s->sinks ? from : last), s->window, s->sinks);
    }
    for (size_t i = keep; i < s->pages.size(); i++) p->give(s->pages[i]);
    s->pages.resize(keep);
    s->len = len;
    return RNB_B200_OK;
}

int rnb_b200_kv_pages_release(rnb_b200_kv_pages *p, int32_t seq, int32_t window, int32_t sinks) {
    if (!p) return null_arg();
    if (window < 1 || sinks < 0) return fail(RNB_B200_VALIDATION_FAILED, "KV pages: window must be at least 1 and sinks at least 0, got %d and %d", window, sinks);
    std::lock_guard<std::mutex> g(p->mutex);
    rnb_b200_kv_pages::Seq *s = p->find(seq);
    if (!s) return no_seq(seq);
    const int64_t size = p->page_size, first = (sinks + size - 1) / size, unseen = (int64_t)s->len - window + 1;   // positions below `unseen`
    for (int64_t i = first; (i + 1) * size <= unseen; i++) {
        p->give(s->pages[i]);
        s->pages[i] = -1;
    }
    s->window = window;
    s->sinks = sinks;
    return RNB_B200_OK;
}

int rnb_b200_kv_pages_free(rnb_b200_kv_pages *p, int32_t seq) {
    if (!p) return null_arg();
    std::lock_guard<std::mutex> g(p->mutex);
    rnb_b200_kv_pages::Seq *s = p->find(seq);
    if (!s) return no_seq(seq);
    for (int32_t page : s->pages) p->give(page);
    *s = {};
    return RNB_B200_OK;
}

int rnb_b200_kv_pages_compact(rnb_b200_kv_pages *p, int32_t *src, int32_t *dst, size_t cap, size_t *n_copies) {
    if (!p || !n_copies || (cap && (!src || !dst))) return null_arg();
    return guarded([&] {
        std::lock_guard<std::mutex> g(p->mutex);
        const int32_t used = p->n_pages - (int32_t)p->free_heap.size();
        std::vector<int32_t> to(p->n_pages, -1);   // where a page at the end of the pool goes
        size_t n = 0;
        for (int32_t page = used; page < p->n_pages; page++) n += p->holders[page] > 0;
        *n_copies = n;
        if (n > cap) return fail(RNB_B200_VALIDATION_FAILED, "KV pages: %zu pages to move, room for %zu", n, cap);
        size_t i = 0;
        for (int32_t page = used, hole = 0; page < p->n_pages; page++) {
            if (p->holders[page] == 0) continue;
            while (p->holders[hole] > 0) hole++;   // as many holes below `used` as pages behind it
            src[i] = page;
            dst[i++] = to[page] = hole;
            p->holders[hole] = p->holders[page];
            p->holders[page] = 0;
        }
        for (auto &s : p->seqs)
            for (int32_t &page : s.pages)
                if (page >= 0 && to[page] >= 0) page = to[page];
        for (int32_t k = used; k < p->n_pages; k++) p->free_heap[k - used] = k;
        return RNB_B200_OK;
    });
}

int rnb_b200_kv_pages_tables(const rnb_b200_kv_pages *p, const int32_t *seqs, size_t n, int32_t *table, size_t stride, int32_t *kv_len) {
    if (!p || (n && (!seqs || !(table || kv_len)))) return null_arg();
    std::lock_guard<std::mutex> g(p->mutex);
    rnb_b200_kv_pages *q = const_cast<rnb_b200_kv_pages *>(p);
    for (size_t i = 0; i < n; i++) {
        const rnb_b200_kv_pages::Seq *s = q->find(seqs[i]);
        if (!s) return no_seq(seqs[i]);
        if (table && s->pages.size() > stride) return fail(RNB_B200_VALIDATION_FAILED, "KV pages: sequence %d has %zu pages, a row of the table %zu entries", seqs[i], s->pages.size(), stride);
    }
    for (size_t i = 0; i < n; i++) {
        const rnb_b200_kv_pages::Seq &s = *q->find(seqs[i]);
        if (table) std::fill(std::copy(s.pages.begin(), s.pages.end(), table + i * stride), table + (i + 1) * stride, -1);
        if (kv_len) kv_len[i] = s.len;
    }
    return RNB_B200_OK;
}

}  // extern "C"
