// tb_kvpool.cu — host bookkeeping of the paged cache: which sequence holds
// which pages (include/tb_gguf_dequant.h part 4, tb_cuda_kv_pool_*).
//
// Pages are counted by the sequences that hold them.  A fork shares every page
// and raises the counts; the first extension of a sequence whose part-filled
// last page is shared gives it a page of its own, to be filled by
// tb_cuda_kv_copy_dev.  Full shared pages are never written again, so they
// stay shared.  Free pages are handed out lowest first (a min-heap), which
// keeps the pool dense; compaction moves the highest pages in use into the
// lowest free ones.  No CUDA call is made here.
#include <algorithm>
#include <climits>
#include <cstdio>
#include <functional>
#include <new>
#include <vector>

#include "../../include/tb_gguf_dequant.h"

namespace {

struct Seq {
    bool live = false;
    int len = 0;
    std::vector<int> pages;
};

struct Pool {
    int n_pages = 0, page_size = 0;
    std::vector<int> refs;        // sequences that hold each page
    std::vector<int> free_heap;   // min-heap of pages with no holder
    std::vector<Seq> seqs;

    Seq *at(int id)
    {
        return id >= 0 && id < static_cast<int>(seqs.size()) && seqs[id].live ? &seqs[id] : nullptr;
    }
    int take()
    {
        std::pop_heap(free_heap.begin(), free_heap.end(), std::greater<int>());
        const int p = free_heap.back();
        free_heap.pop_back();
        refs[p] = 1;
        return p;
    }
    void drop(int p)   // free_heap has room for every page, so this never allocates
    {
        if (--refs[p] == 0) {
            free_heap.push_back(p);
            std::push_heap(free_heap.begin(), free_heap.end(), std::greater<int>());
        }
    }
    int new_slot()   // may throw; a slot that is not live yet changes nothing
    {
        for (size_t i = 0; i < seqs.size(); ++i)
            if (!seqs[i].live) return static_cast<int>(i);
        if (seqs.size() >= static_cast<size_t>(INT_MAX)) return -1;
        seqs.emplace_back();
        return static_cast<int>(seqs.size()) - 1;
    }
};

Pool *pool_of(void *p) { return static_cast<Pool *>(p); }

}  // namespace

extern "C" {

void *tb_cuda_kv_pool_create(int n_pages, int page_size)
{
    if (n_pages <= 0 || page_size <= 0 || page_size % 16 || page_size > 65536) return nullptr;
    Pool *p = nullptr;
    try {
        p = new Pool;
        p->n_pages = n_pages;
        p->page_size = page_size;
        p->refs.assign(static_cast<size_t>(n_pages), 0);
        p->free_heap.resize(static_cast<size_t>(n_pages));
        for (int i = 0; i < n_pages; ++i) p->free_heap[i] = i;   // ascending: a min-heap
        return p;
    } catch (const std::exception &e) {
        fprintf(stderr, "[tb_cuda] kv_pool_create: %s\n", e.what());
        delete p;
        return nullptr;
    }
}

void tb_cuda_kv_pool_destroy(void *pool) { delete pool_of(pool); }

int tb_cuda_kv_pool_new(void *pool)
{
    if (!pool) return -1;
    try {
        const int id = pool_of(pool)->new_slot();
        if (id >= 0) {
            Seq &s = pool_of(pool)->seqs[id];
            s.live = true;
            s.len = 0;
            s.pages.clear();
        }
        return id;
    } catch (const std::exception &e) {
        fprintf(stderr, "[tb_cuda] kv_pool_new: %s\n", e.what());
        return -1;
    }
}

int tb_cuda_kv_pool_fork(void *pool, int seq)
{
    if (!pool || !pool_of(pool)->at(seq)) return -1;
    Pool &p = *pool_of(pool);
    try {
        const int id = p.new_slot();
        if (id < 0) return -1;
        Seq &to = p.seqs[id];
        const Seq &from = p.seqs[seq];   // after new_slot, which may move the vector
        to.pages = from.pages;
        to.len = from.len;
        to.live = true;
        for (int pg : to.pages) ++p.refs[pg];
        return id;
    } catch (const std::exception &e) {
        fprintf(stderr, "[tb_cuda] kv_pool_fork: %s\n", e.what());
        return -1;
    }
}

int tb_cuda_kv_pool_extend(void *pool, int seq, int n, int *src, int *dst)
{
    if (!pool || n < 0) return -1;
    Pool &p = *pool_of(pool);
    Seq *s = p.at(seq);
    if (!s || n > INT_MAX - s->len) return -1;
    const int len = s->len + n;
    const size_t want = (static_cast<size_t>(len) + p.page_size - 1) / p.page_size;
    const bool own = n > 0 && s->len % p.page_size != 0 && p.refs[s->pages.back()] > 1;
    if (own && (!src || !dst)) return -1;
    if (want - s->pages.size() + (own ? 1 : 0) > p.free_heap.size()) return -1;
    try {
        s->pages.reserve(want);
    } catch (const std::exception &e) {
        fprintf(stderr, "[tb_cuda] kv_pool_extend: %s\n", e.what());
        return -1;
    }
    if (own) {
        *src = s->pages.back();
        *dst = p.take();
        p.drop(*src);
        s->pages.back() = *dst;
    }
    while (s->pages.size() < want) s->pages.push_back(p.take());
    s->len = len;
    return own ? 1 : 0;
}

int tb_cuda_kv_pool_extend_all(void *pool, const int *seqs, const int *n, int count, int *src, int *dst)
{
    if (!pool || count < 0 || (count > 0 && (!seqs || !n || !src || !dst))) return -1;
    Pool &p = *pool_of(pool);
    struct Step {
        int len;        // before
        size_t pages;
        int from;       // the shared page that got a copy, -1: none
    };
    std::vector<Step> done;
    try {
        done.reserve(static_cast<size_t>(count));
    } catch (const std::exception &e) {
        fprintf(stderr, "[tb_cuda] kv_pool_extend_all: %s\n", e.what());
        return -1;
    }
    int copies = 0;
    for (int i = 0; i < count; ++i) {
        const Seq *s = p.at(seqs[i]);
        const Step before{s ? s->len : 0, s ? s->pages.size() : 0, -1};
        int a = -1, b = -1;
        const int r = tb_cuda_kv_pool_extend(pool, seqs[i], n[i], &a, &b);
        if (r >= 0) {
            done.push_back(before);
            if (r == 1) done.back().from = src[copies] = a, dst[copies] = b, ++copies;
            continue;
        }
        for (int k = i - 1; k >= 0; --k) {   // what the ones before it took goes back, last first
            Seq &t = p.seqs[seqs[k]];
            while (t.pages.size() > done[k].pages) {
                p.drop(t.pages.back());
                t.pages.pop_back();
            }
            if (done[k].from >= 0) {
                p.drop(t.pages.back());
                ++p.refs[done[k].from];   // still held by the sequences that it was shared with
                t.pages.back() = done[k].from;
            }
            t.len = done[k].len;
        }
        return -1;
    }
    return copies;
}

int tb_cuda_kv_pool_truncate(void *pool, int seq, int len)
{
    if (!pool) return 0;
    Pool &p = *pool_of(pool);
    Seq *s = p.at(seq);
    if (!s || len < 0 || len > s->len) return 0;
    const size_t want = (static_cast<size_t>(len) + p.page_size - 1) / p.page_size;
    while (s->pages.size() > want) {
        p.drop(s->pages.back());
        s->pages.pop_back();
    }
    s->len = len;
    return 1;
}

int tb_cuda_kv_pool_free(void *pool, int seq)
{
    if (!tb_cuda_kv_pool_truncate(pool, seq, 0)) return 0;
    pool_of(pool)->seqs[seq].live = false;
    return 1;
}

int tb_cuda_kv_pool_compact(void *pool, int *src, int *dst, int cap)
{
    if (!pool || cap < 0 || (cap > 0 && (!src || !dst))) return -1;
    Pool &p = *pool_of(pool);
    try {
        std::vector<int> holes(p.free_heap);
        std::sort(holes.begin(), holes.end());
        std::vector<int> to(static_cast<size_t>(p.n_pages), -1);
        int n = 0;
        int hi = p.n_pages - 1;
        for (size_t h = 0; h < holes.size() && n < cap; ++h) {
            while (hi >= 0 && p.refs[hi] == 0) --hi;
            if (hi < holes[h]) break;
            src[n] = hi;
            dst[n] = holes[h];
            to[hi] = holes[h];
            ++n;
            --hi;
        }
        if (n == 0) return 0;
        for (int i = 0; i < n; ++i) {
            p.refs[dst[i]] = p.refs[src[i]];
            p.refs[src[i]] = 0;
        }
        for (Seq &s : p.seqs)
            for (int &pg : s.pages)
                if (to[pg] >= 0) pg = to[pg];
        p.free_heap.clear();   // keeps its capacity
        for (int i = 0; i < p.n_pages; ++i)
            if (p.refs[i] == 0) p.free_heap.push_back(i);
        return n;
    } catch (const std::exception &e) {
        fprintf(stderr, "[tb_cuda] kv_pool_compact: %s\n", e.what());
        return -1;
    }
}

int tb_cuda_kv_pool_len(void *pool, int seq)
{
    Seq *s = pool ? pool_of(pool)->at(seq) : nullptr;
    return s ? s->len : -1;
}

int tb_cuda_kv_pool_pages(void *pool, int seq, int *pages, int cap)
{
    Seq *s = pool ? pool_of(pool)->at(seq) : nullptr;
    if (!s || (cap > 0 && !pages)) return -1;
    const int n = static_cast<int>(s->pages.size());
    for (int i = 0; i < n && i < cap; ++i) pages[i] = s->pages[i];
    return n;
}

int tb_cuda_kv_pool_free_pages(void *pool)
{
    return pool ? static_cast<int>(pool_of(pool)->free_heap.size()) : -1;
}

}  // extern "C"
