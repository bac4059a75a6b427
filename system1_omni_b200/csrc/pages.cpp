// Who owns which page of a paged cache: the host's side of the page tables (append with copy on
// write, fork, truncate, compact). Plain bookkeeping, no device calls; the copies that it asks for
// are s1_pages_copy's.
#include <algorithm>
#include <exception>
#include <vector>

#include "s1_executor.h"

namespace {

struct Pages {
    int page_tokens, max_seq_pages;
    std::vector<int> free;              // page numbers, taken from the back
    std::vector<int> users;             // sequences that name a page
    std::vector<std::vector<int>> seq;  // a sequence's pages
    std::vector<int> tokens;            // and its tokens

    bool has(int s) const { return s >= 0 && s < (int)seq.size(); }
    int take() {
        const int p = free.back();
        free.pop_back();
        users[p] = 1;
        return p;
    }
    void drop(int p) {
        if (--users[p] == 0) free.push_back(p);  // within the capacity it was made with
    }
};

Pages* of(void* p) { return static_cast<Pages*>(p); }

}  // namespace

extern "C" int s1_pages_create(int n_pages, int page_tokens, int max_seqs, int max_seq_pages, void** pages) {
    if (!pages || n_pages <= 0 || page_tokens <= 0 || max_seqs <= 0 || max_seq_pages <= 0) return S1_ERR_ARGUMENT;
    if ((long long)max_seq_pages * page_tokens > 0x7fffffffLL) return S1_ERR_ARGUMENT;
    *pages = nullptr;
    try {
        Pages* p = new Pages;
        *pages = p;
        p->page_tokens = page_tokens;
        p->max_seq_pages = max_seq_pages;
        p->free.resize(n_pages);
        for (int i = 0; i < n_pages; i++) p->free[i] = n_pages - 1 - i;
        p->users.assign(n_pages, 0);
        p->seq.resize(max_seqs);
        p->tokens.assign(max_seqs, 0);
    } catch (const std::exception&) {
        delete of(*pages);
        *pages = nullptr;
        return S1_ERR_PAGES;
    }
    return 0;
}

extern "C" void s1_pages_destroy(void* pages) { delete of(pages); }

extern "C" int s1_pages_append(void* pages, int seq, int tokens, int* src, int* dst, int cap, int* n_copies) {
    Pages* p = of(pages);
    if (!p || !p->has(seq) || tokens < 0 || cap < 0 || (cap > 0 && (!src || !dst)) || !n_copies) return S1_ERR_ARGUMENT;
    std::vector<int>& own = p->seq[seq];
    const long long want = (long long)p->tokens[seq] + tokens;
    const long long need = (want + p->page_tokens - 1) / p->page_tokens;
    // the tokens would land in a page that someone else reads
    const bool copy = tokens > 0 && p->tokens[seq] % p->page_tokens != 0 && p->users[own.back()] > 1;
    if (need > p->max_seq_pages || need - (long long)own.size() + copy > (long long)p->free.size() || (copy && cap < 1)) return S1_ERR_PAGES;
    try {
        own.reserve((size_t)need);
    } catch (const std::exception&) {
        return S1_ERR_PAGES;
    }
    *n_copies = copy;
    if (copy) {
        src[0] = own.back();
        own.back() = dst[0] = p->take();
        p->users[src[0]]--;
    }
    while ((long long)own.size() < need) own.push_back(p->take());
    p->tokens[seq] = (int)want;
    return 0;
}

extern "C" int s1_pages_fork(void* pages, int from, int to) {
    Pages* p = of(pages);
    if (!p || !p->has(from) || !p->has(to) || from == to || !p->seq[to].empty()) return S1_ERR_ARGUMENT;
    try {
        p->seq[to] = p->seq[from];
    } catch (const std::exception&) {
        p->seq[to].clear();
        return S1_ERR_PAGES;
    }
    for (int page : p->seq[to]) p->users[page]++;
    p->tokens[to] = p->tokens[from];
    return 0;
}

extern "C" int s1_pages_truncate(void* pages, int seq, int tokens) {
    Pages* p = of(pages);
    if (!p || !p->has(seq) || tokens < 0 || tokens > p->tokens[seq]) return S1_ERR_ARGUMENT;
    const size_t keep = ((size_t)tokens + p->page_tokens - 1) / p->page_tokens;
    std::vector<int>& own = p->seq[seq];
    while (own.size() > keep) {
        p->drop(own.back());
        own.pop_back();
    }
    p->tokens[seq] = tokens;
    return 0;
}

extern "C" int s1_pages_compact(void* pages, int* src, int* dst, int cap, int* n_copies) {
    Pages* p = of(pages);
    if (!p || cap < 0 || (cap > 0 && (!src || !dst)) || !n_copies) return S1_ERR_ARGUMENT;
    const int total = (int)p->users.size(), used = total - (int)p->free.size();
    // used pages at or behind place `used` move into the free places before it, in ascending order
    int moves = 0;
    for (int i = used; i < total; i++) moves += p->users[i] > 0;
    if (moves > cap) return S1_ERR_PAGES;
    std::vector<int> place;
    try {
        place.assign(total, -1);
    } catch (const std::exception&) {
        return S1_ERR_PAGES;
    }
    *n_copies = moves;
    int hole = 0, n = 0;
    for (int i = used; i < total; i++) {
        if (p->users[i] == 0) continue;
        while (p->users[hole] > 0) hole++;
        src[n] = i;
        dst[n++] = place[i] = hole;
        p->users[hole] = p->users[i];
        p->users[i] = 0;
    }
    for (std::vector<int>& own : p->seq)
        for (int& page : own)
            if (place[page] >= 0) page = place[page];
    for (int i = 0; i < total - used; i++) p->free[i] = total - 1 - i;  // the lowest is taken first
    return 0;
}

extern "C" int s1_pages_table(void* pages, int seq, int n, int* table, int table_pages, int* len) {
    Pages* p = of(pages);
    if (!p || seq < 0 || n < 0 || n > (int)p->seq.size() - seq || (table && table_pages <= 0)) return S1_ERR_ARGUMENT;
    if (table)
        for (int i = 0; i < n; i++)
            if (p->seq[seq + i].size() > (size_t)table_pages) return S1_ERR_ARGUMENT;
    for (int i = 0; i < n; i++) {
        const std::vector<int>& own = p->seq[seq + i];
        if (table) {
            int* row = table + (size_t)i * table_pages;
            std::copy(own.begin(), own.end(), row);
            std::fill(row + own.size(), row + table_pages, -1);
        }
        if (len) len[i] = p->tokens[seq + i];
    }
    return 0;
}

extern "C" int s1_pages_free_count(void* pages) { return pages ? (int)of(pages)->free.size() : 0; }
