// Which page of the pool belongs to which sequence of a model: tables, reference counts, free pages (host memory only).
#pragma once

#include <algorithm>
#include <cstdint>
#include <vector>

namespace elb {

struct PageBook {
    int page = 0, width = 0;                // positions of a page, pages of a sequence
    std::vector<int> free, refs;            // pages nobody has; users of each page
    std::vector<std::vector<int>> table;    // per sequence
    std::vector<int> len;                   // positions of each sequence

    void init(int page_, int n_pages, int n_seq, int n_ctx) {
        page = page_;
        width = (n_ctx + page - 1) / page;
        refs.assign(size_t(n_pages), 0);
        free.clear();
        for (int p = n_pages - 1; p >= 0; --p) free.push_back(p);
        table.assign(size_t(n_seq), {});
        len.assign(size_t(n_seq), 0);
    }
    int pages_of(int positions) const { return (positions + page - 1) / page; }
    int take() {
        const int p = free.back();
        free.pop_back();
        refs[size_t(p)] = 1;
        return p;
    }
    void drop(int p) {
        if (--refs[size_t(p)] == 0) free.push_back(p);
    }
    // the sequence keeps its first `positions` positions
    void shorten(int s, int positions) {
        auto& t = table[size_t(s)];
        while (int(t.size()) > pages_of(positions)) {
            drop(t.back());
            t.pop_back();
        }
        len[size_t(s)] = std::min(len[size_t(s)], positions);
    }
    // the most free pages that sequence s needs to be written from position p0 (<= len) to p1 (exclusive): new ones, and one for a last page
    // that it keeps in part and shares
    int need(int s, int p0, int p1) const {
        const int kept = std::min(pages_of(p0), int(table[size_t(s)].size()));
        return std::max(0, pages_of(p1) - kept) + (shared_tail(s, p0) ? 1 : 0);
    }
    // Are there pages for count[s] rows of every sequence s from first[s] on? Exactly: with what the sequences themselves give back
    bool fits(const std::vector<int>& first, const std::vector<int>& count) const {
        int64_t most = 0;
        for (size_t s = 0; s < count.size(); ++s)
            if (count[s]) most += need(int(s), first[s], first[s] + count[s]);
        if (most <= int64_t(free.size())) return true;
        PageBook b = *this;
        for (size_t s = 0; s < count.size(); ++s)
            if (count[s]) b.shorten(int(s), first[s]);
        for (size_t s = 0; s < count.size(); ++s) {
            if (!count[s]) continue;
            auto& t = b.table[s];
            if (b.shared_tail(int(s), first[s])) {
                if (b.free.empty()) return false;
                const int mine = b.take();
                b.drop(t.back());
                t.back() = mine;
            }
            while (int(t.size()) < b.pages_of(first[s] + count[s])) {
                if (b.free.empty()) return false;
                t.push_back(b.take());
            }
        }
        return true;
    }
    bool shared_tail(int s, int p0) const { return p0 % page && refs[size_t(table[size_t(s)][size_t(p0 / page)])] > 1; }
    // sequences 0.. go on from parent[s]: who needs a copy of the parent's last page (the rule of elb_kv_reorder_dev)
    std::vector<char> copies(const std::vector<int>& parent) const {
        std::vector<char> seen(parent.size(), 0), copy(parent.size(), 0);
        for (size_t s = 0; s < parent.size(); ++s) {
            const size_t p = size_t(parent[s]);
            copy[s] = seen[p] && len[p] % page;
            seen[p] = 1;
        }
        return copy;
    }
    // spare[s] = a page for every s that needs a copy, else -1: free pages, then those that only sequences which are replaced have. (Copies
    // are made from pages that a first child keeps, so none of the latter is a source.) False: there are too few.
    bool spares(const std::vector<int>& parent, const std::vector<char>& copy, std::vector<int>* spare) const {
        size_t left = size_t(std::count(copy.begin(), copy.end(), char(1)));
        std::vector<int> pages(free.end() - std::ptrdiff_t(std::min(left, free.size())), free.end());
        if (pages.size() < left) {
            std::vector<char> kept(refs.size(), 0);
            for (size_t s = 0; s < parent.size(); ++s) {
                const auto& t = table[size_t(parent[s])];
                const int n = pages_of(len[size_t(parent[s])]) - copy[s];
                for (int i = 0; i < n; ++i) kept[size_t(t[size_t(i)])] = 1;
            }
            for (size_t p = 0; p < refs.size() && pages.size() < left; ++p)
                if (refs[p] && !kept[p]) pages.push_back(int(p));
            if (pages.size() < left) return false;
        }
        spare->assign(parent.size(), -1);
        for (size_t s = 0; s < parent.size(); ++s)
            if (copy[s]) (*spare)[s] = pages[--left];
        return true;
    }
    void reorder(const std::vector<int>& parent, const std::vector<int>& spare) {  // spare: as spares() gave them
        std::vector<std::vector<int>> next(table.size());
        std::vector<int> next_len(len.size());
        for (size_t s = 0; s < parent.size(); ++s) {
            const size_t p = size_t(parent[s]);
            next_len[s] = len[p];
            next[s].assign(table[p].begin(), table[p].begin() + pages_of(len[p]));
            if (spare[s] >= 0) next[s].back() = spare[s];
            for (int pg : next[s]) ++refs[size_t(pg)];
        }
        while (!free.empty() && refs[size_t(free.back())]) free.pop_back();  // (spares come from its end)
        for (auto& t : table)
            for (int pg : t) drop(pg);
        table.swap(next);
        len.swap(next_len);
    }
};

// The rows of an evaluation that is under way: until it has ended well their positions do not count. When it goes out of scope before
// that, its sequences end where its rows began.
struct PagedRows {
    PageBook* book = nullptr;        // null: nothing has been changed yet, or all is done
    std::vector<int> first, count;   // per sequence
    PagedRows() = default;
    PagedRows(const PagedRows&) = delete;
    ~PagedRows() {
        for (size_t s = 0; book && s < count.size(); ++s)
            if (count[s]) book->shorten(int(s), first[s]);
    }
};

}  // namespace elb
