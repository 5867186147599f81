// The page book of a paged model, for tests without a GPU.
#include "../exactinfer_b200/csrc/pages.cuh"

using elb::PageBook;
using elb::PagedRows;

extern "C" {
PageBook* book_new(int page, int n_pages, int n_seq, int n_ctx) {
    auto* b = new PageBook;
    b->init(page, n_pages, n_seq, n_ctx);
    return b;
}
void book_delete(PageBook* b) { delete b; }
int book_free(const PageBook* b) { return int(b->free.size()); }
int book_len(const PageBook* b, int s) { return b->len[size_t(s)]; }
int book_pages(const PageBook* b, int s, int* out) {
    const auto& t = b->table[size_t(s)];
    std::copy(t.begin(), t.end(), out);
    return int(t.size());
}
int book_refs(const PageBook* b, int page) { return b->refs[size_t(page)]; }
void book_drop(PageBook* b, int s) { b->shorten(s, 0); }
// 1: sequences go on from parent[s], spare[s] is the page of its copy or -1; 0: no pages for the copies
int book_reorder(PageBook* b, int n_seq, const int* parent, int* spare) {
    const std::vector<int> from(parent, parent + n_seq);
    std::vector<int> pages;
    if (!b->spares(from, b->copies(from), &pages)) return 0;
    std::copy(pages.begin(), pages.end(), spare);
    b->reorder(from, pages);
    return 1;
}
// An evaluation of count[s] rows from first[s] on: 1 when it fits. `stop` >= 0: it fails when so many sequences have their pages
int book_eval(PageBook* b, int n_seq, const int* first, const int* count, int stop) {
    PagedRows rows;
    rows.first.assign(first, first + n_seq);
    rows.count.assign(count, count + n_seq);
    if (!b->fits(rows.first, rows.count)) return 0;
    rows.book = b;
    for (int s = 0; s < n_seq; ++s)
        if (count[s]) b->shorten(s, first[s]);
    for (int s = 0; s < n_seq; ++s) {
        if (!count[s]) continue;
        if (stop-- == 0) return -1;
        auto& t = b->table[size_t(s)];
        if (b->shared_tail(s, first[s])) {
            const int mine = b->take();
            b->drop(t.back());
            t.back() = mine;
        }
        while (int(t.size()) < b->pages_of(first[s] + count[s])) t.push_back(b->take());
        b->len[size_t(s)] = first[s] + count[s];
    }
    if (stop == 0) return -1;
    rows.book = nullptr;
    return 1;
}
}
