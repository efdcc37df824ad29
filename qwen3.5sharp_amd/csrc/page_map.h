// Host-only: which pages a paged cache's sequences map, and what a call may
// read and write through them.
//
// A sequence is a row of page ids (-1: not mapped) and a length.  A page may
// be mapped by several entries (a prefix that sequences share); such a page
// is read-only: a call that would write a row into it is refused, since the
// row would change under the other entry (the caller maps a copy first).  So
// the rows that one call writes for different sequences are always in
// different pages, and no sequence reads a page that another one writes.
// The device copy of the table holds only ids that passed these checks.
#pragma once

#include <cstddef>
#include <vector>

namespace q35 {

class PageMap {
public:
    enum Result { kOk = 0, kBadSeq, kBadRange, kBadPage, kShared, kUnmapped, kTooLong };

    // Sequences of up to max_rows rows, pages of page_rows.
    PageMap(int n_seqs, int max_rows, int n_pages, int page_rows)
        : n_seqs_(n_seqs), max_rows_(max_rows), max_pages_((max_rows + page_rows - 1) / page_rows), n_pages_(n_pages),
          page_rows_(page_rows), table_((size_t)n_seqs * max_pages_, -1), refs_(n_pages, 0), len_(n_seqs, 0),
          mapped_(n_seqs, 0) {}

    int n_seqs() const { return n_seqs_; }
    int max_rows() const { return max_rows_; }
    int max_pages() const { return max_pages_; }
    int page_rows() const { return page_rows_; }
    int length(int seq) const { return len_[seq]; }
    void set_length(int seq, int len) { len_[seq] = len; }
    int page(int seq, int i) const { return table_[(size_t)seq * max_pages_ + i]; }
    bool has(int seq) const { return seq >= 0 && seq < n_seqs_; }

    // Whether map() would take these arguments.
    Result can_map(int seq, int first, int n, const int* pages) const {
        if (!has(seq)) return kBadSeq;
        if (first < 0 || n < 0 || first > max_pages_ - n) return kBadRange;
        if (pages)
            for (int i = 0; i < n; ++i)
                if (pages[i] < 0 || pages[i] >= n_pages_) return kBadPage;
        return kOk;
    }
    // Entries [first, first + n) of seq become pages[0 .. n) (null: unmapped).
    // Nothing changes unless every argument is good.
    Result map(int seq, int first, int n, const int* pages) {
        const Result r = can_map(seq, first, n, pages);
        if (r != kOk) return r;
        int* t = &table_[(size_t)seq * max_pages_];
        for (int i = 0; i < n; ++i) {
            if (t[first + i] >= 0) --refs_[t[first + i]];
            t[first + i] = pages ? pages[i] : -1;
            if (pages) ++refs_[pages[i]];
        }
        if (!pages) {
            if (n && mapped_[seq] > first) mapped_[seq] = first;
        } else if (first <= mapped_[seq]) {
            while (mapped_[seq] < max_pages_ && t[mapped_[seq]] >= 0) ++mapped_[seq];
        }
        return kOk;
    }

    // Whether a call may read seq's rows [0, length + tokens) and, of these,
    // write the last `tokens`.
    Result usable(int seq, int tokens) const {
        if (!has(seq)) return kBadSeq;
        const long rows = (long)len_[seq] + tokens;
        if (rows > max_rows_) return kTooLong;
        if (rows > (long)mapped_[seq] * page_rows_) return kUnmapped;
        if (tokens > 0)
            for (int i = len_[seq] / page_rows_; i <= (rows - 1) / page_rows_; ++i)
                if (refs_[page(seq, i)] > 1) return kShared;
        return kOk;
    }

    // Whether rows [first, first + n) of seq may be read; `bound`: as far as max_rows goes, mapped or not.
    Result readable(int seq, int first, int n, bool bound) const {
        if (!has(seq)) return kBadSeq;
        if (first > max_rows_ - n) return kTooLong;
        if (!bound && n > 0)
            for (int i = first / page_rows_; i <= (first + n - 1) / page_rows_; ++i)
                if (page(seq, i) < 0) return kUnmapped;
        return kOk;
    }

private:
    int n_seqs_, max_rows_, max_pages_, n_pages_, page_rows_;
    std::vector<int> table_;
    std::vector<int> refs_;     // entries that map a page
    std::vector<int> len_;
    std::vector<int> mapped_;   // entries [0, mapped) are all mapped
};

}  // namespace q35
