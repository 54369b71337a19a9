// A batch over a 4-bit cache, as its kernels (xl_kv.hip, xl_attend.hip) address it: the
// sequences' rows, their tokens' pages, and where a token's codes and scales lie
// (layout and rules: xl_kv_batch in crosslane.h). Plain functions, so that the host's
// tests can walk them with whatever a batch may hold.
#pragma once
#include "xl_format.hpp"

namespace xl {

struct KvBatch {
    uint8_t* pages;
    int64_t page_stride, table_stride;
    const int32_t* table;
    const int32_t* lens;
    const int32_t* starts;
    int dim, kv_heads, page, n_pages, max_pages, n_seqs, rows, max_rows;
    uint32_t page_inv;          // kv_page_inverse(page)
    int* err;
};

// Runs of 16 tokens to pages: run / (page / 16) = run * page_inv >> 32, with page_inv the
// quotient 2^32 / (page / 16) rounded up. It is at most 63 / 64 too large (a page has up to 64 runs), so
// that products of runs up to 2^22 are right. (0: a page is a run.)
XL_HD uint32_t kv_page_inverse(int page) {
    const uint32_t runs = uint32_t(page) / 16;
    return runs > 1 ? uint32_t(((uint64_t(1) << 32) + runs - 1) / runs) : 0u;
}

// Rows of a sequence: the first one, how many, and the sequence's tokens. One whose starts or
// length are out of range (`bad`) has no rows (starts) or no tokens (length).
struct SeqRows {
    int first, n, len;
    bool bad;
};
XL_HD SeqRows seq_rows(const KvBatch& b, int seq) {
    SeqRows r{b.starts[seq], 0, b.lens[seq], false};
    const int end = b.starts[seq + 1];
    if (r.first < 0 || end < r.first || end > b.rows || end - r.first > b.max_rows) {
        r.first = 0;
        r.bad = true;
    } else {
        r.n = end - r.first;
    }
    if (r.len < 0 || r.len > b.max_pages * b.page) {
        r.len = 0;
        r.bad = true;
    }
    return r;
}
// The last sequence that starts at or before row t (the first, if none does).
XL_HD int seq_of(const KvBatch& b, int t) {
    int lo = 0, hi = b.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (b.starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}
// Where the page with a sequence's run of 16 tokens begins, and which run of the page it
// is; -1: the table's entry is no page. run < max_pages * page / 16.
XL_HD int64_t page_at(const KvBatch& b, int seq, uint32_t run, int& run_in_page) {
    const uint32_t col = b.page_inv ? uint32_t((uint64_t(run) * b.page_inv) >> 32) : run;
    run_in_page = int(run - col * uint32_t(b.page >> 4));
    const int id = b.table[int64_t(seq) * b.table_stride + col];
    return uint32_t(id) < uint32_t(b.n_pages) ? int64_t(id) * b.page_stride : -1;
}

// The parts of one kv head in a page of `page` tokens: byte offsets of the keys' scales, the
// values' codes and scales, and the bytes of all four. D: the head's values.
template <int D>
struct Slab {
    static constexpr int G = D / 32;
    int page;
    XL_HD explicit Slab(int p) : page(p) {}
    XL_HD int k_scales() const { return page * (D / 2); }
    XL_HD int v_codes() const { return page * (D / 2 + D / 8); }
    XL_HD int v_scales() const { return page * (D + D / 8); }
    XL_HD int bytes() const { return page * (D + D / 4); }
    // chunk c: dims 8c ..+7 of token `tok` of the page
    XL_HD int k_word(int tok, int c) const { return 4 * (tok * (D / 8) + (c & 3) * G + (c >> 2)); }
    XL_HD int k_scale(int tok, int g) const { return k_scales() + 4 * (tok * G + g); }                       // s, m
    XL_HD int v_half(int tok, int c) const {                                                                 // the second half 4 on
        return v_codes() + 2 * ((tok >> 2) * D + c * 8 + (tok >> 1 & 1) * 4 + (tok & 1));
    }
    XL_HD int v_scale(int tok, int g) const { return v_scales() + 2 * (((tok >> 2) * G + g) * 8 + (tok & 3)); }   // s; m 8 on
};

}  // namespace xl
