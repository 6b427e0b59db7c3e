// Attention of drafted tokens over the paged cache: what its kernels share.
//
// A span is one request's tree of drafted tokens ("nodes"). Its `context` cached positions lie at places 0 .. context - 1 of
// the request's pages, node j at place context + j. Node i sees a cached place p, whose position is p, and node j where bit j
// of its mask is set, whose position is positions[begin + j]; under a window only keys whose position is above its own minus
// the window. The query heads of a group share a kv head: rows (node, head of the group) of one kv head, the head running
// fastest, are one problem, so that a key is read once for all of them.
//
// The keys are cut into `splits` pieces where the rows alone do not fill the GPU; a block then leaves its rows' unnormalised
// sums with their maximum and denominator in scratch, and a second launch joins the pieces in order. There are no atomics:
// the same inputs give the same bits.
#pragma once
#include "common.cuh"

namespace celeg_b200 {

constexpr int kTreeMaxNodes = 256;            // masks are read in words of 32 nodes, eight at most
constexpr long long kTreeMaxPlaces = 0x7fffffffll - 1024;      // a block of keys behind the last place still has a 32-bit number

struct TreeParams {
    const void* q;                 // [tokens, q_row_stride], head h at h * head_dim
    long long q_row_stride;
    void* out;                     // [tokens, q_heads * head_dim]
    const void* k_cache;           // [pages, kv_heads, page_tokens, head_dim]
    const void* v_cache;
    long long page_stride;
    const int* positions;          // [tokens]
    const int* span_begin;         // [spans + 1]
    const int* span_context;       // [spans]
    const unsigned* ancestors;     // [tokens, words]
    const int* block_table;        // [spans, table_columns], rows table_stride apart
    int words, table_stride, pages, tokens, spans, max_nodes;
    int q_heads, kv_heads, group, head_dim, page_tokens, window, splits;
    int page_shift;                // page_tokens = 1 << page_shift, -1: no power of two
    float scale;
    const float* sinks;            // [q_heads] or null
    float cap_in, cap_out;         // capped scores: cap_out tanh(cap_in * raw score), scale / cap and cap; 0: none
    float* part_o;                 // [tokens, q_heads, splits, head_dim]; null with one split
    float* part_ml;                // [tokens, q_heads, splits, 2]: maximum in units of log2, denominator
    int* error_flag;
    int table_columns;             // (behind the others: in their midst, eight ragged requests took 27.5 us instead of 26.9)
};

// One span as a block sees it; nodes 0 where the block has nothing to do, or must not begin: a span outside the launch's sizes
// (error 4), or with places behind its row of the table (error 2), whose rows are left as they were.
struct TreeSpan {
    int begin, nodes, context;
};

// `report`: sets the error flag (once a launch is enough: a join asks again what its pieces' blocks have asked).
__device__ __forceinline__ TreeSpan tree_span(const TreeParams& p, int span, bool report = true) {
    TreeSpan s;
    s.begin = p.span_begin[span];
    s.nodes = p.span_begin[span + 1] - s.begin;
    s.context = p.span_context[span];
    if (s.begin < 0 || s.nodes < 0 || s.begin > p.tokens - s.nodes || s.nodes > p.max_nodes || s.context < 0) {
        if (report && s.nodes != 0) atomicExch(p.error_flag, 4);
        s.nodes = 0;
    }
    const long long places = (long long)p.table_columns * p.page_tokens;
    if (s.nodes > 0 && (long long)s.context + s.nodes > (places < kTreeMaxPlaces ? places : kTreeMaxPlaces)) {
        if (report) atomicExch(p.error_flag, 2);
        s.nodes = 0;
    }
    return s;
}

// The page that holds `place` of a span, -1 (and error 2) where there is none.
__device__ __forceinline__ int tree_page(const TreeParams& p, const int* table, int place) {
    const int logical = place / p.page_tokens;
    const int page = logical < p.table_columns ? table[logical] : -1;
    if (page < 0 || page >= p.pages) {
        atomicExch(p.error_flag, 2);
        return -1;
    }
    return page;
}

// Whether node i (its mask's words, its position) sees the key at `place`, whose position is `key_position`.
__device__ __forceinline__ bool tree_sees(const TreeParams& p, const TreeSpan& s, const unsigned* mask, int position, int place,
                                          int key_position) {
    const int j = place - s.context;
    const bool there = j < 0 || (j < s.nodes && ((__ldg(mask + (j >> 5)) >> (j & 31)) & 1u));
    return there && (p.window == 0 || (long long)key_position > (long long)position - p.window);
}

// The first cached place that a node at `position` may see.
__device__ __forceinline__ int tree_first_place(const TreeParams& p, const TreeSpan& s, int position) {
    if (p.window == 0) return 0;
    const long long first = (long long)position - p.window + 1;
    return (int)max(0ll, min(first, (long long)s.context));
}

}  // namespace celeg_b200
