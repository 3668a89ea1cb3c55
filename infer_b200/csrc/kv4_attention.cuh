// What the two attention kernels over the 4-bit cache share: their parameters, the rows and tokens of a request, the flat
// list of work that is dealt out in equal shares, and the joining of partial results.
#pragma once

#include "kv4.cuh"

namespace fth {
namespace kv4 {

constexpr int kSiteAttention = 42;

struct AttentionParams {
    Cache cache;
    const void* q;
    void* out;
    float* lse;
    int64_t ldq, ldo, tokens;
    const int32_t* table;
    const int32_t* total_lens;
    const int32_t* query_start;
    int requests, max_blocks, max_query, kv_heads, group, causal, window;
    float scale_log2;  // scale * log2(e): scores are kept as exponents of two
    int* status;
    int* counters;     // one per block of threads: arrivals of the parts of the unit that begins in it
    float* partials;   // [block of threads][2][rows of a unit][head_dim + 2]
};

// The rows of one request and what they see.  Row i of n stands at position total - n + i.
struct Request {
    int first_row;  // row of its first query in q
    int queries;
    int rows;       // queries * group: (query, head of the group), heads innermost
    int length;     // tokens that the table can hold
    int total;
};
__device__ __forceinline__ Request LoadRequest(const AttentionParams& p, int b) {
    Request r;
    r.first_row = b;
    int end = b + 1;
    if (p.query_start != nullptr) {
        r.first_row = p.query_start[b];
        end = p.query_start[b + 1];
    }
    const int64_t limit = p.tokens;
    if (r.first_row < 0 || r.first_row >= limit) { r.first_row = 0; end = 0; }
    if (end > limit) end = static_cast<int>(limit);
    int n = end - r.first_row;
    r.total = p.total_lens[b];
    const int given = n < 0 ? 0 : n;
    n = given > p.max_query ? p.max_query : given;
    // rows are the request's last tokens; rows beyond max_query are not computed, the others keep their positions
    r.total -= given - n;
    r.queries = n;
    r.rows = n * p.group;
    const int64_t room = static_cast<int64_t>(p.max_blocks) << p.cache.block_shift;
    r.length = p.total_lens[b] < 0 ? 0 : p.total_lens[b] > room ? static_cast<int>(room) : p.total_lens[b];
    return r;
}
// Tokens [low, high) that query i of the request sees (high <= low: none).
__device__ __forceinline__ void Visible(const AttentionParams& p, const Request& r, int query, int* low, int* high) {
    const int position = r.total - r.queries + query;
    int h = r.length;
    if (p.causal && position + 1 < h) h = position + 1;
    int l = 0;
    if (p.window > 0 && position + 1 > p.window) l = position + 1 - p.window;
    *low = l;
    *high = h;
}
// Token tiles [first, last) of the unit that holds rows [row, row + count) of a request; at least one, so that a unit
// whose rows see nothing is still somebody's to write.
template <int TILE>
__device__ __forceinline__ void UnitTiles(const AttentionParams& p, const Request& r, int row, int count, int* first, int* last) {
    int end = row + count;
    if (end > r.rows) end = r.rows;
    int l0, h0, l1, h1;
    Visible(p, r, row / p.group, &l0, &h0);
    Visible(p, r, (end - 1) / p.group, &l1, &h1);
    *first = l0 / TILE;
    *last = h1 > 0 ? (h1 + TILE - 1) / TILE : 0;
    if (*last <= *first) *last = *first + 1;
}

}  // namespace kv4
}  // namespace fth
