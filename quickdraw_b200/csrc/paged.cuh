// Attention of one new token over a paged cache: what is to be done, and how it is shared out.
#pragma once
#include "common.cuh"

namespace qd {

struct PagedParams {
    const void* q; const void* gate; const void* k; const void* v;
    long long q_row, q_head, gate_row, gate_head, page_stride, row_stride, head_stride, table_stride;   // in elements
    const int* table; const int* lengths;
    void* out;                          // [batch, heads, dim]
    float* partial;                     // [pair][most][heads of a chunk][dim + 2]: weighted values, maximum, sum
    int batch, heads, kv_heads, dim, pages, page, width, window, sinks;
    int group, chunk, chunks;           // query heads of a key/value head; of them at a time; how often
    int unit, most;                     // positions of a unit; parts of a pair, at most
    float scale;                        // of the scores, times log2(e)
};

// What a sequence of n positions sees: the i-th of `seen` is at i, or, behind the first `sinks`, at i + skip.
struct Span { int seen, skip; };
QD_DEVINL Span paged_span(const PagedParams& p, int b) {
    const int n = min(max(p.lengths[b], 0), p.width * p.page);
    Span s{n, 0};
    if (p.window > 0 && (long long)n > (long long)p.window + p.sinks) { s.seen = p.window + p.sinks; s.skip = n - s.seen; }
    return s;
}
QD_DEVINL int paged_position(const PagedParams& p, int i, int skip) { return i < p.sinks ? i : i + skip; }

// A sequence is cut into parts by its own length, the number of (sequence, key/value head, chunk of heads) triples and that of blocks alone, so that
// its result does not depend on its neighbours: as if all of the batch were as long, each block gets one part, or, if that is a long one, several
// equal ones, because beside other lengths smaller parts are shared out more evenly.
constexpr int kPagedRound = 4, kPagedRounds = 16;
static __host__ __device__ __forceinline__ int paged_parts(int seen, int unit, long long pairs, int blocks) {
    if (seen <= 0) return 0;
    const long long n = (seen + unit - 1) / unit, share = (n * pairs + blocks - 1) / blocks;
    long long rounds = share / kPagedRound;
    rounds = rounds < 1 ? 1 : rounds > kPagedRounds ? kPagedRounds : rounds;
    const long long per = (share + rounds - 1) / rounds;
    return (int)((n + per - 1) / per);
}
// An upper bound of it over all lengths (n * rounds / share <= rounds * blocks / pairs, rounded up).
static __host__ __device__ __forceinline__ int paged_most(long long pairs, int blocks) {
    return (int)((long long)kPagedRounds * blocks / (pairs > 0 ? pairs : 1)) + 1;
}

}  // namespace qd
