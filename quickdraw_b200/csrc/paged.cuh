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
    int q_whole;                        // queries in 16-byte pieces
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

template <typename T> QD_DEVINL float paged_load(const T* p) { return (float)*p; }
template <> QD_DEVINL float paged_load<bf16>(const bf16* p) { return __bfloat162float(*p); }
template <typename T> QD_DEVINL void paged_store(T* p, float v);
template <> QD_DEVINL void paged_store<float>(float* p, float v) { *p = v; }
template <> QD_DEVINL void paged_store<bf16>(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int kPagedSeqs = 1024;        // sequences of a launch

// The sequences' parts, in front of one another: before[b] pieces (a part of a pair each) belong to the sequences below b.
template <int THREADS>
QD_DEVINL int paged_schedule(const PagedParams& p, int* before, int* seen) {
    __shared__ int sums[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = p.kv_heads * p.chunks;
    int total = 0;
    for (int base = 0; base < p.batch; base += THREADS) {
        const int b = base + tid;
        int sum = 0;
        if (b < p.batch) {
            seen[b] = paged_span(p, b).seen;
            sum = each * paged_parts(seen[b], p.unit, (long long)p.batch * each, (int)gridDim.x);
        }
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += up;
        }
        if (lane == 31) sums[warp] = sum;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < THREADS / 32; ++w) { if (w < warp) sum += sums[w]; all += sums[w]; }
        if (b < p.batch) before[b + 1] = total + sum;
        total += all;
        __syncthreads();
    }
    if (tid == 0) before[0] = 0;
    __syncthreads();
    return total;
}

struct Piece { int b, kvh, head0, heads, t0, t1, skip, part, parts, pair; };
QD_DEVINL Piece paged_piece(const PagedParams& p, const int* before, const int* seen, int r) {
    int lo = 0;
    for (int hi = p.batch; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= r) lo = mid; else hi = mid;
    }
    Piece a;
    const int each = p.kv_heads * p.chunks, n = seen[lo], at = r - before[lo];
    a.b = lo;
    a.parts = (before[lo + 1] - before[lo]) / each;
    const int pair = at / a.parts, per = ((n + p.unit - 1) / p.unit + a.parts - 1) / a.parts * p.unit;
    a.part = at - pair * a.parts;
    a.kvh = pair / p.chunks;
    const int chunk = pair - a.kvh * p.chunks;
    a.head0 = a.kvh * p.group + chunk * p.chunk;
    a.heads = min(p.chunk, p.group - chunk * p.chunk);
    a.pair = lo * each + pair;
    a.t0 = a.part * per;
    a.t1 = min(n, a.t0 + per);
    a.skip = p.window > 0 && n == p.window + p.sinks ? min(max(p.lengths[lo], 0), p.width * p.page) - n : 0;
    return a;
}

template <typename T>
QD_DEVINL void paged_put(const PagedParams& p, int b, int head, int f, float v) {
    if (p.gate) v *= sigmoid_precise(paged_load((const T*)p.gate + b * p.gate_row + head * p.gate_head + f));
    paged_store((T*)p.out + ((long long)b * p.heads + head) * p.dim + f, v);
}

}  // namespace qd
