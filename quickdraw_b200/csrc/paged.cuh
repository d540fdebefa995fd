// Attention of one new token over a paged cache: what is to be done, and how it is shared out.
#pragma once
#include "common.cuh"

namespace qd {

struct PagedParams {
    const void* q; const void* gate; const void* k; const void* v;
    long long q_row, q_head, gate_row, gate_head, page_stride, row_stride, head_stride, table_stride;   // in elements
    const int* table; const int* lengths;
    void* out;                          // [batch, heads, dim]
    float* partial; float2* stats;      // [pair][most][heads of a chunk][dim]: weighted values; [pair][most][heads of a chunk]: maximum, sum
    int batch, heads, kv_heads, dim, pages, page, width, window, sinks;
    int group, chunk, chunks;           // query heads of a key/value head; of them at a time; how often
    int unit, most;                     // positions of a unit; parts of a pair, at most
    int q_whole;                        // queries in 16-byte pieces
    float scale;                        // of the scores, times log2(e)
};

// What a sequence of n positions sees: the i-th of `seen` is at i, or, behind the first `sinks`, at i + skip.
struct Span { int seen, skip; };
QD_DEVINL Span paged_span(const PagedParams& p, int b) {
    const int n = min(max(__ldcg(p.lengths + b), 0), p.width * p.page);
    Span s{n, 0};
    if (p.window > 0 && (long long)n > (long long)p.window + p.sinks) { s.seen = p.window + p.sinks; s.skip = n - s.seen; }
    return s;
}
QD_DEVINL int paged_position(const PagedParams& p, int i, int skip) { return i < p.sinks ? i : i + skip; }

// A sequence is cut into parts by its own length, the number of (sequence, key/value head, chunk of heads) triples and that of workers alone, so that
// its result does not depend on its neighbours: as if all of the batch were as long, each worker gets one part, or, if that is a long one, several
// equal ones, because beside other lengths smaller parts are shared out more evenly.
constexpr int kPagedLeast = 4, kPagedRound = 8, kPagedRounds = 4;
static __host__ __device__ __forceinline__ int paged_most(long long pairs, int workers) {
    const long long most = (long long)kPagedRounds * workers / pairs;
    return most < 1 ? 1 : (int)most;
}
static __host__ __device__ __forceinline__ int paged_parts(int seen, int unit, int pairs, int workers) {
    if (seen <= 0) return 0;
    const int n = (seen - 1) / unit + 1;
    const float share = (float)n * (float)pairs / (float)workers;                 // units of a worker, if all were as long
    const int rounds = share < 2.f * kPagedRound ? 1 : share < (float)kPagedRounds * kPagedRound ? (int)(share / kPagedRound) : kPagedRounds;
    const int parts = rounds * workers / pairs;                                   // (at most kPagedRounds * workers)
    int per = parts > 1 ? (n + parts - 1) / parts : n;
    if (per < kPagedLeast) per = kPagedLeast;
    return (n + per - 1) / per;
}

template <typename T> QD_DEVINL float paged_load(const T* p) { return (float)*p; }
template <> QD_DEVINL float paged_load<bf16>(const bf16* p) { return __bfloat162float(*p); }
template <typename T> QD_DEVINL void paged_store(T* p, float v);
template <> QD_DEVINL void paged_store<float>(float* p, float v) { *p = v; }
template <> QD_DEVINL void paged_store<bf16>(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int kPagedSeqs = 256;        // sequences of a launch

// The parts of all sequences, those of the largest parts first.
struct PagedOrder {
    int before[kPagedSeqs + 1];         // pieces (a part of a pair each) in front of the i-th sequence's
    int seen[kPagedSeqs];               // rows that it sees
    uint8_t sequence[kPagedSeqs];
};
template <int THREADS>
QD_DEVINL int paged_schedule(const PagedParams& p, PagedOrder& o, int workers) {
    __shared__ int sums[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = p.kv_heads * p.chunks;
    // units of a part (in `before`, for a moment), and how many sequences have larger ones
    for (int b = tid; b < p.batch; b += THREADS) {
        const int n = paged_span(p, b).seen, parts = paged_parts(n, p.unit, p.batch * each, workers);
        o.before[b] = parts ? ((n - 1) / p.unit + parts) / parts : 0;
    }
    __syncthreads();
    constexpr int kEach = (kPagedSeqs + THREADS - 1) / THREADS;
    int rank[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int b = j * THREADS + tid, per = b < p.batch ? o.before[b] : 0;
        rank[j] = 0;
        if (b < p.batch)
            for (int z = 0; z < p.batch; ++z) rank[j] += o.before[z] > per || (o.before[z] == per && z < b);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int b = j * THREADS + tid;
        if (b < p.batch) { o.sequence[rank[j]] = (uint8_t)b; o.seen[rank[j]] = paged_span(p, b).seen; }
    }
    __syncthreads();
    int total = 0;
    for (int base = 0; base < p.batch; base += THREADS) {
        const int i = base + tid;
        int sum = i < p.batch ? each * paged_parts(o.seen[i], p.unit, p.batch * each, workers) : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += up;
        }
        if (lane == 31) sums[warp] = sum;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < THREADS / 32; ++w) { if (w < warp) sum += sums[w]; all += sums[w]; }
        if (i < p.batch) o.before[i + 1] = total + sum;
        total += all;
        __syncthreads();
    }
    if (tid == 0) o.before[0] = 0;
    __syncthreads();
    return total;
}
// Rounds of pieces, one a worker, to and fro, so that who had a larger one takes a smaller one next: the piece after piece r.
QD_DEVINL int paged_next(int r, int workers) {
    const int round = r / workers;
    return 2 * (round + 1) * workers - 1 - r;
}

struct Piece { int b, kvh, head0, heads, t0, t1, skip, part, parts, pair; };
QD_DEVINL Piece paged_piece(const PagedParams& p, const PagedOrder& o, int r) {
    int lo = 0;
    for (int hi = p.batch; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (o.before[mid] <= r) lo = mid; else hi = mid;
    }
    Piece a;
    const int each = p.kv_heads * p.chunks, n = o.seen[lo], at = r - o.before[lo];
    a.b = o.sequence[lo];
    a.parts = (o.before[lo + 1] - o.before[lo]) / each;
    const int pair = at / a.parts, per = ((n + p.unit - 1) / p.unit + a.parts - 1) / a.parts * p.unit;
    a.part = at - pair * a.parts;
    a.kvh = pair / p.chunks;
    const int chunk = pair - a.kvh * p.chunks;
    a.head0 = a.kvh * p.group + chunk * p.chunk;
    a.heads = min(p.chunk, p.group - chunk * p.chunk);
    a.pair = a.b * each + pair;
    a.t0 = a.part * per;
    a.t1 = min(n, a.t0 + per);
    a.skip = p.window > 0 && n == p.window + p.sinks ? min(max(__ldcg(p.lengths + a.b), 0), p.width * p.page) - n : 0;
    return a;
}

QD_DEVINL long long paged_place(const PagedParams& p, const Piece& a, int h) { return ((long long)a.pair * p.most + a.part) * p.chunk + h; }

template <typename T>
QD_DEVINL void paged_put(const PagedParams& p, int b, int head, int f, float v) {
    if (p.gate) v *= sigmoid_precise(paged_load((const T*)p.gate + b * p.gate_row + head * p.gate_head + f));
    paged_store((T*)p.out + ((long long)b * p.heads + head) * p.dim + f, v);
}

}  // namespace qd
