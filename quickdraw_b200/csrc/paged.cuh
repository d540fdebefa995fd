// Attention of one new token over a paged cache: what is to be done, and how it is shared out.
#pragma once
#include "common.cuh"

namespace qd {

// Of the current device, asked for once: -1 where there is none.
constexpr int kDevices = 64;
static inline int current_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kDevices ? dev : -1;
}
static inline int device_blocks() {
    static int known[kDevices];
    const int dev = current_device();
    if (dev < 0) return 148;
    if (!known[dev]) {
        int sms = 0;
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        known[dev] = sms > 0 ? sms : 148;
    }
    return known[dev];
}
// A kernel's limit of dynamic shared memory, raised once per device (`raised`: of this kernel).
template <typename... KArgs>
static inline bool raise_smem(void (*kernel)(KArgs...), size_t bytes, bool (&raised)[kDevices]) {
    const int dev = current_device();
    if (dev < 0) return false;
    if (!raised[dev]) raised[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess;
    return raised[dev];
}

// Two numbers in one instruction.
QD_DEVINL float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
QD_DEVINL float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
QD_DEVINL float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// A sequence is cut into parts by its own length, the number of (sequence, key/value head, chunk of heads) triples and that of workers alone, so that
// its result does not depend on its neighbours: as if all of the batch were as long, so that they fill some rounds of workers in least time (a part
// costs `kPagedFixed` units beside its own: its state is written, read and joined); of cuts that are within 1 / 16 of it the finest, because beside
// other lengths smaller parts are shared out more evenly.
constexpr int kPagedCuts = 6;
constexpr float kPagedFixed = 1.f;
// parts of a sequence (their reciprocal), rounds of workers; the most parts of any, 0: one each, whose results the parts' kernel writes itself
struct PagedCuts { float each[kPagedCuts], rounds[kPagedCuts]; int most; };
// Caches of at most kPagedWhole units are not cut (a second launch costs more than it would save: one sequence of 256 positions 8.8 us instead of 9.0,
// 200 of them 22.6 instead of 31; 512 positions 12.7 instead of 9.2), nor are those of more pairs than the finest cut has workers.
constexpr int kPagedWhole = 4;
static inline PagedCuts paged_cuts(long long pairs, int workers, long long units) {
    constexpr int kRounds[kPagedCuts] = {1, 2, 3, 4, 6, 8};
    PagedCuts c{};
    if (units <= kPagedWhole || pairs >= (long long)kRounds[kPagedCuts - 1] * workers) return c;
    c.most = 1;
    for (int i = 0; i < kPagedCuts; ++i) {
        long long parts = (long long)kRounds[i] * workers / pairs;
        if (parts < 1) parts = 1;
        c.each[i] = 1.f / (float)parts;
        c.rounds[i] = (float)((pairs * parts + workers - 1) / workers);
        c.most = (int)parts + 1;                                                  // (one more than the rounding of `each` may make of it)
    }
    return c;
}
static __device__ __forceinline__ int paged_parts(const PagedCuts& c, int seen, int unit) {
    if (c.most == 0) return 1;
    if (seen <= 0) return 0;
    const int n = (seen - 1) / unit + 1;
    float per[kPagedCuts], cost[kPagedCuts], least = INFINITY;
#pragma unroll
    for (int i = 0; i < kPagedCuts; ++i) {
        per[i] = ceilf((float)n * c.each[i]);
        cost[i] = c.rounds[i] * (per[i] + kPagedFixed);
        least = fminf(least, cost[i]);
    }
    int best = n;
#pragma unroll
    for (int i = 0; i < kPagedCuts; ++i)
        if (cost[i] <= least * 1.0625f) best = (int)per[i];
    return (n + best - 1) / best;
}

struct PagedParams {
    const void* q; const void* gate; const void* k; const void* v;
    long long q_row, q_head, gate_row, gate_head, page_stride, row_stride, head_stride, table_stride;   // in elements
    const int* table; const int* lengths;
    void* out;                          // [batch, heads, dim]
    float* partial; float2* stats;      // [pair][most][heads of a chunk][dim]: weighted means; [pair][most][heads of a chunk]: maximum, sum
    int batch, heads, kv_heads, dim, pages, page, width, window, sinks;
    int group, chunk, chunks;           // query heads of a key/value head; of them at a time; how often
    int unit;                           // positions of a unit
    PagedCuts cuts;
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

template <typename T> QD_DEVINL float paged_load(const T* p) { return (float)*p; }
template <> QD_DEVINL float paged_load<bf16>(const bf16* p) { return __bfloat162float(*p); }
template <typename T> QD_DEVINL void paged_store(T* p, float v);
template <> QD_DEVINL void paged_store<float>(float* p, float v) { *p = v; }
template <> QD_DEVINL void paged_store<bf16>(bf16* p, float v) { *p = __float2bfloat16_rn(v); }


// Pieces (a part of a pair each) in front of each sequence's, and the rows that it sees.  Where there is more than a piece for each worker and not too
// many sequences, those of the largest parts are first.
constexpr int kPagedSorted = 128;
template <int N> struct PagedOrder {
    int before[N + 1], seen[N], sorted;
    uint8_t sequence[kPagedSorted];
};
template <int N, int THREADS>
QD_DEVINL int paged_schedule(const PagedParams& p, PagedOrder<N>& o, int workers) {
    __shared__ int sums[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = p.kv_heads * p.chunks;
    // pieces of the i-th sequence, given by `count`, summed up in order
    const auto sum_up = [&](const auto& count) {
        int total = 0;
        for (int base = 0; base < p.batch; base += THREADS) {
            const int i = base + tid;
            int sum = i < p.batch ? each * count(i) : 0;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += up;
            }
            if (p.batch > 32) {
                if (lane == 31) sums[warp] = sum;
                __syncthreads();
                int all = 0;
#pragma unroll
                for (int w = 0; w < THREADS / 32; ++w) { const int of = sums[w]; if (w < warp) sum += of; all += of; }
                if (i < p.batch) o.before[i + 1] = total + sum;
                total += all;
                __syncthreads();
            } else if (i < p.batch) o.before[i + 1] = sum;              // (one warp's)
        }
        if (tid == 0) o.before[0] = 0;
        __syncthreads();
        return o.before[p.batch];
    };
    if (tid == 0) o.sorted = 0;
    int mine = 0, parts = 0;
    const int total = sum_up([&](int b) {
        mine = paged_span(p, b).seen;
        o.seen[b] = mine;
        return parts = paged_parts(p.cuts, mine, p.unit);
    });
    if (total <= workers || p.batch > kPagedSorted || p.batch > THREADS || p.batch == 1) return total;
    int* per = o.before;                                                // units of a part, for a moment
    __syncthreads();
    if (tid < kPagedSorted) per[tid] = tid < p.batch && parts ? ((mine - 1) / p.unit + parts) / parts : -1;
    __syncthreads();
    int rank = 0;
    if (tid < p.batch)
        for (int z = 0; z < p.batch; z += 4) {                          // (behind the last: -1)
            const int4 of = *reinterpret_cast<const int4*>(per + z);
            const int own = per[tid];
            rank += of.x > own || (of.x == own && z < tid);
            rank += of.y > own || (of.y == own && z + 1 < tid);
            rank += of.z > own || (of.z == own && z + 2 < tid);
            rank += of.w > own || (of.w == own && z + 3 < tid);
        }
    __syncthreads();
    if (tid < p.batch) { o.sequence[rank] = (uint8_t)tid; o.seen[rank] = mine; }
    if (tid == 0) o.sorted = 1;
    __syncthreads();
    return sum_up([&](int i) { return paged_parts(p.cuts, o.seen[i], p.unit); });
}
// Rounds of pieces, one a worker, to and fro, so that who had a larger one takes a smaller one next: the piece after piece r.
QD_DEVINL int paged_next(int r, int workers) { return 2 * (r / workers + 1) * workers - 1 - r; }

// a / b of numbers below 2^24
QD_DEVINL int paged_quotient(int a, int b) {
    int q = (int)__fdividef((float)a, (float)b);
    const int rest = a - q * b;
    q += rest >= b ? 1 : 0;
    return rest < 0 ? q - 1 : q;
}
struct Piece { int at, b, kvh, head0, heads, t0, t1, skip, part, pair; };
// Piece r, of no sequence in front of the `from`-th.
template <int N>
QD_DEVINL Piece paged_piece(const PagedParams& p, const PagedOrder<N>& o, int r, int from) {
    int lo = from;
    for (int hi = p.batch; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (o.before[mid] <= r) lo = mid; else hi = mid;
    }
    Piece a;
    const int each = p.kv_heads * p.chunks, n = o.seen[lo], at = r - o.before[lo], parts = paged_quotient(o.before[lo + 1] - o.before[lo], each);
    const int pair = paged_quotient(at, parts), per = ((n - 1) / p.unit + parts) / parts * p.unit;
    a.at = lo;
    a.b = o.sorted ? o.sequence[lo] : lo;
    a.part = at - pair * parts;
    a.kvh = p.chunks == 1 ? pair : paged_quotient(pair, p.chunks);
    const int chunk = pair - a.kvh * p.chunks;
    a.head0 = a.kvh * p.group + chunk * p.chunk;
    a.heads = min(p.chunk, p.group - chunk * p.chunk);
    a.pair = a.b * each + pair;
    a.t0 = a.part * per;
    a.t1 = min(n, a.t0 + per);
    a.skip = p.window > 0 && n == p.window + p.sinks ? min(max(__ldcg(p.lengths + a.b), 0), p.width * p.page) - n : 0;
    return a;
}

QD_DEVINL long long paged_place(const PagedParams& p, const Piece& a, int h) { return ((long long)a.pair * p.cuts.most + a.part) * p.chunk + h; }

template <typename T>
QD_DEVINL void paged_put(const PagedParams& p, int b, int head, int f, float v) {
    if (p.gate) v *= sigmoid_precise(paged_load((const T*)p.gate + b * p.gate_row + head * p.gate_head + f));
    paged_store((T*)p.out + ((long long)b * p.heads + head) * p.dim + f, v);
}

}  // namespace qd
