// Pages of a key-value cache that sequences share by reference counts: rows set aside, sequences forked, the pool compacted.
//
// Which page goes where is decided by one cluster of blocks (a barrier between its phases, no launch); a second launch, of the whole GPU, moves the
// bytes.  A request for a page gets the lowest free one, in the order of the requests, so that tables do not depend on the order of any atomics
// (reference counts are whole numbers: their sums do not either).
#include "common.cuh"

namespace qd {
namespace {

constexpr int kBlocks = 8, kThreads = 1024, kWarps = kThreads / 32;
enum { kMoves = 0, kCounts = 16, kCounts2 = 32, kLists = 48 };          // words of the scratch: number of moves, blocks' counts, lists

struct Move { int from, to, rows; };

QD_DEVINL void cluster_sync() {
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
QD_DEVINL int read_now(const int* p) { return __ldcg(p); }              // written by another block of the cluster

// Exclusive sum over the block in thread order; the total in *all.
QD_DEVINL int block_before(int v, int* all, int* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
    }
    __syncthreads();                                                    // the previous use of `sums` is over
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < kWarps; ++w) { if (w < warp) before += sums[w]; total += sums[w]; }
    *all = total;
    return before + sum - v;
}

// The places i of [first, last) with test(i), in ascending order, over all blocks of the cluster: found(rank, i) for ranks below `most`; how many
// there are.  A block takes a run of places, a warp a run of the block's.  counts: kBlocks words, not used before in this launch.
template <typename Test, typename Found>
QD_DEVINL int cluster_list(int first, int last, int most, int* counts, int* sums, const Test& test, const Found& found) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, runs = kBlocks * kWarps;
    const int per = ((last - first + runs - 1) / runs + 31) & ~31;
    const int run = (int)blockIdx.x * kWarps + warp;
    const long long from = first + (long long)run * per;
    const int lo = (int)(from < last ? from : last), hi = (int)(from + per < last ? from + per : last);
    int mine = 0;
    for (int base = lo; base < hi; base += 32) mine += __popc(__ballot_sync(0xffffffffu, base + lane < hi && test(base + lane)));
    int all;
    int rank = block_before(lane == 0 ? mine : 0, &all, sums);
    if (threadIdx.x == 0) counts[blockIdx.x] = all;
    cluster_sync();
    int total = 0;
    for (int b = 0; b < kBlocks; ++b) { const int c = read_now(counts + b); if (b < (int)blockIdx.x) rank += c; total += c; }
    rank = __shfl_sync(0xffffffffu, rank, 0);
    for (int base = lo; base < hi && rank < most; base += 32) {
        const bool is = base + lane < hi && test(base + lane);
        const unsigned all_of = __ballot_sync(0xffffffffu, is);
        const int r = rank + __popc(all_of & ((1u << lane) - 1u));
        if (is && r < most) found(r, base + lane);
        rank += __popc(all_of);
    }
    return total;
}

QD_DEVINL bool is_page(int e, int pages) { return e >= 0 && e < pages; }

struct ForkParams {
    const int* table; const int* lengths; const int* refs; const int* parents;
    int* table_out; int* lengths_out; int* refs_out; int* scratch; unsigned int* status;
    int sequences, width, pages, page;
};
// Rows and full pages of sequence b after the fork; `parent` is b itself where parents[b] names no sequence.
struct Child { int parent, n, full, rest; bool stays, ends; };
QD_DEVINL Child child_of(const ForkParams& p, int b) {
    Child c;
    const int parent = p.parents[b];
    c.ends = parent == -1;
    c.parent = parent < 0 || parent >= p.sequences ? b : parent;
    c.stays = !c.ends && c.parent == b;
    c.n = c.ends ? 0 : c.stays ? p.lengths[b] : min(max(p.lengths[c.parent], 0), p.width * p.page);
    c.full = c.n / p.page;
    c.rest = c.n - c.full * p.page;
    return c;
}

__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kThreads) fork_kernel(const ForkParams p) {
    chain_enter();
    __shared__ int sums[kWarps];
    const int tid = threadIdx.x, all = kBlocks * kThreads, at = blockIdx.x * kThreads + tid;
    int* first = p.scratch + kLists;                                    // of each sequence: its first child, -1: itself
    int* asks = first + p.sequences;                                    // sequences that need a page, in order
    Move* moves = (Move*)(asks + p.sequences);
    for (int i = at; i < p.pages; i += all) p.refs_out[i] = p.refs[i];
    for (int b = at; b < p.sequences; b += all) first[b] = p.sequences;
    cluster_sync();
    for (int b = at; b < p.sequences; b += all) {
        const Child c = child_of(p, b);
        const int parent = p.parents[b];
        if (parent < -1 || parent >= p.sequences) atomicOr(p.status, QD_STATUS_BAD_ARG);
        if (!c.ends) atomicMin(first + c.parent, c.stays ? -1 : b);
        p.lengths_out[b] = c.n;
    }
    // full pages shared, others dropped; a page that stays in its place needs no count
    for (int b = blockIdx.x; b < p.sequences; b += kBlocks) {
        const Child c = child_of(p, b);
        for (int j = tid; j < p.width; j += kThreads) {
            const int old = p.table[(long long)b * p.width + j];
            const int now = c.stays ? old : j < c.full ? p.table[(long long)c.parent * p.width + j] : -1;
            p.table_out[(long long)b * p.width + j] = now;
            if (now != old) {
                if (is_page(old, p.pages)) atomicSub(p.refs_out + old, 1);
                if (is_page(now, p.pages)) atomicAdd(p.refs_out + now, 1);
            }
        }
    }
    cluster_sync();
    // the page that is not full: to the parent itself or its first child, copies for the others
    if (blockIdx.x == 0) {
        int before = 0;
        for (int base = 0; base < p.sequences; base += kThreads) {
            const int b = base + tid;
            bool asking = false;
            if (b < p.sequences) {
                const Child c = child_of(p, b);
                if (!c.stays && c.rest > 0) {
                    const int tail = p.table[(long long)c.parent * p.width + c.full];
                    asking = read_now(first + c.parent) != b;
                    if (!asking) {
                        p.table_out[(long long)b * p.width + c.full] = tail;
                        if (is_page(tail, p.pages)) atomicAdd(p.refs_out + tail, 1);
                    }
                }
            }
            int found;
            const int rank = before + block_before(asking, &found, sums);
            if (asking) asks[rank] = b;
            before += found;
        }
        if (tid == 0) p.scratch[kMoves] = before;
    }
    cluster_sync();
    const int wanted = read_now(p.scratch + kMoves);
    const int free = cluster_list(0, p.pages, wanted, p.scratch + kCounts, sums, [&](int i) { return read_now(p.refs_out + i) <= 0; },
        [&](int rank, int page) {
            const int b = read_now(asks + rank);
            const Child c = child_of(p, b);
            const int tail = p.table[(long long)c.parent * p.width + c.full];
            p.table_out[(long long)b * p.width + c.full] = page;
            moves[rank] = Move{tail, page, is_page(tail, p.pages) ? c.rest : 0};
        });
    cluster_sync();                                                     // all have read the counts and `wanted`
    const int got = min(wanted, free);
    for (int i = at; i < got; i += all) p.refs_out[read_now(&moves[i].to)] = 1;
    for (int i = got + at; i < wanted; i += all) {                      // no page left: the sequence ends where its full pages do
        const int b = read_now(asks + i);
        p.lengths_out[b] = child_of(p, b).full * p.page;
        atomicOr(p.status, QD_STATUS_NO_PAGE);
    }
    if (at == 0) p.scratch[kMoves] = got;
}

struct CompactParams {
    const int* table; const int* refs; int* table_out; int* refs_out; int* used; int* scratch;
    int entries, pages, page;
};
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kThreads) compact_kernel(const CompactParams p) {
    chain_enter();
    __shared__ int sums[kWarps];
    const int tid = threadIdx.x, all = kBlocks * kThreads, at = blockIdx.x * kThreads + tid;
    int* place = p.scratch + kLists;                                    // of each page: where it goes
    Move* moves = (Move*)(place + p.pages);
    const int used = cluster_list(0, p.pages, 0, p.scratch + kCounts, sums, [&](int i) { return p.refs[i] > 0; }, [](int, int) {});
    for (int i = at; i < p.pages; i += all) { place[i] = i; p.refs_out[i] = p.refs[i]; }
    cluster_list(0, used, p.pages, p.scratch + kCounts + kBlocks, sums, [&](int i) { return p.refs[i] <= 0; },
                 [&](int rank, int i) { moves[rank].to = i; moves[rank].rows = p.page; });
    const int count = cluster_list(used, p.pages, p.pages, p.scratch + kCounts2, sums, [&](int i) { return p.refs[i] > 0; },
                                   [&](int rank, int i) { moves[rank].from = i; });
    cluster_sync();
    for (int i = at; i < count; i += all) {
        const int from = read_now(&moves[i].from), to = read_now(&moves[i].to);
        place[from] = to;
        p.refs_out[to] = p.refs[from];
        p.refs_out[from] = 0;
    }
    cluster_sync();
    for (int i = at; i < p.entries; i += all) {
        const int e = p.table[i];
        p.table_out[i] = is_page(e, p.pages) ? read_now(place + e) : e;
    }
    if (at == 0) { *p.used = used; p.scratch[kMoves] = count; }
}

struct ReserveParams {
    int* table; const int* lengths; int* refs; const int* counts; int* scratch; unsigned int* status;
    int count, sequences, width, pages, page;
};
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kThreads) reserve_kernel(const ReserveParams p) {
    chain_enter();
    __shared__ int sums[kWarps];
    const int tid = threadIdx.x;
    int* asks = p.scratch + kLists;                                     // places of the table that need a page, in order
    if (blockIdx.x == 0) {
        int before = 0;
        for (int base = 0; base < p.sequences; base += kThreads) {
            const int b = base + tid;
            int from = 0, to = 0, need = 0;
            if (b < p.sequences) {
                const int n = p.lengths[b], more = p.counts ? p.counts[b] : p.count;
                if (n < 0 || more < 0 || (long long)n + more > (long long)p.width * p.page) atomicOr(p.status, QD_STATUS_BAD_ARG);
                else if (more > 0) {
                    from = (n + p.page - 1) / p.page;
                    to = (n + more + p.page - 1) / p.page;
                    for (int j = from; j < to; ++j) need += p.table[(long long)b * p.width + j] < 0;
                }
            }
            int found;
            int rank = before + block_before(need, &found, sums);
            for (int j = from; j < to; ++j)
                if (p.table[(long long)b * p.width + j] < 0) asks[rank++] = b * p.width + j;
            before += found;
        }
        if (tid == 0) p.scratch[kMoves] = before;
    }
    cluster_sync();
    const int wanted = read_now(p.scratch + kMoves);
    if (wanted == 0) return;                                            // (of all blocks alike)
    const int free = cluster_list(0, p.pages, wanted, p.scratch + kCounts, sums, [&](int i) { return p.refs[i] <= 0; },
        [&](int rank, int page) {
            p.table[read_now(asks + rank)] = page;
            p.refs[page] = 1;
        });
    if (free < wanted && blockIdx.x == 0 && tid == 0) atomicOr(p.status, QD_STATUS_NO_PAGE);
}

// The moves' rows, of every layer of both pools: a warp per 2 KB, four pieces of a lane in flight.
struct MoveParams {
    char* k; char* v; const int* scratch; const int* list;
    long long page_bytes, layer_bytes, row_bytes;
    int layers, page;
};
__global__ void __launch_bounds__(256) move_kernel(const MoveParams p) {
    chain_enter();
    const int count = p.scratch[kMoves], lane = threadIdx.x & 31;
    const Move* moves = (const Move*)p.list;
    const long long pieces = (p.page * p.row_bytes + 2047) / 2048, each = 2 * p.layers * pieces;
    const long long all = each * count, warps = (long long)gridDim.x * 8;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < all; i += warps) {
        const Move m = moves[i / each];
        const long long in = i % each, bytes = m.rows * p.row_bytes, start = in % pieces * 2048 + lane * 16;
        const int run = (int)(in / pieces), layer = run >> 1;
        char* pool = run & 1 ? p.v : p.k;
        const char* from = pool + m.from * p.page_bytes + layer * p.layer_bytes + start;
        char* to = pool + m.to * p.page_bytes + layer * p.layer_bytes + start;
        uint4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (start + j * 512 < bytes) x[j] = __ldcs((const uint4*)(from + j * 512));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (start + j * 512 < bytes) __stcs((uint4*)(to + j * 512), x[j]);
    }
}

// Rows of one sequence between a contiguous cache and its pages, every layer, keys and values: a warp per row.
struct RowsParams {
    char* k; char* v; char* k_rows; char* v_rows; const int* table; unsigned int* status;
    long long page_bytes, layer_bytes, row_bytes, rows_layer;
    int layers, page, pages, width, first, count, out;
};
__global__ void __launch_bounds__(256) rows_kernel(const RowsParams p) {
    chain_enter();
    const int lane = threadIdx.x & 31;
    const long long all = 2ll * p.layers * p.count, warps = (long long)gridDim.x * 8;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < all; i += warps) {
        const int row = p.first + (int)(i % p.count), run = (int)(i / p.count), layer = run >> 1, page = p.table[row / p.page];
        if (!is_page(page, p.pages)) {
            if (lane == 0) atomicOr(p.status, QD_STATUS_NO_PAGE);
            continue;
        }
        char* pool = (run & 1 ? p.v : p.k) + page * p.page_bytes + layer * p.layer_bytes + row % p.page * p.row_bytes;
        char* rows = (run & 1 ? p.v_rows : p.k_rows) + layer * p.rows_layer + (row - p.first) * p.row_bytes;
        const char* from = p.out ? pool : rows;
        char* to = p.out ? rows : pool;
        for (long long j = lane * 16; j < p.row_bytes; j += 512) *(uint4*)(to + j) = *(const uint4*)(from + j);
    }
}

int sms_of() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms > 0 ? sms : 148;
}
bool whole_pieces(const void* a, const void* b, long long x, long long y, long long z) {
    return !(((uintptr_t)a | (uintptr_t)b) & 15u) && x % 16 == 0 && y % 16 == 0 && z % 16 == 0;
}
int launch_moves(void* k, void* v, long long page_bytes, long long layer_bytes, long long row_bytes, int layers, int page, const int* scratch,
                 const int* list, cudaStream_t stream) {
    MoveParams m{(char*)k, (char*)v, scratch, list, page_bytes, layer_bytes, row_bytes, layers, page};
    return qd_launch(move_kernel, dim3(sms_of() * 8), dim3(256), 0, stream, 3, m);
}

}  // namespace
}  // namespace qd

using namespace qd;

extern "C" long long qd_pages_scratch_words(int sequences, int width, int pages) {
    if (sequences <= 0 || width <= 0 || pages <= 0) return 0;
    const long long fork = 5ll * sequences, compact = 4ll * pages, reserve = (long long)sequences * width;
    return kLists + (fork > compact ? fork > reserve ? fork : reserve : compact > reserve ? compact : reserve);
}

extern "C" int qd_pages_fork(void* k, void* v, long long page_bytes, long long layer_bytes, long long row_bytes, int layers, const int* table,
                             const int* lengths, const int* refs, const int* parents, int* table_out, int* lengths_out, int* refs_out, int* scratch,
                             unsigned int* status, int sequences, int width, int pages, int page, void* stream) {
    QD_CHECK_ARG(k && v && table && lengths && refs && parents && table_out && lengths_out && refs_out && scratch && status);
    QD_CHECK_ARG(table_out != table && lengths_out != lengths && refs_out != refs);
    QD_CHECK_ARG(sequences > 0 && width > 0 && pages > 0 && page > 0 && layers > 0 && row_bytes > 0 && (long long)width * page <= 0x7fffffffll);
    QD_CHECK_ARG(layer_bytes >= page * row_bytes && page_bytes >= layers * layer_bytes);
    if (!whole_pieces(k, v, page_bytes, layer_bytes, row_bytes)) return QD_ERR_UNSUPPORTED;
    ForkParams p{table, lengths, refs, parents, table_out, lengths_out, refs_out, scratch, status, sequences, width, pages, page};
    const int code = qd_launch(fork_kernel, dim3(kBlocks), dim3(kThreads), 0, (cudaStream_t)stream, 3, p);
    if (code != QD_OK) return code;
    return launch_moves(k, v, page_bytes, layer_bytes, row_bytes, layers, page, scratch, scratch + kLists + 2 * sequences, (cudaStream_t)stream);
}

extern "C" int qd_pages_compact(void* k, void* v, long long page_bytes, long long layer_bytes, long long row_bytes, int layers, const int* table,
                                const int* refs, int* table_out, int* refs_out, int* used, int* scratch, int sequences, int width, int pages, int page,
                                void* stream) {
    QD_CHECK_ARG(k && v && table && refs && table_out && refs_out && used && scratch && table_out != table && refs_out != refs);
    QD_CHECK_ARG(sequences > 0 && width > 0 && pages > 0 && page > 0 && layers > 0 && row_bytes > 0 && (long long)sequences * width <= 0x7fffffffll - 8192);
    QD_CHECK_ARG(layer_bytes >= page * row_bytes && page_bytes >= layers * layer_bytes);
    if (!whole_pieces(k, v, page_bytes, layer_bytes, row_bytes)) return QD_ERR_UNSUPPORTED;
    CompactParams p{table, refs, table_out, refs_out, used, scratch, sequences * width, pages, page};
    const int code = qd_launch(compact_kernel, dim3(kBlocks), dim3(kThreads), 0, (cudaStream_t)stream, 3, p);
    if (code != QD_OK) return code;
    return launch_moves(k, v, page_bytes, layer_bytes, row_bytes, layers, page, scratch, scratch + kLists + pages, (cudaStream_t)stream);
}

extern "C" int qd_pages_reserve(int* table, const int* lengths, int* refs, const int* counts, int count, int* scratch, unsigned int* status,
                                int sequences, int width, int pages, int page, void* stream) {
    QD_CHECK_ARG(table && lengths && refs && scratch && status && (counts || count >= 0));
    QD_CHECK_ARG(sequences > 0 && width > 0 && pages > 0 && page > 0 && (long long)sequences * width <= 0x7fffffffll);
    ReserveParams p{table, lengths, refs, counts, scratch, status, count, sequences, width, pages, page};
    return qd_launch(reserve_kernel, dim3(kBlocks), dim3(kThreads), 0, (cudaStream_t)stream, 3, p);
}

extern "C" int qd_pages_rows(void* k, void* v, long long page_bytes, long long layer_bytes, long long row_bytes, void* k_rows, void* v_rows,
                             long long rows_layer_bytes, const int* table, unsigned int* status, int layers, int width, int pages, int page, int first,
                             int count, int out, void* stream) {
    QD_CHECK_ARG(k && v && k_rows && v_rows && table && status && layers > 0 && width > 0 && pages > 0 && page > 0 && first >= 0 && count >= 0);
    QD_CHECK_ARG((long long)first + count <= (long long)width * page && row_bytes > 0 && layer_bytes >= page * row_bytes);
    if (!whole_pieces(k, v, page_bytes, layer_bytes, row_bytes) || !whole_pieces(k_rows, v_rows, rows_layer_bytes, 0, 0)) return QD_ERR_UNSUPPORTED;
    if (count == 0) return QD_OK;
    RowsParams p{(char*)k, (char*)v, (char*)k_rows, (char*)v_rows, table, status, page_bytes, layer_bytes, row_bytes, rows_layer_bytes,
                 layers, page, pages, width, first, count, out};
    const long long blocks = (2ll * layers * count + 7) / 8, most = sms_of() * 8;
    return qd_launch(rows_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, (cudaStream_t)stream, 3, p);
}
