// Pages of a key-value cache that sequences share by reference counts: rows set aside, sequences forked, the pool compacted.
//
// Which page goes where is decided by one block or one cluster of blocks (a barrier between its phases, no launch); a second launch, of the whole GPU,
// moves the bytes.  The first is a handful of dependent reads: 4 us for 4 sequences of 14 pages, 7 for 128 of 35 (11 and 20 with every phase through
// global memory and a cluster for any size).  A request for a page gets the lowest free one, in the order of the requests, so that tables do not depend on the order of any atomics
// (reference counts are whole numbers: their sums do not either).
#include "paged.cuh"

namespace qd {
namespace {

constexpr int kBlocks = 8, kThreads = 1024, kWarps = kThreads / 32;
enum { kMoves = 0, kCounts = 16, kMark = 24, kLists = 32 };             // words of the scratch: number of moves, blocks' counts, a number, lists

struct Move { int from, to, rows; };

// BLOCKS 1: a block by itself, for what a block goes through in a few rounds; 8: a cluster.
template <int BLOCKS> QD_DEVINL void all_sync() {
    __syncthreads();
    if (BLOCKS > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
    const int of = sums[lane];                                          // (a warp for every lane)
    int before = lane < warp ? of : 0, total = of;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, d);
        total += __shfl_xor_sync(0xffffffffu, total, d);
    }
    *all = total;
    return before + sum - v;
}

// The places i of [0, last) with test(i), in ascending order, over all blocks: a block takes a run of places, a warp a run of the block's.  After
// `count` and a barrier, `before` is the number of such places in front of the warp's, `total` that of all.
struct Run { int lo, hi, before, total; };
template <int BLOCKS, typename Test>
QD_DEVINL Run list_count(int last, int* counts, int* sums, const Test& test) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = ((last + BLOCKS * kWarps - 1) / (BLOCKS * kWarps) + 31) & ~31;
    const long long from = (long long)((int)blockIdx.x * kWarps + warp) * per;
    Run r;
    r.lo = (int)(from < last ? from : last);
    r.hi = (int)(from + per < last ? from + per : last);
    int mine = 0;
    for (int base = r.lo; base < r.hi; base += 32) mine += __popc(__ballot_sync(0xffffffffu, base + lane < r.hi && test(base + lane)));
    r.before = __shfl_sync(0xffffffffu, block_before(lane == 0 ? mine : 0, &r.total, sums), 0);
    if (BLOCKS > 1) {
        if (threadIdx.x == 0) counts[blockIdx.x] = r.total;
        all_sync<BLOCKS>();
        const int all = lane < BLOCKS ? read_now(counts + lane) : 0;
        int front = lane < (int)blockIdx.x ? all : 0, total = all;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            front += __shfl_xor_sync(0xffffffffu, front, d);
            total += __shfl_xor_sync(0xffffffffu, total, d);
        }
        r.before += front;
        r.total = total;
    }
    return r;
}
// found(rank, i) for the warp's places with test(i), ranks below `most`.
template <typename Test, typename Found>
QD_DEVINL void list_found(const Run& r, int most, const Test& test, const Found& found) {
    const int lane = threadIdx.x & 31;
    int rank = r.before;
    for (int base = r.lo; base < r.hi && rank < most; base += 32) {
        const bool is = base + lane < r.hi && test(base + lane);
        const unsigned all = __ballot_sync(0xffffffffu, is);
        const int mine = rank + __popc(all & ((1u << lane) - 1u));
        if (is && mine < most) found(mine, base + lane);
        rank += __popc(all);
    }
}

QD_DEVINL bool is_page(int e, int pages) { return e >= 0 && e < pages; }

struct ForkParams {
    const int* table; const int* lengths; const int* refs; const int* parents;
    int* table_out; int* lengths_out; int* refs_out; int* scratch; unsigned int* status;
    int sequences, width, pages, page;
};
// What concerns the sequences alone every block works out for itself, in shared memory; the blocks meet for the reference counts.
template <int BLOCKS>
QD_DEVINL void fork_pages(const ForkParams& p) {
    extern __shared__ int fork_smem[];
    __shared__ int sums[kWarps];
    const int S = p.sequences, tid = threadIdx.x, all = BLOCKS * kThreads, at = blockIdx.x * kThreads + tid;
    int *parent_of = fork_smem, *rows = parent_of + S, *first = rows + S, *asks = first + S;       // parent (itself where none is named; -1: ends), rows,
    Move* moves = (Move*)(p.scratch + kLists);                                                    // first child (-1: itself), sequences that ask for a page
    for (int i = at; i < p.pages; i += all) p.refs_out[i] = p.refs[i];
    for (int b = tid; b < S; b += kThreads) {
        const int parent = p.parents[b];
        if (parent < -1 || parent >= S) { if (blockIdx.x == 0) atomicOr(p.status, QD_STATUS_BAD_ARG); }
        parent_of[b] = parent < -1 || parent >= S ? b : parent;
        rows[b] = p.lengths[b];
        first[b] = S;
    }
    all_sync<BLOCKS>();
    for (int b = tid; b < S; b += kThreads)
        if (parent_of[b] >= 0) atomicMin(first + parent_of[b], parent_of[b] == b ? -1 : b);
    __syncthreads();
    const auto length = [&](int b) {                                    // of b after the fork
        const int parent = parent_of[b];
        return parent < 0 ? 0 : parent == b ? rows[b] : min(max(rows[parent], 0), p.width * p.page);
    };
    // full pages shared, the page that is not full for the parent itself or its first child, others dropped; a page that stays in its place needs no count
    for (long long i = at; i < (long long)S * p.width; i += all) {
        const int b = (int)(i / p.width), j = (int)(i - (long long)b * p.width), parent = parent_of[b], old = p.table[i];
        int now = old;
        if (parent != b) {
            const int n = length(b), full = n / p.page;
            const bool mine = j < full || (j == full && n > full * p.page && first[parent] == b);
            now = mine ? p.table[(long long)parent * p.width + j] : -1;
        }
        p.table_out[i] = now;
        if (now != old) {
            if (is_page(old, p.pages)) atomicSub(p.refs_out + old, 1);
            if (is_page(now, p.pages)) atomicAdd(p.refs_out + now, 1);
        }
    }
    int wanted = 0;
    for (int base = 0; base < S; base += kThreads) {
        const int b = base + tid, parent = b < S ? parent_of[b] : -1, n = b < S ? length(b) : 0;
        // (a parent without that page, of which nothing is seen, has children without it: a free page would show them what its last owner left)
        const bool asking = parent >= 0 && parent != b && n % p.page != 0 && first[parent] != b && is_page(p.table[(long long)parent * p.width + n / p.page], p.pages);
        if (b < S && blockIdx.x == 0) p.lengths_out[b] = n;
        int found;
        const int rank = wanted + block_before(asking, &found, sums);
        if (asking) asks[rank] = b;
        wanted += found;
    }
    all_sync<BLOCKS>();
    const auto free_page = [&](int i) { return read_now(p.refs_out + i) <= 0; };
    const Run run = list_count<BLOCKS>(p.pages, p.scratch + kCounts, sums, free_page);
    list_found(run, wanted, free_page, [&](int rank, int page) {
        const int b = asks[rank], parent = parent_of[b], n = length(b), full = n / p.page;
        p.table_out[(long long)b * p.width + full] = page;
        p.refs_out[page] = 1;                                           // (looked at by this warp alone)
        moves[rank] = Move{p.table[(long long)parent * p.width + full], page, n - full * p.page};
    });
    if (blockIdx.x) return;
    const int got = min(wanted, run.total);
    for (int i = got + tid; i < wanted; i += kThreads) {                // no page left: the sequence ends where its full pages do
        p.lengths_out[asks[i]] = length(asks[i]) / p.page * p.page;
        atomicOr(p.status, QD_STATUS_NO_PAGE);
    }
    if (tid == 0) p.scratch[kMoves] = got;
}
__global__ void __launch_bounds__(kThreads) fork_block_kernel(const ForkParams p) {
    chain_enter();
    fork_pages<1>(p);
}
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kThreads) fork_cluster_kernel(const ForkParams p) {
    chain_enter();
    fork_pages<kBlocks>(p);
}

struct CompactParams {
    const int* table; const int* refs; int* table_out; int* refs_out; int* used; int* scratch;
    int entries, pages, page;
};
template <int BLOCKS>
QD_DEVINL void compact_pages(const CompactParams& p) {
    __shared__ int sums[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, all = BLOCKS * kThreads, at = blockIdx.x * kThreads + tid;
    int* place = p.scratch + kLists;                                    // of a page that moves: where it goes
    Move* moves = (Move*)(place + p.pages);
    const auto taken = [&](int i) { return p.refs[i] > 0; };
    const Run run = list_count<BLOCKS>(p.pages, p.scratch + kCounts, sums, taken);
    const int used = run.total;
    // pages in use among the first `used`: the warp that has the border counts to it
    if (used == 0 && at == 0) p.scratch[kMark] = 0;
    if (run.lo < used && run.hi >= used) {
        int count = run.before;
        for (int base = run.lo; base < used; base += 32) count += __popc(__ballot_sync(0xffffffffu, base + lane < used && taken(base + lane)));
        if (lane == 0) p.scratch[kMark] = count;
    }
    all_sync<BLOCKS>();
    const int front = read_now(p.scratch + kMark), count = used - front;
    int rank = run.before;
    for (int base = run.lo; base < run.hi; base += 32) {
        const int i = base + lane, refs = i < run.hi ? p.refs[i] : 0;
        const unsigned is = __ballot_sync(0xffffffffu, refs > 0);
        const int in_front = rank + __popc(is & ((1u << lane) - 1u));
        rank += __popc(is);
        if (i >= run.hi) continue;
        if (i < used && refs <= 0) { moves[i - in_front].to = i; moves[i - in_front].rows = p.page; }       // a free one: as many in front as are not in use
        else if (i >= used && refs > 0) moves[in_front - front].from = i;
        else p.refs_out[i] = refs;
    }
    all_sync<BLOCKS>();
    for (int i = at; i < count; i += all) {
        const int from = read_now(&moves[i].from), to = read_now(&moves[i].to);
        place[from] = to;
        p.refs_out[to] = p.refs[from];
        p.refs_out[from] = 0;
    }
    all_sync<BLOCKS>();
    for (int i = at; i < p.entries; i += all) {
        const int e = p.table[i];
        p.table_out[i] = e >= used && e < p.pages && p.refs[e] > 0 ? read_now(place + e) : e;
    }
    if (at == 0) { *p.used = used; p.scratch[kMoves] = count; }
}
__global__ void __launch_bounds__(kThreads) compact_block_kernel(const CompactParams p) {
    chain_enter();
    compact_pages<1>(p);
}
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kThreads) compact_cluster_kernel(const CompactParams p) {
    chain_enter();
    compact_pages<kBlocks>(p);
}

struct ReserveParams {
    int* table; const int* lengths; int* refs; const int* counts; int* scratch; unsigned int* status;
    int count, sequences, width, pages, page, begun;
};
// One block, or (many pages) a cluster whose blocks all list the requests.
template <int BLOCKS>
QD_DEVINL void reserve_pages(const ReserveParams& p) {
    __shared__ int sums[kWarps];
    const int tid = threadIdx.x;
    int* asks = p.scratch + kLists;                                     // places of the table that need a page, in order
    int wanted = 0;
    for (int base = 0; base < p.sequences; base += kThreads) {
        const int b = base + tid;
        int from = 0, to = 0, need = 0;
        if (b < p.sequences) {
            const int n = p.lengths[b], more = p.counts ? p.counts[b] : p.count;
            if (n < 0 || more < 0 || (long long)n + more > (long long)p.width * p.page) {
                if (blockIdx.x == 0) atomicOr(p.status, QD_STATUS_BAD_ARG);
            } else if (more > 0) {
                from = n ? (n - 1) / p.page + 1 : 0;
                to = (n + more - 1) / p.page + 1;                           // (no sum passes the table's rows)
                // a page in whose middle the sequence is cannot be made up for (what was to be in front is lost), nor are the rows to come there
                if (p.begun && blockIdx.x == 0 && n % p.page && !is_page(read_now(p.table + (long long)b * p.width + n / p.page), p.pages))
                    atomicOr(p.status, QD_STATUS_NO_PAGE);
                for (int j = from; j < to; ++j) need += read_now(p.table + (long long)b * p.width + j) < 0;
            }
        }
        int found;
        int rank = wanted + block_before(need, &found, sums);
        if (blockIdx.x == 0 && need > 0)
            for (int j = from; j < to; ++j)
                if (read_now(p.table + (long long)b * p.width + j) < 0) asks[rank++] = b * p.width + j;
        wanted += found;
    }
    if (wanted == 0) return;                                            // (of all blocks alike)
    all_sync<BLOCKS>();
    const auto free_page = [&](int i) { return read_now(p.refs + i) <= 0; };
    const Run run = list_count<BLOCKS>(p.pages, p.scratch + kCounts, sums, free_page);
    list_found(run, wanted, free_page, [&](int rank, int page) {
        p.table[read_now(asks + rank)] = page;
        p.refs[page] = 1;
    });
    if (run.total < wanted && blockIdx.x == 0 && tid == 0) atomicOr(p.status, QD_STATUS_NO_PAGE);
}
__global__ void __launch_bounds__(kThreads) reserve_block_kernel(const ReserveParams p) {
    chain_enter();
    reserve_pages<1>(p);
}
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kThreads) reserve_cluster_kernel(const ReserveParams p) {
    chain_enter();
    reserve_pages<kBlocks>(p);
}

// The moves' rows, of every layer of both pools: a warp per 2 KB, four pieces of a lane in flight.  Bound by HBM: 1.38 GB in 215 us (6.4 TB/s), 72 MB
// in pieces of one page 16 us.
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

// What a block goes through in a few rounds.
bool few(long long entries, long long pages) { return entries <= 8 * kThreads && pages <= 16 * kThreads; }
bool whole_pieces(const void* a, const void* b, long long x, long long y, long long z) {
    return !(((uintptr_t)a | (uintptr_t)b) & 15u) && x % 16 == 0 && y % 16 == 0 && z % 16 == 0;
}
int launch_moves(void* k, void* v, long long page_bytes, long long layer_bytes, long long row_bytes, int layers, int page, const int* scratch,
                 const int* list, cudaStream_t stream) {
    MoveParams m{(char*)k, (char*)v, scratch, list, page_bytes, layer_bytes, row_bytes, layers, page};
    return qd_launch(move_kernel, dim3(device_blocks() * 8), dim3(256), 0, stream, 3, m);
}

}  // namespace
}  // namespace qd

using namespace qd;

extern "C" long long qd_pages_scratch_words(int sequences, int width, int pages) {
    if (sequences <= 0 || width <= 0 || pages <= 0) return 0;
    const long long fork = 3ll * sequences, compact = 4ll * pages, reserve = (long long)sequences * width;
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
    const size_t smem = 16ull * sequences;
    if (smem > 200 * 1024) return QD_ERR_UNSUPPORTED;
    const bool alone = few((long long)sequences * width, pages);
    static bool raised_block[kDevices], raised_cluster[kDevices];
    if (smem > 40 * 1024 && !(alone ? raise_smem(fork_block_kernel, 200 * 1024, raised_block) : raise_smem(fork_cluster_kernel, 200 * 1024, raised_cluster)))
        return QD_ERR_LAUNCH;                                              // (what is declared counts too)
    const int code = alone ? qd_launch(fork_block_kernel, dim3(1), dim3(kThreads), smem, (cudaStream_t)stream, 3, p)
                           : qd_launch(fork_cluster_kernel, dim3(kBlocks), dim3(kThreads), smem, (cudaStream_t)stream, 3, p);
    if (code != QD_OK) return code;
    return launch_moves(k, v, page_bytes, layer_bytes, row_bytes, layers, page, scratch, scratch + kLists, (cudaStream_t)stream);
}

extern "C" int qd_pages_compact(void* k, void* v, long long page_bytes, long long layer_bytes, long long row_bytes, int layers, const int* table,
                                const int* refs, int* table_out, int* refs_out, int* used, int* scratch, int sequences, int width, int pages, int page,
                                void* stream) {
    QD_CHECK_ARG(k && v && table && refs && table_out && refs_out && used && scratch && table_out != table && refs_out != refs);
    QD_CHECK_ARG(sequences > 0 && width > 0 && pages > 0 && page > 0 && layers > 0 && row_bytes > 0 && (long long)sequences * width <= 0x7fffffffll - 8192);
    QD_CHECK_ARG(layer_bytes >= page * row_bytes && page_bytes >= layers * layer_bytes);
    if (!whole_pieces(k, v, page_bytes, layer_bytes, row_bytes)) return QD_ERR_UNSUPPORTED;
    CompactParams p{table, refs, table_out, refs_out, used, scratch, sequences * width, pages, page};
    const int code = few((long long)sequences * width, pages) ? qd_launch(compact_block_kernel, dim3(1), dim3(kThreads), 0, (cudaStream_t)stream, 3, p)
                                                              : qd_launch(compact_cluster_kernel, dim3(kBlocks), dim3(kThreads), 0, (cudaStream_t)stream, 3, p);
    if (code != QD_OK) return code;
    return launch_moves(k, v, page_bytes, layer_bytes, row_bytes, layers, page, scratch, scratch + kLists + pages, (cudaStream_t)stream);
}

extern "C" int qd_pages_reserve(int* table, const int* lengths, int* refs, const int* counts, int count, int* scratch, unsigned int* status,
                                int sequences, int width, int pages, int page, int begun, void* stream) {
    QD_CHECK_ARG(table && lengths && refs && scratch && status && (counts || count >= 0));
    QD_CHECK_ARG(sequences > 0 && width > 0 && pages > 0 && page > 0 && (long long)sequences * width <= 0x7fffffffll);
    ReserveParams p{table, lengths, refs, counts, scratch, status, count, sequences, width, pages, page, begun};
    return few(sequences, pages) ? qd_launch(reserve_block_kernel, dim3(1), dim3(kThreads), 0, (cudaStream_t)stream, 3, p)
                                 : qd_launch(reserve_cluster_kernel, dim3(kBlocks), dim3(kThreads), 0, (cudaStream_t)stream, 3, p);
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
    const long long blocks = (2ll * layers * count + 7) / 8, most = device_blocks() * 8;
    return qd_launch(rows_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, (cudaStream_t)stream, 3, p);
}
