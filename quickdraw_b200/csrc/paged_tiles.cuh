// Attention over pages, a tile of positions at a time: who works on what, and how the tiles come.  What is done with a tile is given by a class Work:
//   Type, kDim (columns, at least the head dimension), kHeads (query heads, a multiple of eight), kTile (positions), kWarps, kAhead (tiles on their way),
//   kSeqs (sequences of a launch), begin(queries), scores(keys, rows, scale), values(values), leave(n, state, stats).
#pragma once
#include "paged.cuh"

#include <type_traits>

namespace qd {

QD_DEVINL void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// constant offsets stay in the instruction
template <int TO, int FROM> QD_DEVINL void cp_async16_at(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0 + %3], [%1 + %4], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(TO), "n"(FROM) : "memory");
}
template <int I, int N, typename F> QD_DEVINL void static_loop(const F& f) {
    if constexpr (I < N) { f(std::integral_constant<int, I>{}); static_loop<I + 1, N>(f); }
}
QD_DEVINL void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
QD_DEVINL void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
template <int N> QD_DEVINL void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// exp2 of a difference to a running maximum that may be -inf (nothing seen yet)
QD_DEVINL float weight_of(float s, float top) { return exp2f(s - (top == -INFINITY ? 0.f : top)); }
// What weights are taken times.  They are up to 2^8 (see the Work): the sum of as many as a warp meets (2^24) times the largest value stays below the
// largest number, and what is joined after it are means.  (Of values below 2^-94 bits are lost instead.)
constexpr float kPagedWeight = 0x1p-32f;

// 1 / x of a normal number, off by 2^-23 at most
QD_DEVINL float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four or eight elements from a place that may not be on a 16-byte boundary.
QD_DEVINL uint4 paged_load16(const float* src) {
    return make_uint4(__float_as_uint(src[0]), __float_as_uint(src[1]), __float_as_uint(src[2]), __float_as_uint(src[3]));
}
QD_DEVINL uint4 paged_load16(const bf16* src) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (uint32_t)__bfloat16_as_ushort(src[2 * e]) | (uint32_t)__bfloat16_as_ushort(src[2 * e + 1]) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Four warps take a part, every fourth tile each, through rings of their own whose slots hold the keys or the values of a tile: nothing in the loop
// waits for another warp.  At the end of a part the four join their states (alone a warp would write four times as many, 8 KB each for eight heads of
// 256) while the block's other groups keep the loads going.
//
// Long caches are bound by HBM: 4 sequences of 100 000 to 131 072 positions, 32 heads on 8 of 128, 1.82 GB in 284 us with the join (6.4 TB/s); 32 of 8192,
// 16 on 2 of 256, 537 MB in 94.  Of other lengths (32 up to 8192, 282 MB, 57 us) a tenth goes to parts that end at different times; some 9 us go to the
// launches, the lengths, the first look into the table and the first rows, one after the other.  What it took, us for those three: parts cut by blocks
// whose warps joined by the tree, straight code that missed the instruction cache at every part 366 / - / 137; their states through the free slot 317 / 121
// / 84; warps by themselves 293 / 103 / 74; copies by whole lines (64 bytes of eight rows an instruction cost a tenth) 280 / 104 / 65; four warps a part,
// offsets in the instructions, rescaling only by 2^8: 283 / 94 / 60; largest parts first 282 / 94 / 56.
constexpr int kPagedGroup = 4;
template <class W> struct PagedTiles {
    static constexpr int kThreads = W::kWarps * 32, kGroups = W::kWarps / kPagedGroup, kSize = sizeof(typename W::Type), kSlots = 2 * W::kAhead + 1;
    static constexpr int kRow = W::kDim * kSize, kSlot = W::kTile * kRow, kRing = kSlots * kSlot, kQ = W::kHeads * kRow;
    static constexpr int kQueries = W::kWarps * kRing, kStats = kQueries + kGroups * 2 * kQ, kSpare = kStats + W::kWarps * W::kHeads * 8;       // offsets
    static constexpr int kSmem = kSpare + W::kWarps * W::kSpare;
    static constexpr int kStride = kPagedGroup * W::kTile, kLook = 32 / W::kTile;      // between two tiles of a warp; tiles of a look into the table
    static_assert(8 * W::kDim * 4 <= kSlot, "eight heads' state fits the slot that is free");
};

template <class W>
__global__ void __launch_bounds__(PagedTiles<W>::kThreads, 1) paged_tiles_kernel(const PagedParams p) {
    using S = PagedTiles<W>;
    using T = typename W::Type;
    constexpr int D = W::kDim, kPiece = 16 / S::kSize;                 // elements of 16 bytes
    chain_enter();
    extern __shared__ __align__(128) unsigned char paged_smem[];
    __shared__ __align__(16) PagedOrder<W::kSeqs> order;
    __shared__ uint8_t freed[W::kWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = warp / kPagedGroup, among = warp % kPagedGroup;
    unsigned char* own = paged_smem + warp * S::kRing;
    const uint32_t ring = smem_u32(own), queries = smem_u32(paged_smem) + S::kQueries + group * 2 * S::kQ;
    float2* stats = reinterpret_cast<float2*>(paged_smem + S::kStats) + group * kPagedGroup * W::kHeads;       // [warp of the group][head]: maximum, sum
    const int total = paged_schedule<W::kSeqs, S::kThreads>(p, order, (int)gridDim.x * S::kGroups);
    const int step = (int)gridDim.x * S::kGroups, mine = group * (int)gridDim.x + (int)blockIdx.x;             // neighbouring parts lie on different SMs
    if (mine >= total) return;
    const auto meet = [&]() { named_barrier(1 + group, kPagedGroup * 32); };

    // ---- queries, pieces turned as the tiles'; two buffers, the next part's on their way during this one
    constexpr int kRowPieces = D / kPiece, kQPieces = W::kHeads * kRowPieces, kQEach = (kQPieces + kPagedGroup * 32 - 1) / (kPagedGroup * 32);
    const auto q_fetch = [&](const Piece& a, int buffer) {
        const T* first = (const T*)p.q + a.b * p.q_row + a.head0 * p.q_head;
#pragma unroll
        for (int j = 0; j < kQEach; ++j) {
            const int i = (j * kPagedGroup + among) * 32 + lane, h = i / kRowPieces, piece = i % kRowPieces;
            if (kQPieces % (kPagedGroup * 32) && i >= kQPieces) break;
            const uint32_t at = buffer * S::kQ + h * S::kRow + ((piece ^ (h & 7)) << 4);
            const bool there = h < a.heads && piece * kPiece < p.dim;
            const T* src = there ? first + h * p.q_head + piece * kPiece : (const T*)p.q;
            if (p.q_whole) cp_async16(queries + at, src, there ? 16 : 0);
            else *reinterpret_cast<uint4*>(paged_smem + S::kQueries + group * 2 * S::kQ + at) = there ? paged_load16(src) : make_uint4(0, 0, 0, 0);
        }
    };

    // ---- what the warp loads next: a lane's page is looked up ahead (a look takes longer than a tile when HBM is busy)
    struct Look { int entry, row, kvh, tiles; };                       // a lane's position; tiles of the warp among the 32 positions
    Piece ahead = paged_piece(p, order, mine, 0), a = ahead;
    q_fetch(a, 0);
    cp_async_commit();
    int next = mine, c = ahead.t0 + among * W::kTile;
    const auto look_up = [&]() {
        while (c >= ahead.t1 && next < total) {
            next = paged_next(next, step);
            if (next < total) { ahead = paged_piece(p, order, next, ahead.at); c = ahead.t0 + among * W::kTile; }
        }
        Look k{-1, 0, ahead.kvh, 1};
        if (next >= total) return k;
        k.tiles = S::kLook == 2 ? (c + S::kStride < ahead.t1 ? 2 : 1) : min(S::kLook, (ahead.t1 - c + S::kStride - 1) / S::kStride);
        const int i = c + lane % W::kTile + lane / W::kTile * S::kStride;
        if (i < ahead.t1) {
            const int position = paged_position(p, i, ahead.skip), at = position / p.page;
            k.row = position - at * p.page;
            k.entry = __ldcg(p.table + ahead.b * p.table_stride + at);
        }
        c += S::kLook * S::kStride;
        return k;
    };
    Look later = look_up();
    long long off = 0;                 // a lane's row, in elements
    uint32_t there = 0;                // which of the 32 rows there are
    int at = 0, end = 0;               // the tile's rows among them; behind the last tile's
    const auto advance = [&]() {
        at += W::kTile;
        if (at < end) return;
        const bool page = later.entry >= 0 && later.entry < p.pages;
        off = page ? later.entry * p.page_stride + later.row * p.row_stride + later.kvh * p.head_stride : 0;
        there = __ballot_sync(0xffffffffu, page);
        end = later.tiles * W::kTile;
        at = 0;
        later = look_up();
    };
    // Eight lanes copy a line of a row, four rows an instruction.  Piece i of row r lies at piece i ^ (r & 7): a place of the lane's and a constant.
    const int lr = lane >> 3, lq = lane & 7, pieces = p.dim / kPiece;
    const uint32_t turn = lr * S::kRow + ((lq ^ lr) << 4);
    const auto load = [&](int slot, const void* pool) {
        const uint32_t to = ring + slot * S::kSlot + turn, to_odd = to ^ 64;
        const T* const first = (const T*)pool + lq * kPiece;
        if (p.dim == D)
            static_loop<0, W::kTile / 4>([&](auto four) {
                const T* src = first + __shfl_sync(0xffffffffu, off, at + 4 * four + lr);
                const int size = (there >> (at + 4 * four + lr) & 1) << 4;
                static_loop<0, S::kRow / 128>([&](auto j) { cp_async16_at<4 * four * S::kRow + j * 128, j * 128>(four & 1 ? to_odd : to, src, size); });
            });
        else                            // columns past the head dimension: zeros (no byte is read there)
            static_loop<0, W::kTile / 4>([&](auto four) {
                const T* src = first + __shfl_sync(0xffffffffu, off, at + 4 * four + lr);
                const int size = (there >> (at + 4 * four + lr) & 1) << 4;
                static_loop<0, S::kRow / 128>([&](auto j) {
                    cp_async16_at<4 * four * S::kRow + j * 128, j * 128>(four & 1 ? to_odd : to, src, 8 * j + lq < pieces ? size : 0);
                });
            });
        cp_async_commit();
    };
    constexpr uint32_t kMask = W::kTile == 32 ? ~0u : (1u << (W::kTile & 31)) - 1u;
    advance();
    uint32_t rows_of[W::kAhead + 1];                                   // which rows of the tiles on their way are there
#pragma unroll
    for (int i = 0; i < W::kAhead; ++i) {
        rows_of[i] = there >> at & kMask;
        load(2 * i, p.k);
        load(2 * i + 1, p.v);
        advance();
    }
    cp_async_wait<2 * W::kAhead>();
    meet();

    int slot = 0, buffer = 0;
    const auto next_slot = [&]() { slot = slot == S::kSlots - 1 ? 0 : slot + 1; };
    const auto free_slot = [&]() { return slot == 0 ? S::kSlots - 1 : slot - 1; };        // read in the previous step
    W work(lane, smem_u32(paged_smem) + S::kSpare + warp * W::kSpare);
    for (int r = mine, following; r < total; r = following, buffer ^= 1) {
        following = paged_next(r, step);
        Piece b = a;
        work.begin(queries + buffer * S::kQ);
        if (following < total) { b = paged_piece(p, order, following, a.at); q_fetch(b, buffer ^ 1); }
#pragma unroll 1
        for (int i = a.t0 + among * W::kTile; i < a.t1; i += S::kStride) {
            cp_async_wait<S::kSlots - 2>();
            __syncwarp();
            rows_of[W::kAhead] = there >> at & kMask;
            load(free_slot(), p.k);
            const uint32_t keys = ring + slot * S::kSlot;
            next_slot();
            work.scores(keys, rows_of[0], p.scale);
            cp_async_wait<S::kSlots - 2>();
            __syncwarp();
            load(free_slot(), p.v);
            advance();
            const uint32_t values = ring + slot * S::kSlot;
            next_slot();
            work.values(values);
#pragma unroll
            for (int j = 0; j < W::kAhead; ++j) rows_of[j] = rows_of[j + 1];
        }
        // the next queries came with the first tile that this part sent for: behind more tiles than are on their way they have been waited for
        if (a.t1 - a.t0 <= (W::kAhead * kPagedGroup + among) * W::kTile) cp_async_wait_all();
        // ---- the four states, eight heads at a time, each in the slot that its warp has free: [head][column], columns of heads 2 t and 2 t + 1 turned by
        // 8 t (four heads' columns meet 32 banks); joined to means, no larger than the largest value
        if (lane == 0) freed[warp] = (uint8_t)free_slot();
#pragma unroll
        for (int n = 0; n < W::kHeads / 8; ++n) {
            work.leave(n, reinterpret_cast<float*>(own + free_slot() * S::kSlot), stats + among * W::kHeads + n * 8);
            meet();
#pragma unroll
            for (int i = among * 32 + lane; i < 8 * (D / 4); i += kPagedGroup * 32) {
                const int eighth = i / (D / 4), h = n * 8 + eighth, f = i % (D / 4) * 4, place = eighth * D + (f ^ ((eighth >> 1) << 3));
                if (h >= a.heads || f >= p.dim) continue;
                float2 of[kPagedGroup];
                float top = -INFINITY, den = 0.f;
#pragma unroll
                for (int w = 0; w < kPagedGroup; ++w) { of[w] = stats[w * W::kHeads + h]; top = fmaxf(top, of[w].x); }
#pragma unroll
                for (int w = 0; w < kPagedGroup; ++w) { of[w].x = of[w].y == 0.f ? 0.f : exp2f(of[w].x - top); den += of[w].x * of[w].y; }
                float4 mean = make_float4(0.f, 0.f, 0.f, 0.f);
                const float inverse = den == 0.f ? 0.f : reciprocal(den);
#pragma unroll
                for (int w = 0; w < kPagedGroup; ++w) {
                    const float share = of[w].x * inverse;
                    const int other = group * kPagedGroup + w;
                    const float4 v = *reinterpret_cast<const float4*>(paged_smem + other * S::kRing + freed[other] * S::kSlot + place * 4);
                    mean.x += share * v.x; mean.y += share * v.y; mean.z += share * v.z; mean.w += share * v.w;
                }
                if (p.cuts.most) {
                    *reinterpret_cast<float4*>(p.partial + paged_place(p, a, h) * p.dim + f) = mean;
                    if (f == 0) p.stats[paged_place(p, a, h)] = make_float2(top, den);
                } else {
                    const float v[4] = {mean.x, mean.y, mean.z, mean.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) paged_put<T>(p, a.b, a.head0 + h, f + e, v[e]);
                }
            }
            meet();                                                                     // the states are read, the next queries there
        }
        a = b;
    }
    cp_async_wait<0>();
}

}  // namespace qd
