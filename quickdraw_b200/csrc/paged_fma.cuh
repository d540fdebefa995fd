// fp32 tiles in fp32 arithmetic: a position's columns over LANES lanes, eight a lane, all query heads of the part in each.
#pragma once
#include "paged_tiles.cuh"

namespace qd {

// HEADS (4 or 8) query heads.  What bounds it is the number of instructions, 2 * HEADS * 4 of them multiply-adds for two rows' eight columns; so a sum
// over lanes is taken for all heads at once, each step halving the heads that a lane still carries, and weights go through shared memory.  48 sequences
// that see 1028 rows, 16 heads on 4 of 64 (99 MB, from HBM): 28 us; 20 up to 3000, 32 on 8 of 128 (249 MB): 60; 16 up to 8000, 32 on 1 of 256 (138 MB, four
// passes over eight heads): 111, where arithmetic is all (134 with one multiply-add an instruction).
template <int D, int HEADS> struct PagedFma {
    using Type = float;
    static constexpr int kDim = D, kHeads = 8, kTile = 8, kSeqs = 256;
    static constexpr bool kNarrow = D == 64 && HEADS == 4;               // state and queries fit 128 registers but for five words: 28.2 us of the first, 29.4 by eight warps, 8 on 8 of 64 (370 MB) 73 and 80; eight heads of 64 would not, 79 for 35
    static constexpr int kWarps = kNarrow ? 16 : 8, kAhead = D == 256 ? 1 : D == 128 || kNarrow ? 2 : 4;
    static constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kSteps = kTile / kAtOnce;        // lanes of a position, positions at once
    static constexpr int kSpare = kAtOnce > 1 ? kTile * 8 * 4 : 0;
    const int lane, own, part, column;       // own: the head whose sums the lane gets; part: which of the positions at once; first columns: column and D / 2 + column
    const uint32_t weights;                  // shared memory: [position][8] (where a warp has all of a position, from lane to lane)
    float2 q[HEADS][4], acc[HEADS][4];       // by twos: one instruction for two
    float x[kSteps], m, l;       // scores, then weights, m and l of head `own`

    QD_DEVINL PagedFma(int lane, uint32_t spare) : lane(lane),
        own(HEADS == 8 ? (lane & 1) * 4 + (lane >> 1 & 1) * 2 + (lane >> 2 & 1) : (lane & 1) * 2 + (lane >> 1 & 1)),
        part(lane / kLanes), column(lane % kLanes * 4), weights(spare) {}

    QD_DEVINL float4 shared4(uint32_t at) const {
        float4 v;
        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
        return v;
    }
    // Eight columns of a row of a tile.
    QD_DEVINL void row8(uint32_t tile, int row, float2 (&v)[4]) const {
        const uint32_t at = tile + row * (D * 4) + (((lane % kLanes) ^ (row & 7)) << 4);
        const float4 a = shared4(at), b = shared4(at + D * 2);               // (kLanes pieces further: a multiple of eight)
        v[0] = make_float2(a.x, a.y); v[1] = make_float2(a.z, a.w); v[2] = make_float2(b.x, b.y); v[3] = make_float2(b.z, b.w);
    }
    QD_DEVINL void begin(uint32_t queries) {
#pragma unroll
        for (int h = 0; h < HEADS; ++h) row8(queries, h, q[h]);
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[h][j] = make_float2(0.f, 0.f);
        m = -INFINITY; l = 0.f;
    }
    static QD_DEVINL constexpr int lane_of(int h) { return HEADS == 8 ? (h >> 2) + (h & 2) + (h & 1) * 4 : (h >> 1) + (h & 1) * 2; }       // that gets head h
    // The sums over a position's lanes of v[h], that of head `own` here.
    QD_DEVINL float sum_up(float (&v)[HEADS]) const {
        int d = 1;
#pragma unroll
        for (int count = HEADS / 2; count > 0; count >>= 1, d <<= 1) {
            const bool upper = lane & d;
#pragma unroll
            for (int i = 0; i < count; ++i) {
                const float keep = upper ? v[i + count] : v[i], give = upper ? v[i] : v[i + count];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
            }
        }
#pragma unroll
        for (int e = HEADS; e < kLanes; e <<= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], e);
        return v[0];
    }
    QD_DEVINL void scores(uint32_t keys, uint32_t rows, float scale) {
        float top = -INFINITY;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            float2 k[4];
            float v[HEADS];
            row8(keys, s * kAtOnce + part, k);
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                float2 sum = mul2(q[h][0], k[0]);
#pragma unroll
                for (int j = 1; j < 4; ++j) sum = fma2(q[h][j], k[j], sum);
                v[h] = sum.x + sum.y;
            }
            x[s] = sum_up(v);
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            x[s] = rows >> (s * kAtOnce + part) & 1 ? x[s] * scale : -INFINITY;
            top = fmaxf(top, x[s]);
        }
#pragma unroll
        for (int e = kLanes; e < 32; e <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, e));
        // the reference moves when the maximum is 2^8 above it: weights of up to 2^8 lose nothing, and few tiles rescale
        if (__any_sync(0xffffffffu, top > m + 8.f)) {
            top = fmaxf(m, top);
            const float fix = weight_of(m, top);
            m = top;
            l *= fix;
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                const float of = __shfl_sync(0xffffffffu, fix, lane_of(h));
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[h][j] = mul2(acc[h][j], make_float2(of, of));
            }
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            x[s] = weight_of(x[s], m) * kPagedWeight;
            l += x[s];
            if (kAtOnce > 1 && lane % kLanes < HEADS)
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(weights + ((s * kAtOnce + part) * 8 + own) * 4), "f"(x[s]) : "memory");
        }
        if (kAtOnce > 1) __syncwarp();
    }
    QD_DEVINL void values(uint32_t values) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int row = s * kAtOnce + part;
            float2 v[4];
            float w[8];
            row8(values, row, v);
            if constexpr (kAtOnce > 1) {
                const float4 a = shared4(weights + row * 32), b = HEADS == 8 ? shared4(weights + row * 32 + 16) : a;
                w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
            } else {
#pragma unroll
                for (int h = 0; h < HEADS; ++h) w[h] = __shfl_sync(0xffffffffu, x[s], lane_of(h));
            }
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[h][j] = fma2(make_float2(w[h], w[h]), v[j], acc[h][j]);
        }
    }
    QD_DEVINL void leave(int, float* state, float2* stats) {
#pragma unroll
        for (int e = kLanes; e < 32; e <<= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, e);
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[h][j].x += __shfl_xor_sync(0xffffffffu, acc[h][j].x, e);
                    acc[h][j].y += __shfl_xor_sync(0xffffffffu, acc[h][j].y, e);
                }
        }
        if (lane < HEADS) stats[own] = make_float2(m, l);
        if (part == 0) {
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                float* to = state + h * D + (column ^ ((h >> 1) << 3));
                *reinterpret_cast<float4*>(to) = make_float4(acc[h][0].x, acc[h][0].y, acc[h][1].x, acc[h][1].y);
                *reinterpret_cast<float4*>(to + D / 2) = make_float4(acc[h][2].x, acc[h][2].y, acc[h][3].x, acc[h][3].y);
            }
        }
    }
};

}  // namespace qd
