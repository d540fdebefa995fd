// bf16 tiles on the tensor cores (mma.sync: eight query heads fill its columns, 16 of 128 rows of a tcgen05 tile would be used): scores S = K Q^T,
// weights, O^T += V^T P^T, positions or columns as rows and eight heads as columns.
#pragma once
#include "paged_tiles.cuh"

namespace qd {

template <int AT = 0> QD_DEVINL void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at), "n"(AT) : "memory");
}
template <int AT> QD_DEVINL void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at), "n"(AT) : "memory");
}
QD_DEVINL uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
QD_DEVINL void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
QD_DEVINL uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}
QD_DEVINL uint32_t high_halves(float lo, float hi) { return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632); }
QD_DEVINL float rest_of(float x) { return fmaxf(x - __uint_as_float(__float_as_uint(x) & 0xffff0000u), x * 0x1p-20f); }

template <int D, int NT> struct PagedMma {
    using Type = bf16;
    static constexpr int kDim = D, kHeads = NT * 8, kTile = 16, kWarps = D == 64 ? 16 : 8, kAhead = D == 256 ? 1 : 2, kSpare = 0;
    static constexpr int kSeqs = D == 256 && NT == 2 ? 192 : 1024;     // (what memory has room for)
    const int lane, g, t;
    const uint32_t key_turn, value_turn;
    static constexpr bool kHeld = NT == 1 || D == 128;                 // queries in registers (24 heads of 128 on a key head, 28 x 12307 positions: 122.7 us, 130.5 read for each tile); sixteen heads of 64 (five words lie outside of the registers as it is) or 256 find no room
    uint32_t q_row, q4[kHeld ? NT * D / 32 : 1][4];
    float acc[NT][D / 16][4], m[NT][2], l[NT][2];                      // columns g and g + 8 of every sixteen, heads 2 t and 2 t + 1
    uint32_t hi[NT][2], lo[NT][2];

    QD_DEVINL PagedMma(int lane, uint32_t) : lane(lane), g(lane >> 2), t(lane & 3),
        key_turn((lane & 15) * (D * 2) + ((((lane >> 4) ^ (lane & 3)) | (lane & 4)) << 4)),
        value_turn(((lane & 7) + ((lane >> 4) << 3)) * (D * 2) + ((((lane >> 3 & 1) ^ (lane & 3)) | (lane & 4)) << 4)) {}

    QD_DEVINL void begin(uint32_t queries) {
        q_row = queries + (lane & 7) * (D * 2);
        if (kHeld) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < D / 32; ++k) ldmatrix4(q4[n * D / 32 + k], q_row + n * 8 * (D * 2) + (((4 * k + (lane >> 3)) ^ (lane & 7)) << 4));
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
        }
    }

    // Scores and weights of positions g and g + 8.
    QD_DEVINL void scores(uint32_t keys, uint32_t rows, float scale) {
        // scores of positions g and g + 8, heads 2 t and 2 t + 1
        float s[NT][2][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][0][e] = s[n][1][e] = 0.f;
        // (places as they were loaded: two bits of the piece are the lane's, one turns with kk, the rest are constants)
        const uint32_t key_at = keys + key_turn;
        static_loop<0, D / 32>([&](auto k) {
            uint32_t ka[4], kb[4];
            const uint32_t at = k & 1 ? key_at ^ 64 : key_at;
            ldmatrix4<(k >> 1) * 128>(ka, at);
            ldmatrix4<(k >> 1) * 128>(kb, at ^ 32);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t (&q)[4] = q4[kHeld ? n * D / 32 + k : 0];
                if (!kHeld) ldmatrix4(q, q_row + n * 8 * (D * 2) + (((4 * k + (lane >> 3)) ^ (lane & 7)) << 4));
                mma16816(s[n][0], ka, q[0], q[1]);
                mma16816(s[n][1], kb, q[2], q[3]);
            }
        });
        const bool in0 = rows >> g & 1, in1 = rows >> (g + 8) & 1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (e < 2 ? in0 : in1) ? (s[n][0][e] + s[n][1][e]) * scale : -INFINITY;
            float top0 = fmaxf(x[0], x[2]), top1 = fmaxf(x[1], x[3]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, d));
                top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, d));
            }
            // the reference moves when the maximum is 2^8 above it: weights of up to 2^8 lose nothing, and few tiles rescale
            if (__any_sync(0xffffffffu, top0 > m[n][0] + 8.f || top1 > m[n][1] + 8.f)) {
                top0 = fmaxf(m[n][0], top0);
                top1 = fmaxf(m[n][1], top1);
                const float fix0 = weight_of(m[n][0], top0), fix1 = weight_of(m[n][1], top1);
                m[n][0] = top0; m[n][1] = top1;
                l[n][0] *= fix0; l[n][1] *= fix1;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) { acc[n][d][0] *= fix0; acc[n][d][1] *= fix1; acc[n][d][2] *= fix0; acc[n][d][3] *= fix1; }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = weight_of(x[e], m[n][e & 1]) * kPagedWeight;
            l[n][0] += x[0] + x[2];
            l[n][1] += x[1] + x[3];
            // weights in two bf16 pieces (sixteen bits): one alone would be off by as much as the result's own rounding.  The first is cut off, not rounded,
            // and the second is at least 2^-20 of the weight: zero or a negative number times an infinite value would make NaN of an infinite mean
            hi[n][0] = transposed(high_halves(x[0], x[1])); hi[n][1] = transposed(high_halves(x[2], x[3]));
            lo[n][0] = transposed(pack2(rest_of(x[0]), rest_of(x[1])));
            lo[n][1] = transposed(pack2(rest_of(x[2]), rest_of(x[3])));
        }
    }
    QD_DEVINL void values(uint32_t values) {
        const uint32_t value_at = values + value_turn;
        static_loop<0, D / 16>([&](auto d) {
            uint32_t va[4];
            ldmatrix4_trans<(d >> 2) * 128>(va, value_at ^ ((d & 1) * 32 + (d >> 1 & 1) * 64));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mma16816(acc[n][d], va, hi[n][0], hi[n][1]);
                mma16816(acc[n][d], va, lo[n][0], lo[n][1]);
            }
        });
    }
    QD_DEVINL void leave(int n, float* state, float2* stats) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
            const int h = 2 * t + e;
            if (g == 0) stats[h] = make_float2(m[n][e], l[n][e]);
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int up = 0; up < 2; ++up) state[h * D + ((d * 16 + up * 8 + g) ^ (t << 3))] = acc[n][d][2 * up + e];
        }
    }
};

}  // namespace qd
