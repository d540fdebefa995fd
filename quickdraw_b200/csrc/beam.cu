// Beam search: the best continuations of every group of beams, and the beams' states put in the order of their parents.
//
// A continuation of beam i by token v counts score[i] + x[i, v] - log sum_w exp x[i, w].  Within a beam the order is that of the logits, so a first
// kernel takes, of each piece of a row, the largest logits, the maximum and the sum of exponentials, and a second one joins the pieces, adds up in 64
// bits (sums of different beams lie next to one another) and merges the beams.
#include "paged_tiles.cuh"

namespace qd {
namespace {

constexpr int kMostBeams = 32, kMostSplits = 32;

// Keys order as (value, lower index first); NaN cannot occur among rows that count.
QD_DEVINL unsigned long long logit_key(float v, int index) {
    uint32_t bits = __float_as_uint(v);
    if (bits == 0x80000000u) bits = 0u;
    const uint32_t order = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return ((unsigned long long)order << 32) | (0xffffffffu - (uint32_t)index);
}
QD_DEVINL float key_logit(unsigned long long key) {
    const uint32_t order = (uint32_t)(key >> 32);
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
QD_DEVINL int key_index(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }
template <typename T> QD_DEVINL float logit_of(T v);
template <> QD_DEVINL float logit_of<float>(float v) { return v; }
template <> QD_DEVINL float logit_of<bf16>(bf16 v) { return __bfloat162float(v); }

struct SelectParams {
    const void* logits; long long row_stride;                 // elements from a row to the next
    const float* scores; const uint8_t* finished;
    unsigned long long* keys;                                 // [row][split][candidates], descending; 0: none
    double2* sums;                                            // [row][split]: maximum, sum of exp(x - maximum)
    float* scores_out; int* parents_out; long long* tokens_out;
    int batch, beams, vocab, candidates, splits, eos, placed, fp32;
};

QD_DEVINL float exp_base2(float x) {             // (results below 2^-126 are zero)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The largest of three.
QD_DEVINL float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Descending order of 32 keys, one a lane.
QD_DEVINL unsigned long long warp_sorted(unsigned long long key, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, d);
            const bool upper = lane & d, ascending = lane & size;               // (of the last round: lane & 32, never)
            key = (other > key) != (upper != ascending) ? other : key;
        }
    return key;
}

// A block per piece of a row, one pass: sixteen logits a thread at a time, their maximum and sum of exponentials, and a list of the keys above a bound that
// `candidates` keys seen so far reach.  The bound comes from the lanes' largest keys of the first chunk, and again where more than a few threads have a key
// above it; it rises to the candidates-th of the list when that grows.  32 x 8 rows of 151936 with the merge: 40 us fp32 (156 MB; 35 with no keys
// and no exponentials to take) and 40 bf16; fp32 43 with the next chunk in registers (fewer blocks an SM) and a second barrier in every chunk that
// has a key.  Two chunks ahead took 42 (fewer blocks), a warp with a list of its own ten more (eight first chunks instead of one), 256 threads seven more.
// 4 x 32 rows: 65 to 68 us, 98 with a first bound from each warp alone (a fifth of the chunk is above it).
constexpr int kPartThreads = 128, kPartEach = 16, kPartMany = 32, kPartPending = 16, kPartSlack = 4;
template <typename T> constexpr size_t part_ring() { return 2 * kPartThreads * kPartEach * sizeof(T); }
template <typename T>
QD_DEVINL double2 part_of_row(const T* x, int lo, int hi, int K, unsigned long long* part_list, unsigned char* ring, unsigned long long* out) {
    // part_list (part_bytes) has room for K + kPartSlack keys, for those of kPartPending threads and for what a chunk can add: kPartMany threads' keys, or
    // those of K lanes of each warp.  ring: part_ring bytes on 16.  out: the K largest keys, 0 behind the last
    __shared__ unsigned long long bounds[2 * (kPartThreads / 32)];
    __shared__ double2 sums[kPartThreads / 32];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) count = 0;
    // the thread's j-th logit of the chunk from `base`: four pieces of 16 bytes of fp32, two of bf16; the first chunk begins on a piece in front of `lo`
    constexpr int kRun = sizeof(T) == 4 ? 4 : 8;
    const auto place = [&](int base, int j) { return base + j / kRun * (kRun * kPartThreads) + tid * kRun + j % kRun; };
    constexpr int kChunk = kPartThreads * kPartEach, kBytes = kChunk * (int)sizeof(T);
    const uint32_t own = smem_u32(ring) + tid * 16;
    const int start = lo - (int)((reinterpret_cast<uintptr_t>(x + lo) & 15u) / sizeof(T));
    const auto whole = [&](int base) { return base >= lo && base <= hi - kChunk; };             // (of all threads alike)
    const auto is_there = [&](int at) { return at >= lo && at < hi; };
    const auto fetch = [&](int base, int slot) {
        if (whole(base)) {
#pragma unroll
            for (int j = 0; j < kPartEach / kRun; ++j) cp_async16(own + slot * kBytes + j * (kPartThreads * 16), x + place(base, j * kRun), 16);
        }
        cp_async_commit();
    };
    const auto take = [&](int base, int slot, float (&v)[kPartEach]) {
        if (whole(base)) {
#pragma unroll
            for (int j = 0; j < kPartEach; j += kRun) {
                uint32_t w[4];
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(own + slot * kBytes + j / kRun * (kPartThreads * 16)) : "memory");
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (sizeof(T) == 4) v[j + e] = __uint_as_float(w[e]);
                    else { v[j + 2 * e] = __uint_as_float(w[e] << 16); v[j + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < kPartEach; ++j) v[j] = is_there(place(base, j)) ? logit_of(x[place(base, j)]) : -INFINITY;
        }
    };
    // the K largest of the list, in order: a thread counts for its keys how many are larger
    const auto keep = [&](unsigned long long* into, int n) {
        for (int i = tid; i < n; i += kPartThreads) {
            const unsigned long long key = part_list[i];
            int rank = 0, z = 0;
#pragma unroll 4
            for (; z + 1 < n; z += 2) {
                const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(part_list + z);
                rank += (two.x > key) + (two.y > key);
            }
            if (z < n) rank += part_list[z] > key;
            if (rank < K) into[rank] = key;
        }
    };
    float top = -INFINITY;
    double sum = 0.0;                  // of sums of sixteen: 32 bits would lose a ten-millionth with every few terms
    unsigned long long bound = 0;
    float least = -INFINITY;           // the bound's logit
    int pending = 0;                   // threads that have put keys into the list since its length was looked at
    fetch(start, 0);
    __syncthreads();
    for (int base = start, slot = 0; base < hi; base += kChunk, slot ^= 1) {
        float v[kPartEach], most = -INFINITY;
        cp_async_wait<0>();
        take(base, slot, v);
        fetch(base + kChunk, slot ^ 1);
#pragma unroll
        for (int j = 0; j < kPartEach; j += 2) most = max3(most, v[j], v[j + 1]);
        // (terms of up to e^2 lose nothing, and few chunks rescale)
        if (most > top + 2.f) { sum *= (double)exp_base2((top - most) * 1.4426950408889634f); top = most; }
        const float shift = top == -INFINITY ? 0.f : top;
        float2 e[kPartEach / 2];
#pragma unroll
        for (int j = 0; j < kPartEach / 2; ++j) {                               // (NaN and infinity go on)
            e[j] = mul2(add2(make_float2(v[2 * j], v[2 * j + 1]), make_float2(-shift, -shift)), make_float2(1.4426950408889634f, 1.4426950408889634f));
            e[j] = make_float2(exp_base2(e[j].x), exp_base2(e[j].y));
        }
#pragma unroll
        for (int d = kPartEach / 4; d > 0; d >>= 1)
#pragma unroll
            for (int j = 0; j < d; ++j) e[j] = add2(e[j], e[j + d]);
        sum += (double)(e[0].x + e[0].y);
        const bool hit = most >= least;
        const int above = __syncthreads_count(hit);
        if (above == 0) continue;
        const auto key_of = [&](int j) { return is_there(place(base, j)) ? logit_key(v[j], place(base, j)) : 0; };       // other places: none
        if (above > kPartMany) {
            unsigned long long mine = 0;
#pragma unroll
            for (int j = 0; j < kPartEach; ++j) mine = key_of(j) > mine ? key_of(j) : mine;
            // K keys are as large as a warp's K-th, and as the least of all warps' shares of K
            constexpr int kAll = kPartThreads / 32;
            const unsigned long long sorted = warp_sorted(mine, lane), kth = __shfl_sync(0xffffffffu, sorted, K - 1), share = __shfl_sync(0xffffffffu, sorted, (K - 1) / kAll);
            if (lane == 0) { bounds[warp] = kth; bounds[kAll + warp] = share; }
            __syncthreads();
            unsigned long long least_share = bounds[kAll];
#pragma unroll
            for (int w = 0; w < kAll; ++w) {
                bound = bounds[w] > bound ? bounds[w] - 1 : bound;
                least_share = bounds[kAll + w] < least_share ? bounds[kAll + w] : least_share;
            }
            bound = least_share > bound ? least_share - 1 : bound;
            if (bound) least = key_logit(bound);
        }
        if (hit) {
            unsigned mask = 0;
#pragma unroll
            for (int j = 0; j < kPartEach; ++j) mask |= v[j] >= least ? 1u << j : 0u;
            for (; mask; mask &= mask - 1u) {
                const int j = __ffs(mask) - 1, at = place(base, j);
                if (!is_there(at)) continue;
                const T* from = whole(base) ? (const T*)(ring + tid * 16 + slot * kBytes + j / kRun * (kPartThreads * 16)) + j % kRun : x + at;
                const unsigned long long key = logit_key(logit_of(*from), at);
                if (key > bound) part_list[atomicAdd(&count, 1)] = key;
            }
        }
        pending += above;
        if (pending <= kPartPending) continue;
        pending = 0;
        __syncthreads();
        const int n = count;
        if (n > K + kPartSlack) {                                                   // (a thread counts n keys: often and few is less than seldom and many)
            keep(out, n);                                                       // (the results' place serves as scratch)
            __syncthreads();
            if (tid < K) part_list[tid] = out[tid];
            bound = out[K - 1];
            least = key_logit(bound);
            if (tid == 0) count = K;
            __syncthreads();
        }
    }
    __syncthreads();
    const int n = count;
    for (int k = n + tid; k < K; k += kPartThreads) out[k] = 0;
    keep(out, n);
    // sums of the threads to the block's largest
    const float warp_top = warp_max(top);
    if (lane == 0) sums[warp].x = warp_top;
    __syncthreads();
    float all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kPartThreads / 32; ++w) all = fmaxf(all, (float)sums[w].x);
    sum = sum == 0.0 ? 0.0 : sum * exp((double)top - (double)all);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) sums[warp].y = sum;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kPartThreads / 32; ++w) total += sums[w].y;
    return make_double2((double)all, total);
}
static size_t part_bytes(int candidates) {
    return sizeof(unsigned long long) * (candidates + kPartSlack + kPartEach * (kPartPending + (kPartMany > kPartThreads / 32 * candidates ? kPartMany : kPartThreads / 32 * candidates)));
}
template <typename T>
__global__ void __launch_bounds__(kPartThreads) select_part_kernel(const SelectParams p) {
    chain_enter();
    extern __shared__ __align__(16) unsigned long long select_list[];
    const int row = blockIdx.y, split = blockIdx.x, each = p.vocab / 8;
    if (p.finished && p.finished[row]) return;
    const int lo = (int)((long long)each * split / p.splits) * 8, hi = split + 1 == p.splits ? p.vocab : (int)((long long)each * (split + 1) / p.splits) * 8;
    const long long at = (long long)row * p.splits + split;
    const double2 sum = part_of_row<T>((const T*)p.logits + row * p.row_stride, lo, hi, p.candidates, select_list + part_ring<T>() / 8, (unsigned char*)select_list, p.keys + at * p.candidates);
    if (threadIdx.x == 0) p.sums[at] = sum;
}

// The first block's shared memory, from any block of the cluster.
QD_DEVINL uint32_t of_first_block(const void* mine) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(mine)));
    return at;
}
QD_DEVINL void store_there(uint32_t at, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(v) : "memory"); }
QD_DEVINL void store_there(uint32_t at, int v) { asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
QD_DEVINL unsigned load_there(uint32_t at) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
QD_DEVINL void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// A cluster per group: a warp joins a beam's pieces, then the first block puts all beams' continuations in order.
//
// Sums of 32-bit exponentials (2^-22 each from the instruction, as much from its argument, twice that from sums of sixteen) leave a beam's log-sum-exp
// known to 2^-20.  Where one of the best is nearer than 2^-18 to another beam's continuation, both beams' sums are taken again in 64 bits by all blocks,
// until no such beams are left: the choice is then that of 64 bits.  Of 16 beams that happens to one group in some fifty.
constexpr int kMergeBlocks = 8, kMergeThreads = 128;
struct MergeShared {                                          // of the first block, but for `piece`
    double best[kMostBeams], partial[kMostBeams][kMergeBlocks], piece[kMergeThreads / 32];
    int order[kMostBeams];
    float top[kMostBeams];
    unsigned near;
};
// What a beam has to offer, into the first block's lists: n of its largest keys, in any order, the K largest among them (by a warp).
QD_DEVINL void offer(const SelectParams& p, MergeShared& shared, double* total, int* token, int group, int beam, bool finished, bool counts, float top, double lse,
                     const unsigned long long* list, int n) {
    const int K = p.candidates, lane = threadIdx.x & 31;
    const uint32_t totals = of_first_block(total + beam * K), tokens = of_first_block(token + beam * K);
    const double score = (double)p.scores[(long long)group * p.beams + beam];
    if (lane == 0) store_there(of_first_block(&shared.top[beam]), __float_as_int(top));
    if (finished || !counts) {
        for (int k = lane; k < K; k += 32) {
            // the end at no cost, and what never follows, in the order of the tokens
            int t = k;
            double v = -INFINITY;
            if (counts) {
                t = k == 0 ? p.eos : k - 1 + (k - 1 >= p.eos);
                if (k == 0) v = score;
            }
            store_there(totals + k * 8, v);
            store_there(tokens + k * 4, t < p.vocab ? t : -1);
        }
    } else {
        for (int k = lane; k < n; k += 32) {
            const unsigned long long key = list[k];
            int rank = 0;
            for (int z = 0; z < n; ++z) rank += list[z] > key;
            if (rank < K) {
                store_there(totals + rank * 8, score + ((double)key_logit(key) - lse));
                store_there(tokens + rank * 4, key_index(key));
            }
        }
        for (int k = n + lane; k < K; k += 32) store_there(tokens + k * 4, -1);
    }
    __syncwarp();
}
// The choice from all beams' lists, after a barrier of the cluster.
QD_DEVINL void choose(const SelectParams& p, MergeShared& shared, double* total, int* token, int group, int block) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = p.candidates;
    const auto finished = [&](int i) { return p.finished && p.finished[(long long)group * p.beams + i]; };
    for (unsigned known = 0;;) {
        if (block == 0) {
            // the shared.best of the beams' heads, K times; a lane has a beam's list, of equal ones the first beam's is taken
            if (warp == 0) {
                int at = 0;
                const auto head_of = [&]() -> unsigned long long {              // orders like the doubles; 0: none
                    if (lane >= p.beams || at >= K || token[lane * K + at] < 0) return 0;
                    const long long bits = __double_as_longlong(total[lane * K + at] + 0.0);
                    return bits < 0 ? ~(unsigned long long)bits : (unsigned long long)bits | 1ull << 63;
                };
                unsigned long long head = head_of();
                for (int k = 0; k < K; ++k) {
                    const unsigned high = __reduce_max_sync(0xffffffffu, (unsigned)(head >> 32));
                    const unsigned low = __reduce_max_sync(0xffffffffu, (unsigned)(head >> 32) == high ? (unsigned)head : 0u);
                    const int who = __ffs(__ballot_sync(0xffffffffu, head == ((unsigned long long)high << 32 | low))) - 1;
                    if (lane == who) {
                        shared.best[k] = total[lane * K + at];
                        shared.order[k] = lane * K + at;
                        ++at;
                        head = head_of();
                    }
                }
            }
            if (tid == 0) shared.near = 0;
            __syncthreads();
            for (int c = tid; c < p.beams * K; c += kMergeThreads) {
                if (token[c] < 0 || total[c] < shared.best[K - 1] - 0x1p-17) continue;
                for (int k = 0; k < K; ++k) {
                    const unsigned both = 1u << c / K | 1u << shared.order[k] / K;
                    if (c / K != shared.order[k] / K && fabs(shared.best[k] - total[c]) < 0x1p-18 && (both & ~known)) atomicOr(&shared.near, both & ~known);      // (-inf - -inf is not)
                }
            }
        }
        __syncthreads();
        cluster_sync();
        const unsigned again = load_there(of_first_block(&shared.near));
        if (again == 0) break;
        known |= again;
        for (int i = 0; i < p.beams; ++i) {
            if (!(again >> i & 1) || finished(i)) continue;
            const long long at = ((long long)group * p.beams + i) * p.row_stride;
            const float top = __uint_as_float(load_there(of_first_block(&shared.top[i])));
            double sum = 0.0;
            for (int v = (int)((long long)p.vocab * block / kMergeBlocks) + tid; v < (int)((long long)p.vocab * (block + 1) / kMergeBlocks); v += kMergeThreads)
                sum += exp((double)(p.fp32 ? ((const float*)p.logits)[at + v] : logit_of(((const bf16*)p.logits)[at + v])) - (double)top);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lane == 0) shared.piece[warp] = sum;
            __syncthreads();
            if (tid == 0) {
                for (int w = 1; w < kMergeThreads / 32; ++w) sum += shared.piece[w];
                store_there(of_first_block(&shared.partial[i][block]), sum);
            }
            __syncthreads();
        }
        cluster_sync();
        if (block == 0) {
            for (int i = warp; i < p.beams; i += kMergeThreads / 32) {
                if (!(again >> i & 1) || finished(i)) continue;
                const long long row = (long long)group * p.beams + i;
                const float top = shared.top[i];
                double sum = 0.0;
                for (int z = 0; z < kMergeBlocks; ++z) sum += shared.partial[i][z];
                const double exact = (double)top + log(sum);
                for (int k = lane; k < K; k += 32) {
                    const int t = token[i * K + k];
                    if (t < 0) continue;
                    const float logit = p.fp32 ? ((const float*)p.logits)[row * p.row_stride + t] : logit_of(((const bf16*)p.logits)[row * p.row_stride + t]);
                    total[i * K + k] = (double)p.scores[row] + ((double)logit - exact);
                }
            }
            __syncthreads();
        }
    }
    cluster_sync();                                                             // all have looked at `near`
    if (block || warp) return;
    const int chosen = lane < K ? shared.order[lane] : 0, parent = chosen / K;
    int place = lane;
    if (p.placed) {
        // a beam's shared.best continuation takes the beam's place, the others the places left, in shared.order
        const unsigned same = __match_any_sync(0xffffffffu, lane < K ? parent : 64 + lane);
        const bool leads = lane < K && (same & ((1u << lane) - 1u)) == 0;
        const unsigned taken = __reduce_or_sync(0xffffffffu, leads ? 1u << parent : 0u);
        const unsigned rest = __ballot_sync(0xffffffffu, lane < K && !leads);
        if (leads) place = parent;
        else {
            int skip = __popc(rest & ((1u << lane) - 1u));
            unsigned left = ~taken;
            for (; skip > 0; --skip) left &= left - 1u;
            place = __ffs(left) - 1;
        }
    }
    if (lane < K) {
        const long long o = (long long)group * K + place;
        p.scores_out[o] = (float)shared.best[lane];
        p.parents_out[o] = group * p.beams + parent;
        p.tokens_out[o] = token[chosen];
    }
}

__global__ void __cluster_dims__(kMergeBlocks, 1, 1) __launch_bounds__(kMergeThreads) select_merge_kernel(const SelectParams p) {
    chain_enter();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");       // waited for before the first access to another block's memory
    extern __shared__ __align__(16) unsigned char merge_smem[];
    __shared__ MergeShared shared;
    const int block = blockIdx.x % kMergeBlocks, group = blockIdx.x / kMergeBlocks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int K = p.candidates, lists = p.splits < K ? p.splits : K;
    double* total = reinterpret_cast<double*>(merge_smem);                                  // [beams][K], descending
    int* token = reinterpret_cast<int*>(total + p.beams * K);                               // [beams][K], -1: none
    unsigned long long* list = reinterpret_cast<unsigned long long*>(total + p.beams * K + (p.beams * K + 1) / 2) + (size_t)warp * lists * K;
    const int beam = block + warp * kMergeBlocks;                                           // the warp's
    const long long row = (long long)group * p.beams + beam;
    const bool there = beam < p.beams, finished = there && p.finished && p.finished[row];
    float top = -INFINITY;
    double lse = 0.0;
    bool counts = there && isfinite(p.scores[row]);
    int n = 0;
    if (there && !finished) {
        const unsigned long long* keys = p.keys + row * p.splits * K;
        const int deep = (K + p.splits - 1) / p.splits, pieces = (K + deep - 1) / deep;
        const unsigned long long head = lane < p.splits ? keys[lane * K + deep - 1] : 0;
        const double2 s = lane < p.splits ? p.sums[row * p.splits + lane] : make_double2(-INFINITY, 0.0);
        top = warp_max((float)s.x);
        const bool odd = __any_sync(0xffffffffu, lane < p.splits && (s.x != s.x || s.y != s.y));
        double sum = s.y == 0.0 ? 0.0 : s.y * exp(s.x - (double)top);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        lse = (double)top + log(sum);
        counts = counts && !odd && isfinite(lse);
        // `pieces` of them have `deep` keys each, K or more in all, that are no smaller than the largest bound for which that is so: keys below it are out
        const unsigned long long bound = __shfl_sync(0xffffffffu, warp_sorted(head, lane), pieces - 1);
        for (int k = lane; counts && k < (p.splits * K + 31) / 32 * 32; k += 32) {
            const unsigned long long key = k < p.splits * K ? keys[k] : 0;
            const bool in = key && key >= bound;
            const unsigned all = __ballot_sync(0xffffffffu, in);
            if (in) list[n + __popc(all & ((1u << lane) - 1u))] = key;
            n += __popc(all);
        }
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (there) offer(p, shared, total, token, group, beam, finished, counts, top, lse, list, n);
    cluster_sync();
    choose(p, shared, total, token, group, block);
}

// Rows of one chunk: the blocks of a group's cluster take its beams' rows themselves, one after the other, and no second launch is needed (which costs
// the host 5 us with its scratch; on the device 500 tokens of 16 x 16 beams take 17.9 instead of 17.7 us, 4096 of 1 x 4 9.9 instead of 10.4, but of 16 x 16
// 27 instead of 19).
constexpr int kShortVocab = kPartThreads * kPartEach;
template <typename T>
__global__ void __cluster_dims__(kMergeBlocks, 1, 1) __launch_bounds__(kMergeThreads) select_short_kernel(const SelectParams p) {
    static_assert(kMergeThreads == kPartThreads, "a block is both");
    chain_enter();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");       // waited for before the first access to another block's memory
    extern __shared__ __align__(16) unsigned char merge_smem[];
    __shared__ MergeShared shared;
    constexpr int kRows = kMostBeams / kMergeBlocks;
    __shared__ unsigned long long keys[kRows][kMostBeams];
    __shared__ double2 sums[kRows];
    const int block = blockIdx.x % kMergeBlocks, group = blockIdx.x / kMergeBlocks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = p.candidates;
    double* total = reinterpret_cast<double*>(merge_smem);                                  // [beams][K], descending
    int* token = reinterpret_cast<int*>(total + p.beams * K);                               // [beams][K], -1: none
    unsigned long long* list = reinterpret_cast<unsigned long long*>(merge_smem + (p.beams * K * 12 + 15) / 16 * 16);
    const auto finished = [&](int i) { return p.finished && p.finished[(long long)group * p.beams + i]; };
    for (int i = 0; block + i * kMergeBlocks < p.beams; ++i) {
        const int beam = block + i * kMergeBlocks;
        if (finished(beam)) continue;
        const long long row = (long long)group * p.beams + beam;
        const double2 sum = part_of_row<T>((const T*)p.logits + row * p.row_stride, 0, p.vocab, K, list + part_ring<T>() / 8, (unsigned char*)list, keys[i]);
        if (threadIdx.x == 0) sums[i] = sum;
        __syncthreads();
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int beam = block + warp * kMergeBlocks;
    if (beam < p.beams) {
        const double2 s = finished(beam) ? make_double2(0.0, 1.0) : sums[warp];
        const double lse = s.x + log(s.y);
        const bool counts = isfinite(p.scores[(long long)group * p.beams + beam]) && isfinite(lse);
        const int n = __popc(__ballot_sync(0xffffffffu, lane < K && keys[warp][lane] != 0));
        offer(p, shared, total, token, group, beam, finished(beam), counts, (float)s.x, lse, keys[warp], n);
    }
    cluster_sync();
    choose(p, shared, total, token, group, block);
}

// state[b] = old state[parents[b]] (-1: zeros; a row that is its own parent is not touched), for up to four tensors at once.  A thread owns a column of
// one unit of all rows, so nothing but its own order of reads and writes matters: a source that is itself overwritten is read first, into shared
// memory; the others are read once and written to all their children.  64 rows of 26 MB, 26 of them moved (1.06 GB): 179 us (5.9 TB/s); all rows through
// shared memory took 454.
struct ReorderParams {
    char* state[4]; long long row[4]; long long stride[4]; long long slices[5];
    const int* parents; unsigned int* status;
    int count, rows, held;                                    // tensors; sequences; bytes for rows that are read ahead
};
constexpr int kReorderThreads = 256, kReorderHeld = 24 * 1024, kReorderAtOnce = 4;
template <typename U>
__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const ReorderParams p) {
    grid_dependency_wait();            // without chain_enter(): kernels further on may fetch a state ahead of their own wait
    extern __shared__ __align__(16) unsigned char reorder_smem[];
    U* held = reinterpret_cast<U*>(reorder_smem);                                          // [source][thread]
    int* first = reinterpret_cast<int*>(reorder_smem + p.held);                      // [rows + 2]: of each source (the last: zeros) its first child's place
    int* child = first + p.rows + 2;                                                       // [rows]
    int* source = child + p.rows;                                                          // [rows]: sources with children: from the front those that stay, from the back the others
    __shared__ int stay, leave, sums[kReorderThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, S = p.rows;
    const auto parent_of = [&](int b) {
        const int parent = p.parents[b];
        if (parent >= -1 && parent < S) return parent < 0 ? S : parent;
        if (blockIdx.x == 0) atomicOr(p.status, QD_STATUS_BAD_ARG);
        return b;
    };
    for (int i = tid; i < S + 2; i += kReorderThreads) first[i] = 0;
    if (tid == 0) stay = leave = 0;
    __syncthreads();
    for (int b = tid; b < S; b += kReorderThreads) {
        const int parent = parent_of(b);
        if (parent != b) atomicAdd(first + parent + 1, 1);
    }
    __syncthreads();
    int before = 0;                                           // counts to places
    for (int base = 0; base < S + 2; base += kReorderThreads) {
        const int i = base + tid;
        int sum = i < S + 2 ? first[i] : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += up;
        }
        if (lane == 31) sums[warp] = sum;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < kReorderThreads / 32; ++w) { if (w < warp) sum += sums[w]; all += sums[w]; }
        if (i < S + 2) first[i] = before + sum;
        before += all;
        __syncthreads();
    }
    for (int b = tid; b < S; b += kReorderThreads) {
        const int parent = parent_of(b);
        if (parent != b) child[atomicAdd(first + parent, 1)] = b;           // (the order among the children changes nothing)
    }
    __syncthreads();
    for (int i = tid; i < S; i += kReorderThreads) {                        // first[i] is now the end of source i's children, first[i - 1] their start
        if (first[i] == (i ? first[i - 1] : 0)) continue;
        if (parent_of(i) == i) source[atomicAdd(&stay, 1)] = i;
        else source[S - 1 - atomicAdd(&leave, 1)] = i;
    }
    __syncthreads();
    const int stays = stay, leaves = leave, zeros = S ? first[S - 1] : 0, zeros_end = first[S];
    if (before == 0) return;
    const int room = p.held / (int)sizeof(U), columns = leaves == 0 || room / leaves >= kReorderThreads ? kReorderThreads : room / leaves;
    for (long long slice = blockIdx.x; slice < p.slices[p.count]; slice += gridDim.x) {
        int t = 0;
        while (slice >= p.slices[t + 1]) ++t;
        const long long units = p.row[t] / (long long)sizeof(U), from = (slice - p.slices[t]) * kReorderThreads;
        const auto at = [&](int b, long long unit) -> U* { return reinterpret_cast<U*>(p.state[t] + b * p.stride[t]) + unit; };
        for (int base = 0; base < kReorderThreads; base += columns) {      // (one round, unless many overwritten rows have to be held)
            const long long unit = from + base + tid;
            if (tid >= columns || base + tid >= kReorderThreads || unit >= units) continue;
            for (int i = 0; i < leaves; ++i) held[i * columns + tid] = *at(source[S - 1 - i], unit);
            for (int i = 0; i < stays; i += kReorderAtOnce) {
                U x[kReorderAtOnce];
#pragma unroll
                for (int j = 0; j < kReorderAtOnce; ++j)
                    if (i + j < stays) x[j] = *at(source[i + j], unit);
#pragma unroll
                for (int j = 0; j < kReorderAtOnce; ++j) {
                    if (i + j >= stays) continue;
                    const int who = source[i + j];
                    for (int c = who ? first[who - 1] : 0; c < first[who]; ++c) *at(child[c], unit) = x[j];
                }
            }
            for (int i = 0; i < leaves; ++i) {
                const int who = source[S - 1 - i];
                const U x = held[i * columns + tid];
                for (int c = who ? first[who - 1] : 0; c < first[who]; ++c) *at(child[c], unit) = x;
            }
            for (int c = zeros; c < zeros_end; ++c) *at(child[c], unit) = U{};
        }
    }
}

template <typename U>
int reorder_launch(const ReorderParams& p, dim3 grid, size_t smem, cudaStream_t stream) {
    static bool raised[kDevices];
    if (smem > 40 * 1024 && !raise_smem(reorder_kernel<U>, 200 * 1024, raised)) return QD_ERR_LAUNCH;        // (what is declared counts too)
    return qd_launch(reorder_kernel<U>, grid, dim3(kReorderThreads), smem, stream, 3, p);
}

template <typename T>
int short_launch(const SelectParams& p, size_t part, cudaStream_t stream) {
    const size_t smem = part + part_ring<T>() + (p.beams * p.candidates * 12 + 15) / 16 * 16;              // at most 47 KB, beside what is declared
    static bool raised[kDevices];
    if (smem > 40 * 1024 && !raise_smem(select_short_kernel<T>, 48 * 1024, raised)) return QD_ERR_LAUNCH;
    return qd_launch(select_short_kernel<T>, dim3(p.batch * kMergeBlocks), dim3(kMergeThreads), smem, stream, 3, p);
}

int splits_of(long long rows, int vocab) {
    const long long want = device_blocks() * 8ll / rows, most = vocab / 2048;
    const long long s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s > kMostSplits ? kMostSplits : s);
}

}  // namespace
}  // namespace qd

using namespace qd;

extern "C" long long qd_beam_scratch_bytes(int batch, int beams, int vocab, int candidates) {
    if (batch <= 0 || beams <= 0 || vocab <= kShortVocab || candidates <= 0) return 0;
    const long long rows = (long long)batch * beams;
    return rows * splits_of(rows, vocab) * (candidates * 8ll + 16);
}

extern "C" int qd_beam_select(const void* logits, long long row_stride, int is_fp32, const float* scores, const void* finished, int eos, float* scores_out,
                              int* parents_out, void* tokens_out, void* scratch, int batch, int beams, int vocab, int candidates, int placed, void* stream) {
    QD_CHECK_ARG(logits && scores && scores_out && parents_out && tokens_out && (scratch || vocab <= kShortVocab) && batch > 0 && beams > 0 && vocab > 0 && candidates > 0);
    QD_CHECK_ARG((long long)beams * vocab >= candidates && (!finished || (eos >= 0 && eos < vocab)) && (!placed || candidates == beams));
    QD_CHECK_ARG(((uintptr_t)scratch & 15u) == 0 && vocab <= 0x7fffffff - 4096);           // (a chunk's places are 32-bit numbers)
    if (beams > kMostBeams || candidates > kMostBeams || (long long)batch * beams > 65535) return QD_ERR_UNSUPPORTED;
    SelectParams p;
    const long long rows = (long long)batch * beams;
    p.logits = logits; p.row_stride = row_stride; p.scores = scores; p.finished = (const uint8_t*)finished;
    p.splits = splits_of(rows, vocab);
    p.sums = (double2*)scratch;
    p.keys = (unsigned long long*)(p.sums + rows * p.splits);
    p.scores_out = scores_out; p.parents_out = parents_out; p.tokens_out = (long long*)tokens_out;
    p.batch = batch; p.beams = beams; p.vocab = vocab; p.candidates = candidates; p.eos = eos; p.placed = placed; p.fp32 = is_fp32;
    if ((uintptr_t)logits % (is_fp32 ? 4 : 2)) return QD_ERR_UNSUPPORTED;
    const size_t part = part_bytes(candidates);
    const dim3 grid(p.splits, (unsigned)rows);
    const cudaStream_t on = (cudaStream_t)stream;
    if (vocab <= kShortVocab) return is_fp32 ? short_launch<float>(p, part, on) : short_launch<bf16>(p, part, on);
    const int code = is_fp32 ? qd_launch(select_part_kernel<float>, grid, dim3(kPartThreads), part + part_ring<float>(), on, 3, p)
                             : qd_launch(select_part_kernel<bf16>, grid, dim3(kPartThreads), part + part_ring<bf16>(), on, 3, p);
    if (code != QD_OK) return code;
    const int lists = p.splits < candidates ? p.splits : candidates;
    const size_t smem = 8ull * (beams * candidates + (beams * candidates + 1) / 2 + (size_t)(kMergeThreads / 32) * lists * candidates);       // at most 44 KB
    return qd_launch(select_merge_kernel, dim3(batch * kMergeBlocks), dim3(kMergeThreads), smem, on, 3, p);
}

extern "C" int qd_reorder_states(void* state0, long long row0, long long stride0, void* state1, long long row1, long long stride1, void* state2,
                                 long long row2, long long stride2, void* state3, long long row3, long long stride3, const int* parents,
                                 unsigned int* status, int sequences, void* stream) {
    QD_CHECK_ARG(parents && status && sequences > 0);
    ReorderParams p;
    void* const states[4] = {state0, state1, state2, state3};
    const long long rows[4] = {row0, row1, row2, row3}, strides[4] = {stride0, stride1, stride2, stride3};
    uintptr_t align = 0;
    p.count = 0;
    for (int i = 0; i < 4; ++i) {
        if (!states[i] || rows[i] == 0) continue;
        QD_CHECK_ARG(rows[i] > 0 && (sequences == 1 || strides[i] >= rows[i]));
        p.state[p.count] = (char*)states[i]; p.row[p.count] = rows[i]; p.stride[p.count] = strides[i];
        align |= (uintptr_t)states[i] | (uintptr_t)rows[i] | (uintptr_t)strides[i];
        ++p.count;
    }
    if (p.count == 0) return QD_OK;
    p.parents = parents; p.status = status; p.rows = sequences;
    const int unit = align % 16 == 0 ? 16 : align % 4 == 0 ? 4 : align % 2 == 0 ? 2 : 1;
    if (sequences > 7000) return QD_ERR_UNSUPPORTED;                         // (at least a column of every row is held)
    p.held = 16 * sequences > kReorderHeld ? 16 * sequences : kReorderHeld;
    const size_t smem = p.held + sizeof(int) * (3ull * sequences + 2);
    p.slices[0] = 0;
    for (int i = 0; i < p.count; ++i) p.slices[i + 1] = p.slices[i] + (p.row[i] / unit + kReorderThreads - 1) / kReorderThreads;
    const long long most = (long long)device_blocks() * (smem > 27 * 1024 ? 4 : 8);
    const dim3 grid((unsigned)(p.slices[p.count] < most ? p.slices[p.count] : most));
    const cudaStream_t on = (cudaStream_t)stream;
    return unit == 16 ? reorder_launch<uint4>(p, grid, smem, on) : unit == 4 ? reorder_launch<uint32_t>(p, grid, smem, on)
                      : unit == 2 ? reorder_launch<uint16_t>(p, grid, smem, on) : reorder_launch<uint8_t>(p, grid, smem, on);
}
