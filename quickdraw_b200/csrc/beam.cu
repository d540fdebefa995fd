// Beam search: the best continuations of every group of beams, and the beams' states put in the order of their parents.
//
// A continuation of beam i by token v counts score[i] + x[i, v] - log sum_w exp x[i, w].  Within a beam the order is that of the logits, so a first
// kernel takes, of each piece of a row, the largest logits, the maximum and the sum of exponentials, and a second one joins the pieces, adds up in 64
// bits (sums of different beams lie next to one another) and merges the beams.
#include "common.cuh"

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
QD_DEVINL unsigned long long warp_most(unsigned long long k) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, d);
        k = other > k ? other : k;
    }
    return k;
}

template <typename T> QD_DEVINL float logit_of(T v);
template <> QD_DEVINL float logit_of<float>(float v) { return v; }
template <> QD_DEVINL float logit_of<bf16>(bf16 v) { return __bfloat162float(v); }

struct SelectParams {
    const void* logits; long long row_stride;                 // elements from a row to the next
    const float* scores; const uint8_t* finished;
    unsigned long long* keys;                                 // [row][split][candidates], descending; 0: none
    float2* sums;                                             // [row][split]: maximum, sum of exp(x - maximum)
    float* scores_out; int* parents_out; long long* tokens_out;
    int batch, beams, vocab, candidates, splits, eos, placed;
};

constexpr int kPartThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kPartThreads) select_part_kernel(const SelectParams p) {
    chain_enter();
    __shared__ float red[kPartThreads / 32];
    __shared__ unsigned long long best[kPartThreads / 32];
    const int row = blockIdx.y, split = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (p.finished && p.finished[row]) return;
    const T* x = (const T*)p.logits + row * p.row_stride;
    const int lo = (int)((long long)p.vocab * split / p.splits), hi = (int)((long long)p.vocab * (split + 1) / p.splits);
    float top = -INFINITY, sum = 0.f;
    for (int i = lo + tid; i < hi; i += kPartThreads) top = fmaxf(top, logit_of(x[i]));
    top = warp_max(top);
    if (lane == 0) red[warp] = top;
    __syncthreads();
    for (int w = 0; w < kPartThreads / 32; ++w) top = fmaxf(top, red[w]);
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kPartThreads) {
        const float v = logit_of(x[i]);
        sum += v == -INFINITY ? 0.f : expf(v - top);          // (NaN and infinity go on)
    }
    sum = warp_sum(sum);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        float all = 0.f;
        for (int w = 0; w < kPartThreads / 32; ++w) all += red[w];
        p.sums[(long long)row * p.splits + split] = make_float2(top, all);
    }
    unsigned long long last = ~0ull, *keys = p.keys + ((long long)row * p.splits + split) * p.candidates;
    for (int k = 0; k < p.candidates; ++k) {
        unsigned long long mine = 0;
        for (int i = lo + tid; i < hi; i += kPartThreads) {
            const unsigned long long key = logit_key(logit_of(x[i]), i);
            if (key < last && key > mine) mine = key;
        }
        mine = warp_most(mine);
        __syncthreads();
        if (lane == 0) best[warp] = mine;
        __syncthreads();
        for (int w = 0; w < kPartThreads / 32; ++w) mine = best[w] > mine ? best[w] : mine;
        last = mine;
        if (tid == 0) keys[k] = mine;
    }
}

// A block per group: a warp joins a beam's pieces, then one warp merges the beams, a lane each.
constexpr int kMergeWarps = 8;
__global__ void __launch_bounds__(kMergeWarps * 32) select_merge_kernel(const SelectParams p) {
    chain_enter();
    extern __shared__ __align__(16) unsigned char merge_smem[];
    const int group = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = p.candidates;
    double* total = reinterpret_cast<double*>(merge_smem);                                  // [beams][K], descending
    unsigned long long* lists = reinterpret_cast<unsigned long long*>(total + p.beams * K) + (size_t)warp * p.splits * K;
    int* token = reinterpret_cast<int*>(reinterpret_cast<unsigned long long*>(total + p.beams * K) + (size_t)kMergeWarps * p.splits * K);   // -1: none
    for (int i = warp; i < p.beams; i += kMergeWarps) {
        const long long row = (long long)group * p.beams + i;
        const float score = p.scores[row];
        const bool done = p.finished && p.finished[row];
        double lse = 0.0;
        bool counts = isfinite(score);
        if (!done) {
            const float2 s = lane < p.splits ? p.sums[row * p.splits + lane] : make_float2(-INFINITY, 0.f);
            const float top = warp_max(s.x);
            const bool odd = __any_sync(0xffffffffu, lane < p.splits && (s.x != s.x || s.y != s.y));
            double sum = s.y == 0.f ? 0.0 : (double)s.y * exp((double)s.x - (double)top);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            lse = (double)top + log(sum);
            counts = counts && !odd && isfinite(lse);
        }
        if (done || !counts) {
            // the end at no cost, and what never follows, in the order of the tokens
            for (int k = lane; k < K; k += 32) {
                int t = k;
                double v = -INFINITY;
                if (done && counts) {
                    t = k == 0 ? p.eos : k - 1 + (k - 1 >= p.eos);
                    if (k == 0) v = score;
                }
                total[i * K + k] = v;
                token[i * K + k] = t < p.vocab ? t : -1;
            }
            continue;
        }
        for (int k = lane; k < p.splits * K; k += 32) lists[k] = p.keys[row * p.splits * K + k];
        __syncwarp();
        int at = 0;
        unsigned long long head = lane < p.splits ? lists[lane * K] : 0;
        for (int k = 0; k < K; ++k) {
            const unsigned long long most = warp_most(head);
            if (lane == 0) {
                total[i * K + k] = (double)score + ((double)key_logit(most) - lse);
                token[i * K + k] = most ? key_index(most) : -1;
            }
            if (most && head == most) { ++at; head = at < K ? lists[lane * K + at] : 0; }
        }
        __syncwarp();
    }
    __syncthreads();
    if (warp) return;
    int at = 0, parent = 0, chosen = 0;
    double best = 0.0;
    for (int k = 0; k < K; ++k) {
        const bool has = lane < p.beams && at < K && token[lane * K + at] >= 0;
        const double mine = has ? total[lane * K + at] : 0.0;
        double v = mine;
        int who = has ? lane : 32;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const double ov = __shfl_xor_sync(0xffffffffu, v, d);
            const int ow = __shfl_xor_sync(0xffffffffu, who, d);
            if (ow < 32 && (who == 32 || ov > v || (ov == v && ow < who))) { v = ov; who = ow; }
        }
        const int t = __shfl_sync(0xffffffffu, has ? token[lane * K + at] : 0, who & 31);
        if (lane == who) ++at;
        if (lane == k) { best = v; parent = who & 31; chosen = t; }
    }
    int place = lane;
    if (p.placed) {
        // a beam's best continuation takes the beam's place, the others the places left, in order
        const unsigned active = __ballot_sync(0xffffffffu, lane < K);
        const unsigned same = __match_any_sync(0xffffffffu, lane < K ? parent : 64 + lane);
        const bool leads = lane < K && (same & ((1u << lane) - 1u)) == 0;
        const unsigned taken = __reduce_or_sync(0xffffffffu, leads ? 1u << parent : 0u);
        const unsigned rest = __ballot_sync(0xffffffffu, lane < K && !leads);
        (void)active;
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
        p.scores_out[o] = (float)best;
        p.parents_out[o] = group * p.beams + parent;
        p.tokens_out[o] = chosen;
    }
}

// state[b] = old state[parents[b]] (-1: zeros; a row that is its own parent is not touched), for up to four tensors at once.  A block takes a column
// of some bytes of all rows: it loads the rows that others copy, then writes, so that no row is read after it is overwritten.
struct ReorderParams {
    char* state[4]; long long row[4]; long long stride[4]; long long slices[5];
    const int* parents; unsigned int* status;
    int count, rows, width;                                   // tensors; sequences; units of a slice
};
template <typename U>
__global__ void __launch_bounds__(256) reorder_kernel(const ReorderParams p) {
    grid_dependency_wait();            // without chain_enter(): kernels further on may fetch a state ahead of their own wait
    extern __shared__ __align__(16) unsigned char reorder_smem[];
    U* held = reinterpret_cast<U*>(reorder_smem);                                          // [rows][width]
    int* parents = reinterpret_cast<int*>(held + (size_t)p.rows * p.width);                // itself: not moved
    int* needed = parents + p.rows;
    const int tid = threadIdx.x;
    for (int b = tid; b < p.rows; b += blockDim.x) {
        int parent = p.parents[b];
        if (parent < -1 || parent >= p.rows) { if (blockIdx.x == 0) atomicOr(p.status, QD_STATUS_BAD_ARG); parent = b; }
        parents[b] = parent;
        needed[b] = 0;
    }
    __syncthreads();
    for (int b = tid; b < p.rows; b += blockDim.x)
        if (parents[b] >= 0 && parents[b] != b) needed[parents[b]] = 1;
    for (long long slice = blockIdx.x; slice < p.slices[p.count]; slice += gridDim.x) {
        int t = 0;
        while (slice >= p.slices[t + 1]) ++t;
        const long long first = (slice - p.slices[t]) * p.width, left = p.row[t] / (long long)sizeof(U) - first;
        const int wide = (int)(left < p.width ? left : p.width);
        __syncthreads();
        for (int i = tid; i < p.rows * p.width; i += blockDim.x) {
            const int b = i / p.width, c = i - b * p.width;
            if (c < wide && needed[b]) held[i] = reinterpret_cast<const U*>(p.state[t] + b * p.stride[t])[first + c];
        }
        __syncthreads();
        for (int i = tid; i < p.rows * p.width; i += blockDim.x) {
            const int b = i / p.width, c = i - b * p.width, parent = parents[b];
            if (c < wide && parent != b) reinterpret_cast<U*>(p.state[t] + b * p.stride[t])[first + c] = parent < 0 ? U{} : held[parent * p.width + c];
        }
    }
}

template <typename U>
int reorder_launch(const ReorderParams& p, dim3 grid, size_t smem, cudaStream_t stream) {
    if (smem > 48 * 1024 && cudaFuncSetAttribute(reorder_kernel<U>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != cudaSuccess) return QD_ERR_LAUNCH;
    return qd_launch(reorder_kernel<U>, grid, dim3(256), smem, stream, 3, p);
}

int beam_sms() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms > 0 ? sms : 148;
}
int splits_of(long long rows, int vocab) {
    const long long want = beam_sms() / rows, most = vocab / 2048;
    const long long s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s > kMostSplits ? kMostSplits : s);
}

}  // namespace
}  // namespace qd

using namespace qd;

extern "C" long long qd_beam_scratch_bytes(int batch, int beams, int vocab, int candidates) {
    if (batch <= 0 || beams <= 0 || vocab <= 0 || candidates <= 0) return 0;
    const long long rows = (long long)batch * beams;
    return rows * splits_of(rows, vocab) * (candidates * 8ll + 8);
}

extern "C" int qd_beam_select(const void* logits, long long row_stride, int is_fp32, const float* scores, const void* finished, int eos, float* scores_out,
                              int* parents_out, void* tokens_out, void* scratch, int batch, int beams, int vocab, int candidates, int placed, void* stream) {
    QD_CHECK_ARG(logits && scores && scores_out && parents_out && tokens_out && scratch && batch > 0 && beams > 0 && vocab > 0 && candidates > 0);
    QD_CHECK_ARG((long long)beams * vocab >= candidates && (!finished || (eos >= 0 && eos < vocab)) && (!placed || candidates == beams));
    QD_CHECK_ARG(((uintptr_t)scratch & 7u) == 0);
    if (beams > kMostBeams || candidates > kMostBeams || (long long)batch * beams > 65535) return QD_ERR_UNSUPPORTED;
    SelectParams p;
    const long long rows = (long long)batch * beams;
    p.logits = logits; p.row_stride = row_stride; p.scores = scores; p.finished = (const uint8_t*)finished;
    p.splits = splits_of(rows, vocab);
    p.keys = (unsigned long long*)scratch;
    p.sums = (float2*)(p.keys + rows * p.splits * candidates);
    p.scores_out = scores_out; p.parents_out = parents_out; p.tokens_out = (long long*)tokens_out;
    p.batch = batch; p.beams = beams; p.vocab = vocab; p.candidates = candidates; p.eos = eos; p.placed = placed;
    int code = is_fp32 ? qd_launch(select_part_kernel<float>, dim3(p.splits, (unsigned)rows), dim3(kPartThreads), 0, (cudaStream_t)stream, 3, p)
                       : qd_launch(select_part_kernel<bf16>, dim3(p.splits, (unsigned)rows), dim3(kPartThreads), 0, (cudaStream_t)stream, 3, p);
    if (code != QD_OK) return code;
    const size_t smem = (size_t)beams * candidates * 12 + (size_t)kMergeWarps * p.splits * candidates * 8;
    if (smem > 48 * 1024 && cudaFuncSetAttribute(select_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024) != cudaSuccess) return QD_ERR_LAUNCH;
    return qd_launch(select_merge_kernel, dim3(batch), dim3(kMergeWarps * 32), smem, (cudaStream_t)stream, 3, p);
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
    const long long room = 160 * 1024 - 8ll * sequences, width = room / ((long long)sequences * unit);
    if (width < 1) return QD_ERR_UNSUPPORTED;
    p.width = (int)(width < 512 / unit ? width : 512 / unit);
    p.slices[0] = 0;
    for (int i = 0; i < p.count; ++i) p.slices[i + 1] = p.slices[i] + (p.row[i] / unit + p.width - 1) / p.width;
    const size_t smem = (size_t)sequences * p.width * unit + 8ull * sequences;
    const long long most = (long long)beam_sms() * 8;
    const dim3 grid((unsigned)(p.slices[p.count] < most ? p.slices[p.count] : most));
    const cudaStream_t on = (cudaStream_t)stream;
    return unit == 16 ? reorder_launch<uint4>(p, grid, smem, on) : unit == 4 ? reorder_launch<uint32_t>(p, grid, smem, on)
                      : unit == 2 ? reorder_launch<uint16_t>(p, grid, smem, on) : reorder_launch<uint8_t>(p, grid, smem, on);
}
