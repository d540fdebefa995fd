// Attention of one new token of every sequence over keys and values in pages:
//   out[b, h] = sum_p softmax_p(scale q[b, h] . k[p]) v[p],   row p of sequence b in pool[table[b][p / page]][p mod page],
// over the positions p that the sequence sees (all, or the first few and a window), times sigmoid(gate) where given.
#include "paged_fma.cuh"
#include "paged_mma.cuh"

namespace qd {
namespace {

// The means of a (sequence, head)'s parts joined, 32 * EACH columns by WARPS warps that take every WARPS-th part; a sequence that sees nothing gets zeros.
constexpr int kJoinWarps = 8;
template <typename T, int EACH, int WARPS>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const PagedParams p) {
    chain_enter();
    __shared__ float state[WARPS][EACH * 32 + 2];
    const int tid = threadIdx.x, warp = WARPS == 1 ? 0 : tid >> 5, lane = tid & 31, each = p.kv_heads * p.chunks, column = blockIdx.y * EACH * 32 + lane;
    const int row = WARPS == 1 ? (int)blockIdx.x * kJoinWarps + (tid >> 5) : (int)blockIdx.x;
    if (row >= p.batch * p.heads) return;
    const int b = row / p.heads, head = row - b * p.heads, kvh = head / p.group, in = head - kvh * p.group;
    const long long place = ((long long)b * each + kvh * p.chunks + in / p.chunk) * p.cuts.most * p.chunk + in % p.chunk;
    const float* src = p.partial + place * p.dim + column;
    // (read while the length is on its way; what lies behind the last part is not used)
    int mine = warp + lane * WARPS;                                    // a lane's part
    float2 of = mine < p.cuts.most ? p.stats[place + (long long)mine * p.chunk] : make_float2(0.f, 0.f);
    const int parts = paged_parts(p.cuts, paged_span(p, b).seen, p.unit);
    float top = -INFINITY, den = 0.f, mean[EACH] = {};
    for (int base = warp; base < parts; base += 32 * WARPS) {
        if (base != warp) of = mine < parts ? p.stats[place + (long long)mine * p.chunk] : of;
        if (mine >= parts) of = make_float2(-INFINITY, 0.f);
        const float now = fmaxf(top, warp_max(of.x)), shift = now == -INFINITY ? 0.f : now;
        const float w = of.y == 0.f ? 0.f : exp2f(of.x - shift) * of.y, before = den * exp2f(top - shift);
        top = now;
        den = before + warp_sum(w);
        const float inverse = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
        for (int j = 0; j < EACH; ++j) mean[j] *= before * inverse;
        const int count = min(32, (parts - base + WARPS - 1) / WARPS);
#pragma unroll (EACH > 2 ? 2 : 16)
        for (int i = 0; i < count; ++i) {
            const float share = __shfl_sync(0xffffffffu, w * inverse, i);
            const float* from = src + (long long)(base + i * WARPS) * p.chunk * p.dim;
#pragma unroll
            for (int j = 0; j < EACH; ++j)
                if (column + j * 32 < p.dim) mean[j] += share * from[j * 32];
        }
        mine += 32 * WARPS;
    }
    if constexpr (WARPS == 1) {
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            if (column + j * 32 < p.dim) paged_put<T>(p, b, head, column + j * 32, mean[j]);
    } else {
#pragma unroll
    for (int j = 0; j < EACH; ++j) state[warp][j * 32 + lane] = mean[j];
    if (lane == 0) { state[warp][EACH * 32] = top; state[warp][EACH * 32 + 1] = den; }
    __syncthreads();
    const int f = blockIdx.y * EACH * 32 + tid;
    if (tid >= EACH * 32 || f >= p.dim) return;
    float all = -INFINITY, sum = 0.f, v = 0.f, share[WARPS];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) all = fmaxf(all, state[w][EACH * 32]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        const float of_w = state[w][EACH * 32 + 1];
        share[w] = of_w == 0.f ? 0.f : exp2f(state[w][EACH * 32] - all) * of_w;
        sum += share[w];
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += share[w] * inverse * state[w][tid];
    paged_put<T>(p, b, head, f, v);
    }
}

// Query heads at a time.
int chunk_of(int group, bool fp32) {
    const int most = fp32 || group <= 8 ? 8 : 16;
    return group < most ? group : most;
}
// The work on a tile for a head dimension, a type and a number of heads at a time: go(Work).
template <typename Go>
auto with_work(int dim, int chunk, bool fp32, const Go& go) {
    if (fp32)
        return chunk <= 4 ? dim <= 64 ? go((PagedFma<64, 4>*)nullptr) : dim <= 128 ? go((PagedFma<128, 4>*)nullptr) : go((PagedFma<256, 4>*)nullptr)
                          : dim <= 64 ? go((PagedFma<64, 8>*)nullptr) : dim <= 128 ? go((PagedFma<128, 8>*)nullptr) : go((PagedFma<256, 8>*)nullptr);
    return chunk <= 8 ? dim <= 64 ? go((PagedMma<64, 1>*)nullptr) : dim <= 128 ? go((PagedMma<128, 1>*)nullptr) : go((PagedMma<256, 1>*)nullptr)
                      : dim <= 64 ? go((PagedMma<64, 2>*)nullptr) : dim <= 128 ? go((PagedMma<128, 2>*)nullptr) : go((PagedMma<256, 2>*)nullptr);
}
struct Plan { int seqs, workers, unit; };          // sequences of a launch, groups of warps that take parts, positions of a unit
Plan plan_of(int dim, int chunk, bool fp32) {
    return with_work(dim, chunk, fp32, [](auto* work) {
        using W = std::remove_pointer_t<decltype(work)>;
        return Plan{W::kSeqs, device_blocks() * PagedTiles<W>::kGroups, PagedTiles<W>::kStride};
    });
}
template <class W>
int tiles_launch(const PagedParams& p, cudaStream_t stream) {
    constexpr int kSmem = PagedTiles<W>::kSmem;
    static bool raised[kDevices];
    if (!raise_smem(paged_tiles_kernel<W>, kSmem, raised)) return QD_ERR_LAUNCH;
    return qd_launch(paged_tiles_kernel<W>, dim3(device_blocks()), dim3(PagedTiles<W>::kThreads), kSmem, stream, 3, p);
}

// By the number of rows: 32 columns of a row a block, a row a block, a row a warp.
template <typename T>
int join_launch(const PagedParams& p, int blocks, cudaStream_t stream) {
    const int rows = p.heads * p.batch;
    if (2 * rows <= blocks) return qd_launch(paged_join_kernel<T, 1, kJoinWarps>, dim3(rows, (p.dim + 31) / 32), dim3(kJoinWarps * 32), 0, stream, 3, p);
    if (rows <= 4 * blocks) return qd_launch(paged_join_kernel<T, 8, kJoinWarps>, dim3(rows), dim3(kJoinWarps * 32), 0, stream, 3, p);
    return qd_launch(paged_join_kernel<T, 8, 1>, dim3((rows + kJoinWarps - 1) / kJoinWarps), dim3(kJoinWarps * 32), 0, stream, 3, p);
}
int paged_launch(const PagedParams& p, bool fp32, cudaStream_t stream) {
    const int code = with_work(p.dim, p.chunk, fp32, [&](auto* work) { return tiles_launch<std::remove_pointer_t<decltype(work)>>(p, stream); });
    if (code != QD_OK || p.cuts.most == 0) return code;
    return fp32 ? join_launch<float>(p, device_blocks(), stream) : join_launch<bf16>(p, device_blocks(), stream);
}

}  // namespace
}  // namespace qd

using namespace qd;

extern "C" long long qd_paged_attention_floats(int batch, int heads, int kv_heads, int dim, int positions) {
    if (positions < 0 || batch <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || dim <= 0) return 0;
    const int group = heads / kv_heads;
    long long most = 0;
    for (int fp32 = 0; fp32 < 2; ++fp32) {
        const int chunk = chunk_of(group, fp32), chunks = (group + chunk - 1) / chunk;
        const Plan plan = plan_of(dim, chunk, fp32);
        for (const int some : {batch < plan.seqs ? batch : plan.seqs, batch % plan.seqs}) {          // whole launches and the last one
            if (!some) continue;
            const long long pairs = (long long)some * kv_heads * chunks, floats = pairs * paged_cuts(pairs, plan.workers, (positions - 1ll) / plan.unit + 1).most * chunk * (dim + 2);
            if (floats > most) most = floats;
        }
    }
    return most;
}

extern "C" int qd_paged_attention(const void* q, long long q_row, long long q_head, const void* k, const void* v, long long page_stride,
                                  long long row_stride, long long head_stride, const int* table, long long table_stride, const int* lengths,
                                  const void* gate, long long gate_row, long long gate_head, void* out, float* partial, int batch, int heads,
                                  int kv_heads, int dim, int pages, int page, int width, int window, int sinks, float scale, int is_fp32, void* stream) {
    QD_CHECK_ARG(q && k && v && table && lengths && out);
    QD_CHECK_ARG(batch > 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && dim > 0 && pages > 0 && page > 0 && width > 0);
    QD_CHECK_ARG(window >= 0 && sinks >= 0 && (window > 0 || sinks == 0) && (long long)width * page <= 0x7fffffffll - 4096 && heads <= 65535);
    if (dim > 256 || dim % 8) return QD_ERR_UNSUPPORTED;
    PagedParams p;
    p.q_row = q_row; p.q_head = q_head; p.gate_row = gate_row; p.gate_head = gate_head;
    p.page_stride = page_stride; p.row_stride = row_stride; p.head_stride = head_stride; p.table_stride = table_stride;
    p.k = k; p.v = v; p.partial = partial;
    p.heads = heads; p.kv_heads = kv_heads; p.dim = dim; p.pages = pages; p.page = page; p.width = width;
    const bool all = (long long)window + sinks >= (long long)width * page;      // (their sum fits 32 bits otherwise)
    p.window = all ? 0 : window; p.sinks = all ? 0 : sinks;
    p.group = heads / kv_heads; p.chunk = chunk_of(p.group, is_fp32); p.chunks = (p.group + p.chunk - 1) / p.chunk;
    const Plan plan = plan_of(dim, p.chunk, is_fp32);
    p.unit = plan.unit; p.scale = scale * 1.4426950408889634f;
    const int size = is_fp32 ? 4 : 2;
    p.q_whole = !(((uintptr_t)q | (uintptr_t)(q_row * size) | (uintptr_t)(q_head * size)) & 15u);
    if (((uintptr_t)partial | (uintptr_t)k | (uintptr_t)v | (uintptr_t)(page_stride * size) | (uintptr_t)(row_stride * size) | (uintptr_t)(head_stride * size)) & 15u) return QD_ERR_UNSUPPORTED;
    for (int b = 0; b < batch; b += plan.seqs) {                 // (the scratch is used again in stream order)
        p.batch = batch - b < plan.seqs ? batch - b : plan.seqs;
        const long long pairs = (long long)p.batch * kv_heads * p.chunks;
        p.cuts = paged_cuts(pairs, plan.workers, ((p.window ? (long long)p.window + p.sinks : (long long)width * page) - 1) / plan.unit + 1);
        QD_CHECK_ARG(partial || p.cuts.most == 0);
        p.stats = (float2*)(p.partial + pairs * p.cuts.most * p.chunk * dim);
        p.q = (const char*)q + b * q_row * size;
        p.gate = gate ? (const char*)gate + b * gate_row * size : nullptr;
        p.out = (char*)out + (long long)b * heads * dim * size;
        p.table = table + b * table_stride; p.lengths = lengths + b;
        const int code = paged_launch(p, is_fp32 != 0, (cudaStream_t)stream);
        if (code != QD_OK) return code;
    }
    return QD_OK;
}
