// Attention of one new token of every sequence over keys and values in pages:
//   out[b, h] = sum_p softmax_p(scale q[b, h] . k[p]) v[p],   row p of sequence b in pool[table[b][p / page]][p mod page],
// over the positions p that the sequence sees (all, or the first few and a window), times sigmoid(gate) where given.
#include "paged.cuh"

#include <type_traits>

namespace qd {
namespace {

template <typename T> QD_DEVINL float paged_load(const T* p) { return (float)*p; }
template <> QD_DEVINL float paged_load<bf16>(const bf16* p) { return __bfloat162float(*p); }
template <typename T> QD_DEVINL void paged_store(T* p, float v);
template <> QD_DEVINL void paged_store<float>(float* p, float v) { *p = v; }
template <> QD_DEVINL void paged_store<bf16>(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int kSeqs = 1024;             // sequences of a launch

// The sequences' parts, in front of one another: before[b] pieces (a part of a pair each) belong to the sequences below b.
template <int THREADS>
QD_DEVINL int paged_schedule(const PagedParams& p, int* before) {
    __shared__ int sums[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = p.kv_heads * p.chunks;
    int total = 0;
    for (int base = 0; base < p.batch; base += THREADS) {
        const int b = base + tid;
        int sum = b < p.batch ? each * paged_parts(paged_span(p, b).seen, p.unit, (long long)p.batch * each, (int)gridDim.x) : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += up;
        }
        if (lane == 31) sums[warp] = sum;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < THREADS / 32; ++w) { if (w < warp) sum += sums[w]; all += sums[w]; }
        if (b < p.batch) before[b + 1] = total + sum;
        total += all;
        __syncthreads();
    }
    if (tid == 0) before[0] = 0;
    __syncthreads();
    return total;
}

struct Piece { int b, kvh, head0, heads, t0, t1, skip, part, parts; long long pair; };
QD_DEVINL Piece paged_piece(const PagedParams& p, const int* before, int r) {
    int lo = 0;
    for (int hi = p.batch; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= r) lo = mid; else hi = mid;
    }
    Piece a;
    const int each = p.kv_heads * p.chunks;
    const Span s = paged_span(p, lo);
    a.b = lo;
    a.parts = (before[lo + 1] - before[lo]) / each;
    const int at = r - before[lo], pair = at / a.parts, units = (s.seen + p.unit - 1) / p.unit;
    a.part = at - pair * a.parts;
    a.kvh = pair / p.chunks;
    const int chunk = pair - a.kvh * p.chunks;
    a.head0 = a.kvh * p.group + chunk * p.chunk;
    a.heads = min(p.chunk, p.group - chunk * p.chunk);
    a.pair = (long long)lo * each + pair;
    a.t0 = min(s.seen, (int)((long long)units * a.part / a.parts) * p.unit);
    a.t1 = min(s.seen, (int)((long long)units * (a.part + 1) / a.parts) * p.unit);
    a.skip = s.skip;
    return a;
}

template <typename T>
QD_DEVINL void paged_put(const PagedParams& p, int b, int head, int f, float v) {
    if (p.gate) v *= sigmoid_precise(paged_load((const T*)p.gate + b * p.gate_row + head * p.gate_head + f));
    paged_store((T*)p.out + ((long long)b * p.heads + head) * p.dim + f, v);
}

// A warp per position, a lane for every 32nd feature, fp32 sums.
constexpr int kPlainWarps = 8, kPlainHeads = 8;
template <typename T>
__global__ void __launch_bounds__(kPlainWarps * 32) paged_plain_kernel(const PagedParams p) {
    chain_enter();
    extern __shared__ __align__(16) float plain_smem[];                // [warps][heads][dim + 2]
    __shared__ int before[kSeqs + 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, stride = p.dim + 2;
    const int total = paged_schedule<kPlainWarps * 32>(p, before);
    for (int r = blockIdx.x; r < total; r += gridDim.x) {
        const Piece a = paged_piece(p, before, r);
        float q[kPlainHeads][8], acc[kPlainHeads][8], m[kPlainHeads], l[kPlainHeads];
#pragma unroll
        for (int h = 0; h < kPlainHeads; ++h) {
            m[h] = -INFINITY; l[h] = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int f = j * 32 + lane;
                acc[h][j] = 0.f;
                q[h][j] = h < a.heads && f < p.dim ? paged_load((const T*)p.q + a.b * p.q_row + (a.head0 + h) * p.q_head + f) : 0.f;
            }
        }
        for (int i = a.t0 + warp; i < a.t1; i += kPlainWarps) {
            const int position = paged_position(p, i, a.skip), page = p.table[a.b * p.table_stride + position / p.page];
            if (page < 0 || page >= p.pages) continue;
            const long long at = page * p.page_stride + position % p.page * p.row_stride + a.kvh * p.head_stride;
            float k[8], v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int f = j * 32 + lane;
                k[j] = f < p.dim ? paged_load((const T*)p.k + at + f) : 0.f;
                v[j] = f < p.dim ? paged_load((const T*)p.v + at + f) : 0.f;
            }
#pragma unroll
            for (int h = 0; h < kPlainHeads; ++h) {
                float dot = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) dot += q[h][j] * k[j];
                const float s = warp_sum(dot) * p.scale, top = fmaxf(m[h], s);
                const float fix = m[h] == -INFINITY ? 0.f : exp2f(m[h] - top), w = s == -INFINITY ? 0.f : exp2f(s - top);
                l[h] = l[h] * fix + w;
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[h][j] = acc[h][j] * fix + w * v[j];
                m[h] = top;
            }
        }
#pragma unroll
        for (int h = 0; h < kPlainHeads; ++h) {
            float* dst = plain_smem + (warp * kPlainHeads + h) * stride;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j * 32 + lane < p.dim) dst[j * 32 + lane] = acc[h][j];
            if (lane == 0) { dst[p.dim] = m[h]; dst[p.dim + 1] = l[h]; }
        }
        __syncthreads();
        for (int i = tid; i < a.heads * p.dim; i += kPlainWarps * 32) {
            const int h = i / p.dim, f = i % p.dim;
            float top = -INFINITY, num = 0.f, den = 0.f;
            for (int w = 0; w < kPlainWarps; ++w) top = fmaxf(top, plain_smem[(w * kPlainHeads + h) * stride + p.dim]);
            for (int w = 0; w < kPlainWarps; ++w) {
                const float* src = plain_smem + (w * kPlainHeads + h) * stride;
                const float g = src[p.dim + 1] == 0.f ? 0.f : exp2f(src[p.dim] - top);
                num += g * src[f];
                den += g * src[p.dim + 1];
            }
            if (a.parts == 1) paged_put<T>(p, a.b, a.head0 + h, f, den == 0.f ? 0.f : num / den);
            else {
                float* dst = p.partial + ((a.pair * p.most + a.part) * p.chunk + h) * stride;
                dst[f] = num;
                if (f == 0) { dst[p.dim] = top; dst[p.dim + 1] = den; }
            }
        }
        __syncthreads();
    }
}

// The parts of a (sequence, head) joined; a sequence that sees nothing gets zeros.
template <typename T>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedParams p, int blocks) {
    chain_enter();
    const int head = blockIdx.x, b = blockIdx.y, each = p.kv_heads * p.chunks;
    const int parts = paged_parts(paged_span(p, b).seen, p.unit, (long long)p.batch * each, blocks);
    if (parts == 1) return;
    const int kvh = head / p.group, in = head - kvh * p.group, stride = p.dim + 2;
    const long long pair = (long long)b * each + kvh * p.chunks + in / p.chunk;
    const float* src = p.partial + (pair * p.most * p.chunk + in % p.chunk) * stride;
    const long long step = (long long)p.chunk * stride;
    for (int f = threadIdx.x; f < p.dim; f += blockDim.x) {
        float top = -INFINITY, num = 0.f, den = 0.f;
        for (int i = 0; i < parts; ++i) top = fmaxf(top, src[i * step + p.dim]);
        for (int i = 0; i < parts; ++i) {
            const float g = src[i * step + p.dim + 1] == 0.f ? 0.f : exp2f(src[i * step + p.dim] - top);
            num += g * src[i * step + f];
            den += g * src[i * step + p.dim + 1];
        }
        paged_put<T>(p, b, head, f, den == 0.f ? 0.f : num / den);
    }
}

int paged_blocks() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms > 0 ? sms : 148;
}
int chunk_of(int group) { return group < kPlainHeads ? group : kPlainHeads; }

template <typename T>
int paged_launch(PagedParams p, cudaStream_t stream) {
    const int blocks = paged_blocks();
    const size_t smem = sizeof(float) * kPlainWarps * kPlainHeads * (p.dim + 2);
    if (cudaFuncSetAttribute(paged_plain_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 72 * 1024) != cudaSuccess) return QD_ERR_LAUNCH;
    int code = qd_launch(paged_plain_kernel<T>, dim3(blocks), dim3(kPlainWarps * 32), smem, stream, 3, p);
    if (code == QD_OK) code = qd_launch(paged_join_kernel<T>, dim3(p.heads, p.batch), dim3(p.dim < 256 ? (p.dim + 31) / 32 * 32 : 256), 0, stream, 3, p, blocks);
    return code;
}

}  // namespace
}  // namespace qd

using namespace qd;

extern "C" long long qd_paged_attention_floats(int batch, int heads, int kv_heads, int dim) {
    if (batch <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || dim <= 0) return 0;
    const int group = heads / kv_heads, chunk = chunk_of(group), chunks = (group + chunk - 1) / chunk, few = batch < kSeqs ? batch : kSeqs;
    const long long pairs = (long long)few * kv_heads * chunks, rest = (long long)(batch % kSeqs) * kv_heads * chunks;
    const int blocks = paged_blocks();
    const long long whole = pairs * paged_most(pairs, blocks), last = batch > kSeqs && rest ? rest * paged_most(rest, blocks) : 0;
    return (whole > last ? whole : last) * chunk * (dim + 2);
}

extern "C" int qd_paged_attention(const void* q, long long q_row, long long q_head, const void* k, const void* v, long long page_stride,
                                  long long row_stride, long long head_stride, const int* table, long long table_stride, const int* lengths,
                                  const void* gate, long long gate_row, long long gate_head, void* out, float* partial, int batch, int heads,
                                  int kv_heads, int dim, int pages, int page, int width, int window, int sinks, float scale, int is_fp32, void* stream) {
    QD_CHECK_ARG(q && k && v && table && lengths && out && partial);
    QD_CHECK_ARG(batch > 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && dim > 0 && pages > 0 && page > 0 && width > 0);
    QD_CHECK_ARG(window >= 0 && sinks >= 0 && (window > 0 || sinks == 0) && (long long)width * page <= 0x7fffffffll - 4096 && heads <= 65535);
    if (dim > 256 || dim % 8) return QD_ERR_UNSUPPORTED;
    PagedParams p;
    p.q_row = q_row; p.q_head = q_head; p.gate_row = gate_row; p.gate_head = gate_head;
    p.page_stride = page_stride; p.row_stride = row_stride; p.head_stride = head_stride; p.table_stride = table_stride;
    p.k = k; p.v = v; p.partial = partial;
    p.heads = heads; p.kv_heads = kv_heads; p.dim = dim; p.pages = pages; p.page = page; p.width = width; p.window = window; p.sinks = sinks;
    p.group = heads / kv_heads; p.chunk = chunk_of(p.group); p.chunks = (p.group + p.chunk - 1) / p.chunk;
    p.unit = 32; p.scale = scale * 1.4426950408889634f;
    const int size = is_fp32 ? 4 : 2;
    for (int b = 0; b < batch; b += kSeqs) {                 // (the scratch is used again in stream order)
        p.batch = batch - b < kSeqs ? batch - b : kSeqs;
        p.most = paged_most((long long)p.batch * kv_heads * p.chunks, paged_blocks());
        p.q = (const char*)q + b * q_row * size;
        p.gate = gate ? (const char*)gate + b * gate_row * size : nullptr;
        p.out = (char*)out + (long long)b * heads * dim * size;
        p.table = table + b * table_stride; p.lengths = lengths + b;
        const int code = is_fp32 ? paged_launch<float>(p, (cudaStream_t)stream) : paged_launch<bf16>(p, (cudaStream_t)stream);
        if (code != QD_OK) return code;
    }
    return QD_OK;
}
