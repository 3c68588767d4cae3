// b200_kv_append: new key and value rows into a paged cache.
#include <cuda_runtime.h>

#include "q4gemv.h"
#include "serve_dev.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 256;

struct AppendArgs {
    KvView kv;
    const char *k_new, *v_new;
    long long token_stride, head_stride;  // bytes
    const int *offsets, *seen;
    int *positions;
    float *weights;
    long long aux_stride;
    int *lengths_out, *seen_out;
    int n_tokens;
    bool in_place;          // lengths_out or seen_out is what other CTAs still read
    unsigned *ticket;
};

// Eight consecutive elements, as the copy's unit: 16 bytes of a 16-bit type,
// 32 of float32.
template <typename T>
struct Eight {
    uint4 v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Eight<T> load8(const char *p) {
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    return r;
}
template <typename T>
__device__ __forceinline__ void store8(char *p, const Eight<T> &s) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4 *>(p)[i] = s.v[i];
}
// To nearest even, two to a word.
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename Src, typename Dst>
__device__ __forceinline__ Eight<Dst> convert(const Eight<Src> &s) {
    if constexpr (sizeof(Src) == sizeof(Dst)) {
        return s;
    } else {
        const auto f = [](uint32_t u) { return __uint_as_float(u); };
        Eight<Dst> d;
        d.v[0].x = pack2(f(s.v[0].x), f(s.v[0].y), Dst());
        d.v[0].y = pack2(f(s.v[0].z), f(s.v[0].w), Dst());
        d.v[0].z = pack2(f(s.v[1].x), f(s.v[1].y), Dst());
        d.v[0].w = pack2(f(s.v[1].z), f(s.v[1].w), Dst());
        return d;
    }
}

// Sequence b's first row, of those that there are.
__device__ __forceinline__ int row_from(const AppendArgs &a, int b) { return min(max(a.offsets[b], 0), a.n_tokens); }

// The copy is bound by memory: a thread takes eight elements of a row of k and
// of v, of kTokens tokens, and has asked for all of them before the CTA looks
// up where they go (sequence, length, page: reads that wait for one another,
// done by one thread per token). Consecutive threads write consecutive bytes of
// a row. 23000 rows of 8 heads of 128 bfloat16 (190 MB in and out): 37 us with
// the launch, 5.2 TB/s; with the lookups first, and in every thread, 41. One row
// for each of 64 sequences: the launch.
template <typename Src, typename Dst>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const AppendArgs a) {
    constexpr int kTokens = sizeof(Src) == 4 ? 2 : 4;
    __shared__ long long s_row[kThreads * kTokens / 8];   // a token's row of head 0, -1: none
    __shared__ int s_slot[kThreads * kTokens / 8], s_seq[kThreads * kTokens / 8], s_pos[kThreads * kTokens / 8];
    const int per_row = a.kv.head_dim / 8;
    const int units = a.kv.n_head_kv * per_row;      // of a token
    const int lane_units = min(units, kThreads);
    const int tokens = min(kThreads / lane_units, kThreads / 8);   // side by side in a CTA
    const int ty = threadIdx.x / lane_units, tx = threadIdx.x - ty * lane_units;
    const int slots = a.kv.cols * a.kv.page_size;
    const long long first = static_cast<long long>(blockIdx.x) * tokens * kTokens;
    const int count = static_cast<int>(min(static_cast<long long>(tokens) * kTokens, a.n_tokens - first));
    for (int u0 = 0; u0 < units; u0 += lane_units) {
        const int u = u0 + tx, h = u / per_row, c = u - h * per_row;
        const bool on = ty < tokens && u < units;
        Eight<Src> k[kTokens], v[kTokens];
#pragma unroll
        for (int x = 0; x < kTokens; ++x) {
            if (!on || ty + x * tokens >= count) break;
            const long long src = (first + ty + x * tokens) * a.token_stride + h * a.head_stride + c * static_cast<int>(sizeof(Src)) * 8;
            k[x] = load8<Src>(a.k_new + src);
            v[x] = load8<Src>(a.v_new + src);
        }
        if (u0 == 0) {
            if (static_cast<int>(threadIdx.x) < count) {
                const int t = static_cast<int>(first) + static_cast<int>(threadIdx.x);
                int b = t, i = 0;
                if (a.offsets) {
                    int lo = 0, hi = a.kv.batch;     // offsets[lo] <= t < offsets[hi]
                    while (hi - lo > 1) {
                        const int mid = (lo + hi) >> 1;
                        if (a.offsets[mid] <= t) lo = mid; else hi = mid;
                    }
                    b = lo;
                    const int from = row_from(a, lo);
                    i = t < from || t >= row_from(a, lo + 1) ? -1 : t - from;   // -1: no sequence has this row
                }
                const int at = kv_length(a.kv, b), slot = i < 0 || i >= slots - at ? -1 : at + i;
                s_seq[threadIdx.x] = b;
                s_slot[threadIdx.x] = slot;
                s_pos[threadIdx.x] = (a.seen ? a.seen[b] : at) + i;
                s_row[threadIdx.x] = slot < 0 ? -1 : kv_row(a.kv, b, 0, slot);
            }
            __syncthreads();
        }
#pragma unroll
        for (int x = 0; x < kTokens; ++x) {
            const int j = ty + x * tokens;
            if (!on || j >= count) break;
            if (s_row[j] >= 0) {
                const long long dst = s_row[j] + h * a.kv.head_stride + c * static_cast<int>(sizeof(Dst)) * 8;
                store8<Dst>(a.kv.k + dst, convert<Src, Dst>(k[x]));
                store8<Dst>(a.kv.v + dst, convert<Src, Dst>(v[x]));
            }
            if (c == 0 && s_slot[j] >= 0) {
                const long long aux = (static_cast<long long>(s_seq[j]) * a.kv.n_head_kv + h) * a.aux_stride + s_slot[j];
                if (a.positions) a.positions[aux] = s_pos[j];
                if (a.weights) a.weights[aux] = 0.0f;
            }
        }
    }
    // The new lengths: where they replace the old ones, only when every CTA
    // has read those.
    if (!a.lengths_out && !a.seen_out) return;
    if (a.in_place ? !last_cta(a.ticket, gridDim.x) : blockIdx.x != 0) return;
    for (int b = threadIdx.x; b < a.kv.batch; b += kThreads) {
        const int n = a.offsets ? max(row_from(a, b + 1) - row_from(a, b), 0) : 1;
        const int at = kv_length(a.kv, b);
        const int seen = a.seen ? a.seen[b] : at;
        if (a.lengths_out) a.lengths_out[b] = at + min(n, slots - at);
        if (a.seen_out) a.seen_out[b] = seen + n;
    }
}

template <typename Src, typename Dst>
cudaError_t launch(const AppendArgs &a, cudaStream_t stream) {
    const int units = a.kv.n_head_kv * a.kv.head_dim / 8;
    const int side = kThreads / (units < kThreads ? units : kThreads);
    const int tokens = (side < kThreads / 8 ? side : kThreads / 8) * (sizeof(Src) == 4 ? 2 : 4);
    const int grid = a.n_tokens > 0 ? (a.n_tokens + tokens - 1) / tokens : 1;
    kv_append_kernel<Src, Dst><<<grid, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

int kv_validate(const b200_kv_t *kv, const char **why) {
    const auto bad = [why](const char *w) { *why = w; return kErrInval; };
    if (!kv) return bad("null cache");
    if (kv->dtype < B200_F32 || kv->dtype > B200_BF16) return bad("unknown cache type");
    if (kv->batch < 1 || kv->batch > 65535) return bad("batch must be in [1, 65535]");
    if (kv->n_pages < 1 || kv->page_size < 1) return bad("n_pages and page_size must be positive");
    if (kv->n_head_kv < 1 || kv->n_head_kv > 1024) return bad("n_head_kv must be in [1, 1024]");
    if (kv->head_dim < 8 || kv->head_dim % 8 || kv->head_dim > kMaxHeadDim)
        return bad("head_dim must be a multiple of 8 in [8, 256]");
    if (kv->table_cols < 1 || static_cast<int64_t>(kv->table_cols) * kv->page_size > kMaxSlots)
        return bad("table_cols * page_size must be in [1, 1048576]");
    if (kv->table_stride < kv->table_cols) return bad("table_stride is below table_cols");
    if (!kv->k || !kv->v || !kv->table || !kv->lengths) return bad("null address");
    const int es = esize(kv->dtype);
    if (kv->page_stride < 0 || kv->head_stride < 0 || kv->row_stride < 0) return bad("strides must not be negative");
    if (kv->k % 16 || kv->v % 16 || kv->page_stride * es % 16 || kv->head_stride * es % 16 || kv->row_stride * es % 16)
        return bad("cache addresses and strides must be multiples of 16 bytes");
    if (kv->table % 4 || kv->lengths % 4) return bad("table and lengths must be 4-byte aligned");
    return 0;
}

KvView kv_view(const b200_kv_t *kv) {
    const int es = esize(kv->dtype);
    KvView v;
    v.k = reinterpret_cast<char *>(kv->k);
    v.v = reinterpret_cast<char *>(kv->v);
    v.page_stride = kv->page_stride * es;
    v.head_stride = kv->head_stride * es;
    v.row_stride = kv->row_stride * es;
    v.table = reinterpret_cast<const int *>(kv->table);
    v.table_stride = kv->table_stride;
    v.lengths = reinterpret_cast<const int *>(kv->lengths);
    v.n_pages = kv->n_pages;
    v.page_size = kv->page_size;
    v.n_head_kv = kv->n_head_kv;
    v.head_dim = kv->head_dim;
    v.cols = kv->table_cols;
    v.batch = kv->batch;
    return v;
}

int kv_append_validate(const b200_kv_t *kv, const b200_kv_append_t *a, const char **why) {
    if (int rc = kv_validate(kv, why)) return rc;
    const auto bad = [why](const char *w) { *why = w; return kErrInval; };
    if (!a) return bad("null arguments");
    if (a->dtype != B200_F32 && a->dtype != kv->dtype) return bad("new rows must be float32 or of the cache's type");
    if (a->n_tokens < 0) return bad("n_tokens must not be negative");
    if (!a->offsets && a->n_tokens != kv->batch) return bad("without offsets there is one row per sequence");
    if (a->n_tokens > 0 && (!a->k_new || !a->v_new)) return bad("null address");
    const int es = esize(a->dtype);
    if (a->token_stride < 0 || a->head_stride < 0) return bad("strides must not be negative");
    if (a->k_new % 16 || a->v_new % 16 || a->token_stride * es % 16 || a->head_stride * es % 16)
        return bad("new rows' addresses and strides must be multiples of 16 bytes");
    if ((a->positions || a->weights) && a->aux_stride < static_cast<int64_t>(kv->table_cols) * kv->page_size)
        return bad("aux_stride is below the cache's slots");
    if (a->offsets % 4 || a->seen % 4 || a->positions % 4 || a->weights % 4 || a->lengths_out % 4 || a->seen_out % 4)
        return bad("offsets, seen, positions, weights and the outputs must be 4-byte aligned");
    return 0;
}

cudaError_t kv_append_launch(const b200_kv_t *kv, const b200_kv_append_t *p, void *scratch, cudaStream_t stream) {
    AppendArgs a;
    const int es = esize(p->dtype);
    a.kv = kv_view(kv);
    a.k_new = reinterpret_cast<const char *>(p->k_new);
    a.v_new = reinterpret_cast<const char *>(p->v_new);
    a.token_stride = p->token_stride * es;
    a.head_stride = p->head_stride * es;
    a.offsets = reinterpret_cast<const int *>(p->offsets);
    a.seen = reinterpret_cast<const int *>(p->seen);
    a.positions = reinterpret_cast<int *>(p->positions);
    a.weights = reinterpret_cast<float *>(p->weights);
    a.aux_stride = p->aux_stride;
    a.lengths_out = reinterpret_cast<int *>(p->lengths_out);
    a.seen_out = reinterpret_cast<int *>(p->seen_out);
    a.n_tokens = p->n_tokens;
    const uint64_t seen = p->seen ? p->seen : kv->lengths;
    a.in_place = (p->lengths_out && (p->lengths_out == kv->lengths || p->lengths_out == seen)) ||
                 (p->seen_out && (p->seen_out == kv->lengths || p->seen_out == seen));
    a.ticket = static_cast<unsigned *>(scratch);
    if (kv->dtype == B200_F32) return launch<float, float>(a, stream);
    if (kv->dtype == B200_F16)
        return p->dtype == B200_F32 ? launch<float, __half>(a, stream) : launch<__half, __half>(a, stream);
    return p->dtype == B200_F32 ? launch<float, __nv_bfloat16>(a, stream)
                                : launch<__nv_bfloat16, __nv_bfloat16>(a, stream);
}

}  // namespace b200
