// b200_kv_attend: attention of one new token per sequence over a paged cache.
#include <cuda_runtime.h>

#include "q4gemv.h"
#include "serve_dev.cuh"

namespace b200 {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;

struct AttendArgs {
    KvView kv;
    const char *q;
    char *out;
    long long q_batch, q_head, out_batch, out_head;  // elements
    int n_head, group;
    float scale;
    float *lse;           // [batch][n_head], the caller's or the workspace's; NULL: not wanted
    const float *weights;
    float *weights_out;
    long long aux_stride;
    float decay;
};

// One CTA per query head of a sequence; a warp takes every kWarps-th slot, a
// lane every 32nd element of the row. One pass with a running maximum and sum
// per warp, joined at the end.
template <typename Q, typename T>
__global__ void __launch_bounds__(kThreads) kv_attend_kernel(const AttendArgs a) {
    __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][kMaxHeadDim];
    const int head = blockIdx.x, b = blockIdx.y, h = head / a.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = a.kv.head_dim;
    const Q *q = reinterpret_cast<const Q *>(a.q) + b * a.q_batch + head * a.q_head;
    float qv[kMaxHeadDim / 32], o[kMaxHeadDim / 32];
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i) {
        qv[i] = lane + 32 * i < d ? to_float(q[lane + 32 * i]) * a.scale : 0.0f;
        o[i] = 0.0f;
    }
    const int n = kv_length(a.kv, b);
    float m = -INFINITY, l = 0.0f;
    for (int slot = warp; slot < n; slot += kWarps) {
        const long long row = kv_row(a.kv, b, h, slot);
        if (row < 0) continue;
        const T *k = reinterpret_cast<const T *>(a.kv.k + row), *v = reinterpret_cast<const T *>(a.kv.v + row);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kMaxHeadDim / 32; ++i)
            if (lane + 32 * i < d) s = fmaf(qv[i], to_float(k[lane + 32 * i]), s);
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(kAllLanes, s, x);
        if (s == -INFINITY) continue;
        const float m1 = fmaxf(m, s), old = expf(m - m1), p = expf(s - m1);
        m = m1;
        l = l * old + p;
#pragma unroll
        for (int i = 0; i < kMaxHeadDim / 32; ++i)
            if (lane + 32 * i < d) o[i] = fmaf(p, to_float(v[lane + 32 * i]), o[i] * old);
    }
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i) s_o[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float top = -INFINITY, sum = 0.0f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
    for (int w = 0; w < kWarps; ++w) sum += top == -INFINITY ? 0.0f : s_l[w] * expf(s_m[w] - top);
    Q *out = reinterpret_cast<Q *>(a.out) + b * a.out_batch + head * a.out_head;
    for (int i = threadIdx.x; i < d; i += kThreads) {
        float v = 0.0f;
        for (int w = 0; w < kWarps; ++w) v += top == -INFINITY ? 0.0f : s_o[w][i] * expf(s_m[w] - top);
        out[i] = from_float<Q>(top == -INFINITY ? 0.0f : v / sum);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[static_cast<long long>(b) * a.n_head + head] = top == -INFINITY ? -INFINITY : top + logf(sum);
}

// The softmax's weights again, from the rows and the log-sums: one warp per slot.
template <typename Q, typename T>
__global__ void __launch_bounds__(kThreads) kv_weights_kernel(const AttendArgs a) {
    const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, d = a.kv.head_dim;
    const int n = kv_length(a.kv, b);
    for (int slot = blockIdx.x * kWarps + (threadIdx.x >> 5); slot < n; slot += gridDim.x * kWarps) {
        const long long row = kv_row(a.kv, b, h, slot);
        float w = 0.0f;
        for (int g = 0; row >= 0 && g < a.group; ++g) {
            const int head = h * a.group + g;
            const Q *q = reinterpret_cast<const Q *>(a.q) + b * a.q_batch + head * a.q_head;
            const T *k = reinterpret_cast<const T *>(a.kv.k + row);
            float s = 0.0f;
            for (int i = lane; i < d; i += 32) s = fmaf(to_float(q[i]) * a.scale, to_float(k[i]), s);
            for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(kAllLanes, s, x);
            if (s != -INFINITY) w += expf(s - a.lse[static_cast<long long>(b) * a.n_head + head]);
        }
        const long long aux = (static_cast<long long>(b) * a.kv.n_head_kv + h) * a.aux_stride + slot;
        if (lane == 0) a.weights_out[aux] = (a.weights ? a.decay * a.weights[aux] : 0.0f) + w;
    }
}

template <typename Q, typename T>
cudaError_t launch(const AttendArgs &a, cudaStream_t stream) {
    kv_attend_kernel<Q, T><<<dim3(a.n_head, a.kv.batch), kThreads, 0, stream>>>(a);
    if (cudaError_t e = cudaGetLastError()) return e;
    if (!a.weights_out) return cudaSuccess;
    kv_weights_kernel<Q, T><<<dim3(32, a.kv.n_head_kv, a.kv.batch), kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

int kv_attend_validate(const b200_kv_t *kv, const b200_kv_attend_t *a, const char **why) {
    if (int rc = kv_validate(kv, why)) return rc;
    const auto bad = [why](const char *w) { *why = w; return kErrInval; };
    if (!a) return bad("null arguments");
    if (a->dtype != kv->dtype && !(a->dtype == B200_F32 && kv->dtype == B200_F16))
        return bad("q must be of the cache's type, or float32 with a float16 cache");
    if (a->n_head < 1 || a->n_head % kv->n_head_kv) return bad("n_head must be a multiple of n_head_kv");
    if (a->n_head / kv->n_head_kv > 256) return bad("at most 256 query heads read one cache head");
    if (!a->q || !a->out) return bad("null address");
    if (a->q_batch_stride < 0 || a->q_head_stride < 0 || a->out_batch_stride < 0 || a->out_head_stride < 0)
        return bad("strides must not be negative");
    const int es = esize(a->dtype);
    if (a->q % es || a->out % es || a->lse % 4 || a->weights % 4 || a->weights_out % 4)
        return bad("addresses must be aligned to their elements");
    if (!(a->scale - a->scale == 0.0f)) return bad("scale must be finite");
    if (a->weights_out) {
        if (a->aux_stride < static_cast<int64_t>(kv->table_cols) * kv->page_size)
            return bad("aux_stride is below the cache's slots");
        if (!(a->decay - a->decay == 0.0f)) return bad("decay must be finite");
        if (!a->workspace || a->workspace % 16 || a->workspace_bytes < b200_kv_attend_workspace(kv, a->n_head))
            return bad("weights_out needs a workspace of b200_kv_attend_workspace() bytes, 16-byte aligned");
    } else if (a->weights) {
        return bad("weights without weights_out");
    }
    return 0;
}

size_t serve_scratch_bytes() { return 256; }

cudaError_t kv_attend_launch(const b200_kv_t *kv, const b200_kv_attend_t *p, void *, cudaStream_t stream) {
    AttendArgs a;
    a.kv = kv_view(kv);
    a.q = reinterpret_cast<const char *>(p->q);
    a.out = reinterpret_cast<char *>(p->out);
    a.q_batch = p->q_batch_stride;
    a.q_head = p->q_head_stride;
    a.out_batch = p->out_batch_stride;
    a.out_head = p->out_head_stride;
    a.n_head = p->n_head;
    a.group = p->n_head / kv->n_head_kv;
    a.scale = p->scale;
    a.weights = reinterpret_cast<const float *>(p->weights);
    a.weights_out = reinterpret_cast<float *>(p->weights_out);
    a.lse = reinterpret_cast<float *>(p->lse ? p->lse : a.weights_out ? p->workspace : 0);
    a.aux_stride = p->aux_stride;
    a.decay = p->decay;
    if (kv->dtype == B200_F32) return launch<float, float>(a, stream);
    if (kv->dtype == B200_BF16) return launch<__nv_bfloat16, __nv_bfloat16>(a, stream);
    return p->dtype == B200_F32 ? launch<float, __half>(a, stream) : launch<__half, __half>(a, stream);
}

}  // namespace b200

extern "C" uint64_t b200_kv_attend_workspace(const b200_kv_t *kv, int n_head) {
    if (!kv || kv->batch < 1 || n_head < 1) return 0;
    return static_cast<uint64_t>(kv->batch) * static_cast<uint64_t>(n_head) * 4;
}
