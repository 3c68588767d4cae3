// b200_sample: the next token of each row of logits.
#include <cuda_runtime.h>

#include "common.cuh"
#include "serve_dev.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kUnitBits = 40;                  // a token's largest weight is 2^40
constexpr int kShareBits = 24;                 // u and top_p count in 2^-24

using u64 = unsigned long long;

struct SampleArgs {
    const char *logits;
    long long row_stride;   // elements
    int n;
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *u;
    int *token;
    float *logprob;
};

// Order-preserving unsigned form of a logit: NaN as -infinity, -0 as 0.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

// 2^((x - top) c), 1 at the top itself (where x - top or c may not be finite).
// No fused multiply-add: the weight is the same wherever it is computed.
__device__ __forceinline__ float exponent(float x, float top, float c) {
    return x == top ? 0.0f : x == -INFINITY ? -INFINITY : __fmul_rn(__fsub_rn(x, top), c);
}
__device__ __forceinline__ u64 units(float e) { return static_cast<u64>(e * static_cast<float>(1ull << kUnitBits)); }

// floor(share * total / 2^24), total < 2^62, and the same rounded up.
__device__ __forceinline__ u64 part(u64 share, u64 total) {
    return (total >> kShareBits) * share + (((total & 0xffffff) * share) >> kShareBits);
}
__device__ __forceinline__ u64 part_up(u64 share, u64 total) {
    return part(share, total) + (((total & 0xffffff) * share & 0xffffff) != 0);
}

__device__ __forceinline__ u64 block_sum(u64 v, u64 *s) {
    for (int k = 16; k; k >>= 1) v += __shfl_xor_sync(kFullMask, v, k);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s[threadIdx.x & 31];
    for (int k = 16; k; k >>= 1) v += __shfl_xor_sync(kFullMask, v, k);
    return v;
}

struct Shared {
    u64 mass[256];
    unsigned count[256];
    u64 warp[32];
    u64 before, left;
    uint32_t prefix;
    int index;
};

// The 8-bit digit at which the sum over bins, taken from the highest, first
// reaches s.left (as counts or as masses); narrows s.prefix to it.
template <typename V>
__device__ __forceinline__ void pick_bin(Shared &s, const V *bins, int shift) {
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    u64 c[8], mine = 0;
    for (int j = 0; j < 8; ++j) mine += c[j] = bins[255 - (lane * 8 + j)];
    u64 x = mine;
    for (int k = 1; k < 32; k <<= 1) {
        const u64 y = __shfl_up_sync(kFullMask, x, k);
        if (lane >= k) x += y;
    }
    u64 before = x - mine;
    const u64 left = s.left;
    const unsigned there = __ballot_sync(kFullMask, before < left && left <= x);
    if (lane == __ffs(there) - 1) {
        int j = 0;
        while (before + c[j] < left) before += c[j++];
        s.prefix |= static_cast<uint32_t>(255 - (lane * 8 + j)) << shift;
        s.left = left - before;
    }
}

// One CTA per row.
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
    __shared__ Shared s;
    const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = a.n;
    const T *logits = reinterpret_cast<const T *>(a.logits) + row * a.row_stride;
    const auto at = [&](int i) { return clean(to_float(logits[i])); };

    float top = -INFINITY;
    for (int i = tid; i < n; i += kThreads) top = fmaxf(top, at(i));
    for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, k));
    if (lane == 0) s.count[warp] = __float_as_uint(top);
    if (tid == 0) s.index = n;
    __syncthreads();
    top = __uint_as_float(s.count[lane]);
    for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, k));
    __syncthreads();
    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    if (top == -INFINITY) {
        if (tid == 0) {
            a.token[row] = -1;
            if (a.logprob) a.logprob[row] = -INFINITY;
        }
        return;
    }
    if (!(temp > 0.0f)) {
        for (int i = tid; i < n; i += kThreads)
            if (at(i) == top) {
                atomicMin(&s.index, i);
                break;
            }
        __syncthreads();
        if (tid == 0) {
            a.token[row] = s.index;
            if (a.logprob) a.logprob[row] = 0.0f;
        }
        return;
    }
    const float c = __fdiv_rn(1.44269504088896340736f, temp);
    const float min_p = a.min_p && a.min_p[row] > 0.0f ? a.min_p[row] : 0.0f;
    const auto weight = [&](float x) { return units(exp2f(exponent(x, top, c))); };

    // What the filters keep: keys above `edge`, and the first `ties` at it.
    uint32_t edge = 0;
    u64 ties = 0;
    const int k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < n) {
        if (tid == 0) s.prefix = 0, s.left = static_cast<u64>(k);
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) s.count[tid] = 0;
            __syncthreads();
            const uint32_t prefix = s.prefix, mask = shift == 24 ? 0 : kFullMask << (shift + 8);
            for (int i = tid; i < n; i += kThreads) {
                const uint32_t key = order_key(at(i));
                if ((key & mask) == prefix) atomicAdd(&s.count[(key >> shift) & 255], 1u);
            }
            __syncthreads();
            pick_bin(s, s.count, shift);
            __syncthreads();
        }
        edge = s.prefix;
        ties = s.left;
        __syncthreads();
    }
    const float share_p = a.top_p ? a.top_p[row] : 1.0f;
    const long long p24 = share_p < 1.0f ? __float2ll_rn(fmaxf(share_p, 0.0f) * 16777216.0f) : 1ll << kShareBits;
    if (p24 < 1ll << kShareBits) {
        u64 sum = 0, at_edge = 0;
        for (int i = tid; i < n; i += kThreads) {
            const float x = at(i);
            const uint32_t key = order_key(x);
            if (key > edge) sum += weight(x);
            else if (key == edge) at_edge = weight(x);
        }
        sum = block_sum(sum, s.warp);
        // every tie weighs the same: one thread's is all that is needed
        if (tid == 0) s.before = 0;
        __syncthreads();
        if (at_edge) s.before = at_edge;
        __syncthreads();
        at_edge = s.before * ties;
        u64 need = part_up(static_cast<u64>(p24), sum + at_edge);
        if (need < 1) need = 1;
        __syncthreads();
        if (tid == 0) s.prefix = 0, s.left = need;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) s.mass[tid] = 0;
            __syncthreads();
            const uint32_t prefix = s.prefix, mask = shift == 24 ? 0 : kFullMask << (shift + 8);
            for (int i = tid; i < n; i += kThreads) {
                const float x = at(i);
                const uint32_t key = order_key(x);
                if (key > edge && (key & mask) == prefix) {
                    const u64 w = weight(x);
                    if (w) atomicAdd(&s.mass[(key >> shift) & 255], w);
                }
            }
            if (tid == 0 && at_edge && (edge & mask) == prefix) atomicAdd(&s.mass[(edge >> shift) & 255], at_edge);
            __syncthreads();
            pick_bin(s, s.mass, shift);
            __syncthreads();
        }
        edge = s.prefix;
        const u64 left = s.left;
        const uint32_t u = edge ^ (edge >> 31 ? 0x80000000u : 0xffffffffu);
        const u64 w = weight(__uint_as_float(u));
        ties = (left + w - 1) / w;
        __syncthreads();
    }
    if (min_p > 1.0f) edge = order_key(top), ties = 1;

    // The kept weight of each warp's stretch of the row, and where u falls.
    const int per_warp = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
    const int i0 = min(warp * per_warp, n), i1 = min(i0 + per_warp, n);
    u64 sum = 0, equal = 0, w_edge = 0;
    const auto kept = [&](float x, u64 *w, bool *tie) {
        const uint32_t key = order_key(x);
        *w = 0;
        *tie = false;
        if (key < edge) return;
        const float e = exp2f(exponent(x, top, c));
        if (e < min_p && x != top) return;
        *w = units(e);
        *tie = key == edge;
    };
    for (int i = i0 + lane; i < i1; i += 32) {
        u64 w;
        bool tie;
        kept(at(i), &w, &tie);
        if (tie) ++equal, w_edge = w;
        else sum += w;
    }
    for (int x = 16; x; x >>= 1) {
        sum += __shfl_xor_sync(kFullMask, sum, x);
        equal += __shfl_xor_sync(kFullMask, equal, x);
        w_edge = max(w_edge, __shfl_xor_sync(kFullMask, w_edge, x));
    }
    if (lane == 0) s.warp[warp] = equal;
    __syncthreads();
    u64 ties_before = 0;
    for (int j = 0; j < warp; ++j) ties_before += s.warp[j];
    const u64 mine = ties > ties_before ? min(equal, ties - ties_before) : 0;
    sum += mine * w_edge;
    __syncthreads();
    if (lane == 0) s.warp[warp] = sum;
    __syncthreads();
    u64 before = 0, total = 0;
    for (int j = 0; j < kWarps; ++j) {
        if (j < warp) before += s.warp[j];
        total += s.warp[j];
    }
    const float u = a.u[row];
    const u64 share = u > 0.0f ? static_cast<u64>(fminf(u, 1.0f - 0x1p-24f) * 16777216.0f) : 0;
    const u64 target = part(share, total);
    if (before <= target && target < before + sum) {
        u64 run = before, seen = ties_before;
        for (int base = i0; base < i1; base += 32) {
            const int i = base + lane;
            u64 w = 0;
            bool tie = false;
            float x = -INFINITY;
            if (i < i1) kept(x = at(i), &w, &tie);
            const unsigned eq = __ballot_sync(kFullMask, tie);
            if (tie && seen + __popc(eq & ((1u << lane) - 1)) >= ties) w = 0;
            u64 upto = w;
            for (int j = 1; j < 32; j <<= 1) {
                const u64 y = __shfl_up_sync(kFullMask, upto, j);
                if (lane >= j) upto += y;
            }
            const unsigned hit = __ballot_sync(kFullMask, run + upto > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    a.token[row] = i;
                    if (a.logprob)
                        a.logprob[row] = exponent(x, top, c) * 0.693147180559945309417f -
                                         logf(static_cast<float>(total) * (1.0f / static_cast<float>(1ull << kUnitBits)));
                }
                break;
            }
            run += __shfl_sync(kFullMask, upto, 31);
            seen += __popc(eq);
        }
    }
}

}  // namespace

int sample_validate(const b200_sample_t *s, const char **why) {
    const auto bad = [why](const char *w) { *why = w; return kErrInval; };
    if (!s) return bad("null arguments");
    if (s->dtype < B200_F32 || s->dtype > B200_BF16) return bad("unknown logits type");
    if (s->batch < 1 || s->batch > 65535) return bad("batch must be in [1, 65535]");
    if (s->n_vocab < 1 || s->n_vocab > kMaxVocab) return bad("n_vocab must be in [1, 4194304]");
    if (s->row_stride < s->n_vocab && s->batch > 1) return bad("row_stride is below n_vocab");
    if (!s->logits || !s->u || !s->token) return bad("null address");
    if (s->logits % esize(s->dtype) || s->temperature % 4 || s->top_k % 4 || s->top_p % 4 || s->min_p % 4 || s->u % 4 ||
        s->token % 4 || s->logprob % 4)
        return bad("addresses must be aligned to their elements");
    return 0;
}

cudaError_t sample_launch(const b200_sample_t *p, cudaStream_t stream) {
    SampleArgs a;
    a.logits = reinterpret_cast<const char *>(p->logits);
    a.row_stride = p->row_stride;
    a.n = p->n_vocab;
    a.temperature = reinterpret_cast<const float *>(p->temperature);
    a.top_k = reinterpret_cast<const int *>(p->top_k);
    a.top_p = reinterpret_cast<const float *>(p->top_p);
    a.min_p = reinterpret_cast<const float *>(p->min_p);
    a.u = reinterpret_cast<const float *>(p->u);
    a.token = reinterpret_cast<int *>(p->token);
    a.logprob = reinterpret_cast<float *>(p->logprob);
    if (p->dtype == B200_F32) sample_kernel<float><<<p->batch, kThreads, 0, stream>>>(a);
    else if (p->dtype == B200_F16) sample_kernel<__half><<<p->batch, kThreads, 0, stream>>>(a);
    else sample_kernel<__nv_bfloat16><<<p->batch, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace b200
