// b200_rope: rotary positions of queries and keys, and the store of keys and
// values into a paged cache.
#include <cuda_runtime.h>

#include <cmath>
#include <limits>

#include "common.cuh"
#include "q4gemv.h"
#include "serve_dev.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;         // of a CTA

// One of q, k, v: rows in and out, in bytes.
struct Side {
    const char *in = nullptr;
    char *out = nullptr;
    long long in_token = 0, in_head = 0, out_token = 0, out_head = 0;
    int heads = 0, out_dtype = 0;
    bool stored = false;               // out is a pool: its row is the token's slot
};

struct RopeArgs {
    Side side[3];                      // q, k, v; v is only copied
    int n_tokens, head_dim, rot, tokens;
    const int *positions;
    const unsigned long long *freqs;
    float mscale;
    const long long *slots;
    int n_pages, page_size;
    long long page_stride;
    // items of a row and rows of a token: x / n = x * magic >> 32 for x * n < 2^32 and n > 1
    int per_row[3];
    unsigned row_magic[3], head_magic[3];
};

__device__ __forceinline__ int divide(int x, int n, unsigned magic) { return n == 1 ? x : static_cast<int>(__umulhi(x, magic)); }

// cos and sin of a phase in units of 2^-64 turns. The phase is a whole number,
// so nothing of a far position's angle is lost; its nearest quarter turn is
// taken off exactly, what is left is at most an eighth.
__device__ __forceinline__ float2 cos_sin(unsigned long long phase) {
    const unsigned quarter = static_cast<unsigned>((phase + (1ull << 61)) >> 62);
    const long long rest = static_cast<long long>(phase - (static_cast<unsigned long long>(quarter) << 62));
    const float t = static_cast<float>(static_cast<int>(rest >> 30)) * 0x1p-33f;   // half turns
    float s, c;
    sincospif(t, &s, &c);
    const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
    return make_float2(quarter == 1 || quarter == 2 ? -x : x, quarter >= 2 ? -y : y);
}

template <typename T, int V>
__device__ __forceinline__ void load(const char *p, float *v) {
    if constexpr (V == 8) {
        uint4 w[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
        const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
    } else {
        v[0] = to_float(*reinterpret_cast<const T *>(p));
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_as(char *p, const float *v) {
    if constexpr (V == 8) {
        uint4 w[sizeof(T) / 2];
        T *e = reinterpret_cast<T *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_float<T>(v[i]);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4 *>(p)[i] = w[i];
    } else {
        *reinterpret_cast<T *>(p) = from_float<T>(v[0]);
    }
}

template <int V>
__device__ __forceinline__ void store(char *row, int i, int dtype, const float *v) {
    if (dtype == B200_F32) store_as<float, V>(row + i * 4, v);
    else if (dtype == B200_F16) store_as<__half, V>(row + i * 2, v);
    else store_as<__nv_bfloat16, V>(row + i * 2, v);
}

// What bounds it: memory, for long prompts. 16384 tokens (32 and 8 heads of 128
// bfloat16, 336 MB): 61 us, 5.5 TB/s; 3001 tokens of 24 heads of 80 with 32
// rotated elements, into pages (69 MB): 20 us, 3.5 TB/s, with the call's 15 us
// hidden; 64 tokens: the call, 14 us (6.5 on the GPU, a chain of positions, rows
// and stores). Four tokens to a CTA share the cosines' start; one or two, which
// short calls need to fill the GPU, take 79 and 67 us for the first. No
// division: with them the second took 27 us.
//
// A CTA takes `tokens` tokens: their cosines and sines once into shared memory,
// then items of V pairs (or, behind the rotated part and in v, of 8 elements)
// of all their heads, consecutive threads on consecutive bytes of a row. The
// thread that reads a pair writes it, so a row may be turned in place.
template <typename T, int V, bool kNext>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeArgs a) {
    extern __shared__ float2 s_cs[];                   // [tokens][rot / 2]
    __shared__ long long s_row[kMaxTokens];            // byte offset of a token's row of a pool's head 0; -1: none
    const int half = a.rot / 2, first = blockIdx.x * a.tokens, tokens = min(a.tokens, a.n_tokens - first);
    for (int i = threadIdx.x; i < tokens * half; i += kThreads) {
        const int t = i / half, f = i - t * half;
        const long long p = a.positions[first + t];
        float2 cs = cos_sin(static_cast<unsigned long long>(p) * a.freqs[f]);
        s_cs[i] = make_float2(cs.x * a.mscale, cs.y * a.mscale);
    }
    if (a.slots && static_cast<int>(threadIdx.x) < tokens) {
        const long long s = a.slots[first + threadIdx.x];
        const long long page = s / a.page_size;
        s_row[threadIdx.x] = s >= 0 && page < a.n_pages ? page * a.page_stride + (s - page * a.page_size) * a.side[1].out_token : -1;
    }
    __syncthreads();
    const int turned = half / V;
#pragma unroll
    for (int part = 0; part < 3; ++part) {
        const Side &s = a.side[part];
        if (!s.in) continue;
        const int per_row = a.per_row[part], items = per_row * s.heads * tokens;
#pragma unroll 1
        for (int i = threadIdx.x; i < items; i += kThreads) {
            const int r = divide(i, per_row, a.row_magic[part]), c = i - r * per_row;
            const int t = divide(r, s.heads, a.head_magic[part]), h = r - t * s.heads;
            const char *in = s.in + (first + t) * s.in_token + h * s.in_head;
            char *out;
            if (s.stored) {
                const long long row = s_row[t];
                if (row < 0) continue;
                out = s.out + row + h * s.out_head;
            } else {
                out = s.out + (first + t) * s.out_token + h * s.out_head;
            }
            constexpr int kEs = sizeof(T);
            if (part == 2) {
                float v[8];
                load<T, 8>(in + c * 8 * kEs, v);
                store<8>(out, c * 8, s.out_dtype, v);
            } else if (c < turned) {
                const float2 *cs = s_cs + t * half + c * V;
                float x[V], y[V], u[V], w[V];
                if constexpr (kNext && V == 8) {
                    float e[16];
                    load<T, 8>(in + c * 16 * kEs, e);
                    load<T, 8>(in + (c * 16 + 8) * kEs, e + 8);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float2 z = cs[j];
                        u[j] = e[2 * j] * z.x - e[2 * j + 1] * z.y;
                        w[j] = e[2 * j + 1] * z.x + e[2 * j] * z.y;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[2 * j] = u[j], e[2 * j + 1] = w[j];
                    store<8>(out, c * 16, s.out_dtype, e);
                    store<8>(out, c * 16 + 8, s.out_dtype, e + 8);
                } else {
                    const int i0 = kNext ? 2 * c : c * V, i1 = kNext ? 2 * c + 1 : half + c * V;
                    load<T, V>(in + i0 * kEs, x);
                    load<T, V>(in + i1 * kEs, y);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float2 z = cs[j];
                        u[j] = x[j] * z.x - y[j] * z.y;
                        w[j] = y[j] * z.x + x[j] * z.y;
                    }
                    store<V>(out, i0, s.out_dtype, u);
                    store<V>(out, i1, s.out_dtype, w);
                }
            } else {
                float v[V];
                const int at = a.rot + (c - turned) * V;
                load<T, V>(in + at * kEs, v);
                store<V>(out, at, s.out_dtype, v);
            }
        }
    }
}

template <typename T>
cudaError_t launch(RopeArgs &a, bool interleaved, cudaStream_t stream) {
    const int smem = a.tokens * a.rot / 2 * static_cast<int>(sizeof(float2));
    const int grid = (a.n_tokens - 1) / a.tokens + 1;
    // eight pairs of a row at a time need rows cut at multiples of 16 bytes
    const bool wide = a.rot % 16 == 0;
    for (int i = 0; i < 3; ++i) {
        a.per_row[i] = i == 2 ? a.head_dim / 8 : wide ? a.rot / 16 + (a.head_dim - a.rot) / 8 : a.rot / 2 + a.head_dim - a.rot;
        a.row_magic[i] = static_cast<unsigned>((1ull << 32) / static_cast<unsigned>(a.per_row[i])) + 1;
        a.head_magic[i] = a.side[i].heads ? static_cast<unsigned>((1ull << 32) / static_cast<unsigned>(a.side[i].heads)) + 1 : 0;
    }
    if (interleaved) {
        if (wide) rope_kernel<T, 8, true><<<grid, kThreads, smem, stream>>>(a);
        else rope_kernel<T, 1, true><<<grid, kThreads, smem, stream>>>(a);
    } else {
        if (wide) rope_kernel<T, 8, false><<<grid, kThreads, smem, stream>>>(a);
        else rope_kernel<T, 1, false><<<grid, kThreads, smem, stream>>>(a);
    }
    return cudaGetLastError();
}

}  // namespace

int rope_validate(const b200_kv_t *kv, const b200_rope_t *a, const char **why) {
    if (kv)
        if (int rc = kv_validate(kv, why)) return rc;
    const auto bad = [why](const char *w) { *why = w; return kErrInval; };
    if (!a) return bad("null arguments");
    if (a->dtype < B200_F32 || a->dtype > B200_BF16 || a->out_dtype < B200_F32 || a->out_dtype > B200_BF16)
        return bad("unknown type");
    if (a->dtype != B200_F32 && a->out_dtype != a->dtype) return bad("16-bit rows stay of their type");
    if (a->n_tokens < 0) return bad("n_tokens must not be negative");
    if (a->n_tokens == 0) return 0;
    if (a->head_dim < 8 || a->head_dim % 8 || a->head_dim > kMaxHeadDim)
        return bad("head_dim must be a multiple of 8 in [8, 256]");
    if (a->rot_dim < 2 || a->rot_dim % 2 || a->rot_dim > a->head_dim) return bad("rot_dim must be even, in [2, head_dim]");
    if (!(a->mscale - a->mscale == 0.0f)) return bad("mscale must be finite");
    if (!a->q && !a->k) return bad("neither q nor k");
    if (!a->positions || !a->freqs) return bad("null address");
    if (a->positions % 4 || a->freqs % 8 || a->slots % 8) return bad("positions, freqs and slots must be aligned");
    const int es = esize(a->dtype), eo = esize(a->out_dtype);
    const auto rows_ok = [](uint64_t at, int64_t token, int64_t head, int size) {
        return token >= 0 && head >= 0 && at % 16 == 0 && token * size % 16 == 0 && head * size % 16 == 0;
    };
    // in place, the thread that reads a pair writes it only where a row's elements stay where they are
    const auto moved = [&](uint64_t in, int64_t token, int64_t head, uint64_t out, int64_t to_token, int64_t to_head, int heads) {
        return in == out && (a->dtype != a->out_dtype || (a->n_tokens > 1 && token != to_token) || (heads > 1 && head != to_head));
    };
    const char *in_place = "rows in place keep their type and strides";
    const auto meet = [a](int64_t token, int64_t head, int heads) {
        return (a->n_tokens > 1 && token < a->head_dim) || (heads > 1 && head < a->head_dim);
    };
    const char *apart = "rows of an output must not overlap";
    const char *aligned = "rows' addresses and strides must be multiples of 16 bytes and not negative";
    if (a->q) {
        if (a->n_head < 1 || a->n_head > 4096) return bad("n_head must be in [1, 4096]");
        if (!a->q_out) return bad("q without q_out");
        if (!rows_ok(a->q, a->q_token_stride, a->q_head_stride, es) ||
            !rows_ok(a->q_out, a->q_out_token_stride, a->q_out_head_stride, eo))
            return bad(aligned);
        if (meet(a->q_out_token_stride, a->q_out_head_stride, a->n_head)) return bad(apart);
        if (moved(a->q, a->q_token_stride, a->q_head_stride, a->q_out, a->q_out_token_stride, a->q_out_head_stride, a->n_head))
            return bad(in_place);
    }
    if (a->k) {
        if (a->n_head_kv < 1 || a->n_head_kv > 4096) return bad("n_head_kv must be in [1, 4096]");
        if (!rows_ok(a->k, a->k_token_stride, a->k_head_stride, es)) return bad(aligned);
        if (!kv) {
            if (!a->k_out) return bad("k without k_out or a cache");
            if (!rows_ok(a->k_out, a->k_out_token_stride, a->k_out_head_stride, eo)) return bad(aligned);
            if (meet(a->k_out_token_stride, a->k_out_head_stride, a->n_head_kv)) return bad(apart);
            if (moved(a->k, a->k_token_stride, a->k_head_stride, a->k_out, a->k_out_token_stride, a->k_out_head_stride,
                      a->n_head_kv))
                return bad(in_place);
        }
    }
    if (kv) {
        if (!a->k) return bad("a cache without k");
        if (a->n_head_kv != kv->n_head_kv || a->head_dim != kv->head_dim) return bad("k must have the cache's heads and head_dim");
        if (a->dtype != B200_F32 && a->dtype != kv->dtype) return bad("k must be float32 or of the cache's type");
        if (!a->slots) return bad("a cache without slots");
        if (a->v && !rows_ok(a->v, a->v_token_stride, a->v_head_stride, es)) return bad(aligned);
    } else if (a->v || a->slots) {
        return bad("v and slots need a cache");
    }
    return 0;
}

cudaError_t rope_launch(const b200_kv_t *kv, const b200_rope_t *p, cudaStream_t stream) {
    if (p->n_tokens == 0) return cudaSuccess;
    RopeArgs a{};
    const int es = esize(p->dtype), eo = esize(p->out_dtype);
    if (p->q)
        a.side[0] = Side{reinterpret_cast<const char *>(p->q), reinterpret_cast<char *>(p->q_out), p->q_token_stride * es,
                         p->q_head_stride * es, p->q_out_token_stride * eo, p->q_out_head_stride * eo, p->n_head,
                         p->out_dtype, false};
    if (p->k) {
        Side s{reinterpret_cast<const char *>(p->k), reinterpret_cast<char *>(p->k_out), p->k_token_stride * es,
               p->k_head_stride * es, p->k_out_token_stride * eo, p->k_out_head_stride * eo, p->n_head_kv, p->out_dtype,
               false};
        if (kv) {
            const KvView v = kv_view(kv);
            s.out = v.k;
            s.out_token = v.row_stride;
            s.out_head = v.head_stride;
            s.out_dtype = kv->dtype;
            s.stored = true;
            a.n_pages = v.n_pages;
            a.page_size = v.page_size;
            a.page_stride = v.page_stride;
            a.slots = reinterpret_cast<const long long *>(p->slots);
            if (p->v) {
                a.side[2] = s;
                a.side[2].in = reinterpret_cast<const char *>(p->v);
                a.side[2].out = v.v;
                a.side[2].in_token = p->v_token_stride * es;
                a.side[2].in_head = p->v_head_stride * es;
            }
        }
        a.side[1] = s;
    }
    a.n_tokens = p->n_tokens;
    a.head_dim = p->head_dim;
    a.rot = p->rot_dim;
    a.positions = reinterpret_cast<const int *>(p->positions);
    a.freqs = reinterpret_cast<const unsigned long long *>(p->freqs);
    a.mscale = p->mscale;
    a.tokens = p->n_tokens >= 1024 ? 4 : 1;
    if (p->dtype == B200_F32) return launch<float>(a, p->interleaved != 0, stream);
    if (p->dtype == B200_F16) return launch<__half>(a, p->interleaved != 0, stream);
    return launch<__nv_bfloat16>(a, p->interleaved != 0, stream);
}

int rope_freqs(uint64_t *freqs, int rot_dim, double base, const float *factors, int scaling, double factor,
               double context, double low, double high, const char **why) {
    const auto bad = [why](const char *w) { *why = w; return kErrInval; };
    const auto positive = [](double x) { return x > 0 && x - x == 0; };
    if (!freqs) return bad("null address");
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > kMaxHeadDim) return bad("rot_dim must be even, in [2, 256]");
    if (!positive(base)) return bad("base must be positive");
    if (scaling < B200_ROPE_PLAIN || scaling > B200_ROPE_YARN) return bad("unknown scaling");
    if (scaling != B200_ROPE_PLAIN && !positive(factor)) return bad("factor must be positive");
    if (scaling >= B200_ROPE_BANDS && (!positive(context) || !positive(low) || !positive(high) || low >= high))
        return bad("context, low and high must be positive, low below high");
    if (scaling == B200_ROPE_YARN && base <= 1) return bad("base must be above 1");
    const double pi = 3.14159265358979323846;
    // the pair that makes `turns` turns in `context` positions
    const auto pair = [&](double turns) { return rot_dim * std::log(context / (turns * 2 * pi)) / (2 * std::log(base)); };
    double from = 0, to = 1;
    if (scaling == B200_ROPE_YARN) {
        from = std::fmax(std::floor(pair(high)), 0.0);
        to = std::fmin(std::ceil(pair(low)), rot_dim - 1.0);
    }
    // in 64 bits: times a position of 31 bits, a double's 53 would leave 2^-25 of a turn
    using Real = long double;
    static_assert(std::numeric_limits<Real>::digits >= 64);
    const Real round = 2 * 3.14159265358979323846264338327950288L;
    for (int i = 0; i < rot_dim / 2; ++i) {
        Real f = std::pow(static_cast<Real>(base), static_cast<Real>(-2 * i) / rot_dim);
        if (factors) {
            if (!positive(factors[i])) return bad("factors must be positive");
            f /= factors[i];
        }
        Real slow = 0;                                 // share of the divided frequency
        if (scaling == B200_ROPE_LINEAR) slow = 1;
        if (scaling == B200_ROPE_BANDS) slow = 1 - (context * f / round - low) / (static_cast<Real>(high) - low);
        if (scaling == B200_ROPE_YARN) slow = (i - from) / std::fmax(static_cast<Real>(to) - from, static_cast<Real>(0.001));
        slow = std::fmin(std::fmax(slow, static_cast<Real>(0)), static_cast<Real>(1));
        if (scaling != B200_ROPE_PLAIN) f = f / factor * slow + f * (1 - slow);
        Real turns = f / round;
        turns -= std::floor(turns);
        const Real units = std::round(std::ldexp(turns, 64));
        freqs[i] = units >= 0x1p64L ? 0 : static_cast<uint64_t>(units);
    }
    return 0;
}

}  // namespace b200
