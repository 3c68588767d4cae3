// b200_rms_norm: residual addition, root-mean-square norm and Q8_0 rows.
#include <cuda_runtime.h>

#include "common.cuh"
#include "q4gemv.h"
#include "serve_dev.cuh"

namespace b200 {

namespace {

constexpr int kMaxNorm = 32768, kMaxThreads = 1024;   // a block of so many has 64 registers a thread
// Outputs above half of the 126 MB L2 are written past it (16384 rows of 4096 bfloat16 with their residual, 268 MB
// written: 96 us, and 104 without), smaller ones are left there for the matrix that reads them.
constexpr long long kStreamBytes = 64 << 20;

struct NormArgs {
    const char *x, *residual;
    char *residual_out, *out;
    const float *weight;
    uint8_t *q8;
    long long x_stride, residual_stride, residual_out_stride, out_stride, q8_stride;  // bytes
    int residual_dtype, out_dtype, k, round_mode;
    float eps;
};

template <typename T>
__device__ __forceinline__ void load8(const char *p, float *v) {
    uint4 w[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = reinterpret_cast<const uint4 *>(p)[i];
    const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
}
template <typename T, bool kStream>
__device__ __forceinline__ void store8(char *p, const float *v) {
    uint4 w[sizeof(T) / 2];
    T *e = reinterpret_cast<T *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_float<T>(v[i]);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
        if (kStream) __stcs(reinterpret_cast<uint4 *>(p) + i, w[i]);
        else reinterpret_cast<uint4 *>(p)[i] = w[i];
    }
}
template <bool kStream>
__device__ __forceinline__ void store8(char *row, int i, int dtype, const float *v) {
    if (dtype == B200_F32) store8<float, kStream>(row + i * 4, v);
    else if (dtype == B200_F16) store8<__half, kStream>(row + i * 2, v);
    else store8<__nv_bfloat16, kStream>(row + i * 2, v);
}

// A CTA per row, J times eight elements in each thread's registers: one pass
// over memory, which bounds it (16384 rows of 4096 bfloat16 with their residual,
// 537 MB: 96 us, 5.6 TB/s, with two units a thread; one 99, four 102). One row:
// 4.5 us on the GPU, less than the call. Four neighbouring threads hold a Q8_0
// block.
template <typename T, int J, bool kStream>
__global__ void __maxnreg__(65536 / kMaxThreads) rms_norm_kernel(const NormArgs a) {
    __shared__ float s_sum[32];
    const int row = blockIdx.x, threads = blockDim.x, tid = threadIdx.x, units = a.k / 8;
    const char *x = a.x + row * a.x_stride;
    float v[J][8];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int u = tid + j * threads;
        if (u < units) load8<T>(x + u * 8 * static_cast<int>(sizeof(T)), v[j]);
    }
    if (a.residual) {
        const char *r = a.residual + row * a.residual_stride;
        char *ro = a.residual_out + row * a.residual_out_stride;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int u = tid + j * threads;
            if (u >= units) break;
            float e[8];
            if (a.residual_dtype == B200_F32) load8<float>(r + u * 32, e);
            else load8<T>(r + u * 8 * static_cast<int>(sizeof(T)), e);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] += e[i];
            if (a.residual_out) store8<kStream>(ro, u * 8, a.residual_dtype, v[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        if (tid + j * threads >= units) break;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(v[j][i], v[j][i], sum);
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(kFullMask, sum, i);
    if (threads > 32) {
        if ((tid & 31) == 0) s_sum[tid >> 5] = sum;
        __syncthreads();
        sum = (tid & 31) < threads / 32 ? s_sum[tid & 31] : 0.0f;
#pragma unroll
        for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(kFullMask, sum, i);
    }
    const float scale = __frsqrt_rn(sum / static_cast<float>(a.k) + a.eps);
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int u = tid + j * threads;
        const bool on = u < units;
        float y[8], w[8];
        if (on) load8<float>(reinterpret_cast<const char *>(a.weight) + u * 32, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = on ? v[j][i] * scale * w[i] : 0.0f;
        if (on && a.out) store8<kStream>(a.out + row * a.out_stride, u * 8, a.out_dtype, y);
        if (a.q8) {                        // uniform; units is a multiple of 4, so four threads are all on or all off
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(y[i]));
            m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 1));
            m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 2));
            const float d = __fdiv_rn(m, 127.0f);
            const float inv = d == 0.0f ? 0.0f : __fdiv_rn(1.0f, d);
            uint32_t q[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                q[i >> 2] |= (static_cast<uint32_t>(q8_round(__fmul_rn(y[i], inv), a.round_mode)) & 0xffu) << (8 * (i & 3));
            if (on) {
                uint8_t *o = a.q8 + row * a.q8_stride;
                reinterpret_cast<uint32_t *>(o)[2 * u] = q[0];
                reinterpret_cast<uint32_t *>(o)[2 * u + 1] = q[1];
                if ((u & 3) == 0) reinterpret_cast<float *>(o + a.k)[u >> 2] = __half2float(__float2half_rn(d));
            }
        }
    }
}

template <typename T, bool kStream>
cudaError_t launch(const NormArgs &a, int rows, cudaStream_t stream) {
    const int units = a.k / 8;
    // two units a thread where rows are many and there is enough to hide latency, else one
    int threads = (units + 31) / 32 * 32;
    int j = 1;
    while (threads > kMaxThreads || (rows >= 2048 && threads > 256 && j < 2)) {
        j *= 2;
        threads = ((units + j - 1) / j + 31) / 32 * 32;
    }
    if (j == 1) rms_norm_kernel<T, 1, kStream><<<rows, threads, 0, stream>>>(a);
    else if (j == 2) rms_norm_kernel<T, 2, kStream><<<rows, threads, 0, stream>>>(a);
    else rms_norm_kernel<T, 4, kStream><<<rows, threads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const NormArgs &a, int rows, bool past_l2, cudaStream_t stream) {
    return past_l2 ? launch<T, true>(a, rows, stream) : launch<T, false>(a, rows, stream);
}

}  // namespace

int rms_norm_validate(const b200_rms_norm_t *a, const char **why) {
    const auto bad = [why](const char *w) { *why = w; return kErrInval; };
    if (!a) return bad("null arguments");
    if (a->dtype < B200_F32 || a->dtype > B200_BF16) return bad("unknown type");
    if (a->n_rows < 0) return bad("n_rows must not be negative");
    if (a->n_rows == 0) return 0;
    if (a->k < 8 || a->k % 8 || a->k > kMaxNorm) return bad("k must be a multiple of 8 in [8, 32768]");
    if (a->q8 && a->k % 32) return bad("q8 needs k to be a multiple of 32");
    if (!(a->eps >= 0.0f) || !(a->eps - a->eps == 0.0f)) return bad("eps must be finite and not negative");
    if (!a->x || !a->weight) return bad("null address");
    if (!a->out && !a->q8 && !a->residual_out) return bad("no output");
    if (a->residual && a->residual_dtype != a->dtype && a->residual_dtype != B200_F32)
        return bad("residual must be of x's type or float32");
    if (a->residual_out && !a->residual) return bad("residual_out without residual");
    if (a->out && a->out_dtype != a->dtype && (a->dtype != B200_F32 || a->out_dtype < B200_F32 || a->out_dtype > B200_BF16))
        return bad("out must be of x's type, or of any with float32");
    const auto rows_ok = [](uint64_t at, int64_t stride, int size) { return stride >= 0 && at % 16 == 0 && stride * size % 16 == 0; };
    const int es = esize(a->dtype), er = esize(a->residual_dtype);
    if (!rows_ok(a->x, a->x_stride, es) || a->weight % 16 || (a->residual && !rows_ok(a->residual, a->residual_stride, er)) ||
        (a->residual_out && !rows_ok(a->residual_out, a->residual_out_stride, er)) ||
        (a->out && !rows_ok(a->out, a->out_stride, esize(a->out_dtype))))
        return bad("addresses and strides must be multiples of 16 bytes and not negative");
    if (a->n_rows > 1 && ((a->out && a->out_stride < a->k) || (a->residual_out && a->residual_out_stride < a->k)))
        return bad("rows of an output must not overlap");
    // a CTA reads its row before it writes it, so a row in place must be its own; the sum is written element by element
    // before all of the row has been read
    const int eo = esize(a->out_dtype);
    const auto moves = [a](int64_t from, int64_t to) { return a->n_rows > 1 && from != to; };
    if ((a->out && a->out == a->x && moves(a->x_stride * es, a->out_stride * eo)) ||
        (a->out && a->out == a->residual && moves(a->residual_stride * er, a->out_stride * eo)) ||
        (a->residual_out && a->residual_out == a->residual && moves(a->residual_stride, a->residual_out_stride)) ||
        (a->residual_out && a->residual_out == a->x && (er != es || moves(a->x_stride, a->residual_out_stride))))
        return bad("rows in place must stay where they are");
    if (a->out && a->out == a->residual_out) return bad("out and residual_out must differ");
    if (a->q8 && (a->q8 % 4 || a->q8_stride % 4 || a->q8_stride < a->k + a->k / 8))
        return bad("q8 rows must be 4-byte aligned and hold k + k / 8 bytes");
    return 0;
}

cudaError_t rms_norm_launch(const b200_rms_norm_t *p, int round_mode, cudaStream_t stream) {
    if (p->n_rows == 0) return cudaSuccess;
    NormArgs a;
    const int es = esize(p->dtype), er = p->residual ? esize(p->residual_dtype) : 4;
    a.x = reinterpret_cast<const char *>(p->x);
    a.residual = reinterpret_cast<const char *>(p->residual);
    a.residual_out = reinterpret_cast<char *>(p->residual_out);
    a.out = reinterpret_cast<char *>(p->out);
    a.weight = reinterpret_cast<const float *>(p->weight);
    a.q8 = reinterpret_cast<uint8_t *>(p->q8);
    a.x_stride = p->x_stride * es;
    a.residual_stride = p->residual_stride * er;
    a.residual_out_stride = p->residual_out_stride * er;
    a.out_stride = p->out ? p->out_stride * esize(p->out_dtype) : 0;
    a.q8_stride = p->q8_stride;
    a.residual_dtype = p->residual_dtype;
    a.out_dtype = p->out_dtype;
    a.k = p->k;
    a.round_mode = round_mode;
    a.eps = p->eps;
    const long long written = static_cast<long long>(p->n_rows) * p->k * ((p->residual_out ? er : 0) + (p->out ? esize(p->out_dtype) : 0));
    if (p->dtype == B200_F32) return launch<float>(a, p->n_rows, written > kStreamBytes, stream);
    if (p->dtype == B200_F16) return launch<__half>(a, p->n_rows, written > kStreamBytes, stream);
    return launch<__nv_bfloat16>(a, p->n_rows, written > kStreamBytes, stream);
}

}  // namespace b200
