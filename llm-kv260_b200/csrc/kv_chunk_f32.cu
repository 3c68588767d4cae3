// b200_kv_attend_chunk on the float32 units.
#include <cuda_runtime.h>

#include "kv_chunk.cuh"

namespace b200 {
namespace chunk {

namespace {

constexpr int kM = 64, kN = 64, kThreads = 256;
constexpr int kCost = 1;               // units that a tile's begin and end take

template <int kDim>
struct Smem {
    float q[kM][kDim + 4], k[kN][kDim + 4], v[kN][kDim + 4], p[kM][kN + 4];
    long long row[kN];                 // byte offset of a slot's row, -1: not there
    Shared<kThreads> find;
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

// 64 rows by 64 slots at a time, 16 x 16 threads: a thread has the scores of
// rows 4 ty + i and slots tx + 16 j, and of the output the columns 4 tx + 64 j.
// One pass over the slots with the running maximum m and sum l of each row.
template <int kDim>
__global__ void __launch_bounds__(kThreads, 1) f32_kernel(const Args a) {
    extern __shared__ char smem_raw[];
    Smem<kDim> &s = *reinterpret_cast<Smem<kDim> *>(smem_raw);
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, d = a.kv.head_dim;
    Stretch st = find<kM, kN, kCost, kThreads>(a, &s.find);
    if (tid == 0) a.joints[blockIdx.x].first = -1;
    if (st.left == 0) return;
    Sequence q = sequence(a, st.b);
    int tile = st.tile, head = st.head, skip = st.skip;
    if (skip > kCost && tid == 0 && st.first + 1 == static_cast<int>(blockIdx.x))
        a.joints[blockIdx.x] = Joint{st.first, st.last, q.from, q.n, tile, head};
#pragma unroll 1
    for (;;) {
        const Fragment f = fragment<kM, kN, kCost>(a, q, tile, skip, st.left);
        const int row0 = f.row0, rows = f.rows;
        if (f.u1 > f.u0) {
        for (int i = tid; i < kM * (kDim / 8); i += kThreads) {
            const int r = i / (kDim / 8), c = i % (kDim / 8) * 8;
            float v[8] = {};
            if (row0 + r < rows && c < d) {
                const int token = (row0 + r) / a.group, h = row0 + r - token * a.group;
                load8<float>(a.q + (q.from + token) * a.q_token + (head * a.group + h) * a.q_head + c * static_cast<int>(sizeof(float)), v);
            }
            *reinterpret_cast<float4 *>(&s.q[r][c]) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4 *>(&s.q[r][c + 4]) = make_float4(v[4], v[5], v[6], v[7]);
        }
        int at[4];                                     // the slots that rows stand at
        float m[4], l[4], o[4][kDim / 16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row0 + ty * 4 + i;
            at[i] = r < rows ? f.first + r / a.group : -1;
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < kDim / 16; ++j) o[i][j] = 0.0f;
        }
#pragma unroll 1
        for (int u = f.u0; u < f.u1; ++u) {
            __syncthreads();
            if (tid < kN) {
                const int slot = u * kN + tid;
                s.row[tid] = slot < q.length ? kv_row(a.kv, q.b, head, slot) : -1;
            }
            __syncthreads();
            for (int i = tid; i < kN * (kDim / 8); i += kThreads) {
                const int r = i / (kDim / 8), c = i % (kDim / 8) * 8;
                float x[8] = {}, y[8] = {};
                if (s.row[r] >= 0 && c < d) {
                    load8<float>(a.kv.k + s.row[r] + c * static_cast<int>(sizeof(float)), x);
                    load8<float>(a.kv.v + s.row[r] + c * static_cast<int>(sizeof(float)), y);
                }
                *reinterpret_cast<float4 *>(&s.k[r][c]) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4 *>(&s.k[r][c + 4]) = make_float4(x[4], x[5], x[6], x[7]);
                *reinterpret_cast<float4 *>(&s.v[r][c]) = make_float4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<float4 *>(&s.v[r][c + 4]) = make_float4(y[4], y[5], y[6], y[7]);
            }
            __syncthreads();
            float t[4][4] = {};
#pragma unroll 4
            for (int c = 0; c < kDim; c += 4) {
                float4 x[4], y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4 *>(&s.q[ty * 4 + i][c]);
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4 *>(&s.k[tx + 16 * j][c]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        t[i][j] = fmaf(x[i].w, y[j].w, fmaf(x[i].z, y[j].z, fmaf(x[i].y, y[j].y, fmaf(x[i].x, y[j].x, t[i][j]))));
            }
            const bool edge = (u + 1) * kN - 1 > f.last_all || u * kN < f.first_all;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float top = -INFINITY;
                bool dead[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int slot = u * kN + tx + 16 * j;
                    dead[j] = s.row[tx + 16 * j] < 0 || slot > at[i] || (a.window && slot <= at[i] - a.window);
                    t[i][j] = dead[j] ? -INFINITY : t[i][j] * a.scale;
                    top = fmaxf(top, t[i][j]);
                }
#pragma unroll
                for (int x = 8; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, x));
                const float m1 = fmaxf(m[i], top), ref = m1 == -INFINITY ? 0.0f : m1;
                const float keep = exp2f(m[i] - ref);
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float p = exp2f(t[i][j] - ref);
                    s.p[ty * 4 + i][tx + 16 * j] = p;
                    sum += p;
                }
#pragma unroll
                for (int x = 8; x; x >>= 1) sum += __shfl_xor_sync(kFullMask, sum, x);
                l[i] = fmaf(l[i], keep, sum);
                m[i] = m1;
#pragma unroll
                for (int j = 0; j < kDim / 16; ++j) o[i][j] *= keep;
            }
            __syncwarp();                              // a row's 16 threads are in one warp
#pragma unroll 2
            for (int n = 0; n < kN; n += 4) {
                float4 p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4 *>(&s.p[ty * 4 + i][n]);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
#pragma unroll
                    for (int j = 0; j < kDim / 64; ++j) {
                        const float4 v = *reinterpret_cast<const float4 *>(&s.v[n + x][4 * tx + 64 * j]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float w = x == 0 ? p[i].x : x == 1 ? p[i].y : x == 2 ? p[i].z : p[i].w;
                            if (edge && w == 0.0f) continue;           // not seen: whatever the value is
                            o[i][4 * j] = fmaf(w, v.x, o[i][4 * j]);
                            o[i][4 * j + 1] = fmaf(w, v.y, o[i][4 * j + 1]);
                            o[i][4 * j + 2] = fmaf(w, v.z, o[i][4 * j + 2]);
                            o[i][4 * j + 3] = fmaf(w, v.w, o[i][4 * j + 3]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = ty * 4 + i;
            if (row0 + r >= rows) break;
            const int token = (row0 + r) / a.group, h = head * a.group + row0 + r - token * a.group;
            if (f.whole) {
                const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
                char *out = a.out + (q.from + token) * a.out_token + h * a.out_head;
#pragma unroll
                for (int j = 0; j < kDim / 64; ++j)
                    if (4 * tx + 64 * j < d)
                        store4<float>(out + (4 * tx + 64 * j) * static_cast<int>(sizeof(float)),
                                   make_float4(o[i][4 * j] * inv, o[i][4 * j + 1] * inv, o[i][4 * j + 2] * inv, o[i][4 * j + 3] * inv));
                if (a.lse && tx == 0)
                    a.lse[static_cast<long long>(q.from + token) * a.n_head + h] = (m[i] + log2f(l[i])) * kLn2;
            } else {
                float *part = a.parts + (2ll * blockIdx.x + f.begins) * part_floats(kM, kDim);
#pragma unroll
                for (int j = 0; j < kDim / 64; ++j)
                    *reinterpret_cast<float4 *>(part + r * kDim + 4 * tx + 64 * j) =
                        make_float4(o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]);
                if (tx == 0) {
                    part[kM * kDim + r] = m[i];
                    part[kM * kDim + kM + r] = l[i];
                }
            }
        }
        }
        st.left -= f.used;
        if (st.left <= 0) break;
        skip = 0;
        next_tile<kM>(a, q, tile, head);
        __syncthreads();
    }
}

int grid_of(int) { return sm_count(); }

template <int kDim>
cudaError_t launch(const Args &a, cudaStream_t stream) {
    const auto fn = f32_kernel<kDim>;
    const int smem = static_cast<int>(sizeof(Smem<kDim>)), grid = grid_of(kDim);
    if (!ensure_smem(reinterpret_cast<const void *>(fn), smem)) return cudaGetLastError();
    fn<<<grid, kThreads, smem, stream>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? e : launch_join<float, kM, kDim>(a, grid, stream);
}

}  // namespace

Shape f32_shape(int head_dim) {
    const int dim = (head_dim + 63) / 64 * 64;
    return Shape{grid_of(dim), part_floats(kM, dim) * 4};
}

cudaError_t f32_launch(const Args &a, cudaStream_t stream) {
    if (a.kv.head_dim <= 64) return launch<64>(a, stream);
    if (a.kv.head_dim <= 128) return launch<128>(a, stream);
    if (a.kv.head_dim <= 192) return launch<192>(a, stream);
    return launch<256>(a, stream);
}

}  // namespace chunk
}  // namespace b200
