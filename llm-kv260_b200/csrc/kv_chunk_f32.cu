// b200_kv_attend_chunk in float32 throughout, on the float32 units: every bit of
// queries and cache counts. (Three bfloat16 parts of each operand hold them too,
// and six products of parts at the fifth-generation tensor cores' 16-bit rate,
// 273 TFLOP/s, would leave the float32 units' 75 behind; that is not built.) What
// bounds it: float32 operations and the shared-memory reads that feed them (16
// of 128 bytes for 128 operations of a warp), with 8 warps an SM. 2000 tokens, 32
// heads of 128, 8 of the cache: 946 us, 35 TFLOP/s, 47 % of what the units can
// do (990 with the test for values not seen in the inner loop, 1080 with four
// rows to a thread, 1230 with two numbers to an instruction); 35 TFLOP/s with
// heads of 256.
#include <cuda_runtime.h>

#include <type_traits>

#include "kv_chunk.cuh"

namespace b200 {
namespace chunk {

namespace {

constexpr int kN = 64, kThreads = 256;
// Rows of a thread: eight, half as many reads for an operation as four, where a tile of 128 rows fits shared memory.
__host__ __device__ constexpr int rows_of(int dim) { return dim <= 128 ? 8 : 4; }
constexpr int kCost = 1;               // units that a tile's begin and end take
constexpr uint32_t kHidden = 0x80000000;   // weight of a slot that the row does not see: -0, beside the 0 of one too small to count

template <int kDim>
struct Smem {
    static constexpr int kM = 16 * rows_of(kDim);
    float q[kM][kDim + 4], k[kN][kDim + 4], v[kN][kDim + 4], p[kM][kN + 4];
    long long row[2][kN];              // byte offset of a slot's row, -1: not there
    Shared<kThreads> find;
};

// 64 slots by 128 rows (64) at a time, 16 x 16 threads: a thread has the scores
// of rows 8 ty + i (4 ty + i) and slots tx + 16 j, and of the output the columns
// 4 tx + 64 j.
// One pass over the slots with the running maximum m and sum l of each row.
template <int kDim>
__global__ void __launch_bounds__(kThreads, 1) f32_kernel(const Args a) {
    extern __shared__ char smem_raw[];
    Smem<kDim> &s = *reinterpret_cast<Smem<kDim> *>(smem_raw);
    constexpr int kRows = rows_of(kDim), kM = 16 * kRows;
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
        // Keys of the next unit come while this one's weights and outputs are computed, values while the next one's scores
        // are; the rows are looked up a unit before.
        const int *table = a.kv.table + q.b * a.kv.table_stride;
        int page = -1;
        const auto ask = [&](int u) {
            const int slot = u * kN + tid;
            page = -1;
            if (tid < kN && u < f.u1 && slot < q.length) page = table[static_cast<int>((slot * a.page_magic) >> 40)];
        };
        const auto place = [&](int u) {
            if (tid >= kN) return;
            const int slot = u * kN + tid, col = static_cast<int>((slot * a.page_magic) >> 40);
            const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(a.kv.n_pages);
            s.row[u & 1][tid] = there ? page * a.kv.page_stride + (slot - col * a.kv.page_size) * a.kv.row_stride : -1;
        };
        const auto copy = [&](const char *from, float (&to)[kN][kDim + 4], int u) {
            if (u < f.u1) {
#pragma unroll 4
                for (int i = tid; i < kN * (kDim / 4); i += kThreads) {
                    const int r = i / (kDim / 4), c = i % (kDim / 4) * 4;
                    const long long at = s.row[u & 1][r];
                    const bool there = at >= 0 && c < d;
                    copy16(smem_addr(&to[r][c]), from + (there ? at + c * 4 : 0), there);
                }
            }
            cp_async_commit();
        };
        const char *k_head = a.kv.k + head * a.kv.head_stride, *v_head = a.kv.v + head * a.kv.head_stride;
        ask(f.u0);
        place(f.u0);
        ask(f.u0 + 1);
        __syncthreads();
        copy(k_head, s.k, f.u0);
        copy(v_head, s.v, f.u0);
        for (int i = tid; i < kM * (kDim / 4); i += kThreads) {
            const int r = i / (kDim / 4), c = i % (kDim / 4) * 4;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (row0 + r < rows && c < d) {
                const int token = (row0 + r) / a.group, h = row0 + r - token * a.group;
                v = *reinterpret_cast<const float4 *>(a.q + (q.from + token) * a.q_token + (head * a.group + h) * a.q_head + c * 4);
            }
            *reinterpret_cast<float4 *>(&s.q[r][c]) = v;
        }
        int at[kRows];                                     // the slots that rows stand at
        float m[kRows], l[kRows], o[kRows][kDim / 16];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = row0 + ty * kRows + i;
            at[i] = r < rows ? f.first + r / a.group : -1;
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < kDim / 16; ++j) o[i][j] = 0.0f;
        }
#pragma unroll 1
        for (int u = f.u0; u < f.u1; ++u) {
            cp_async_wait<1>();                        // the keys; the values may be on their way
            __syncthreads();
            const long long *row = s.row[u & 1];
            place(u + 1);
            ask(u + 2);
            float t[kRows][4] = {};
#pragma unroll 4
            for (int c = 0; c < kDim; c += 4) {
                float4 x[kRows], y[4];
#pragma unroll
                for (int i = 0; i < kRows; ++i) x[i] = *reinterpret_cast<const float4 *>(&s.q[ty * kRows + i][c]);
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4 *>(&s.k[tx + 16 * j][c]);
#pragma unroll
                for (int i = 0; i < kRows; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        t[i][j] = fmaf(x[i].w, y[j].w, fmaf(x[i].z, y[j].z, fmaf(x[i].y, y[j].y, fmaf(x[i].x, y[j].x, t[i][j]))));
            }
            __syncthreads();                           // the keys have been read
            copy(k_head, s.k, u + 1);
            const bool edge = (u + 1) * kN - 1 > f.last_all || u * kN < f.first_all;
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                float top = -INFINITY;
                bool dead[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int slot = u * kN + tx + 16 * j;
                    dead[j] = row[tx + 16 * j] < 0 || slot > at[i] || (a.window && slot <= at[i] - a.window);
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
                    const float p = dead[j] ? __uint_as_float(kHidden) : exp2f(t[i][j] - ref);
                    s.p[ty * kRows + i][tx + 16 * j] = p;
                    sum += p;
                }
#pragma unroll
                for (int x = 8; x; x >>= 1) sum += __shfl_xor_sync(kFullMask, sum, x);
                l[i] = fmaf(l[i], keep, sum);
                m[i] = m1;
#pragma unroll
                for (int j = 0; j < kDim / 16; ++j) o[i][j] *= keep;
            }
            cp_async_wait<1>();                        // the values
            __syncthreads();
            const auto outputs = [&](auto at_edge) {
                constexpr bool kEdge = decltype(at_edge)::value;
#pragma unroll 2
                for (int n = 0; n < kN; n += 4) {
                    float4 p[kRows];
#pragma unroll
                    for (int i = 0; i < kRows; ++i) p[i] = *reinterpret_cast<const float4 *>(&s.p[ty * kRows + i][n]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
#pragma unroll
                        for (int j = 0; j < kDim / 64; ++j) {
                            const float4 v = *reinterpret_cast<const float4 *>(&s.v[n + x][4 * tx + 64 * j]);
#pragma unroll
                            for (int i = 0; i < kRows; ++i) {
                                const float w = x == 0 ? p[i].x : x == 1 ? p[i].y : x == 2 ? p[i].z : p[i].w;
                                if (kEdge && __float_as_uint(w) == kHidden) continue;      // whatever the value is
                                o[i][4 * j] = fmaf(w, v.x, o[i][4 * j]);
                                o[i][4 * j + 1] = fmaf(w, v.y, o[i][4 * j + 1]);
                                o[i][4 * j + 2] = fmaf(w, v.z, o[i][4 * j + 2]);
                                o[i][4 * j + 3] = fmaf(w, v.w, o[i][4 * j + 3]);
                            }
                        }
                    }
                }
            };
            if (edge) outputs(std::true_type{});
            else outputs(std::false_type{});
            __syncthreads();                           // the values have been read
            copy(v_head, s.v, u + 1);
        }
        cp_async_wait<0>();
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = ty * kRows + i;
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

template <int kDim>
cudaError_t launch(const Args &a, cudaStream_t stream) {
    const auto fn = f32_kernel<kDim>;
    const int smem = static_cast<int>(sizeof(Smem<kDim>)), grid = sm_count();
    if (!ensure_smem(reinterpret_cast<const void *>(fn), smem)) return cudaGetLastError();
    fn<<<grid, kThreads, smem, stream>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? e : launch_join<float, 16 * rows_of(kDim), kDim>(a, grid, stream);
}

}  // namespace

Shape f32_shape(int head_dim) {
    const int dim = (head_dim + 63) / 64 * 64;
    return Shape{1, part_floats(16 * rows_of(dim), dim) * 4};
}

cudaError_t f32_launch(const Args &a, cudaStream_t stream) {
    if (a.kv.head_dim <= 64) return launch<64>(a, stream);
    if (a.kv.head_dim <= 128) return launch<128>(a, stream);
    if (a.kv.head_dim <= 192) return launch<192>(a, stream);
    return launch<256>(a, stream);
}

}  // namespace chunk
}  // namespace b200
