// What the kernels of b200_kv_attend_chunk share: how the work is dealt out,
// and the parts of tiles that several CTAs compute.
//
// The query heads that read a cache head and a sequence's new tokens are packed
// into rows, row = token * group + head of the group; M consecutive rows are a
// tile. A tile sees a range of slots, cut into units of N, and what it takes to
// begin and end it counts as C more units before them. All units, in the order
// cache head, sequence, tile, slot, are dealt out in equal stretches to the CTAs
// of a grid that fits the GPU at once, whatever the lengths, which only the
// device knows; a stretch that ends among a tile's C leaves all of it to the
// next. A tile that lies in more than one stretch is joined by a second kernel
// from the parts (m, l, O) that the CTAs leave in the workspace, in the order of
// its slots, so that the result does not depend on timing.
#pragma once

#include "common.cuh"
#include "serve_dev.cuh"

namespace b200 {
namespace chunk {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// A tile whose units begin in an earlier CTA's stretch, as the join needs it;
// first >= 0 only in the first such CTA's.
struct Joint {
    int first, last;       // the CTAs that have parts of it
    int from, n;           // the sequence's rows of q
    int tile, head;
};

struct Args {
    KvView kv;
    unsigned long long page_magic;     // slot / page_size = slot * page_magic >> 40 (slot < 2^20)
    const char *q;
    char *out;
    float *lse;
    const int *offsets;
    long long q_token, q_head, out_token, out_head;  // bytes
    int n_tokens, n_head, group, window;
    unsigned group_magic;              // x / group = x * group_magic >> 32 for x * group < 2^32, a group of 1 apart
    float scale;                       // times log2(e)
    Joint *joints;                     // [grid]
    float *parts;                      // [grid][2] parts: O [M][dim], m [M], l [M]
    unsigned *status;
};

// Floats of a part.
__host__ __device__ constexpr long long part_floats(int m, int dim) { return static_cast<long long>(m) * (dim + 2); }

struct Sequence {
    int b, from, n, length;            // its rows of q, slots in use
};

__device__ __forceinline__ Sequence sequence(const Args &a, int b) {
    Sequence s;
    s.b = b;
    s.from = min(max(a.offsets[b], 0), a.n_tokens);
    s.n = max(min(max(a.offsets[b + 1], 0), a.n_tokens) - s.from, 0);
    s.length = kv_length(a.kv, b);
    return s;
}

// The units of a tile: first and how many (at least one, so that its rows are
// written). Packed rows fit 31 bits: there are at most 2^30 query heads in a call.
template <int M, int N>
__device__ __forceinline__ int2 units_of(const Args &a, int n, int length, int tile) {
    const int i1 = min(n - 1, ((tile + 1) * M - 1) / a.group);
    const int hi = max(length - n + i1 + 1, 0);
    const int lo = a.window ? max(0, length - n + tile * M / a.group - a.window + 1) : 0;
    const int u0 = min(lo, hi) / N;
    return make_int2(u0, max((hi + N - 1) / N - u0, 1));
}

// Inclusive sum over the CTA of T threads; *total is all of it.
template <int T>
__device__ __forceinline__ int scan(int x, int *s_warp, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
        const int u = __shfl_up_sync(kFullMask, x, i);
        if (lane >= i) x += u;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int w = lane < T / 32 ? s_warp[lane] : 0;
    const int own = w;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
        const int u = __shfl_up_sync(kFullMask, w, i);
        if (lane >= i) w += u;
    }
    *total = __shfl_sync(kFullMask, w, 31);
    return x + __shfl_sync(kFullMask, w - own, warp);
}

// Where a CTA's stretch begins and how long it is.
struct Stretch {
    long long left;                    // units
    int head, b, tile, skip;           // its first unit is the skip-th of that tile, its C included
    int first, last;                   // CTAs with units of that tile, its C not included
};

// A stretch's part of one tile.
struct Fragment {
    int used;                          // units of the stretch
    int u0, u1;                        // slots by N; none where they are equal
    int row0, rows;                    // first packed row, all of the sequence's
    int first;                         // the slot of the first new token
    bool begins, whole;                // has the tile's first unit, has all of them
    int last_all, first_all;           // slots that every row sees lie between
};

template <int M, int N, int C>
__device__ __forceinline__ Fragment fragment(const Args &a, const Sequence &q, int tile, int skip, long long left) {
    Fragment f;
    const int2 all = units_of<M, N>(a, q.n, q.length, tile);
    const int end = static_cast<int>(min(static_cast<long long>(all.y + C), skip + left)), from = max(skip - C, 0);
    f.used = end - skip;
    f.u0 = all.x + from;
    f.u1 = all.x + max(end - C, from);
    f.row0 = tile * M;
    f.rows = q.n * a.group;
    f.first = q.length - q.n;
    f.begins = from == 0;
    f.whole = f.u1 - f.u0 == all.y;
    f.last_all = f.first + f.row0 / a.group;
    f.first_all = a.window ? f.first + min(f.rows - 1, f.row0 + M - 1) / a.group - a.window + 1 : 0;
    return f;
}

template <int T>
struct Shared {
    int warp[32], tiles[T], n[T], length[T];
    int b, tile, skip, count;
    long long before;                  // units before the tile
};

// Found by the whole CTA (T threads): sums of the tiles' units, T tiles at a
// time, first for their total, then up to the stretch's first. A thread has a
// tile, found by a search in the sums of the tiles of T sequences.
template <int M, int N, int C, int T>
__device__ __forceinline__ Stretch find(const Args &a, Shared<T> *s) {
    const int tid = threadIdx.x;
    long long sum = 0, target = -1, units = 0, begin = 0, end = 0, ctas = 0;
    int head = 0;
    struct Mine {
        int b, tile, count;
        long long before;
        bool any;
    } mine{};
    const auto keep = [&](const Mine &x) {
        if (!x.any || target < x.before || target >= x.before + x.count) return;
        s->b = x.b;
        s->tile = x.tile;
        s->count = x.count;
        s->skip = static_cast<int>(target - x.before);
        s->before = x.before;
    };
    int rounds = 0;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        long long run = 0;
#pragma unroll 1
        for (int base = 0; base < a.kv.batch; base += T) {
            int tiles = 0;
            if (base + tid < a.kv.batch) {
                const Sequence q = sequence(a, base + tid);
                tiles = (q.n * a.group + M - 1) / M;
                s->n[tid] = q.n;
                s->length[tid] = q.length;
            }
            int total;
            const int upto = scan<T>(tiles, s->warp, &total);
            s->tiles[tid] = upto;
            __syncthreads();
#pragma unroll 1
            for (int k0 = 0; k0 < total; k0 += T) {
                const int k = k0 + tid;
                int lo = 0, count = 0, tile = 0;
                if (k < total) {
                    int hi = min(T, a.kv.batch - base) - 1;
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        if (s->tiles[mid] > k) hi = mid; else lo = mid + 1;
                    }
                    tile = k - (lo ? s->tiles[lo - 1] : 0);
                    count = units_of<M, N>(a, s->n[lo], s->length[lo], tile).y + C;
                }
                int all;
                const int to = scan<T>(count, s->warp, &all);
                mine = Mine{base + lo, tile, count, run + to - count, k < total};
                if (pass) keep(mine);
                run += all;
                ++rounds;
            }
            __syncthreads();
        }
        if (pass == 0) {
            sum = run;
            units = sum * a.kv.n_head_kv;
            ctas = min(static_cast<long long>(gridDim.x), units);      // each with a unit at least
            if (blockIdx.x >= ctas) return Stretch{0, 0, 0, 0, 0, 0, 0};
            begin = units * blockIdx.x / ctas;
            end = units * (blockIdx.x + 1) / ctas;
            head = static_cast<int>(begin / sum);
            target = begin - head * sum;
            if (rounds == 1) {             // every thread still has the only tile it saw
                keep(mine);
                break;
            }
        }
    }
    __syncthreads();
    Stretch r;
    r.left = end - begin;
    r.head = head;
    r.b = s->b;
    r.tile = s->tile;
    r.skip = s->skip;
    const long long u0 = head * sum + s->before + C, u1 = u0 + s->count - C - 1;
    r.first = static_cast<int>(((u0 + 1) * ctas - 1) / units);
    r.last = static_cast<int>(((u1 + 1) * ctas - 1) / units);
    return r;
}

// The next tile: of the sequence, of the next sequence that has rows, of the next head.
template <int M>
__device__ __forceinline__ void next_tile(const Args &a, Sequence &q, int &tile, int &head) {
    if (++tile * M < q.n * a.group) return;
    tile = 0;
    int b = q.b;
    do {
        if (++b == a.kv.batch) b = 0, ++head;
        q = sequence(a, b);
    } while (q.n == 0);
}

// 16 bytes from global memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Byte of the 16-byte piece c of row r in a tile of `rows` rows, 64 16-bit columns beside 64.
__device__ __forceinline__ uint32_t piece(int rows, int r, int c) {
    return static_cast<uint32_t>((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <typename T>
__device__ __forceinline__ void store4(char *p, float4 v) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = v;
    } else {
        T e[4] = {from_float<T>(v.x), from_float<T>(v.y), from_float<T>(v.z), from_float<T>(v.w)};
        *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(e);
    }
}

constexpr int kJoinRows = 8;             // CTAs of 8 warps to a tile

// A split tile's rows from their parts, a warp for each: with m the largest of
// the parts', out = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i.
template <typename T, int M, int kDim>
__global__ void __launch_bounds__(256) join_kernel(const Args a) {
    pdl_wait_prior_grid();
    const Joint j = a.joints[blockIdx.x];
    if (j.first < 0) return;
    const int lane = threadIdx.x & 31;
    // the first CTA's stretch ends with its part, the others' begin with theirs
    const auto part = [&](int c) { return a.parts + (2ll * c + (c == j.first)) * part_floats(M, kDim); };
#pragma unroll 1
    for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < M; r += kJoinRows * 8) {
        const int row = j.tile * M + r;
        if (row >= j.n * a.group) return;
        const int i = row / a.group, h = j.head * a.group + row - i * a.group;
        // a lane's parts' references, and the largest
        float m = -INFINITY;
        for (int c = j.first + lane; c <= j.last; c += 32) {
            const float x = part(c)[M * kDim + r];
            m = x > m || x != x ? x : m;   // NaN stays
        }
#pragma unroll
        for (int x = 16; x; x >>= 1) {
            const float y = __shfl_xor_sync(kFullMask, m, x);
            m = y > m || y != y ? y : m;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        constexpr int kPer = (kDim + 127) / 128;
        float l = 0.0f;
        float4 o[kPer] = {};
#pragma unroll 4
        for (int c = j.first; c <= j.last; ++c) {
            const float *p = part(c);
            const float w = exp2f(p[M * kDim + r] - ref);
            l = fmaf(w, p[M * kDim + M + r], l);
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int at = k * 128 + lane * 4;
                if (at >= kDim) break;
                const float4 x = *reinterpret_cast<const float4 *>(p + static_cast<long long>(r) * kDim + at);
                // a value that is not finite and seen counts however small its part's weight is, 0 included
                o[k] = make_float4(fmaf(w, x.x, o[k].x), fmaf(w, x.y, o[k].y), fmaf(w, x.z, o[k].z), fmaf(w, x.w, o[k].w));
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        char *out = a.out + (j.from + i) * a.out_token + h * a.out_head;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int at = k * 128 + lane * 4;
            if (at < a.kv.head_dim) store4<T>(out + at * static_cast<int>(sizeof(T)), make_float4(o[k].x * inv, o[k].y * inv, o[k].z * inv, o[k].w * inv));
        }
        if (a.lse && lane == 0) a.lse[static_cast<long long>(j.from + i) * a.n_head + h] = (m + log2f(l)) * kLn2;
    }
}

template <typename T, int M, int kDim>
cudaError_t launch_join(const Args &a, int grid, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid, kJoinRows);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<T, M, kDim>, a);
}

// Each launches calls of its types: kv_chunk_mma.cu those with 16-bit queries,
// kv_chunk_split.cu float32 queries with a float16 cache, kv_chunk_f32.cu all in
// float32; CTAs to an SM and bytes of a part of its tiles for the workspace.
struct Shape {
    int ctas;
    long long part;
};
Shape mma_shape(int head_dim);
cudaError_t mma_launch(const Args &a, int kv_dtype, cudaStream_t stream);
Shape split_shape(int head_dim);
cudaError_t split_launch(const Args &a, cudaStream_t stream);
Shape f32_shape(int head_dim);
cudaError_t f32_launch(const Args &a, cudaStream_t stream);

}  // namespace chunk
}  // namespace b200
