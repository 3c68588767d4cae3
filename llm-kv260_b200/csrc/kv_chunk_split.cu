// b200_kv_attend_chunk for float32 queries and a float16 cache.
//
// Both products run on the tensor cores (mma.sync, warp by warp, 16 rows each)
// with the float32 operand in two parts of float16, x = high + 2^-11 low, 22
// bits: S = Qh K^T + 2^-11 Ql K^T and O = Ph V + 2^-11 Pl V. The factor keeps the
// low part a normal number wherever the high part is one. A row's queries are
// multiplied by a power of two first, the largest to [2^14, 2^15), so that an
// element 2^-j of it keeps 22 bits, or 50 - j where that is less; the scale
// takes it back. A unit's weights are taken relative to its own largest, which
// becomes 2^15, so those down to 2^-29 of it keep 22 bits; smaller ones, which
// matter where larger ones meet small values, take products of their own, 2^29
// times larger, until none is left (one more round for scores that differ by 20
// to 40 nats within 64 slots, none for most). The tensor cores cut sums off at
// 24 bits instead of rounding them, so the small parts are summed first, S in
// sums of its own for both parts, and a unit's 64 slots are added to the output
// outside of them: eight cuts of S and four of what a unit adds, each below
// 2^-24 (40 tokens behind 8000 slots: 5.1e-7 of the output's norm off the exact
// one; behind 120000: 5.3e-7).
//
// What bounds it: the products, twice as many as in 16 bits and at the rate of
// mma.sync, 255 registers and with them 8 warps an SM, two CTAs up to head_dim
// 128. 4 chunks of 100 to 333 tokens behind up to 2000 slots (24 heads, 8 of the
// cache, 128): 201 us, 114 TFLOP/s of the float32 products' (307 us with one CTA
// to an SM, 802 on the float32 units); 2000 tokens from the start, 32 heads: 311
// us, 105 TFLOP/s, with scores that differ by tens of nats within 64 slots 760.
#include <cuda_runtime.h>

#include "kv_chunk.cuh"

namespace b200 {
namespace chunk {

namespace {

constexpr int kM = 64, kN = 64, kThreads = 128;
constexpr int kCost = 2;               // units that a tile's begin and end take
constexpr float kTop = 15.0f;          // a unit's largest weight is 2^15, in float16's range with its low part's 2^14
constexpr float kLeast = 0x1p-14f, kRound = 0x1p29f;   // of a round of products the least weight, and what the next one's grow by
constexpr float kLow = 0x1p11f;        // factor of the low parts
// The reference m of l and O is a maximum of some time ago: it moves, and they are multiplied, where it is passed by 2^8.
constexpr float kSlack = 8.0f;

template <int kDim>
struct Smem {
    __half q[2][kM * kDim];            // high and low parts
    __half kv[2][2][kN * kDim];        // keys and values of two units
    long long row[2][kN];              // byte offset of a slot's row, -1: not there
    int shift[kM];                     // exponents that the queries were multiplied by
    Shared<kThreads> find;
};

__device__ __forceinline__ void load_matrices(uint32_t (&v)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void load_matrices_turned(uint32_t (&v)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void multiply(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }

// Two CTAs to an SM of 228 KB, of which each takes 1 KB for itself.
static_assert(2 * (sizeof(Smem<128>) + 1024) <= 228 * 1024);

template <int kDim>
__global__ void __launch_bounds__(kThreads, kDim <= 128 ? 2 : 1) split_kernel(const Args a) {
    extern __shared__ __align__(128) char smem_raw[];
    Smem<kDim> &s = *reinterpret_cast<Smem<kDim> *>(smem_raw);
    constexpr int kPieces = kDim / 8;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, d = a.kv.head_dim, filled = d / 8;
    Stretch st = find<kM, kN, kCost, kThreads>(a, &s.find);
    if (tid == 0) a.joints[blockIdx.x].first = -1;
    if (st.left == 0) return;
    Sequence q = sequence(a, st.b);
    int tile = st.tile, head = st.head, skip = st.skip;
    if (skip > kCost && tid == 0 && st.first + 1 == static_cast<int>(blockIdx.x))
        a.joints[blockIdx.x] = Joint{st.first, st.last, q.from, q.n, tile, head};
    const uint32_t q_at = smem_addr(s.q), kv_at = smem_addr(s.kv);
#pragma unroll 1
    for (;;) {
        const Fragment f = fragment<kM, kN, kCost>(a, q, tile, skip, st.left);
        if (f.u1 > f.u0) {
        const char *k_head = a.kv.k + head * a.kv.head_stride, *v_head = a.kv.v + head * a.kv.head_stride;
        // A unit's rows are looked up a unit ahead, and its copies asked for two ahead.
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
        const auto copy = [&](int u) {
            if (u < f.u1) {
                const uint32_t to = kv_at + (u & 1) * (2 * kN * kDim * 2);
#pragma unroll 4
                for (int i = tid; i < kN * kPieces; i += kThreads) {
                    const int r = i / kPieces, c = i % kPieces;
                    const long long at = s.row[u & 1][r];
                    const bool there = at >= 0 && c < filled;
                    const long long off = there ? at + c * 16 : 0;
                    copy16(to + piece(kN, r, c), k_head + off, there);
                    copy16(to + kN * kDim * 2 + piece(kN, r, c), v_head + off, there);
                }
            }
            cp_async_commit();
        };
        ask(f.u0);
        place(f.u0);
        ask(f.u0 + 1);
        __syncthreads();
        copy(f.u0);
        place(f.u0 + 1);
        ask(f.u0 + 2);
        // The queries, two threads to a row: the largest, its power of two, both parts.
        {
            const int r = tid >> 1, side = tid & 1;
            const bool there = f.row0 + r < f.rows;
            const int token = (f.row0 + r) / a.group, h = head * a.group + f.row0 + r - token * a.group;
            const float *src = reinterpret_cast<const float *>(a.q + (q.from + token) * a.q_token + h * a.q_head);
            float top = 0.0f;
            for (int c = side * 4; there && c < d; c += 8) {
                const float4 x = *reinterpret_cast<const float4 *>(src + c);
                top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
            }
            top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
            int e = 0;                                 // top * 2^e in [2^14, 2^15); what is not finite stays as it is
            if (top > 0.0f && top < INFINITY) e = min(max(14 - ilogbf(top), -126), 126);
            const float by = __int_as_float((127 + e) << 23);
            if (side == 0) s.shift[r] = e;
            for (int c = side; c < kPieces; c += 2) {
                float x[8] = {};
                if (there && c < filled) {
                    const float4 u = *reinterpret_cast<const float4 *>(src + c * 8), v = *reinterpret_cast<const float4 *>(src + c * 8 + 4);
                    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
                }
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float y0 = x[2 * k] * by, y1 = x[2 * k + 1] * by;
                    hi[k] = pack(y0, y1);
                    const float2 z = unpack(hi[k]);
                    const float l0 = (y0 - z.x) * kLow, l1 = (y1 - z.y) * kLow;
                    lo[k] = pack(l0 - l0 == 0.0f ? l0 : 0.0f, l1 - l1 == 0.0f ? l1 : 0.0f);
                }
                const uint32_t at = piece(kM, r, c);
                *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(s.q[0]) + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(s.q[1]) + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        __syncthreads();
        copy(f.u0 + 1);
        // This thread's rows: lane / 4 and the 8th behind it, of its warp's 16.
        const int r0 = warp * 16 + (lane >> 2);
        int at[2];
        float scale[2], ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int r = f.row0 + r0 + 8 * x;
            at[x] = r < f.rows ? f.first + r / a.group : -1;
            scale[x] = ldexpf(a.scale, -s.shift[r0 + 8 * x]);
        }
        float o[kDim / 8][4];
#pragma unroll
        for (int n = 0; n < kDim / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        const bool busy = f.row0 + warp * 16 < f.rows;
#pragma unroll 1
        for (int u = f.u0; u < f.u1; ++u) {
            cp_async_wait<1>();
            __syncthreads();
            const uint32_t k_at = kv_at + (u & 1) * (2 * kN * kDim * 2), v_at = k_at + kN * kDim * 2;
            const bool edge = (u + 1) * kN - 1 > f.last_all || u * kN < f.first_all;
            const bool gap = __syncthreads_or(tid < kN && s.row[u & 1][tid] < 0);
            if (edge) {
                // Where rows see different slots, 0 times a value that is not finite must not reach a row that does not see
                // it: such values make NaN of what they enter in the rows that see them, and become 0.
                const auto odd = [](uint32_t x) { return (x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u; };
                uint4 *v = reinterpret_cast<uint4 *>(s.kv[u & 1][1]);
                bool bad = false;
                for (int i = tid; i < kN * kPieces; i += kThreads) {
                    const uint4 w = v[i];
                    bad |= odd(w.x) || odd(w.y) || odd(w.z) || odd(w.w);
                }
                if (__syncthreads_or(bad)) {
#pragma unroll 1
                    for (int c = 0; c < kN; ++c) {
                        const int slot = u * kN + c;
                        bool sees[2];
#pragma unroll
                        for (int x = 0; x < 2; ++x) sees[x] = slot <= at[x] && !(a.window && slot <= at[x] - a.window);
#pragma unroll
                        for (int n = 0; n < kDim / 8; ++n) {
                            const uint32_t w = *reinterpret_cast<const uint32_t *>(reinterpret_cast<const char *>(v) + piece(kN, c, n) + (lane & 3) * 4);
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                if (sees[x] && odd(w & 0xffffu)) o[n][2 * x] = NAN;
                                if (sees[x] && odd(w & 0xffff0000u)) o[n][2 * x + 1] = NAN;
                            }
                        }
                    }
                    __syncthreads();
                    const auto finite = [&](uint32_t w) { return (odd(w & 0xffffu) ? 0u : w & 0xffffu) | (odd(w & 0xffff0000u) ? 0u : w & 0xffff0000u); };
                    for (int i = tid; i < kN * kPieces; i += kThreads) {
                        const uint4 w = v[i];
                        v[i] = make_uint4(finite(w.x), finite(w.y), finite(w.z), finite(w.w));
                    }
                    __syncthreads();
                }
            }
            if (busy) {
                float hi[8][4] = {}, lo[8][4] = {};
#pragma unroll
                for (int k = 0; k < kDim / 16; ++k) {
                    uint32_t qh[4], ql[4];
                    const uint32_t q_piece = piece(kM, warp * 16 + (lane & 15), 2 * k + (lane >> 4));
                    load_matrices(qh, q_at + q_piece);
                    load_matrices(ql, q_at + kM * kDim * 2 + q_piece);
#pragma unroll
                    for (int n = 0; n < 8; n += 2) {
                        uint32_t b[4];
                        load_matrices(b, k_at + piece(kN, n * 8 + (lane & 7) + (lane >> 4) * 8, 2 * k + (lane >> 3 & 1)));
                        multiply(lo[n], ql, b[0], b[1]);
                        multiply(lo[n + 1], ql, b[2], b[3]);
                        multiply(hi[n], qh, b[0], b[1]);
                        multiply(hi[n + 1], qh, b[2], b[3]);
                    }
                }
                bool nan = false;
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        hi[n][k] = fmaf(lo[n][k], 1 / kLow, hi[n][k]) * scale[k >> 1];
                        nan |= hi[n][k] != hi[n][k];
                    }
                if (__any_sync(kFullMask, nan)) {      // an infinite key, perhaps, whose products with both parts differ in sign
#pragma unroll
                    for (int n = 0; n < 8; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int r = f.row0 + r0 + 8 * (k >> 1), slot = n * 8 + (lane & 3) * 2 + (k & 1);
                            if (hi[n][k] == hi[n][k] || r >= f.rows) continue;
                            const int token = r / a.group, h = head * a.group + r - token * a.group;
                            const float *src = reinterpret_cast<const float *>(a.q + (q.from + token) * a.q_token + h * a.q_head);
                            float sum = 0.0f;
                            for (int c = 0; c < d; ++c)
                                sum = fmaf(src[c], __half2float(*reinterpret_cast<const __half *>(reinterpret_cast<const char *>(s.kv[u & 1][0]) + piece(kN, slot, c >> 3) + (c & 7) * 2)), sum);
                            hi[n][k] = sum * a.scale;
                        }
                    __syncwarp();
                }
                if (edge || gap) {
#pragma unroll
                    for (int n = 0; n < 8; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int c = n * 8 + (lane & 3) * 2 + (k & 1), slot = u * kN + c;
                            if (slot > at[k >> 1] || (a.window && slot <= at[k >> 1] - a.window) || s.row[u & 1][c] < 0) hi[n][k] = -INFINITY;
                        }
                }
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    top[0] = fmaxf(top[0], fmaxf(hi[n][0], hi[n][1]));
                    top[1] = fmaxf(top[1], fmaxf(hi[n][2], hi[n][3]));
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    top[x] = fmaxf(top[x], __shfl_xor_sync(kFullMask, top[x], 1));
                    top[x] = fmaxf(top[x], __shfl_xor_sync(kFullMask, top[x], 2));
                }
                if (__any_sync(kFullMask, top[0] > ref[0] + kSlack || top[1] > ref[1] + kSlack)) {
                    float keep[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        // of the warp's rows only those that need it: a row's bits do not depend on another's scores
                        const float next = top[x] > ref[x] + kSlack ? top[x] : ref[x];
                        keep[x] = next == ref[x] ? 1.0f : exp2f(ref[x] - next);
                        ref[x] = next;
                        l[x] *= keep[x];
                    }
#pragma unroll
                    for (int n = 0; n < kDim / 8; ++n) {
                        o[n][0] *= keep[0], o[n][1] *= keep[0];
                        o[n][2] *= keep[1], o[n][3] *= keep[1];
                    }
                }
                // The unit's weights beside its own largest, and what they count in l and O.
                float off[2], factor[2], sum[2] = {0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    off[x] = top[x] == -INFINITY ? 0.0f : top[x] - kTop;
                    factor[x] = top[x] == -INFINITY ? 0.0f : exp2f(off[x] - ref[x]);
                }
                bool small = false;                    // a weight below a round's least, 0 included
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        hi[n][k] = exp2f(hi[n][k] - off[k >> 1]);
                        sum[k >> 1] += hi[n][k];
                        small |= hi[n][k] < kLeast;
                    }
                l[0] = fmaf(sum[0], factor[0], l[0]);
                l[1] = fmaf(sum[1], factor[1], l[1]);
                const auto products = [&](float (&w)[8][4]) {      // O += factor W V
                    uint32_t ph[4][4], pl[4][4];   // the weights as operands of 16 slots each
#pragma unroll
                    for (int n = 0; n < 8; ++n)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t p = pack(w[n][2 * x], w[n][2 * x + 1]);
                            const float2 z = unpack(p);
                            ph[n >> 1][(n & 1) * 2 + x] = p;
                            pl[n >> 1][(n & 1) * 2 + x] = pack((w[n][2 * x] - z.x) * kLow, (w[n][2 * x + 1] - z.y) * kLow);
                        }
#pragma unroll
                    for (int n = 0; n < kDim / 8; n += 2) {
                        float t[2][4] = {};
                        uint32_t b[4][4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            load_matrices_turned(b[k], v_at + piece(kN, k * 16 + (lane & 15), n + (lane >> 4)));
                            multiply(t[0], pl[k], b[k][0], b[k][1]);
                            multiply(t[1], pl[k], b[k][2], b[k][3]);
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) t[0][k] *= 1 / kLow, t[1][k] *= 1 / kLow;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            multiply(t[0], ph[k], b[k][0], b[k][1]);
                            multiply(t[1], ph[k], b[k][2], b[k][3]);
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            o[n][k] = fmaf(t[0][k], factor[k >> 1], o[n][k]);
                            o[n + 1][k] = fmaf(t[1][k], factor[k >> 1], o[n + 1][k]);
                        }
                    }
                };
                // rounds for weights that are too small for this one; none for most
                while (__builtin_expect(__any_sync(kFullMask, small), 0)) {
                    float w[8][4];
                    bool left = false;
                    small = false;
#pragma unroll
                    for (int n = 0; n < 8; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) left |= hi[n][k] > 0.0f && hi[n][k] < kLeast;
                    if (!__any_sync(kFullMask, left)) break;
#pragma unroll
                    for (int n = 0; n < 8; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            w[n][k] = hi[n][k] < kLeast ? 0.0f : hi[n][k];
                            hi[n][k] = hi[n][k] < kLeast ? hi[n][k] * kRound : 0.0f;
                            small |= hi[n][k] < kLeast;
                        }
                    products(w);
                    factor[0] *= 1 / kRound, factor[1] *= 1 / kRound;
                }
                products(hi);
            }
            __syncthreads();                           // the stage and its rows are free
            if (u + 2 < f.u1) {
                place(u + 2);
                ask(u + 3);
            }
            __syncthreads();
            copy(u + 2);
        }
        cp_async_wait<0>();
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            l[x] += __shfl_xor_sync(kFullMask, l[x], 1);
            l[x] += __shfl_xor_sync(kFullMask, l[x], 2);
            const int r = r0 + 8 * x, row = f.row0 + r;
            if (row >= f.rows) continue;
            const int token = row / a.group, h = head * a.group + row - token * a.group;
            if (f.whole) {
                const float inv = l[x] == 0.0f ? 0.0f : 1.0f / l[x];
                char *out = a.out + (q.from + token) * a.out_token + h * a.out_head;
#pragma unroll
                for (int n = 0; n < kDim / 8; ++n)
                    if (n < filled)
                        *reinterpret_cast<float2 *>(out + (n * 8 + (lane & 3) * 2) * 4) = make_float2(o[n][2 * x] * inv, o[n][2 * x + 1] * inv);
                if (a.lse && (lane & 3) == 0)
                    a.lse[static_cast<long long>(q.from + token) * a.n_head + h] = (ref[x] + log2f(l[x])) * kLn2;
            } else {
                float *part = a.parts + (2ll * blockIdx.x + f.begins) * part_floats(kM, kDim);
#pragma unroll
                for (int n = 0; n < kDim / 8; ++n)
                    *reinterpret_cast<float2 *>(part + r * kDim + n * 8 + (lane & 3) * 2) = make_float2(o[n][2 * x], o[n][2 * x + 1]);
                if ((lane & 3) == 0) {
                    part[kM * kDim + r] = ref[x];
                    part[kM * kDim + kM + r] = l[x];
                }
            }
        }
        __syncwarp();
        }
        st.left -= f.used;
        if (st.left <= 0) break;
        skip = 0;
        next_tile<kM>(a, q, tile, head);
        __syncthreads();
    }
}

// As many CTAs as the GPU holds at once: two of four warps to an SM for head_dim
// up to 128, one above.
template <int kDim>
int ctas_of() {
    return resident_ctas(reinterpret_cast<const void *>(split_kernel<kDim>), kThreads, static_cast<int>(sizeof(Smem<kDim>)));
}

template <int kDim>
cudaError_t launch(const Args &a, cudaStream_t stream) {
    const auto fn = split_kernel<kDim>;
    const int smem = static_cast<int>(sizeof(Smem<kDim>)), grid = sm_count() * ctas_of<kDim>();
    if (!ensure_smem(reinterpret_cast<const void *>(fn), smem)) return cudaGetLastError();
    fn<<<grid, kThreads, smem, stream>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? e : launch_join<float, kM, kDim>(a, grid, stream);
}

}  // namespace

Shape split_shape(int head_dim) {
    const int dim = (head_dim + 63) / 64 * 64;
    const int ctas = dim <= 64 ? ctas_of<64>() : dim <= 128 ? ctas_of<128>() : dim <= 192 ? ctas_of<192>() : ctas_of<256>();
    return Shape{ctas, part_floats(kM, dim) * 4};
}

cudaError_t split_launch(const Args &a, cudaStream_t stream) {
    if (a.kv.head_dim <= 64) return launch<64>(a, stream);
    if (a.kv.head_dim <= 128) return launch<128>(a, stream);
    if (a.kv.head_dim <= 192) return launch<192>(a, stream);
    return launch<256>(a, stream);
}

}  // namespace chunk
}  // namespace b200
