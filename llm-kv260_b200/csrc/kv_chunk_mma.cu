// b200_kv_attend_chunk for 16-bit queries, on the tensor cores.
#include <cuda_runtime.h>

#include "kv_chunk.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace chunk {

namespace {

constexpr int kThreads = 384;          // two warpgroups of softmax, one warp of products, three of copies
constexpr int kCopiers = 96;
constexpr int kLag = 2;                // copies that a copier leaves in flight behind the newest one
constexpr int kColumns = 512;          // of tensor memory
// The reference m trails the maximum by 7 to 15 powers of two: weights stay in
// 2^15 and below, float16's range, and those of 2^-21 of the largest are still
// normal numbers there.
constexpr float kLead = 7.0f, kSlack = 15.0f;

template <int kDim>
struct Plan {
    static constexpr int kTiles = kDim <= 128 ? 2 : 1;     // of 128 rows
    static constexpr int kM = 128 * kTiles, kN = kDim <= 128 ? 128 : 64;
    static constexpr int kStages = kDim <= 64 ? 6 : 4;
    static constexpr int kQBytes = kM * kDim * 2, kStageBytes = kN * kDim * 2;
    static constexpr int kSmem = 1024 + kQBytes + kStages * kStageBytes;
    // columns of tensor memory: scores (and, over them, weights) per tile, or twice of one, then the outputs
    __device__ static constexpr int scores(int i) { return i * kN; }
    __device__ static constexpr int output(int i) { return 256 + i * kDim; }
};

struct Shared0 {
    uint64_t full[6], free[6], q_full, q_free, s_full[2], p_full[2], o_done[2], mask_full[2], mask_free[2], last;
    uint32_t tmem;
    uint32_t mask[2][4];               // a unit's slots that are there
    long long row[2][128];             // byte offsets of their rows
    uint32_t bad[256][8];              // a row's columns that a value which is not finite enters
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack(float lo, float hi, __half) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// An element of the pair that is not finite.
__device__ __forceinline__ bool not_finite(uint32_t w, __half) { return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u; }
__device__ __forceinline__ bool not_finite(uint32_t w, __nv_bfloat16) {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
template <typename T>
__device__ __forceinline__ uint32_t only_finite(uint32_t w) {
    if (not_finite(w & 0xffffu, T())) w &= 0xffff0000u;
    if (not_finite(w & 0xffff0000u, T())) w &= 0xffffu;
    return w;
}

__device__ __forceinline__ bool any_of(uint32_t id, uint32_t threads, bool mine) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(mine)), "r"(id), "r"(threads)
        : "memory");
    return r != 0;
}

// A thread's waits. One that runs out says so in the status word and is the
// last: the thread goes on without waiting, so that it meets every barrier that
// the others meet and the CTA comes to its end.
struct Waiter {
    unsigned *status;
    bool dead = false;
    __device__ __forceinline__ void operator()(uint64_t *bar, int phase) {
        if (!dead) dead = !wait_stage(bar, phase & 1, status);
    }
};

// 16 bytes from global memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Byte of the 16-byte piece c of row r in a tile of `rows` rows.
__device__ __forceinline__ uint32_t piece(int rows, int r, int c) {
    return static_cast<uint32_t>((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// A stretch's part of one tile.
struct Fragment {
    int u0, u1, first;                 // units, the slot of the first new token
    long long row0, rows;              // first packed row, all of the sequence's
    bool whole;
    int last_all, first_all;           // slots that every row sees lie between
};

template <int kM, int kN>
__device__ __forceinline__ Fragment fragment(const Args &a, const Sequence &q, int tile, int skip, long long left) {
    Fragment f;
    const int2 all = units_of<kM, kN>(a, q.n, q.length, tile);
    f.u0 = all.x + skip;
    f.u1 = all.x + static_cast<int>(min(static_cast<long long>(all.y), skip + left));
    f.first = q.length - q.n;
    f.rows = static_cast<long long>(q.n) * a.group;
    f.row0 = static_cast<long long>(tile) * kM;
    f.whole = f.u1 - f.u0 == all.y;
    f.last_all = f.first + static_cast<int>(f.row0 / a.group);
    f.first_all = a.window ? f.first + static_cast<int>(min(f.rows - 1, f.row0 + kM - 1) / a.group) - a.window + 1 : 0;
    return f;
}

// The copies of keys, values and queries into shared memory.
template <typename T, int kDim>
__device__ __forceinline__ void copier(const Args &a, Shared0 &s, char *smem, Stretch st, unsigned *status) {
    using P = Plan<kDim>;
    constexpr int kPieces = kDim / 8;
    const int tid = threadIdx.x - (kThreads - kCopiers), lane = tid & 31;
    const int pieces = (a.kv.head_dim + 15) / 16 * 2, filled = a.kv.head_dim / 8;
    const uint32_t q_at = smem_addr(smem), ring = q_at + P::kQBytes;
    uint64_t *older = nullptr, *newer = nullptr;       // barriers of the copies in flight
    const auto emit = [&](uint64_t *bar) {
        cp_async_commit();
        cp_async_wait<kLag>();
        if (older) {
            fence_async_proxy();
            mbar_arrive(older);
        }
        older = newer;
        newer = bar;
    };
    int item = 0, unit = 0, fragments = 0;
    Sequence q = sequence(a, st.b);
    int tile = st.tile, head = st.head, skip = st.skip;
    Waiter wait{status};
    for (;;) {
        const Fragment f = fragment<P::kM, P::kN>(a, q, tile, skip, st.left);
        const char *k_head = a.kv.k + head * a.kv.head_stride, *v_head = a.kv.v + head * a.kv.head_stride;
        const int *table = a.kv.table + q.b * a.kv.table_stride;
        // a thread looks up two of a unit's slots at most
        int page[2];
        const auto ask = [&](int u) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int slot = u * P::kN + tid + x * kCopiers;
                page[x] = -1;
                if (tid + x * kCopiers < P::kN && slot < q.length)
                    page[x] = table[static_cast<int>((slot * a.page_magic) >> 40)];
            }
        };
        const auto place = [&](int u) {
            const int buf = unit & 1;
            if (unit >= 2) wait(&s.mask_free[buf], (unit >> 1) - 1);
            __syncwarp();
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int r = tid + x * kCopiers, slot = u * P::kN + r;
                const bool there = static_cast<unsigned>(page[x]) < static_cast<unsigned>(a.kv.n_pages);
                const uint32_t word = __ballot_sync(kFullMask, there);
                if (r < P::kN) {
                    const int col = static_cast<int>((slot * a.page_magic) >> 40);
                    s.row[buf][r] = there ? page[x] * a.kv.page_stride + (slot - col * a.kv.page_size) * a.kv.row_stride : -1;
                    if (lane == 0) s.mask[buf][r >> 5] = word;
                }
            }
            named_sync(3, kCopiers);
            if (tid == 0) mbar_arrive(&s.mask_full[buf]);
        };
        ask(f.u0);
        if (fragments) wait(&s.q_free, fragments - 1);
        const int rows = static_cast<int>(min(static_cast<long long>(P::kM), f.rows - f.row0));
        for (int i = tid; i < (rows > 128 ? P::kM : 128) * kPieces; i += kCopiers) {
            const int r = i / kPieces, c = i % kPieces;
            if (c >= pieces) continue;
            const bool there = r < rows && c < filled;
            const char *src = a.q;
            if (there) {
                const int token = static_cast<int>((f.row0 + r) / a.group);
                const int h = static_cast<int>(f.row0 + r - static_cast<long long>(token) * a.group);
                src += (q.from + token) * a.q_token + (head * a.group + h) * a.q_head + c * 16;
            }
            copy16(q_at + (r >> 7) * (128 * kDim * 2) + piece(128, r & 127, c), src, there);
        }
        emit(&s.q_full);
        place(f.u0);
        for (int u = f.u0; u < f.u1; ++u) {
            const int buf = unit & 1;
            if (u + 1 < f.u1) ask(u + 1);
            for (int v = 0; v < 2; ++v) {
                const int stage = item % P::kStages, use = item / P::kStages;
                if (use) wait(&s.free[stage], use - 1);
                const char *src = v ? v_head : k_head;
                const uint32_t dst = ring + stage * P::kStageBytes;
#pragma unroll 8
                for (int i = tid; i < P::kN * kPieces; i += kCopiers) {
                    const int r = i / kPieces, c = i % kPieces;
                    if (c >= pieces) continue;
                    const long long at = s.row[buf][r];
                    const bool there = at >= 0 && c < filled;
                    copy16(dst + piece(P::kN, r, c), there ? src + at + c * 16 : src, there);
                }
                emit(&s.full[stage]);
                ++item;
            }
            ++unit;
            if (u + 1 < f.u1) place(u + 1);
        }
        cp_async_wait<0>();
        fence_async_proxy();
        if (older) mbar_arrive(older);
        if (newer) mbar_arrive(newer);
        older = newer = nullptr;
        ++fragments;
        st.left -= f.u1 - f.u0;
        if (st.left <= 0) break;
        skip = 0;
        next_tile<P::kM>(a, q, tile, head);
    }
}

// The matrix products, issued by one thread. Of a unit j and tile i, in order:
// S_i = Q_i K^T into the columns where the weights of the unit before were, and
// O_i += P_i V once the softmax has put the weights P_i over S_i. Products of
// one thread run in the order of issue, so a tile's next scores cannot overtake
// the use of its weights.
template <typename T, int kDim>
__device__ __forceinline__ void products(const Args &a, Shared0 &s, char *smem, Stretch st, unsigned *status) {
    using P = Plan<kDim>;
    constexpr bool kBf16 = sizeof(T) == 2 && !__is_same(T, __half);
    const int steps = (a.kv.head_dim + 15) / 16;
    const uint32_t score_desc = mma_desc(128, P::kN, kBf16, false), out_desc = mma_desc(128, steps * 16, kBf16, true);
    const uint32_t q_at = smem_addr(smem), ring = q_at + P::kQBytes, tmem = s.tmem;
    int item = 0, fragments = 0;       // copies taken (K, V, K, V ...)
    int put[2] = {0, 0};               // weights taken per buffer
    Sequence q = sequence(a, st.b);
    int tile = st.tile, head = st.head, skip = st.skip;
    Waiter wait{status};
    for (;;) {
        const Fragment f = fragment<P::kM, P::kN>(a, q, tile, skip, st.left);
        const int units = f.u1 - f.u0, tiles = P::kTiles == 2 && f.rows - f.row0 > 128 ? 2 : 1;
        const auto wait_item = [&](int i) { wait(&s.full[i % P::kStages], i / P::kStages); };
        const auto scores = [&](int i, int buf, int k_item) {
            const uint32_t qa = q_at + i * (128 * kDim * 2), kb = ring + (k_item % P::kStages) * P::kStageBytes;
            for (int x = 0; x < steps; ++x)
                mma_ss(tmem + P::scores(buf), smem_desc(qa + (x >> 2) * (128 * 128) + (x & 3) * 32, 16, 1024),
                       smem_desc(kb + (x >> 2) * (P::kN * 128) + (x & 3) * 32, 16, 1024), score_desc, x > 0);
            mma_commit(&s.s_full[buf]);
        };
        const auto outputs = [&](int i, int buf, int v_item, bool add) {
            const uint32_t vb = ring + (v_item % P::kStages) * P::kStageBytes;
#pragma unroll
            for (int x = 0; x < P::kN / 16; ++x)
                mma_ts(tmem + P::output(i), tmem + P::scores(buf) + x * 8, smem_desc(vb + x * 2048, P::kN * 128, 1024), out_desc,
                       add || x > 0);
            mma_commit(&s.o_done[i]);
        };
        wait(&s.q_full, fragments);
        wait_item(item);
        tmem_fence_after();
        for (int i = 0; i < tiles; ++i) scores(i, i, item);
        mma_commit(&s.free[item % P::kStages]);
        if (units == 1) mma_commit(&s.q_free);
        for (int j = 0; j < units; ++j) {
            const int k_next = item + 2 * j + 2, v_now = item + 2 * j + 1;
            const bool more = j + 1 < units;
            if (P::kTiles == 1 && more) {
                wait_item(k_next);
                tmem_fence_after();
                scores(0, (j + 1) & 1, k_next);
                mma_commit(&s.free[k_next % P::kStages]);
                if (j + 2 == units) mma_commit(&s.q_free);
            }
            wait_item(v_now);
            for (int i = 0; i < tiles; ++i) {
                const int buf = P::kTiles == 2 ? i : j & 1;
                wait(&s.p_full[buf], put[buf]++);
                tmem_fence_after();
                outputs(i, buf, v_now, j > 0);
                if (i == tiles - 1) mma_commit(&s.free[v_now % P::kStages]);
                if (P::kTiles == 2 && more) {
                    if (i == 0) {
                        wait_item(k_next);
                        tmem_fence_after();
                    }
                    scores(i, i, k_next);
                    if (i == tiles - 1) {
                        mma_commit(&s.free[k_next % P::kStages]);
                        if (j + 2 == units) mma_commit(&s.q_free);
                    }
                }
            }
        }
        item += 2 * units;
        ++fragments;
        st.left -= units;
        if (st.left <= 0) break;
        skip = 0;
        next_tile<P::kM>(a, q, tile, head);
    }
    mma_commit(&s.last);               // before the tensor memory is given back
    wait(&s.last, 0);
}

// The softmax of one tile's scores and its output, a row to a thread.
template <typename T, int kDim>
__device__ __forceinline__ void softmax(const Args &a, Shared0 &s, char *smem, Stretch st, unsigned *status) {
    using P = Plan<kDim>;
    const int wg = threadIdx.x >> 7, r = threadIdx.x & 127, lane = r & 31;
    const uint32_t lanes = s.tmem + (static_cast<uint32_t>(r >> 5) << 21);
    char *ring = smem + P::kQBytes;
    const int pieces = (a.kv.head_dim + 15) / 16 * 2;
    int unit = 0, item = 0, got[2] = {0, 0}, done = 0;     // units, copies, scores per buffer, outputs of this tile
    Sequence q = sequence(a, st.b);
    int tile = st.tile, head = st.head, skip = st.skip;
    Waiter waiter{status};
    const auto wait = [&](uint64_t *bar, int phase) {
        waiter(bar, phase);
        __syncwarp();
    };
    for (;;) {
        const Fragment f = fragment<P::kM, P::kN>(a, q, tile, skip, st.left);
        const int tiles = P::kTiles == 2 && f.rows - f.row0 > 128 ? 2 : 1;
        const long long row = f.row0 + wg * 128 + r;
        const bool active = wg < tiles;
        const int at = row < f.rows ? f.first + static_cast<int>(row / a.group) : -1;
        float ref = -INFINITY, l = 0.0f;
        bool spoilt = false;           // some row has bits in s.bad
        for (int u = f.u0; u < f.u1; ++u, ++unit, item += 2) {
            const int mb = unit & 1;
            wait(&s.mask_full[mb], unit >> 1);
            uint32_t there[P::kN / 32];
            uint32_t all = 0xffffffffu;
#pragma unroll
            for (int x = 0; x < P::kN / 32; ++x) all &= there[x] = s.mask[mb][x];
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.mask_free[mb]);
            if (!active) continue;
            const bool edge = (u + 1) * P::kN - 1 > f.last_all || u * P::kN < f.first_all;
            const int lo = a.window ? at - a.window + 1 - u * P::kN : 0, hi = at - u * P::kN;   // columns that this row sees
            if (edge) {
                // A value that is not finite must not reach rows that do not see it, and 0 times it would: such values
                // are taken out of the tile, and the rows that see them marked.
                const int v_item = item + 1;
                wait(&s.full[v_item % P::kStages], v_item / P::kStages);
                char *v = ring + (v_item % P::kStages) * P::kStageBytes;
                const int threads = tiles * 128, me = wg * 128 + r;
                bool bad = false;
                for (int i = me; i < P::kN * (kDim / 8); i += threads) {
                    const int n = i / (kDim / 8), c = i % (kDim / 8);
                    if (c >= pieces) continue;
                    const uint4 w = *reinterpret_cast<const uint4 *>(v + piece(P::kN, n, c));
                    bad |= not_finite(w.x, T()) || not_finite(w.y, T()) || not_finite(w.z, T()) || not_finite(w.w, T());
                }
                if (any_of(4, threads, bad)) {
                    if (!spoilt)
                        for (int c = 0; c < 8; ++c) s.bad[me][c] = 0;
                    spoilt = true;
                    for (int n = max(lo, 0); n <= min(hi, P::kN - 1); ++n)
                        for (int c = 0; c < pieces * 4; ++c) {
                            const uint32_t w = *reinterpret_cast<const uint32_t *>(v + piece(P::kN, n, c >> 2) + (c & 3) * 4);
                            const uint32_t low = not_finite(w & 0xffffu, T()), high = not_finite(w & 0xffff0000u, T());
                            s.bad[me][c >> 4] |= (low | high << 1) << (2 * (c & 15));
                        }
                    __syncwarp();
                    named_sync(4, threads);
                    for (int i = me; i < P::kN * (kDim / 8); i += threads) {
                        const int n = i / (kDim / 8), c = i % (kDim / 8);
                        if (c >= pieces) continue;
                        uint4 *w = reinterpret_cast<uint4 *>(v + piece(P::kN, n, c));
                        *w = make_uint4(only_finite<T>(w->x), only_finite<T>(w->y), only_finite<T>(w->z), only_finite<T>(w->w));
                    }
                    fence_async_proxy();
                }
                __syncwarp();
            }
            const int buf = P::kTiles == 2 ? wg : (u - f.u0) & 1;
            wait(&s.s_full[buf], got[buf]++);
            tmem_fence_after();
            uint32_t x[P::kN / 32][32];
#pragma unroll
            for (int i = 0; i < P::kN / 32; ++i) tmem_load32(lanes + P::scores(buf) + i * 32, x[i]);
            tmem_wait_load();
            if (edge || all != 0xffffffffu) {
#pragma unroll
                for (int i = 0; i < P::kN; ++i)
                    if (i < lo || i > hi || !(there[i >> 5] >> (i & 31) & 1)) x[i >> 5][i & 31] = __float_as_uint(-INFINITY);
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < P::kN; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(x[i >> 5][i & 31]));
            const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale;
            if (__any_sync(kFullMask, m > ref + kSlack)) {
                const float next = fmaxf(ref, m - kLead);
                const float keep = next == ref ? 1.0f : ex2(ref - next);
                ref = next;
                l *= keep;
                if (u > f.u0) {
                    wait(&s.o_done[wg], done - 1);
                    tmem_fence_after();
#pragma unroll 1
                    for (int c = 0; c < kDim; c += 32) {
                        uint32_t o[32];
                        tmem_load32(lanes + P::output(wg) + c, o);
                        tmem_wait_load();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                        tmem_store32(lanes + P::output(wg) + c, o);
                    }
                }
            }
            const float off = ref == -INFINITY ? 0.0f : -ref;
            float sum[4] = {};
#pragma unroll
            for (int i = 0; i < P::kN / 64; ++i) {
                uint32_t w[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    const int c = i * 64 + 2 * k;
                    const float p0 = ex2(fmaf(__uint_as_float(x[c >> 5][c & 31]), a.scale, off));
                    const float p1 = ex2(fmaf(__uint_as_float(x[(c + 1) >> 5][(c + 1) & 31]), a.scale, off));
                    sum[(2 * k) & 3] += p0;
                    sum[(2 * k + 1) & 3] += p1;
                    w[k] = pack(p0, p1, T());
                }
                tmem_store32(lanes + P::scores(buf) + i * 32, w);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_wait_store();
            tmem_fence_before();
            mbar_arrive(&s.p_full[buf]);
            ++done;
        }
        if (active) {
            wait(&s.o_done[wg], done - 1);
            tmem_fence_after();
            const float inv = !f.whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const int token = static_cast<int>(row / a.group), h = head * a.group + static_cast<int>(row - static_cast<long long>(token) * a.group);
            char *out = a.out + (q.from + token) * a.out_token + h * a.out_head;
            float *part = a.parts + (2ll * blockIdx.x + (skip == 0)) * part_floats(P::kM, kDim);
            const int pr = wg * 128 + r;
#pragma unroll 1
            for (int c = 0; c < kDim; c += 32) {
                uint32_t o[32];
                tmem_load32(lanes + P::output(wg) + c, o);
                tmem_wait_load();
                if (row < f.rows) {
    #pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
                    if (spoilt) {
                        const uint32_t b = s.bad[pr][c >> 5];
    #pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (b >> i & 1) o[i] = 0x7fffffffu;
                    }
                    if (f.whole) {
    #pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            if (c + i >= a.kv.head_dim) break;
                            uint4 w;
                            w.x = pack(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), T());
                            w.y = pack(__uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]), T());
                            w.z = pack(__uint_as_float(o[i + 4]), __uint_as_float(o[i + 5]), T());
                            w.w = pack(__uint_as_float(o[i + 6]), __uint_as_float(o[i + 7]), T());
                            *reinterpret_cast<uint4 *>(out + (c + i) * 2) = w;
                        }
                    } else {
    #pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4 *>(part + pr * kDim + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
                __syncwarp();
            }
            tmem_fence_before();
            if (row < f.rows) {
                if (!f.whole) {
                    part[P::kM * kDim + pr] = ref;
                    part[P::kM * kDim + P::kM + pr] = l;
                } else if (a.lse) {
                    a.lse[static_cast<long long>(q.from + token) * a.n_head + h] = (ref + log2f(l)) * kLn2;
                }
            }
        }
        st.left -= f.u1 - f.u0;
        if (st.left <= 0) break;
        skip = 0;
        next_tile<P::kM>(a, q, tile, head);
    }
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, 1) mma_kernel(const Args a) {
    using P = Plan<kDim>;
    extern __shared__ char smem_raw[];
    __shared__ Shared0 s;
    char *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5;
    pdl_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < P::kStages; ++i) mbar_init(&s.full[i], kCopiers), mbar_init(&s.free[i], 1);
        mbar_init(&s.q_full, kCopiers);
        mbar_init(&s.q_free, 1);
        mbar_init(&s.last, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_full[i], 128);
            mbar_init(&s.o_done[i], 1);
            mbar_init(&s.mask_full[i], 1);
            mbar_init(&s.mask_free[i], 4 * P::kTiles);
        }
        fence_mbar_init();
        a.joints[blockIdx.x].first = -1;
    }
    if (warp == 8) tmem_alloc(&s.tmem, kColumns);
    const Stretch st = find<P::kM, P::kN, kThreads>(a, reinterpret_cast<Shared<kThreads> *>(smem));
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (st.left > 0) {
        if (tid == 0 && st.skip && st.first + 1 == static_cast<int>(blockIdx.x)) {
            const Sequence q = sequence(a, st.b);
            a.joints[blockIdx.x] = Joint{st.first, st.last, q.from, q.n, st.tile, st.head};
        }
        if (warp < 8) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
            if (warp < 4 * P::kTiles) softmax<T, kDim>(a, s, smem, st, a.status);
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
            if (warp > 8) copier<T, kDim>(a, s, smem, st, a.status);
            else if ((tid & 31) == 0) products<T, kDim>(a, s, smem, st, a.status);
            __syncwarp();
        }
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == 8) tmem_free(s.tmem, kColumns);
}

template <typename T, int kDim>
cudaError_t launch(const Args &a, cudaStream_t stream) {
    const auto fn = mma_kernel<T, kDim>;
    const int grid = sm_count();
    if (!ensure_smem(reinterpret_cast<const void *>(fn), Plan<kDim>::kSmem)) return cudaGetLastError();
    fn<<<grid, kThreads, Plan<kDim>::kSmem, stream>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? e : launch_join<T, Plan<kDim>::kM, kDim>(a, grid, stream);
}

template <typename T>
cudaError_t launch(const Args &a, cudaStream_t stream) {
    if (a.kv.head_dim <= 64) return launch<T, 64>(a, stream);
    if (a.kv.head_dim <= 128) return launch<T, 128>(a, stream);
    if (a.kv.head_dim <= 192) return launch<T, 192>(a, stream);
    return launch<T, 256>(a, stream);
}

}  // namespace

Shape mma_shape(int head_dim) {
    const int dim = (head_dim + 63) / 64 * 64;
    return Shape{sm_count(), part_floats(dim <= 128 ? 256 : 128, dim) * 4};
}

cudaError_t mma_launch(const Args &a, int kv_dtype, cudaStream_t stream) {
    return kv_dtype == B200_BF16 ? launch<__nv_bfloat16>(a, stream) : launch<__half>(a, stream);
}

}  // namespace chunk
}  // namespace b200
