// b200_kv_attend_chunk for 16-bit queries, on the fifth-generation tensor cores.
//
// t = scale log2(e) q . k, out = sum 2^(t - m) v / sum 2^(t - m) with m any
// reference near the running maximum: one pass over the slots, 4 head_dim
// operations for each pair of a packed row and a slot.
//
// A CTA per SM takes two tiles of 128 rows (one where head_dim is above 128) and
// a unit of 128 slots (64) at a time. Its warps have parts: one issues the
// products (tcgen05, scores and outputs in tensor memory, the weights as an
// operand there), a warpgroup per tile turns scores into weights, three warps
// bring keys and values by tensor copies into a ring of two units. While one
// tile's softmax runs, the other's products do.
//
// The weights are rounded to the cache's type, as operands of these products are:
// half a step each, which makes the output's error 0.0021 of its norm in bfloat16
// and 2.4e-4 to 2.9e-4 in float16 where float32 weights leave the output's own
// rounding, 0.0016 and 2.1e-4. Their low parts would be as many products again,
// 3072 cycles for the 2048 below, and conversions for every pair. Sums of weights
// are of what is not rounded, in float32.
//
// What bounds it: the chain of a tile's unit, scores -> weights -> outputs and
// next scores, of which two run side by side: 2250 cycles of softmax and 1000 of
// products, 3330 in all, where the products of both tiles take 2048 and the
// special-function unit, 8.8 cycles for a warp's number beside the products,
// 2250. By GPU and the clock that it then runs at: one prompt of 8192 tokens (32
// heads, 8 of the cache, 128 bfloat16) 594-661 us, 830-925 TFLOP/s of what its
// rows see; 24 users with chunks and single tokens 1250-1510 us, 715-860; 200
// tokens over 120000 slots 348-434 us, 680-850 (and a fifth of the rows idle);
// the prompt with heads of 64 in float16 537 us, 4096 tokens with heads of 192 in
// bfloat16 336, of 256 393 us: 512, 614 and 699 TFLOP/s.
//
// What was measured on the way (prompt / 120000 slots, us): copies of 16 bytes
// by threads 1060 / 600 (pages of fewer than 8 rows still come so); operands of
// the products not constant in the code, 90 cycles each instead of 64: 779 / 358;
// two threads to a row 622 / 425; a warp of products for each tile, which then
// run in step, 812 / 421; a share of the exponentials by a polynomial 720-735 /
// 370; 32 scores at a time 828 / 398; tiles' begin and end not counted where the
// work is dealt out 800 / 350.
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "kv_chunk.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace chunk {

namespace {

// A warpgroup of softmax for each tile, a row to a thread, and one with three
// warps of copies and one that issues the products; and the registers of a
// thread of each, of the 384 * 168 that a CTA begins with.
constexpr int kSoftmaxThreads = 256, kCopiers = 96, kThreads = kSoftmaxThreads + kCopiers + 32;
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(kSoftmaxThreads * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * 168);
constexpr int kCost = 5;                // units that a tile's begin and end take
constexpr int kLeastBox = 8;           // rows of a page that one tensor copy brings at least
constexpr int kColumns = 512;          // of tensor memory: all, so that it begins at address 0
// The reference m trails the maximum by lead to slack powers of two, so weights
// stay in 2^slack and below, and the larger the difference, the more rarely m
// moves. In bfloat16 all other weights are normal numbers whatever the lead. In
// float16, whose range ends at 2^16, a lead of 10 leaves the small ones room: a
// weight of 2^-24 of the largest is still a normal number, a smaller one is off
// by 2^-35 of the largest at most. (A prompt of 8192 tokens in float16 takes 0.4,
// 1.4, 3.3, 5.5 % longer with a lead of 9, 10, 11, 12 than with 7, with heads of
// 64 instead of 128 0.4, 2.7, 9, 15 %.)
template <typename T> struct Lead { static constexpr float lead = 7.0f, slack = 15.0f; };
template <> struct Lead<__half> { static constexpr float lead = 10.0f, slack = 15.75f; };

template <int kDim>
struct Plan {
    static constexpr int kTiles = kDim <= 128 ? 2 : 1;     // of 128 rows
    static constexpr int kM = 128 * kTiles, kN = kDim <= 128 ? 128 : 64;
    static constexpr int kStages = 4;                      // keys and values of two units
    static constexpr int kQBytes = kM * kDim * 2, kStageBytes = kN * kDim * 2;
    static constexpr int kSmem = kQBytes + kStages * kStageBytes;
    // columns of tensor memory: scores (and, over them, weights) per tile, or twice of one, then the outputs
    __device__ static constexpr int scores(int i) { return i * kN; }
    // the weights of 16 slots, two to a column
    __device__ static constexpr int weights(int i, int x) { return i * kN + x * 8; }
    __device__ static constexpr int output(int i) { return 256 + i * kDim; }
};

struct Shared0 {
    uint64_t full[4], free[4], q_full, q_free, s_full[2], p_most[2], p_full[2], o_done[2], last;
    uint32_t tmem;
    int dead;                          // a wait ran out
    long long row[2][128];             // byte offsets of a unit's rows, -1: not there
    uint32_t bad[256][8];              // a row's columns that a value which is not finite enters
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two float32 numbers side by side, for instructions that take two at once.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
    return p;
}
__device__ __forceinline__ void split(Pair p, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
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
// CTA's last: its threads go on without waiting, so that they meet every barrier
// that the others meet and come to their end.
struct Waiter {
    unsigned *status;
    volatile int *dead;                // in shared memory
    __device__ __forceinline__ void operator()(uint64_t *bar, int phase) const {
        if (mbar_try_wait(bar, phase & 1)) return;
        uint64_t t0 = 0;
        for (int n = 1; !mbar_try_wait(bar, phase & 1); ++n) {
            if (n & 63) continue;
            if (*dead) return;
            if (t0 == 0) t0 = globaltimer_ns();
            if (globaltimer_ns() - t0 > kStageTimeoutNs) {
                atomicOr(status, kStatusStageTimeout);
                *dead = 1;
            }
        }
    }
};

// Arrives on `bar` for this thread when the copies that it has asked for are there.
__device__ __forceinline__ void arrive_behind_copies(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// How keys and values come: by tensor copies of `box` rows of a page, or, with
// box 0, by 16 bytes, whatever the pages' size and strides.
struct Maps {
    CUtensorMap k, v;
};

// The copies of keys, values and queries into shared memory. Nothing waits for
// a copy here: its arrival is the barrier's, and the reader's fence hands those
// by 16 bytes to the tensor cores. A tensor copy brings 64 columns of `box` rows;
// a page that is not there is asked for behind the pool's end, which gives
// zeros, as copies by 16 bytes of no source do.
template <typename T, int kDim, bool kBoxes>
__device__ __forceinline__ void copier(const Args &a, const Maps &maps, int box, Shared0 &s, char *smem, Stretch st,
                                       unsigned *status) {
    using P = Plan<kDim>;
    constexpr int kPieces = kDim / 8;
    const int tid = threadIdx.x - kSoftmaxThreads;
    const int pieces = (a.kv.head_dim + 15) / 16 * 2, filled = a.kv.head_dim / 8, columns = (a.kv.head_dim + 63) / 64;
    const uint32_t q_at = smem_addr(smem), ring = q_at + P::kQBytes;
    // Who waits for a stage has to be who fills it: a barrier tells one phase from the next one only, and comes to the one
    // after that without a thread that brings nothing.
    bool issues = !kBoxes || tid == 0;
    for (int n = tid; n < P::kN; n += kCopiers) issues |= kBoxes && (n & (box - 1)) == 0;
    int stage = 0, use = 0, unit = 0, fragments = 0;
    Sequence q = sequence(a, st.b);
    int tile = st.tile, head = st.head, skip = st.skip;
    const Waiter wait{status, &s.dead};
    for (;;) {
        const Fragment f = fragment<P::kM, P::kN, kCost>(a, q, tile, skip, st.left);
        if (f.u1 > f.u0) {
        const char *k_head = a.kv.k + head * a.kv.head_stride, *v_head = a.kv.v + head * a.kv.head_stride;
        const int *table = a.kv.table + q.b * a.kv.table_stride;
        int page[2], asked[2], row[2];                 // of two of this unit's and the next one's slots
        const auto ask = [&](int u) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int n = tid + x * kCopiers, slot = u * P::kN + n;
                asked[x] = -1;
                if (n < P::kN && slot < q.length) asked[x] = table[static_cast<int>((slot * a.page_magic) >> 40)];
            }
        };
        const auto place = [&](int u) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int n = tid + x * kCopiers, slot = u * P::kN + n;
                const bool there = static_cast<unsigned>(asked[x]) < static_cast<unsigned>(a.kv.n_pages);
                page[x] = there ? asked[x] : a.kv.n_pages;
                row[x] = slot - static_cast<int>((slot * a.page_magic) >> 40) * a.kv.page_size;
                if (!kBoxes && n < P::kN) s.row[unit & 1][n] = there ? page[x] * a.kv.page_stride + row[x] * a.kv.row_stride : -1;
            }
            if (!kBoxes) named_sync(3, kCopiers);
        };
        ask(f.u0);
        if (fragments) wait(&s.q_free, fragments - 1);
        const int rows = min(P::kM, f.rows - f.row0);
        const int token0 = f.row0 / a.group, rest = f.row0 - token0 * a.group;
        const char *q_rows = a.q + (q.from + token0) * a.q_token + head * a.group * a.q_head;
#pragma unroll 4
        for (int i = tid; i < (rows > 128 ? P::kM : 128) * kPieces; i += kCopiers) {
            const int r = i / kPieces, c = i % kPieces;
            if (c >= pieces) continue;
            const bool there = r < rows && c < filled;
            const int token = a.group == 1 ? r : static_cast<int>(__umulhi(rest + r, a.group_magic));
            const char *src = q_rows + token * a.q_token + (rest + r - token * a.group) * a.q_head + c * 16;
            copy16(q_at + (r >> 7) * (128 * kDim * 2) + piece(128, r & 127, c), there ? src : a.q, there);
        }
        arrive_behind_copies(&s.q_full);
        place(f.u0);
        for (int u = f.u0; u < f.u1; ++u) {
            const int buf = unit & 1;
            if (u + 1 < f.u1) ask(u + 1);
#pragma unroll 1
            for (int v = 0; v < 2; ++v) {
                if (use && issues) wait(&s.free[stage], use - 1);
                if constexpr (kBoxes) {
                    if (tid == 0) mbar_arrive_expect_tx(&s.full[stage], columns * P::kN * 128);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int n = tid + x * kCopiers;
                        if (n < P::kN && (n & (box - 1)) == 0)
#pragma unroll 1
                            for (int c = 0; c < columns; ++c)
                                tma_load_4d(smem + P::kQBytes + stage * P::kStageBytes + c * (P::kN * 128) + n * 128,
                                            v ? &maps.v : &maps.k, c * 64, row[x], head, page[x], &s.full[stage],
                                            l2_policy_evict_normal());
                    }
                } else {
                    const char *src = v ? v_head : k_head;
                    const uint32_t dst = ring + stage * P::kStageBytes;
#pragma unroll 4
                    for (int i = tid; i < P::kN * kPieces; i += kCopiers) {
                        const int r = i / kPieces, c = i % kPieces;
                        if (c >= pieces) continue;
                        const long long at = s.row[buf][r];
                        const bool there = at >= 0 && c < filled;
                        copy16(dst + piece(P::kN, r, c), src + (there ? at + c * 16 : 0), there);
                    }
                    arrive_behind_copies(&s.full[stage]);
                }
                if (++stage == P::kStages) stage = 0, ++use;
            }
            ++unit;
            if (u + 1 < f.u1) place(u + 1);
        }
        ++fragments;
        }
        st.left -= f.used;
        if (st.left <= 0) break;
        skip = 0;
        next_tile<P::kM>(a, q, tile, head);
    }
    cp_async_commit();
    cp_async_wait<0>();
}

// The matrix products, issued by one warp's elected lane while all of it runs
// the loop. Of a unit j and tile i, in order: O_i += P_i V once the softmax has
// put the weights P_i over the scores, and S_i = Q_i K^T of the next unit into
// the same columns. Products of one thread run in the order of issue, so a
// tile's next scores cannot overtake the use of its weights. (A single tile has
// two buffers of scores, and its next ones come first.) The loop's body exists
// for even and odd units, in which all operands are constants: descriptors that
// have to be computed cost 90 cycles for a product that takes 64.
template <typename T, int kDim, bool kBoxes>
__device__ __forceinline__ void products(const Args &a, Shared0 &s, char *smem, Stretch st, unsigned *status) {
    using P = Plan<kDim>;
    constexpr bool kBf16 = !__is_same(T, __half);
    constexpr int kSteps = P::kN / 16, kMost = kSteps - 2;
    const int steps = (a.kv.head_dim + 15) / 16;
    const uint32_t out_desc = mma_desc(128, steps * 16, kBf16, true);
    const bool lead = elect_one();
    int unit = 0, fragments = 0, used = 0;             // used: weights of a tile taken, a parity each
    Sequence q = sequence(a, st.b);
    int tile = st.tile, head = st.head, skip = st.skip;
    const Waiter wait{status, &s.dead};
    const auto wait_copy = [&](int stage, int phase) {
        wait(&s.full[stage], phase);
        __syncwarp();
        if (!kBoxes) fence_async_proxy();
    };
    // descriptors count in 16 bytes: a step along a row of 128 bytes is 2, the next 64 columns lie a tile's rows further
    const auto scores = [&](auto parity, auto tile_of) {
        constexpr int kG = decltype(parity)::value, kI = decltype(tile_of)::value, kBuf = P::kTiles == 2 ? kI : kG;
        const uint32_t qa = smem_desc(smem_addr(smem) + kI * (128 * kDim * 2), 16);
        const uint32_t kb = smem_desc(smem_addr(smem) + P::kQBytes + 2 * kG * P::kStageBytes, 16);
        const auto step = [&](int x) {
            mma_ss(P::scores(kBuf), qa + (x >> 2) * (128 * 8) + (x & 3) * 2, kb + (x >> 2) * (P::kN * 8) + (x & 3) * 2,
                   mma_desc(128, P::kN, kBf16, false), x > 0);
        };
        if (steps == kDim / 16) {
#pragma unroll
            for (int x = 0; x < kDim / 16; ++x) step(x);
        } else {
#pragma unroll 1
            for (int x = 0; x < steps; ++x) step(x);
        }
        mma_commit(&s.s_full[kBuf]);
    };
    const auto outputs = [&](auto parity, auto tile_of, int from, int to, bool add) {
        constexpr int kG = decltype(parity)::value, kI = decltype(tile_of)::value, kBuf = P::kTiles == 2 ? kI : kG;
        const uint32_t vb = smem_desc(smem_addr(smem) + P::kQBytes + (2 * kG + 1) * P::kStageBytes, P::kN * 128);
#pragma unroll
        for (int x = 0; x < kSteps; ++x)
            if (x >= from && x < to) mma_ts(P::output(kI), P::weights(kBuf, x), vb + x * 128, out_desc, add || x > 0);
    };
    const auto body = [&](auto parity, int tiles, bool add, bool more, bool last_scores) {
        constexpr int kG = decltype(parity)::value;
        using Next = std::integral_constant<int, 1 - kG>;
        const auto tile_body = [&](auto tile_of) {
            constexpr int kI = decltype(tile_of)::value, kBuf = P::kTiles == 2 ? kI : kG;
            const int phase = P::kTiles == 2 ? used >> kI : unit >> 1;
            const bool ends = kI == tiles - 1;
            wait(&s.p_most[kBuf], phase);
            __syncwarp();
            tmem_fence_after();
            if (lead) outputs(parity, tile_of, 0, kMost, add);
            __syncwarp();
            if (P::kTiles == 2 && kI == 0 && more) wait_copy(2 * Next::value, (unit + 1) >> 1);
            wait(&s.p_full[kBuf], phase);
            __syncwarp();
            tmem_fence_after();
            if (lead) {
                outputs(parity, tile_of, kMost, kSteps, true);
                mma_commit(&s.o_done[kI]);
                if (P::kTiles == 2 && more) scores(Next{}, tile_of);
                if (ends) mma_commit(&s.free[2 * kG + 1]);
                if (P::kTiles == 2 && more && ends) {
                    mma_commit(&s.free[2 * Next::value]);
                    if (last_scores) mma_commit(&s.q_free);
                }
            }
            __syncwarp();
            used ^= 1 << kI;
        };
        if (P::kTiles == 1 && more) {
            wait_copy(2 * Next::value, (unit + 1) >> 1);
            if (lead) {
                scores(Next{}, std::integral_constant<int, 0>{});
                mma_commit(&s.free[2 * Next::value]);
                if (last_scores) mma_commit(&s.q_free);
            }
            __syncwarp();
        }
        wait_copy(2 * kG + 1, unit >> 1);
        tile_body(std::integral_constant<int, 0>{});
        if constexpr (P::kTiles == 2)
            if (tiles == 2) tile_body(std::integral_constant<int, 1>{});
    };
    const auto begin = [&](auto parity, int tiles, bool last_scores) {
        constexpr int kG = decltype(parity)::value;
        wait_copy(2 * kG, unit >> 1);
        if (lead) {
            scores(parity, std::integral_constant<int, 0>{});
            if constexpr (P::kTiles == 2)
                if (tiles == 2) scores(parity, std::integral_constant<int, 1>{});
            mma_commit(&s.free[2 * kG]);
            if (last_scores) mma_commit(&s.q_free);
        }
        __syncwarp();
    };
    using Even = std::integral_constant<int, 0>;
    using Odd = std::integral_constant<int, 1>;
    for (;;) {
        const Fragment f = fragment<P::kM, P::kN, kCost>(a, q, tile, skip, st.left);
        if (f.u1 > f.u0) {
        const int units = f.u1 - f.u0, tiles = P::kTiles == 2 && f.rows - f.row0 > 128 ? 2 : 1;
        wait(&s.q_full, fragments);
        __syncwarp();
        fence_async_proxy();
        if (unit & 1) begin(Odd{}, tiles, units == 1);
        else begin(Even{}, tiles, units == 1);
#pragma unroll 1
        for (int j = 0; j < units; ++j, ++unit) {
            if (unit & 1) body(Odd{}, tiles, j > 0, j + 1 < units, j + 2 == units);
            else body(Even{}, tiles, j > 0, j + 1 < units, j + 2 == units);
        }
        ++fragments;
        }
        st.left -= f.used;
        if (st.left <= 0) break;
        skip = 0;
        next_tile<P::kM>(a, q, tile, head);
    }
    if (lead) mma_commit(&s.last);     // before the tensor memory is given back
    __syncwarp();
    wait(&s.last, 0);
    __syncwarp();
}

// The softmax of one tile's scores and its output, a row to a thread.
template <typename T, int kDim, bool kBoxes>
__device__ __forceinline__ void softmax(const Args &a, Shared0 &s, char *smem, Stretch st, unsigned *status) {
    using P = Plan<kDim>;
    constexpr int kRing = P::kStages - 1, kWords = P::kN / 32;
    const int i = threadIdx.x >> 7, r = threadIdx.x & 127, lane = r & 31;      // i: the tile
    const uint32_t lanes = static_cast<uint32_t>(r >> 5) << 21;
    char *ring = smem + P::kQBytes;
    const int pieces = (a.kv.head_dim + 15) / 16 * 2;
    int unit = 0, item = 0, done = 0;  // units, copies, units of this tile
    Sequence q = sequence(a, st.b);
    int tile = st.tile, head = st.head, skip = st.skip;
    const Waiter wait{status, &s.dead};
    const auto arrive = [&](uint64_t *bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    for (;;) {
        const Fragment f = fragment<P::kM, P::kN, kCost>(a, q, tile, skip, st.left);
        if (f.u1 > f.u0) {
        const int tiles = P::kTiles == 2 && f.rows - f.row0 > 128 ? 2 : 1;
        const int row = f.row0 + i * 128 + r;
        const bool active = i < tiles;
        const int at = row < f.rows ? f.first + row / a.group : -1;
        float ref = -INFINITY, l = 0.0f;
        bool spoilt = false;           // some row has bits in s.bad
        // Pages of the tile's slots that are not there are rare: looked for once, and only then per unit.
        const int *table = a.kv.table + q.b * a.kv.table_stride;
        const auto there_of = [&](int slot) {
            return static_cast<unsigned>(table[static_cast<int>((slot * a.page_magic) >> 40)]) < static_cast<unsigned>(a.kv.n_pages);
        };
        bool gaps = false;
        if (active) {
            bool gap = false;
            const int end = min(f.u1 * P::kN, q.length), last = static_cast<int>(((end - 1) * a.page_magic) >> 40);
            if (end > 0)
#pragma unroll 1
                for (int c = static_cast<int>((f.u0 * P::kN * a.page_magic) >> 40) + r; c <= last; c += 128)
                    gap |= static_cast<unsigned>(table[c]) >= static_cast<unsigned>(a.kv.n_pages);
            gaps = any_of(5 + i, 128, gap);
        }
        for (int u = f.u0; u < f.u1; ++u, ++unit, item += 2) {
            if (!active) continue;
            uint32_t there[kWords];
#pragma unroll
            for (int c = 0; c < kWords; ++c) {
                there[c] = 0xffffffffu;
                if (__builtin_expect(gaps, 0)) {
                    const int slot = u * P::kN + c * 32 + lane;
                    there[c] = __ballot_sync(kFullMask, slot < q.length && there_of(slot));
                }
            }
            const bool edge = (u + 1) * P::kN - 1 > f.last_all || u * P::kN < f.first_all;
            const int lo = a.window ? at - a.window + 1 - u * P::kN : 0, hi = at - u * P::kN;   // columns that this row sees
            const int buf = P::kTiles == 2 ? i : unit & 1;
            wait(&s.s_full[buf], P::kTiles == 2 ? done : unit >> 1);
            __syncwarp();
            tmem_fence_after();
            if (__builtin_expect(edge, 0)) {
                // A value that is not finite must not reach rows that do not see it, and 0 times it would: such values
                // are taken out of the tile, and the rows that see them marked. (The scores are there, so the values of
                // two units before were: a phase ahead at most, which is what a barrier can tell.)
                wait(&s.full[(item + 1) & kRing], (item + 1) / P::kStages);
                char *v = ring + ((item + 1) & kRing) * P::kStageBytes;
                // a barrier each for one tile and for two: where a stretch has one tile, the other's warps run ahead
                const int threads = tiles * 128, scan = tiles == 2 ? 2 : 4, me = threadIdx.x, filled = q.length - u * P::kN;
                bool bad = false;
#pragma unroll 1
                for (int x = me; x < P::kN * (kDim / 8); x += threads) {
                    const int n = x / (kDim / 8), c = x % (kDim / 8);
                    if (c >= pieces) continue;
                    uint4 *at_v = reinterpret_cast<uint4 *>(v + piece(P::kN, n, c));
                    if (kBoxes && n >= filled) {       // rows of a page behind the last slot in use
                        *at_v = make_uint4(0, 0, 0, 0);
                        continue;
                    }
                    const uint4 w = *at_v;
                    bad |= not_finite(w.x, T()) || not_finite(w.y, T()) || not_finite(w.z, T()) || not_finite(w.w, T());
                }
                if (kBoxes) fence_async_proxy();
                if (any_of(scan, threads, bad)) {
                    uint32_t *mine = s.bad[me];
                    if (!spoilt)
                        for (int c = 0; c < 8; ++c) mine[c] = 0;
                    spoilt = true;
#pragma unroll 1
                    for (int n = max(lo, 0); n <= min(hi, P::kN - 1); ++n)
#pragma unroll 1
                        for (int c = 0; c < pieces * 4; ++c) {
                            const uint32_t w = *reinterpret_cast<const uint32_t *>(v + piece(P::kN, n, c >> 2) + (c & 3) * 4);
                            const uint32_t low = not_finite(w & 0xffffu, T()), high = not_finite(w & 0xffff0000u, T());
                            mine[c >> 4] |= (low | high << 1) << (2 * (c & 15));
                        }
                    __syncwarp();
                    named_sync(scan, threads);
#pragma unroll 1
                    for (int x = me; x < P::kN * (kDim / 8); x += threads) {
                        const int n = x / (kDim / 8), c = x % (kDim / 8);
                        if (c >= pieces) continue;
                        uint4 *w = reinterpret_cast<uint4 *>(v + piece(P::kN, n, c));
                        *w = make_uint4(only_finite<T>(w->x), only_finite<T>(w->y), only_finite<T>(w->z), only_finite<T>(w->w));
                    }
                    fence_async_proxy();
                    __syncwarp();
                    named_sync(scan, threads);            // before either tile's product
                }
                __syncwarp();
            }
            uint32_t x[kWords][32];
#pragma unroll
            for (int c = 0; c < kWords; ++c) tmem_load32(lanes + P::scores(buf) + c * 32, x[c]);
            tmem_wait_load();
            if (__builtin_expect(edge || gaps, 0)) {
#pragma unroll
                for (int k = 0; k < P::kN; ++k)
                    if (k < lo || k > hi || !(there[k >> 5] >> (k & 31) & 1)) x[k >> 5][k & 31] = __float_as_uint(-INFINITY);
            }
            // The reference moves rarely, so the weights are begun with the one there is while the maximum is found
            // beside them; only where it has to move, and in the first unit, is the maximum first.
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            const auto look = [&](int k) {
                top[k >> 1 & 3] = max3(top[k >> 1 & 3], __uint_as_float(x[k >> 5][k & 31]), __uint_as_float(x[k >> 5][(k & 31) + 1]));
            };
            const Pair scale2 = pair(a.scale, a.scale);
            Pair off2, sum[2];
            uint32_t w[P::kN / 4];
            const auto weigh = [&](int c, bool looks) {        // 32 of the weights
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    Pair p = fma2(pair(__uint_as_float(x[c][2 * k]), __uint_as_float(x[c][2 * k + 1])), scale2, off2);
                    float p0, p1;
                    split(p, p0, p1);
                    p0 = ex2(p0);
                    p1 = ex2(p1);
                    sum[k & 1] = add2(sum[k & 1], pair(p0, p1));
                    w[(c * 16 + k) % (P::kN / 4)] = pack(p0, p1, T());
                    if (looks) {
                        look(c * 32 + 2 * k);
                        look(P::kN / 2 + c * 32 + 2 * k);
                    }
                }
            };
            bool moves = u == f.u0;
            if (__builtin_expect(moves, 0)) {
#pragma unroll
                for (int k = 0; k < P::kN; k += 2) look(k);
            }
            for (;;) {
                if (__builtin_expect(moves, 0)) {
                    const float m = fmaxf(max3(top[0], top[1], top[2]), top[3]) * a.scale;
                    // of the warp's rows only those that need it: a row's bits do not depend on another's scores
                    const float next = m > ref + Lead<T>::slack ? m - Lead<T>::lead : ref;
                    const float keep = next == ref ? 1.0f : ex2(ref - next);
                    ref = next;
                    l *= keep;
                    if (u > f.u0) {
                        wait(&s.o_done[i], done - 1);
                        __syncwarp();
                        tmem_fence_after();
#pragma unroll 1
                        for (int c = 0; c < kDim; c += 32) {
                            uint32_t o[32];
                            tmem_load32(lanes + P::output(i) + c, o);
                            tmem_wait_load();
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                            tmem_store32(lanes + P::output(i) + c, o);
                        }
                    }
                }
                const float off = ref == -INFINITY ? 0.0f : -ref;
                off2 = pair(off, off);
                sum[0] = sum[1] = 0;
#pragma unroll
                for (int c = 0; c < kWords / 2; ++c) weigh(c, true);
                if (moves) break;
                const float m = fmaxf(max3(top[0], top[1], top[2]), top[3]) * a.scale;
                moves = __any_sync(kFullMask, m > ref + Lead<T>::slack);
                if (!moves) break;
            }
            if (P::kTiles == 1 && u > f.u0) {
                // a single tile's scores do not come behind the output of the unit before, and a barrier tells one phase
                // from the next one only
                wait(&s.o_done[i], done - 1);
                __syncwarp();
            }
            if constexpr (P::kN == 128) {
                tmem_store32(lanes + P::weights(buf, 0), w);
            } else {
                tmem_store16(lanes + P::weights(buf, 0), w);
                tmem_wait_store();
                tmem_fence_before();
                arrive(&s.p_most[buf]);
            }
#pragma unroll
            for (int c = kWords / 2; c < kWords; ++c) {
                weigh(c, false);
                uint32_t v[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = w[(c * 16 + k) % (P::kN / 4)];
                tmem_store16(lanes + P::weights(buf, 2 * c), v);
                if (c >= kWords - 2) {                 // the products begin before the last weights are there
                    tmem_wait_store();
                    tmem_fence_before();
                    arrive(c == kWords - 2 ? &s.p_most[buf] : &s.p_full[buf]);
                }
            }
            float s0, s1;
            split(add2(sum[0], sum[1]), s0, s1);
            l += s0 + s1;
            ++done;
        }
        if (active) {
            wait(&s.o_done[i], done - 1);
            __syncwarp();
            tmem_fence_after();
            const float inv = !f.whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const int token = row / a.group, h = head * a.group + row - token * a.group;
            char *out = a.out + (q.from + token) * a.out_token + h * a.out_head;
            float *part = a.parts + (2ll * blockIdx.x + f.begins) * part_floats(P::kM, kDim);
            const int pr = i * 128 + r;
#pragma unroll 1
            for (int c = 0; c < kDim; c += 32) {
                uint32_t o[32];
                tmem_load32(lanes + P::output(i) + c, o);
                tmem_wait_load();
                if (row < f.rows) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * inv);
                    if (spoilt) {
                        const uint32_t b = s.bad[pr][c >> 5];
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (b >> k & 1) o[k] = 0x7fffffffu;
                    }
                    if (f.whole) {
#pragma unroll
                        for (int k = 0; k < 32; k += 8) {
                            if (c + k >= a.kv.head_dim) break;
                            uint4 w;
                            w.x = pack(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), T());
                            w.y = pack(__uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]), T());
                            w.z = pack(__uint_as_float(o[k + 4]), __uint_as_float(o[k + 5]), T());
                            w.w = pack(__uint_as_float(o[k + 6]), __uint_as_float(o[k + 7]), T());
                            *reinterpret_cast<uint4 *>(out + (c + k) * 2) = w;
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            *reinterpret_cast<uint4 *>(part + pr * kDim + c + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
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
            __syncwarp();
        }
        }
        st.left -= f.used;
        if (st.left <= 0) break;
        skip = 0;
        next_tile<P::kM>(a, q, tile, head);
    }
}

template <typename T, int kDim, bool kBoxes>
__global__ void __launch_bounds__(kThreads, 1) mma_kernel(const Args a, const __grid_constant__ Maps maps, int box) {
    using P = Plan<kDim>;
    extern __shared__ __align__(1024) char smem[];
    __shared__ Shared0 s;
    const int tid = threadIdx.x, warp = tid >> 5;
    pdl_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < P::kStages; ++i) mbar_init(&s.full[i], kBoxes ? 1 : kCopiers), mbar_init(&s.free[i], 1);
        mbar_init(&s.q_full, kCopiers);
        mbar_init(&s.q_free, 1);
        mbar_init(&s.last, 1);
        s.dead = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_most[i], 4);
            mbar_init(&s.p_full[i], 4);
            mbar_init(&s.o_done[i], 1);
        }
        fence_mbar_init();
        a.joints[blockIdx.x].first = -1;
    }
    if (warp == kThreads / 32 - 1) tmem_alloc(&s.tmem, kColumns);
    const Stretch st = find<P::kM, P::kN, kCost, kThreads>(a, reinterpret_cast<Shared<kThreads> *>(smem));
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (st.left > 0 && s.tmem == 0) {
        if (tid == 0 && st.skip > kCost && st.first + 1 == static_cast<int>(blockIdx.x)) {
            const Sequence q = sequence(a, st.b);
            a.joints[blockIdx.x] = Joint{st.first, st.last, q.from, q.n, st.tile, st.head};
        }
        if (warp < kSoftmaxThreads / 32) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
            if (warp < 4 * P::kTiles) softmax<T, kDim, kBoxes>(a, s, smem, st, a.status);
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
            if (warp == kThreads / 32 - 1) products<T, kDim, kBoxes>(a, s, smem, st, a.status);
            else copier<T, kDim, kBoxes>(a, maps, box, s, smem, st, a.status);
            __syncwarp();
        }
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (s.dead) {                      // copies that were not waited for land before the memory is another CTA's
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) {}
    }
    if (warp == kThreads / 32 - 1) tmem_free(s.tmem, kColumns);
    if (tid == 0 && (s.tmem != 0 || (smem_addr(smem) & 1023))) atomicOr(a.status, kStatusStageTimeout);   // never
}

// Rows of a page to a tensor copy: the largest power of two that divides the
// page and, with it, every place where a tile's slots change the page.
int box_of(const KvView &kv, int most) {
    const int n = kv.page_size & -kv.page_size;
    return n < most ? n : most;
}

// A cache's rows as the tensor copies see them: [page][head][row][column].
bool map_rows(CUtensorMap *map, const char *rows, const KvView &kv, bool bf16, int box) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    const Encode encode = reinterpret_cast<Encode>(tensor_map_encoder());
    if (!encode) return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(kv.head_dim), static_cast<cuuint64_t>(kv.page_size),
                                static_cast<cuuint64_t>(kv.n_head_kv), static_cast<cuuint64_t>(kv.n_pages)};
    cuuint64_t strides[3] = {static_cast<cuuint64_t>(kv.row_stride), static_cast<cuuint64_t>(kv.head_stride),
                             static_cast<cuuint64_t>(kv.page_stride)};
    for (int i = 0; i < 3; ++i) {
        if (dims[i + 1] == 1) strides[i] = static_cast<cuuint64_t>(kv.head_dim + 7) / 8 * 16;   // not used
        if (strides[i] == 0 || strides[i] >= 1ull << 40) return false;
    }
    const cuuint32_t boxes[4] = {64, static_cast<cuuint32_t>(box), 1, 1}, steps[4] = {1, 1, 1, 1};
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<char *>(rows), dims,
                  strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int kDim, bool kBoxes>
cudaError_t launch(const Args &a, const Maps &maps, int box, cudaStream_t stream) {
    const auto fn = mma_kernel<T, kDim, kBoxes>;
    const int grid = sm_count();
    if (!ensure_smem(reinterpret_cast<const void *>(fn), Plan<kDim>::kSmem)) return cudaGetLastError();
    fn<<<grid, kThreads, Plan<kDim>::kSmem, stream>>>(a, maps, box);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? e : launch_join<T, Plan<kDim>::kM, kDim>(a, grid, stream);
}

template <typename T, int kDim>
cudaError_t launch(const Args &a, cudaStream_t stream) {
    Maps maps{};
    const int box = box_of(a.kv, Plan<kDim>::kN);
    const bool bf16 = !__is_same(T, __half);
    if (box >= kLeastBox && map_rows(&maps.k, a.kv.k, a.kv, bf16, box) && map_rows(&maps.v, a.kv.v, a.kv, bf16, box))
        return launch<T, kDim, true>(a, maps, box, stream);
    return launch<T, kDim, false>(a, maps, 0, stream);
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
    return Shape{1, part_floats(dim <= 128 ? 256 : 128, dim) * 4};
}

cudaError_t mma_launch(const Args &a, int kv_dtype, cudaStream_t stream) {
    return kv_dtype == B200_BF16 ? launch<__nv_bfloat16>(a, stream) : launch<__half>(a, stream);
}

}  // namespace chunk
}  // namespace b200
