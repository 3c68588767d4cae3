// b200_kv_attend: attention of one new token per sequence over a paged cache.
//
// s = scale q . k, out = sum 2^(t - m) v / sum 2^(t - m) with t = s log2(e) and
// m any reference near the running maximum: one pass over the rows, 4 head_dim
// operations per query head for 4 head_dim bytes (16-bit cache), so memory
// bounds it as long as the arithmetic keeps out of the way.
//
// Work: every 16 slots of a cache head (and of one tile of the query heads that
// read it) are a unit. The units of the batch, in the order sequence, head,
// slot, are dealt out in equal stretches to a grid that fits the GPU at once,
// whatever the lengths, which only the device knows. A stretch that begins or
// ends inside a head leaves a part (m, l, O) in scratch; the CTA that comes
// last to a head joins its parts in order, so the result does not depend on
// timing.
//
// Arithmetic: both products run on mma.sync with the rows as the 16-row
// operand and the query heads as the 8 columns: S^T = K Q^T and O^T = V^T P^T.
// A float32 operand is split into a high and a low part of the cache's type,
// and the two go side by side as the columns 2h and 2h + 1 of head h: four heads
// fill a tile of eight columns, and the split costs nothing (float32 caches
// split K and V, too, and run twice). The contraction index may be permuted, so
// a lane's fragments are 16-byte pieces of rows. Each warp copies the units it
// computes to a ring of its own in shared memory (cp.async, whole rows to an
// instruction, swizzled) and reads the pieces back as operands: no barrier
// between warps, no bank conflict, and no transposition but the 8x8 one of P
// (movmatrix).
//
// What bounds it: memory, for long caches. Read once by the kernel, the rows
// come at 5.1-5.4 TB/s (one sequence of 131071 slots, 8 heads of 128 float16:
// 100-105 us on different GPUs; DRAM traffic 1.00 of the rows') and 5.7-6.0 TB/s
// (32 sequences of up to 16384 slots in bfloat16: 190-200 us), of 6.46 measured
// for a copy; a kernel that only
// copies the same pages takes 90 us for the first. The rest is the start (4 us:
// lengths, then table, then rows, each waiting for the one before), the join (5
// us) and SMs that get their rows later than others, always the same ones, by
// up to a fifth. Pieces of 64 bytes of eight rows to an instruction, which need
// no swizzle, took 123 us in that copy where whole rows take 97; the depth of
// the ring (2 to 8 halves) and 2 to 4 CTAs per SM made no difference. For short
// caches the chain of dependent reads is all there is: 10 us with the call
// (200 slots). The tensor pipe is 10 % busy (17 % with float32 rows, whose kernel
// is short of warps: 255 registers, 12 % of the SM's).
#include <cuda_runtime.h>

#include "common.cuh"
#include "q4gemv.h"
#include "serve_dev.cuh"

namespace b200 {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 16;              // slots
constexpr int kShort = 96;             // units of a head beyond which heads are split in any case
constexpr int kMaxCtas = 1024;         // of the grid
constexpr float kLog2e = 1.44269504088896340736f;
// The reference m trails the maximum by lead to slack powers of two, so weights
// stay in 2^slack and below, and the larger the difference, the more rarely m
// moves. Low parts are multiplied by `low`. In float16, whose range ends at 2^16,
// both leave small weights and elements room: low parts are normal numbers
// wherever high ones are, so a weight keeps 22 bits down to 2^-26 of the largest,
// and below that is off by 2^-48 of the largest at most.
template <typename T> struct Range { static constexpr float lead = 7.0f, slack = 15.0f, low = 1.0f; };
template <> struct Range<__half> { static constexpr float lead = 12.0f, slack = 15.75f, low = 0x1p11f; };

struct AttendArgs {
    KvView kv;
    unsigned long long page_magic;     // slot / page_size = slot * page_magic >> 40 (slot < 2^20)
    bool whole_units;                  // page_size % 16 == 0: a unit lies in one page (one lookup and no shuffles:
                                       // 106.5 us where a lookup per row takes 108.5, 16 x 8192 slots)
    const char *q;
    char *out;
    long long q_batch, q_head, out_batch, out_head;  // elements
    int n_head, group, tiles;          // tiles of query heads to a cache head
    float scale;
    float *lse;                        // [batch][n_head] or NULL
    float *scores;                     // weights wanted: t of every slot, [batch][cache head][tile][slot][head of tile]
    float *lse2;                       // and log2 sum 2^t, [batch][cache head][tile][head of tile]
    long long slots;                   // cols * page_size
    unsigned *tickets;
    float *parts;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const char *src, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void sts128_zero(uint32_t a) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t tf32(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}

template <typename T>
__device__ __forceinline__ void mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<float>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo / low in the operand's type: 22 bits of x in float16 (as far as its range goes) and tf32, 16 in bfloat16.
template <typename T>
__device__ __forceinline__ uint32_t split_pair(float x) {   // hi in the low half, lo in the high one
    const T hi = from_float<T>(x), lo = from_float<T>((x - to_float(hi)) * Range<T>::low);
    return static_cast<uint32_t>(*reinterpret_cast<const unsigned short *>(&hi)) |
           static_cast<uint32_t>(*reinterpret_cast<const unsigned short *>(&lo)) << 16;
}
__device__ __forceinline__ void split_tf32(float x, uint32_t *hi, uint32_t *lo) {
    *hi = tf32(x);
    *lo = tf32(x - __uint_as_float(*hi));
}

template <typename T, int D, int NT>
struct Shape {
    static constexpr int kEs = sizeof(T);
    static constexpr int kHeads = 4 * NT;                  // query heads of a tile
    static constexpr int kPieces = D * kEs / 32;           // 16-byte pieces a lane copies of a unit's K (or V)
    static constexpr int kRowPieces = D * kEs / 16;
    static constexpr int kHalf = kPieces * 512;            // bytes of a unit's K (or V)
    static constexpr int kQRow = D * kEs + 64;             // a query row in shared memory: 64 off the same banks
    static constexpr int kFixed = 8 * NT * kQRow + kHeads * D * 4;
    // CTAs per SM: what the registers allow (accumulators of D x heads, and the split of float32 rows).
    static constexpr int kWant = D * NT * (kEs / 2) <= 64 ? 4 : D * NT <= 128 && kEs == 2 ? 3 : 2;
    // Halves (a unit's K, or its V) in flight per warp: what those CTAs leave room for, at least 2 and at most 8;
    // with one CTA per SM where two have no room.
    static constexpr int kRoom = (227 * 1024 / kWant - 1792 - kFixed) / (kWarps * kHalf);
    static constexpr int kCtas = kRoom < 2 ? 1 : kWant;
    static constexpr int kDepth = kRoom > 8 ? 8 : kRoom < 2 ? 3 : kRoom;
    static constexpr int kSmem = kWarps * kDepth * kHalf + kFixed;
    static constexpr int kPart = kHeads * (D + 2);         // floats of a part: O, then m, then l
};

// Row x of a unit keeps its 16-byte piece y at y ^ swizzle(x).
__device__ __forceinline__ int swizzle_k(int row) { return (row & 1) << 2; }
__device__ __forceinline__ int swizzle_v(int row) { return (row >> 1 & 3) << 1; }

// q . k of the unit's row `row`, an element after the other.
template <typename T, typename S>
__device__ __noinline__ float whole_score(const char *k_tile, int row, const char *q_row, int d) {
    constexpr int kPer = 16 / S::kEs;                      // elements of a piece
    const T *k = reinterpret_cast<const T *>(k_tile + row * S::kRowPieces * 16);
    const T *hi = reinterpret_cast<const T *>(q_row), *lo = reinterpret_cast<const T *>(q_row + S::kQRow);
    float sum = 0.0f;
#pragma unroll 1
    for (int i = 0; i < d; ++i) sum = fmaf(to_float(k[i ^ swizzle_k(row) * kPer]), to_float(hi[i]) + to_float(lo[i]) * (1 / Range<T>::low), sum);
    return sum;
}

// A place in the order of units.
struct Cursor {
    int b, s, u, units;     // sequence, head and tile, unit of it, units of the sequence's heads

    __device__ __forceinline__ void advance(const AttendArgs &a, int heads, int by) {
        u += by;
        while (u >= units) {
            u -= units;
            if (++s == heads) {
                s = 0;
                do {
                    if (++b >= a.kv.batch) {
                        units = 0x7fffffff;
                        return;
                    }
                    units = (kv_length(a.kv, b) + kUnit - 1) / kUnit;
                } while (units == 0);
            }
        }
    }
};

// A CTA's share of the units.
struct Stretch {
    long long c0, base, per;  // its first unit; the first unit of the sequence that lies in; units of a CTA
    int count, b;             // its units; that sequence
};

// Where the CTA's stretch lies, into shared memory. Not inlined: the kernel's
// loop gets by with the registers it needs.
__device__ __noinline__ void find_stretch(const int *lengths, int batch, int slots, int heads, Stretch *out) {
    __shared__ long long s_sum[kWarps];
    __shared__ long long s_c0, s_c1, s_base;
    __shared__ int s_b;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const auto units_of = [&](int b) { return b < batch ? (min(max(lengths[b], 0), slots) + kUnit - 1) / kUnit : 0; };
    const auto block_scan = [&](long long v, long long *all) {   // inclusive
        for (int k = 1; k < 32; k <<= 1) {
            const long long y = __shfl_up_sync(kFullMask, v, k);
            if (lane >= k) v += y;
        }
        __syncthreads();
        if (lane == 31) s_sum[warp] = v;
        __syncthreads();
        *all = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) v += s_sum[w];
            *all += s_sum[w];
        }
        return v;
    };
    long long total = 0, mine = 0, upto = 0, all;
    int longest = 0;
    for (int b0 = 0; b0 < batch; b0 += kThreads) {
        const int units = units_of(b0 + tid);
        longest = max(longest, units);
        mine = static_cast<long long>(units) * heads;
        upto = block_scan(mine, &all) + total;
        total += all;
    }
    // Even stretches, or whole heads, the same number to each CTA? A part costs its CTA a fence and a ticket, and
    // another CTA the join, the more time the more CTAs do so at once; whole heads of different lengths leave CTAs
    // idle. Measured, split against whole, heads of 128 elements, 8 to a sequence: one sequence of 160, 320, 640
    // slots 18.4, 14.3, 14.3 against 14.3, 16.4, 20.5 us; 32 of 160, 640, 1280 slots 24.6, 32.8, 45.1 against 16.4,
    // 27.5, 41.0 us. So heads are split where the longest is well over twice the even share.
    long long per = (total + gridDim.x - 1) / gridDim.x;
    if (per < kWarps) per = kWarps;
    const int segments = batch * heads, each = (segments + gridDim.x - 1) / gridDim.x;
    const bool split = __syncthreads_or(longest > kShort || static_cast<long long>(longest) * each > 2 * per + 10);
    const int from = static_cast<int>(min(static_cast<long long>(blockIdx.x) * each, static_cast<long long>(segments)));
    const int to = min(from + each, segments);
    if (tid == 0) {
        s_c0 = split ? min(blockIdx.x * per, total) : total;
        s_c1 = split ? min((blockIdx.x + 1) * per, total) : total;
        s_b = 0;
        s_base = 0;
    }
    __syncthreads();
    // sequence b's n units come behind `before` others
    const auto place = [&](int b, long long n, long long before) {
        if (split) {
            const long long c0 = blockIdx.x * per;
            if (before <= c0 && c0 < before + n) s_b = b, s_base = before;
        } else if (b < batch) {
            const int k = b * heads;
            if (k <= from && from < k + heads) s_c0 = before + n / heads * (from - k), s_b = b, s_base = before;
            if (k <= to && to < k + heads) s_c1 = before + n / heads * (to - k);
        }
    };
    if (batch <= kThreads) {                               // the scan still holds every sequence's place
        place(tid, mine, upto - mine);
    } else {
        long long run = 0;
        for (int b0 = 0; b0 < batch; b0 += kThreads) {
            mine = static_cast<long long>(units_of(b0 + tid)) * heads;
            upto = block_scan(mine, &all) + run;
            place(b0 + tid, mine, upto - mine);
            run += all;
        }
    }
    __syncthreads();
    if (tid == 0) {
        int b = s_b;
        if (s_c0 < s_c1)                                   // a sequence without units has none of the stretch
            while (units_of(b) == 0) ++b;
        *out = Stretch{s_c0, s_base, per, static_cast<int>(s_c1 - s_c0), b};
    }
    __syncthreads();
}

template <typename Q, typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, Shape<T, D, NT>::kCtas)
    kv_attend_kernel(const AttendArgs a) {
    using S = Shape<T, D, NT>;
    constexpr bool kF32 = sizeof(T) == 4;
    constexpr int kKb = S::kPieces / 2;                    // blocks of 64 bytes of a K row
    constexpr int kDb = S::kPieces / 4;                    // blocks of 128 bytes of a V row
    constexpr int kAcc = D / 16;                           // 16-row tiles of O^T
    extern __shared__ __align__(16) char smem[];
    __shared__ Stretch s_stretch;
    __shared__ int s_last;
    __shared__ float s_qs[S::kHeads], s_m[kWarps][S::kHeads], s_l[kWarps][S::kHeads];
    __shared__ float s_M[S::kHeads], s_L[S::kHeads];
    char *s_q = smem + kWarps * S::kDepth * S::kHalf;
    float *s_o = reinterpret_cast<float *>(s_q + 8 * NT * S::kQRow);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
    const int d = a.kv.head_dim, heads = a.kv.n_head_kv * a.tiles;
    const uint32_t ring = smem_addr(smem) + warp * S::kDepth * S::kHalf;

    const auto units_of = [&](int b) { return (kv_length(a.kv, b) + kUnit - 1) / kUnit; };
    find_stretch(a.kv.lengths, a.kv.batch, a.kv.cols * a.kv.page_size, heads, &s_stretch);
    const long long c0 = s_stretch.c0, per = s_stretch.per;
    const int count = s_stretch.count;
    const auto empty_sequences = [&] {
        for (int b = blockIdx.x; b < a.kv.batch; b += gridDim.x) {
            if (kv_length(a.kv, b) > 0) continue;
            for (int i = tid; i < a.n_head * d; i += kThreads) {
                const int h = i / d;
                reinterpret_cast<Q *>(a.out)[b * a.out_batch + h * a.out_head + (i - h * d)] = from_float<Q>(0.0f);
            }
            for (int h = tid; a.lse && h < a.n_head; h += kThreads)
                a.lse[static_cast<long long>(b) * a.n_head + h] = -INFINITY;
        }
    };
    if (count <= 0) {
        empty_sequences();
        return;
    }

    Cursor at;                                             // the first unit of the stretch
    at.b = s_stretch.b;
    at.units = units_of(at.b);
    at.s = static_cast<int>((c0 - s_stretch.base) / at.units);
    at.u = static_cast<int>((c0 - s_stretch.base) - static_cast<long long>(at.s) * at.units);

    // The queries of a tile: warp w has the heads w, w + kWarps. They are asked for before rows are (behind 100 KB of
    // those on their way they would come late): the first tile's here, the next one's while a tile is worked on.
    constexpr int kMine = S::kHeads / kWarps;
    constexpr bool kAhead = kMine * D / 32 <= 8;           // as registers allow
    float qx[kMine][D / 32];
    const auto load_q = [&](const Cursor &at) {
        const int hkv = at.s / a.tiles, tile = at.s - hkv * a.tiles;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int h = tile * S::kHeads + warp + i * kWarps;
            const Q *q = reinterpret_cast<const Q *>(a.q) + at.b * a.q_batch + (hkv * a.group + h) * a.q_head;
#pragma unroll
            for (int k = 0; k < D / 32; ++k) qx[i][k] = h < a.group && lane + 32 * k < d ? to_float(q[lane + 32 * k]) : 0.0f;
        }
    };
    load_q(at);

    // The copying side: units c0 + warp, + kWarps, ... of the stretch, each as K then V.
    Cursor in = at;
    in.advance(a, heads, warp);
    int to_copy = (count - warp + kWarps - 1) / kWarps;
    unsigned long long there = 0;                          // 16 bits per unit in flight: which rows are there
    int flying = 0;
    uint32_t place_in = 0, place_out = 0;                  // ring places, as byte offsets
    // Piece i of a lane is piece i * 32 + lane of the unit's rows, one after the other: whole rows, or half a
    // row of 64 pieces, to an instruction. Row x keeps its piece y at y ^ swizzle(x), so that the fragments'
    // reads below meet no bank twice: 8 lanes read either 4 pieces side by side of rows 2x and 2x + 1 (K), or
    // pieces 2y and 2y + 1 of rows 0, 2, 4, 6 (V).
    constexpr int kRp = S::kRowPieces;
    constexpr int kRows = kRp <= 32 ? 32 / kRp : 1;        // rows to an instruction
    const int my_row = kRp <= 32 ? lane / kRp : 0, my_piece = kRp <= 32 ? lane % kRp : lane;
    const auto piece_row = [&](int i) { return kRp <= 32 ? i * kRows + my_row : i / 2; };
    const auto piece_col = [&](int i) { return kRp <= 32 ? my_piece : (i & 1) * 32 + my_piece; };
    const int row_bytes = d * S::kEs;
    // Rows are read once: they should not push out of the L2 what others will read again (100 against 110 us for
    // 131071 slots of 8 heads; two tiles of query heads that read the same rows: 123 against 131 us).
    const uint64_t policy = l2_policy_evict_first();
    unsigned row_mask;                                     // which of the unit's rows are in use, their page there
    long long row_off;                                     // byte offset of its first row, or of row `lane & 15`; 0, a
                                                           // row that can be read, in place of one that is not there
    const auto lookup = [&] {
        row_mask = 0;
        row_off = 0;
        if (to_copy <= 0) return;
        const int slot = in.u * kUnit + (a.whole_units ? 0 : lane & 15), n = kv_length(a.kv, in.b);
        bool ok = slot < n;
        if (ok) {
            const int col = static_cast<int>(slot * a.page_magic >> 40);
            const int page = a.kv.table[in.b * a.kv.table_stride + col];
            ok = static_cast<unsigned>(page) < static_cast<unsigned>(a.kv.n_pages);
            if (ok) row_off = page * a.kv.page_stride + (in.s / a.tiles) * a.kv.head_stride + (slot - col * a.kv.page_size) * a.kv.row_stride;
        }
        row_mask = a.whole_units ? !ok ? 0 : n - slot >= kUnit ? 0xffffu : (1u << (n - slot)) - 1 : ok;
    };
    const auto copy = [&](const char *pool, const auto &swizzle) {
        const uint32_t dst = ring + place_in;
        if (a.whole_units) {
            // a page holds 16 rows from here; without a page the pool's first row stands in for all
            const long long step = row_mask ? a.kv.row_stride : 0;
            const char *src = pool + row_off + my_row * step;
#pragma unroll
            for (int i = 0; i < S::kPieces; ++i) {
                if (piece_col(i) * 16 < row_bytes)
                    cp_async16(dst + piece_row(i) * kRp * 16 + (piece_col(i) ^ swizzle(piece_row(i))) * 16, src + piece_col(i) * 16, policy);
                if (kRp <= 32 || (i & 1)) src += kRows * step;
            }
        } else {
#pragma unroll
            for (int i = 0; i < S::kPieces; ++i) {
                const char *src = pool + __shfl_sync(kFullMask, row_off, piece_row(i)) + piece_col(i) * 16;
                if (piece_col(i) * 16 < row_bytes)
                    cp_async16(dst + piece_row(i) * kRp * 16 + (piece_col(i) ^ swizzle(piece_row(i))) * 16, src, policy);
            }
        }
    };
    const auto copy_k = [&] {
        if (to_copy > 0) {
            const unsigned rows = a.whole_units ? row_mask : __ballot_sync(kFullMask, row_mask) & 0xffffu;
            there |= static_cast<unsigned long long>(rows) << (16 * flying++);
            copy(a.kv.k, [](int row) { return swizzle_k(row); });
        }
        cp_async_commit();
        place_in = place_in == (S::kDepth - 1) * S::kHalf ? 0 : place_in + S::kHalf;
    };
    const auto copy_v = [&] {
        if (to_copy > 0) {
            copy(a.kv.v, [](int row) { return swizzle_v(row); });
            --to_copy;
            in.advance(a, heads, kWarps);
            lookup();
        }
        cp_async_commit();
        place_in = place_in == (S::kDepth - 1) * S::kHalf ? 0 : place_in + S::kHalf;
    };
    // kDepth - 1 halves ahead: the one that follows when a K (or a V) is taken is known from kDepth.
    constexpr bool kEven = S::kDepth % 2 == 0;
    if (row_bytes < D * S::kEs) {                          // pieces past the row are never copied: zeros
        for (int i = lane; i < S::kDepth * S::kHalf / 16; i += 32) sts128_zero(ring + i * 16);
        __syncwarp();
    }
    lookup();
#pragma unroll
    for (int i = 0; i < S::kDepth - 1; ++i) {
        if (i & 1) copy_v(); else copy_k();
    }
    // Where a lane's fragments lie: K rows r and r + 8, the pieces c of 64-byte blocks (even and odd ones); V rows
    // 2c, 2c + 1, 2c + 8, 2c + 9, the pieces r of 128-byte blocks.
    const uint32_t k_even = r * kRp * 16 + (c ^ swizzle_k(r)) * 16, k_odd = k_even ^ 64;
    const uint32_t v_at = 2 * c * kRp * 16 + (r ^ swizzle_v(2 * c)) * 16;

    pdl_launch_dependents();                               // the weights' kernel may come: it waits for all of this one
    int f = 0;                                             // first unit of the current head's share, from c0 on
    while (f < count) {
        const int head_start = f - at.u, head_end = head_start + at.units, end = min(head_end, count);
        const int hkv = at.s / a.tiles, tile = at.s - hkv * a.tiles;
        const int h0 = hkv * a.group + tile * S::kHeads;   // the tile's first query head
        const int live = min(S::kHeads, a.group - tile * S::kHeads);
        const int n = kv_length(a.kv, at.b);

        // The queries of the tile, split, and the factor that makes t of a product.
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int h = warp + i * kWarps;
            int e = 0;
            // float32 into float16: the head's largest to [2^14, 2^15), so that an element 2^-j of it keeps 22 bits, or
            // 50 - j where that is less
            if (sizeof(Q) == 4 && !kF32) {
                float top = 0.0f;
#pragma unroll
                for (int k = 0; k < D / 32; ++k) top = fmaxf(top, fabsf(qx[i][k]));
                for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, k));
                if (top > 0.0f && top < INFINITY) e = ilogbf(top) - 14;
            }
            char *row = s_q + 2 * (h & 3) * S::kQRow + (h >> 2) * 8 * S::kQRow;
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
                const float v = e ? ldexpf(qx[i][k], -e) : qx[i][k];
                if (kF32) {
                    uint32_t hi, lo;
                    split_tf32(v, &hi, &lo);
                    reinterpret_cast<uint32_t *>(row)[lane + 32 * k] = hi;
                    reinterpret_cast<uint32_t *>(row + S::kQRow)[lane + 32 * k] = lo;
                } else {
                    const uint32_t p = split_pair<T>(v);
                    reinterpret_cast<unsigned short *>(row)[lane + 32 * k] = static_cast<unsigned short>(p);
                    reinterpret_cast<unsigned short *>(row + S::kQRow)[lane + 32 * k] = static_cast<unsigned short>(p >> 16);
                }
            }
            if (lane == 0) s_qs[h] = ldexpf(a.scale * kLog2e, e);
        }
        __syncthreads();
        if (kAhead && head_end < count) {
            Cursor next = at;
            next.advance(a, heads, at.units - at.u);
            load_q(next);
        }

        float m[NT], l[NT], o[kAcc][NT][4], qs[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.0f;
            qs[t] = s_qs[4 * t + c];
#pragma unroll
            for (int i = 0; i < kAcc; ++i) o[i][t][0] = o[i][t][1] = o[i][t][2] = o[i][t][3] = 0.0f;
        }
        const uint32_t qa = smem_addr(s_q) + r * S::kQRow + c * 16;
        for (int g = f + ((warp - f) & (kWarps - 1)); g < end; g += kWarps) {
            const int u = g - head_start;
            // S^T: 16 slots by the tile's columns
            __syncwarp();                                  // every lane has read what is overwritten now
            if (kEven) copy_v(); else copy_k();
            cp_async_wait<S::kDepth - 1>();
            __syncwarp();                                  // and every lane's pieces are there
            float sc[NT][2][4];                            // two chains of products, added up at the end
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[t][0][i] = sc[t][1][i] = 0.0f;
            uint32_t half = ring + place_out;
            place_out = place_out == (S::kDepth - 1) * S::kHalf ? 0 : place_out + S::kHalf;
#pragma unroll
            for (int k = 0; k < kKb; ++k) {
                const uint32_t ka = half + (k & 1 ? k_odd + (k - 1) * 64 : k_even + k * 64);
                const uint4 k0 = lds128(ka), k1 = lds128(ka + 8 * kRp * 16);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint4 q4 = lds128(qa + t * 8 * S::kQRow + k * 64);
                    if constexpr (kF32) {
                        const float x[8] = {__uint_as_float(k0.x), __uint_as_float(k1.x), __uint_as_float(k0.y), __uint_as_float(k1.y),
                                            __uint_as_float(k0.z), __uint_as_float(k1.z), __uint_as_float(k0.w), __uint_as_float(k1.w)};
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) split_tf32(x[i], &hi[i], &lo[i]);
                        float block[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // (added up by ordinary additions: see below)
                        mma<T>(block, lo, q4.x, q4.y);
                        mma<T>(block, lo + 4, q4.z, q4.w);
                        mma<T>(block, hi, q4.x, q4.y);
                        mma<T>(block, hi + 4, q4.z, q4.w);
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[t][k & 1][i] += block[i];
                    } else {
                        const uint32_t a0[4] = {k0.x, k1.x, k0.y, k1.y}, a1[4] = {k0.z, k1.z, k0.w, k1.w};
                        mma<T>(sc[t][0], a0, q4.x, q4.y);
                        mma<T>(sc[t][1], a1, q4.z, q4.w);
                    }
                }
            }
            const unsigned rows = static_cast<unsigned>(there) & 0xffffu;
            there >>= 16;
            --flying;
            // this lane: head c of each column tile, slots r and r + 8
            uint32_t b0[NT], b1[NT], b2[NT], b3[NT];       // P^T as the second product's columns
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const auto whole = [](float hi, float lo) { return fmaf(lo, 1 / Range<T>::low, hi); };
                float t0 = rows >> r & 1 ? whole(sc[t][0][0] + sc[t][1][0], sc[t][0][1] + sc[t][1][1]) * qs[t] : -INFINITY;
                float t1 = rows >> (r + 8) & 1 ? whole(sc[t][0][2] + sc[t][1][2], sc[t][0][3] + sc[t][1][3]) * qs[t] : -INFINITY;
                const float most = m[t] + Range<T>::slack;
                if (__any_sync(kFullMask, !(t0 <= most && t1 <= most))) {
                    // An infinite key element times a low part of 0, or parts of both signs, is NaN where the score is
                    // infinite: such a score is taken again from whole operands. One that stays NaN makes the reference
                    // infinite, and with it all that the head's weights enter: m must not stay at -infinity, which stands
                    // for no slot at all.
                    const char *q_row = s_q + (8 * t + 2 * c) * S::kQRow, *k_tile = smem + (half - smem_addr(smem));
                    if (t0 != t0) t0 = whole_score<T, S>(k_tile, r, q_row, d) * qs[t];
                    if (t1 != t1) t1 = whole_score<T, S>(k_tile, r + 8, q_row, d) * qs[t];
                    float top = t0 == t0 && t1 == t1 ? fmaxf(t0, t1) : INFINITY;
                    for (int k = 4; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, k));
                    const float m1 = fmaxf(m[t], top - Range<T>::lead), old = m1 == -INFINITY ? 1.0f : exp2_fast(m[t] - m1);
                    m[t] = m1;
                    l[t] *= old;
#pragma unroll
                    for (int i = 0; i < kAcc; ++i) o[i][t][0] *= old, o[i][t][1] *= old, o[i][t][2] *= old, o[i][t][3] *= old;
                }
                if (a.scores) {
                    float *dst = a.scores + ((static_cast<long long>(at.b) * heads + at.s) * a.slots + u * kUnit) * S::kHeads + 4 * t + c;
                    if (u * kUnit + r < n) dst[r * S::kHeads] = t0;
                    if (u * kUnit + r + 8 < n) dst[(r + 8) * S::kHeads] = t1;
                }
                const float p0 = t0 == -INFINITY ? 0.0f : exp2_fast(t0 - m[t]);
                const float p1 = t1 == -INFINITY ? 0.0f : exp2_fast(t1 - m[t]);
                l[t] += p0 + p1;
                if constexpr (kF32) {
                    // tf32 columns as two 16-bit planes through the 8x8 transposition
                    uint32_t h0, l0, h1, l1;
                    split_tf32(p0, &h0, &l0);
                    split_tf32(p1, &h1, &l1);
                    const uint32_t u0 = transpose8x8(__byte_perm(h0, l0, 0x7632)), v0 = transpose8x8(__byte_perm(h0, l0, 0x5410));
                    const uint32_t u1 = transpose8x8(__byte_perm(h1, l1, 0x7632)), v1 = transpose8x8(__byte_perm(h1, l1, 0x5410));
                    b0[t] = __byte_perm(v0, u0, 0x5410);
                    b1[t] = __byte_perm(v0, u0, 0x7632);
                    b2[t] = __byte_perm(v1, u1, 0x5410);
                    b3[t] = __byte_perm(v1, u1, 0x7632);
                } else {
                    b0[t] = transpose8x8(split_pair<T>(p0));
                    b1[t] = transpose8x8(split_pair<T>(p1));
                }
            }
            // O^T += V^T P^T. A unit's product is added by an ordinary addition: the tensor cores cut their sums off
            // instead of rounding them, which pulls O (not l) towards 0 with every unit, by 2e-6 of itself in 60 units
            // and by 1.3e-4 in 1800 (131072 slots in one CTA), a fifth of a float16 unit.
            __syncwarp();
            if (kEven) copy_k(); else copy_v();
            cp_async_wait<S::kDepth - 1>();
            __syncwarp();
            half = ring + place_out;
            place_out = place_out == (S::kDepth - 1) * S::kHalf ? 0 : place_out + S::kHalf;
            if (rows != 0xffffu) {                         // what lies in rows that are not there may be NaN
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!(rows >> (2 * c + (j & 1) + (j >> 1) * 8) & 1))
                        for (int k = 0; k < kDb; ++k) sts128_zero(half + v_at + ((j & 1) + (j >> 1) * 8) * kRp * 16 + k * 128);
            }
#pragma unroll
            for (int k = 0; k < kDb; ++k) {
                const uint32_t va4 = half + v_at + k * 128;
                const uint4 x0 = lds128(va4), x1 = lds128(va4 + kRp * 16);
                const uint4 x2 = lds128(va4 + 8 * kRp * 16), x3 = lds128(va4 + 9 * kRp * 16);
                const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
                const uint32_t w2[4] = {x2.x, x2.y, x2.z, x2.w}, w3[4] = {x3.x, x3.y, x3.z, x3.w};
                if constexpr (kF32) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {          // elements 2j and 2j + 1 of the piece
                        const uint32_t lo_rows[4] = {w0[2 * j], w0[2 * j + 1], w1[2 * j], w1[2 * j + 1]};
                        const uint32_t up_rows[4] = {w2[2 * j], w2[2 * j + 1], w3[2 * j], w3[2 * j + 1]};
                        uint32_t hi[4], lo[4], hi2[4], lo2[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            split_tf32(__uint_as_float(lo_rows[i]), &hi[i], &lo[i]);
                            split_tf32(__uint_as_float(up_rows[i]), &hi2[i], &lo2[i]);
                        }
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            float unit[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma<T>(unit, lo, b0[t], b1[t]);
                            mma<T>(unit, lo2, b2[t], b3[t]);
                            mma<T>(unit, hi, b0[t], b1[t]);
                            mma<T>(unit, hi2, b2[t], b3[t]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[2 * k + j][t][i] += unit[i];
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {          // elements 2j and 2j + 1 of the piece
                        const uint32_t va[4] = {__byte_perm(w0[j], w1[j], 0x5410), __byte_perm(w0[j], w1[j], 0x7632),
                                                __byte_perm(w2[j], w3[j], 0x5410), __byte_perm(w2[j], w3[j], 0x7632)};
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            float unit[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma<T>(unit, va, b0[t], b1[t]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[4 * k + j][t][i] += unit[i];
                        }
                    }
                }
            }
        }

        // Join the warps: one reference per head, then the sums in warp order.
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            for (int k = 4; k < 32; k <<= 1) l[t] += __shfl_xor_sync(kFullMask, l[t], k);
            if (r == 0) s_m[warp][4 * t + c] = m[t], s_l[warp][4 * t + c] = l[t];
        }
        __syncthreads();
        float keep[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float top = -INFINITY, sum = 0.0f;
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][4 * t + c]);
            for (int w = 0; w < kWarps; ++w)
                if (s_m[w][4 * t + c] != -INFINITY) sum += s_l[w][4 * t + c] * exp2_fast(s_m[w][4 * t + c] - top);
            keep[t] = m[t] == -INFINITY ? 0.0f : exp2_fast(m[t] - top);
            if (warp == 0 && r == 0) s_M[4 * t + c] = top, s_L[4 * t + c] = sum;
        }
        constexpr int kPer = kF32 ? 4 : 8;                 // consecutive elements a lane holds per V block
        for (int w = 0; w < kWarps; ++w) {
            if (warp == w) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < kAcc; ++i) {
                        const int k = i / (kPer / 2), j = i % (kPer / 2);
                        float2 *dst = reinterpret_cast<float2 *>(s_o + (4 * t + c) * D + k * 8 * kPer + r * kPer + 2 * j);
                        constexpr float kLow = 1 / Range<T>::low;
                        float2 v = make_float2(fmaf(o[i][t][1], kLow, o[i][t][0]) * keep[t], fmaf(o[i][t][3], kLow, o[i][t][2]) * keep[t]);
                        if (w) v.x += dst->x, v.y += dst->y;
                        *dst = v;
                    }
            }
            __syncthreads();
        }

        const bool whole = head_start >= 0 && head_end <= count;
        bool write = whole;
        if (!whole) {
            // A part: the head's first CTA keeps it in its second place, a later one in its first.
            const int first = static_cast<int>((c0 + head_start) / per), last = static_cast<int>((c0 + head_end - 1) / per);
            float *mine = a.parts + (2ll * blockIdx.x + (static_cast<int>(blockIdx.x) == first)) * S::kPart;
            for (int i = tid; i < S::kHeads * D; i += kThreads) __stcg(mine + i, s_o[i]);
            if (tid < S::kHeads) {
                __stcg(mine + S::kHeads * D + tid, s_M[tid]);
                __stcg(mine + S::kHeads * (D + 1) + tid, s_L[tid]);
            }
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                s_last = atomicAdd(a.tickets + first, 1u) == static_cast<unsigned>(last - first);
                if (s_last) a.tickets[first] = 0;
                __threadfence();
            }
            __syncthreads();
            write = s_last;
            if (write) {
                // Each thread joins four elements of a head (or of some), kJoin parts on their way at a time, in order.
                const auto part = [&](int j) { return a.parts + (2ll * j + (j == first)) * S::kPart; };
                constexpr int kItems = S::kHeads * D / 4 > kThreads ? S::kHeads * D / 4 / kThreads : 1, kJoin = kItems > 2 ? 4 : 8;
                float top[kItems], sum[kItems];
                float4 acc[kItems];
                int at4[kItems];                           // (a tile of 64 elements has work for half the threads)
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    top[i] = -INFINITY;
                    sum[i] = 0.0f;
                    acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    at4[i] = min(tid + i * kThreads, S::kHeads * D / 4 - 1);
                }
                for (int j0 = first; j0 <= last; j0 += kJoin) {
                    float pm[kItems][kJoin], pl[kItems][kJoin];
                    float4 v[kItems][kJoin];
#pragma unroll
                    for (int j = 0; j < kJoin; ++j) {
                        const float *p = part(min(j0 + j, last));
#pragma unroll
                        for (int i = 0; i < kItems; ++i) {
                            pm[i][j] = __ldcg(p + S::kHeads * D + at4[i] * 4 / D);
                            pl[i][j] = __ldcg(p + S::kHeads * (D + 1) + at4[i] * 4 / D);
                            v[i][j] = __ldcg(reinterpret_cast<const float4 *>(p) + at4[i]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kItems; ++i) {
                        float next = top[i];
#pragma unroll
                        for (int j = 0; j < kJoin; ++j) next = fmaxf(next, pm[i][j]);
                        const float old = next == -INFINITY ? 0.0f : exp2_fast(top[i] - next);
                        top[i] = next;
                        sum[i] *= old;
                        acc[i].x *= old, acc[i].y *= old, acc[i].z *= old, acc[i].w *= old;
#pragma unroll
                        for (int j = 0; j < kJoin; ++j) {
                            const float w = j0 + j > last || next == -INFINITY ? 0.0f : exp2_fast(pm[i][j] - next);
                            sum[i] = fmaf(pl[i][j], w, sum[i]);
                            acc[i].x = fmaf(v[i][j].x, w, acc[i].x);
                            acc[i].y = fmaf(v[i][j].y, w, acc[i].y);
                            acc[i].z = fmaf(v[i][j].z, w, acc[i].z);
                            acc[i].w = fmaf(v[i][j].w, w, acc[i].w);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    reinterpret_cast<float4 *>(s_o)[at4[i]] = acc[i];   // (what more threads than items write is the same)
                    if (at4[i] * 4 % D == 0) s_M[at4[i] * 4 / D] = top[i], s_L[at4[i] * 4 / D] = sum[i];
                }
                __syncthreads();
            }
        }
        if (write) {
            Q *out = reinterpret_cast<Q *>(a.out) + at.b * a.out_batch + h0 * a.out_head;
            for (int i = tid; i < live * D; i += kThreads) {
                const int h = i / D, k = i - h * D;
                if (k < d) out[h * a.out_head + k] = from_float<Q>(s_M[h] == -INFINITY ? 0.0f : s_o[i] / s_L[h]);
            }
            if (tid < live) {
                const float sum2 = s_M[tid] == -INFINITY ? -INFINITY : s_M[tid] + log2f(s_L[tid]);
                if (a.lse) a.lse[static_cast<long long>(at.b) * a.n_head + h0 + tid] = sum2 * 0.693147180559945309417f;
                if (a.lse2) a.lse2[(static_cast<long long>(at.b) * heads + at.s) * S::kHeads + tid] = sum2;
            }
        }
        f = end;
        if (f < count) {
            at.advance(a, heads, end - head_start - at.u);
            if (!kAhead) load_q(at);
        }
    }
    cp_async_wait<0>();
    empty_sequences();
}

struct WeightArgs {
    KvView kv;
    const float *scores, *lse2, *weights;
    float *weights_out;
    long long slots, aux_stride;
    int group, tiles, heads;           // heads of a tile as the scores hold them
    float decay;
};

// weights_out = decay weights + sum over the query heads of 2^(t - log2 sum
// 2^t), from the scores that the attention left: a thread per slot that the
// table can hold, since the host does not know the lengths (8 sequences of 4300
// slots, attention and weights: 48 us with a table of 4352 slots, 62 with one of
// 131072). It is on the GPU before the attention ends, and has read by then what
// that does not write.
__global__ void __launch_bounds__(256) kv_weights_kernel(const WeightArgs a) {
    const int h = blockIdx.y, b = blockIdx.z, slot = blockIdx.x * 256 + threadIdx.x;
    const long long head = static_cast<long long>(b) * a.kv.n_head_kv + h, aux = head * a.aux_stride + slot;
    const bool on = slot < kv_length(a.kv, b);
    float w = on && a.weights ? a.decay * a.weights[aux] : 0.0f;
    pdl_wait_prior_grid();                                 // the attention's scores and sums
    if (!on) return;
    float sum = 0.0f;
    for (int tile = 0; tile < a.tiles; ++tile) {
        const long long s = head * a.tiles + tile;
        const float4 *t4 = reinterpret_cast<const float4 *>(a.scores + (s * a.slots + slot) * a.heads);
        const float4 *l4 = reinterpret_cast<const float4 *>(a.lse2 + s * a.heads);
        const int live = min(a.heads, a.group - tile * a.heads);
        for (int i = 0; i < live; i += 4) {
            const float4 t = __ldcg(t4 + i / 4), l = __ldcg(l4 + i / 4);
            const float v[4] = {t.x, t.y, t.z, t.w}, lse[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < live && v[j] != -INFINITY) sum += exp2_fast(v[j] - lse[j]);
        }
    }
    a.weights_out[aux] = w + sum;
}

// Query heads of a tile: eight in one pass over the rows, or four where there are no more. (Groups of eight as two
// tiles of four, 16 x 8192 slots: 199 against 121 us; 4 x 1024 slots, from the L2: 22.6 against 26.5 us.) More query
// heads than eight read the rows again for each tile: 8 x 65536 bfloat16 slots of 128 take 76 us for 8 heads on one
// cache head, 117 for 16 and 250 for 40.
int heads_of_tile(int group) { return group <= 4 ? 4 : 8; }
int tiles_of(int group) { return (group + heads_of_tile(group) - 1) / heads_of_tile(group); }

template <typename Q, typename T, int D, int NT>
cudaError_t launch_shape(const AttendArgs &a, cudaStream_t stream) {
    using S = Shape<T, D, NT>;
    const void *fn = reinterpret_cast<const void *>(kv_attend_kernel<Q, T, D, NT>);
    if (!ensure_smem(fn, S::kSmem)) return cudaErrorInvalidValue;
    const int grid = min(sm_count() * resident_ctas(fn, kThreads, S::kSmem), kMaxCtas);
    if (grid < 1) return cudaErrorInvalidConfiguration;
    kv_attend_kernel<Q, T, D, NT><<<grid, kThreads, S::kSmem, stream>>>(a);
    return cudaGetLastError();
}

template <typename Q, typename T>
cudaError_t launch(const AttendArgs &a, cudaStream_t stream) {
    const int d = a.kv.head_dim;
    if (a.group <= 4)
        return d <= 64 ? launch_shape<Q, T, 64, 1>(a, stream)
                       : d <= 128 ? launch_shape<Q, T, 128, 1>(a, stream) : launch_shape<Q, T, 256, 1>(a, stream);
    return d <= 64 ? launch_shape<Q, T, 64, 2>(a, stream)
                   : d <= 128 ? launch_shape<Q, T, 128, 2>(a, stream) : launch_shape<Q, T, 256, 2>(a, stream);
}

// Floats of all parts: two a CTA, of the kernel's padded head size.
uint64_t part_floats(int head_dim, int group) {
    const int d = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    return 2ull * kMaxCtas * heads_of_tile(group) * (d + 2);
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
    if (static_cast<int64_t>(a->n_head) * kv->batch > 1 << 24 ||
        (static_cast<int64_t>(kv->table_cols) * kv->page_size / kUnit + 1) * a->n_head * kv->batch > 1ll << 38)
        return bad("more than 2^24 query heads, or 2^42 slots of theirs, in a call");
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
    } else if (a->weights) {
        return bad("weights without weights_out");
    }
    if (!a->workspace || a->workspace % 16 ||
        a->workspace_bytes < b200_kv_attend_workspace(kv, a->n_head, a->weights_out != 0))
        return bad("needs a workspace of b200_kv_attend_workspace() bytes, 16-byte aligned");
    return 0;
}

size_t serve_scratch_bytes() { return 256 + kMaxCtas * 4; }   // the other calls' tickets come first

cudaError_t kv_attend_launch(const b200_kv_t *kv, const b200_kv_attend_t *p, void *scratch, cudaStream_t stream) {
    AttendArgs a;
    a.kv = kv_view(kv);
    a.page_magic = (1ull << 40) / static_cast<unsigned>(kv->page_size) + 1;
    a.whole_units = kv->page_size % kUnit == 0;
    a.q = reinterpret_cast<const char *>(p->q);
    a.out = reinterpret_cast<char *>(p->out);
    a.q_batch = p->q_batch_stride;
    a.q_head = p->q_head_stride;
    a.out_batch = p->out_batch_stride;
    a.out_head = p->out_head_stride;
    a.n_head = p->n_head;
    a.group = p->n_head / kv->n_head_kv;
    a.tiles = tiles_of(a.group);
    a.scale = p->scale;
    a.lse = reinterpret_cast<float *>(p->lse);
    a.slots = static_cast<long long>(kv->table_cols) * kv->page_size;
    a.tickets = reinterpret_cast<unsigned *>(static_cast<char *>(scratch) + 256);
    a.parts = reinterpret_cast<float *>(p->workspace);
    a.scores = a.lse2 = nullptr;
    const long long rows = static_cast<long long>(kv->batch) * kv->n_head_kv * a.tiles * heads_of_tile(a.group);
    if (p->weights_out) {
        a.scores = a.parts + part_floats(kv->head_dim, a.group);
        a.lse2 = a.scores + rows * a.slots;
    }
    cudaError_t e;
    if (kv->dtype == B200_F32) e = launch<float, float>(a, stream);
    else if (kv->dtype == B200_BF16) e = launch<__nv_bfloat16, __nv_bfloat16>(a, stream);
    else e = p->dtype == B200_F32 ? launch<float, __half>(a, stream) : launch<__half, __half>(a, stream);
    if (e != cudaSuccess || !p->weights_out) return e;
    WeightArgs w;
    w.kv = a.kv;
    w.scores = a.scores;
    w.lse2 = a.lse2;
    w.weights = reinterpret_cast<const float *>(p->weights);
    w.weights_out = reinterpret_cast<float *>(p->weights_out);
    w.slots = a.slots;
    w.aux_stride = p->aux_stride;
    w.group = a.group;
    w.tiles = a.tiles;
    w.heads = heads_of_tile(a.group);
    w.decay = p->decay;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((a.slots + 255) / 256), kv->n_head_kv, kv->batch);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv_weights_kernel, w);
}

}  // namespace b200

extern "C" uint64_t b200_kv_attend_workspace(const b200_kv_t *kv, int n_head, int with_weights) {
    if (!kv || kv->batch < 1 || kv->n_head_kv < 1 || kv->table_cols < 1 || kv->page_size < 1 || n_head < kv->n_head_kv) return 0;
    const int group = n_head / kv->n_head_kv;
    uint64_t n = b200::part_floats(kv->head_dim, group);
    if (with_weights)
        n += static_cast<uint64_t>(kv->batch) * kv->n_head_kv * b200::tiles_of(group) * b200::heads_of_tile(group) *
             (static_cast<uint64_t>(kv->table_cols) * kv->page_size + 1);
    return n * 4;
}
