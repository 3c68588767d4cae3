// b200_sample: the next token of each row of logits.
//
// A row lies in the shared memory of a cluster of CTAs, so its logits are read
// from memory once; where even eight CTAs have no room for it, the later passes
// read it again through the L2. Weights are whole numbers, so every sum is the
// same in any order, and atomics do no harm.
//
// The cut that the filters make is found among few candidates. For top-k, the
// k-th largest of the threads' own maxima bounds the k-th largest logit from
// below; for top-p, a sum over the tokens within 2^-10 of the largest shows
// whether those hold enough weight. The candidates go to one CTA, which orders a
// few each against each, and selects among more by 8-bit digits. A row that they
// do not settle (a flat distribution, a large k) is summed by distance from the
// top over all its tokens first, and the bin that the cut falls in goes to the
// list; one with too many equal logits for that is cut by digits of all its
// keys.
//
// What bounds it: the chain of barriers within a cluster, about a microsecond
// each with the CTAs' skew, and for many rows the instructions of the passes
// (13 a token and pass at least: exponent, power, two halves of the weight). One
// row of 128256, calls behind one another: 10 us without filters, 14 with top-k,
// 27 with top-p alone. 256 such rows: 46 us greedy, 76 without filters, 104 with
// top-k 100, 270 with top-p 0.9 alone (five passes); a mixture 158 (reading them
// takes 20). Whole rows by one CTA each, read again through the L2: 150 for the
// mixture, but slower for greedy rows (63) and for some filters.
#include <cuda_runtime.h>

#include "common.cuh"
#include "serve_dev.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kUnitBits = 40;                  // a token's largest weight is 2^40
constexpr int kShareBits = 24;                 // u and top_p count in 2^-24
constexpr int kList = 4096;                    // candidates
constexpr int kBins = 1024;                    // of the threads' maxima
constexpr int kMaxListK = 2048;                // top_k beyond this goes by the whole row
constexpr float kNear = -10.0f;                // exponents near the top, tried first for top-p
constexpr int kFew = 128;                      // candidates that are ordered each against each
// The sides of these, measured on rows of 128256, one and 64 of them. Listed by the maxima against the whole row:
// k = 1000 24.6 and 51 against 30.7 and 61 us, k = 2000 30.7 and 61 against the same. Near tokens tried first
// against not: top-p 0.5 at a spread of 3.5, 24 and 50 against 35 and 76 us; where they do not do, no more. Each
// against each or digits: k = 100 18.4 and 37 against 20.5 and 41 us, k = 200 22.5 and 47 against 20.5 and 41.

// What a CTA tells the others, each thing in a place of its own.
enum : int {
    kTellTop, kTellFirst, kTellAll, kTellNear, kTellCount, kTellSum, kTellTies, kTellKept,
    kTellCut,                                  // of the counts, and of the weights
    kTellAbove = kTellCut + 2,
    kTellList = kTellAbove + 2,                // of the first list, and as above
    kTold = kTellList + 3,
};

using u64 = unsigned long long;

struct SampleArgs {
    const char *logits;
    long long row_stride;   // elements
    int n;
    int slice;              // 16-byte pieces of a row that a CTA takes
    unsigned *status;       // the device's status word
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

// log2 of a token's weight, 0 at the top itself (where x - top or c may not be
// finite). No fused multiply-add: it is the same wherever it is computed.
__device__ __forceinline__ float exponent(float x, float top, float c) {
    return x == top ? 0.0f : x == -INFINITY ? -INFINITY : __fmul_rn(__fsub_rn(x, top), c);
}
// 2^y, to 2 units in its last place; below 2^-41, where a weight is 0, as 0.
__device__ __forceinline__ float power(float y) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
    return y >= -41.0f ? e : 0.0f;
}
// floor(2^40 e), e <= 1, as (hi - kBase) * 2^23 + (lo - kBase): adding 2^23 with
// rounding down leaves a whole number in the low bits, on the ordinary float
// pipe (a conversion to 64 bits has a small part of its rate). Sums of hi and
// of lo stay apart, in 32 bits, as long as they are short.
constexpr uint32_t kBase = 0x4b000000u;        // bits of 2^23
__device__ __forceinline__ void split_units(float e, uint32_t *hi, uint32_t *lo) {
    const float t = e * 131072.0f, h = __fadd_rd(t, 8388608.0f);
    *hi = __float_as_uint(h);
    *lo = __float_as_uint(__fmaf_rd(t - (h - 8388608.0f), 8388608.0f, 8388608.0f));
}
__device__ __forceinline__ u64 join_units(uint32_t hi, uint32_t lo, uint32_t count) {
    return (static_cast<u64>(hi - count * kBase) << 23) + (lo - count * kBase);
}
__device__ __forceinline__ u64 units(float e) {
    uint32_t hi, lo;
    split_units(e, &hi, &lo);
    return join_units(hi, lo, 1);
}

// floor(share * total / 2^24), total < 2^62, and the same rounded up.
__device__ __forceinline__ u64 part(u64 share, u64 total) {
    return (total >> kShareBits) * share + (((total & 0xffffff) * share) >> kShareBits);
}
__device__ __forceinline__ u64 part_up(u64 share, u64 total) {
    return part(share, total) + (((total & 0xffffff) * share & 0xffffff) != 0);
}

// Another CTA's shared memory (cluster_map addresses).
__device__ __forceinline__ void cluster_store(uint32_t a, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
// The sums over the cluster of two neighbouring values in every CTA, all loads
// on their way at once.
__device__ __forceinline__ void cluster_sum2(const u64 *mine, unsigned ctas, u64 sum[2]) {
    u64 v[kMaxCluster][2];
#pragma unroll
    for (unsigned q = 0; q < kMaxCluster; ++q) {
        v[q][0] = v[q][1] = 0;
        if (q < ctas)
            asm volatile("ld.shared::cluster.v2.u64 {%0, %1}, [%2];" : "=l"(v[q][0]), "=l"(v[q][1]) : "r"(cluster_map(mine, q)) : "memory");
    }
    sum[0] = sum[1] = 0;
#pragma unroll
    for (unsigned q = 0; q < kMaxCluster; ++q) sum[0] += v[q][0], sum[1] += v[q][1];
}
__device__ __forceinline__ void cluster_sum2(const unsigned *mine, unsigned ctas, u64 sum[2]) {
    unsigned v[kMaxCluster][2];
#pragma unroll
    for (unsigned q = 0; q < kMaxCluster; ++q) {
        v[q][0] = v[q][1] = 0;
        if (q < ctas)
            asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v[q][0]), "=r"(v[q][1]) : "r"(cluster_map(mine, q)) : "memory");
    }
    sum[0] = sum[1] = 0;
#pragma unroll
    for (unsigned q = 0; q < kMaxCluster; ++q) sum[0] += v[q][0], sum[1] += v[q][1];
}

struct Yes {
    static constexpr bool value = true;
};
struct No {
    static constexpr bool value = false;
};

struct Shared {
    alignas(16) u64 mass[2][256];       // sums by digit, of this pass and the one before
    alignas(16) u64 sums[kBins];        // sums by distance from the top
    u64 gather[kMaxCluster][kTold];     // what every CTA of the cluster tells the others
    u64 warp[kWarps], warp_ties[kWarps];
    u64 left;
    u64 weight;
    uint32_t prefix;
    unsigned listed;                    // candidates of this CTA
    int bin, last_bin;

    // the threads' maxima by their distance from the top: in the upper half of the sums, which come later
    __device__ __forceinline__ unsigned *bins() { return reinterpret_cast<unsigned *>(sums + kBins / 2); }
};

// Every warp does these sums for itself, from values that the warps (or CTAs)
// left, a lane to each: a loop over them in every thread would cost as much as
// a pass over the row.
template <int kWidth>
__device__ __forceinline__ u64 lanes_scan(u64 v) {   // inclusive, over the first kWidth lanes
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 1; k < kWidth; k <<= 1) {
        const u64 y = __shfl_up_sync(kFullMask, v, k);
        if (lane >= k) v += y;
    }
    return v;
}
template <int kWidth>
__device__ __forceinline__ u64 lanes_sum(u64 v) {    // over each kWidth lanes
#pragma unroll
    for (int k = kWidth / 2; k; k >>= 1) v += __shfl_xor_sync(kFullMask, v, k);
    return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) { return lanes_sum<32>(v); }
__device__ __forceinline__ u64 warps_total(const u64 *s) { return lanes_sum<kWarps>(s[threadIdx.x % kWarps]); }

// Inclusive prefix of one value per thread, and the total.
__device__ __forceinline__ u64 block_scan(u64 v, u64 *s, u64 *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = lanes_scan<32>(v);
    __syncthreads();
    if (lane == 31) s[warp] = v;
    __syncthreads();
    const u64 upto = lanes_scan<kWarps>(s[lane % kWarps]);
    *total = __shfl_sync(kFullMask, upto, kWarps - 1);
    const u64 before = __shfl_sync(kFullMask, upto, warp > 0 ? warp - 1 : 0);
    return warp > 0 ? v + before : v;
}

// The digit at which the sum over 256 bins (from the highest, or the lowest)
// first reaches s.left; narrows s.prefix to it. The first warp's work.
template <bool kFromTop, typename V>
__device__ __forceinline__ void pick_bin(Shared &s, const V *bins, int shift) {
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    u64 c[8], mine = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) mine += c[j] = bins[kFromTop ? 255 - (lane * 8 + j) : lane * 8 + j];
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
        const int bin = lane * 8 + j;
        s.prefix |= static_cast<uint32_t>(kFromTop ? 255 - bin : bin) << shift;
        s.left = left - before;
    }
}

__device__ __forceinline__ unsigned shared_add(uint32_t a, unsigned v) {
    unsigned old;
    asm volatile("atom.shared.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(a), "r"(v) : "memory");
    return old;
}

// Without the old value, and only where `on`: one predicated instruction, so that several are on their way at once.
__device__ __forceinline__ void shared_add_if(uint32_t a, unsigned v, bool on) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p red.shared.add.u32 [%0], %1;\n\t}" ::"r"(a), "r"(v), "r"(static_cast<unsigned>(on))
                 : "memory");
}

// Add w to a 64-bit sum in this CTA's shared memory: its halves are summed by
// 32-bit atomics, which the hardware has, with the low half's carry.
__device__ __forceinline__ void add_mass(u64 *sum, u64 w) {
    const uint32_t a = smem_addr(sum);
    const unsigned lo = static_cast<unsigned>(w), old = shared_add(a, lo);
    const unsigned hi = static_cast<unsigned>(w >> 32) + (old + lo < old);
    if (hi) shared_add(a + 4, hi);
}

// Selection among the N candidates of the list: value(key, idx, &digits) says
// whether a candidate takes part, what it adds, and by which number it is
// ordered; `from` is that number's highest digit's shift.
template <bool kFromTop, typename F>
__device__ __forceinline__ void select_listed(Shared &s, const u64 *list, int n, int from, u64 left, F value) {
    const int tid = threadIdx.x;
    if (tid == 0) s.prefix = 0, s.left = left;
    for (int shift = from; shift >= 0; shift -= 8) {
        if (tid < 256) s.mass[0][tid] = 0;
        __syncthreads();
        const uint32_t prefix = s.prefix, mask = shift == from ? 0 : kFullMask << (shift + 8);
        for (int i = tid; i < n; i += kThreads) {
            uint32_t digits;
            const u64 w = value(list[i], &digits);
            if (w && (digits & mask) == prefix) add_mass(&s.mass[0][digits >> shift & 255], w);
        }
        __syncthreads();
        pick_bin<kFromTop>(s, s.mass[0], shift);
        __syncthreads();
    }
}

__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

template <typename T, bool kCached>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
    constexpr int kVe = 16 / sizeof(T);         // elements of a piece
    extern __shared__ __align__(16) char dyn[];
    __shared__ Shared s;
    __shared__ uint64_t s_bar[kWarps];
    u64 *list = reinterpret_cast<u64 *>(dyn);   // rank 0: kList candidates, key << 32 | index
    uint4 *kept_row = reinterpret_cast<uint4 *>(dyn + kList * 8);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = a.n;
    const unsigned rank = cluster_ctarank();
    unsigned ctas;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    const int row = blockIdx.x / ctas;
    const T *logits = reinterpret_cast<const T *>(a.logits) + row * a.row_stride;
    // Pieces are counted from the 16-byte boundary at or before the row's first element: element i of the row is
    // element i + skew of the pieces.
    const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
    const int pieces = (n + skew + kVe - 1) / kVe;
    const int p0 = min(static_cast<int>(rank) * a.slice, pieces), p1 = min(p0 + a.slice, pieces);
    const uint4 *aligned = reinterpret_cast<const uint4 *>(logits - skew);
    // A warp's pieces lie side by side, so that its tokens do: [w0, w1).
    const int per_warp = (a.slice / kWarps + 31) / 32 * 32;
    const int w0 = min(p0 + warp * per_warp, p1), w1 = min(w0 + per_warp, p1);

    const auto fetch = [&](int p) {             // from memory; what is not of the row is -infinity
        if (p * kVe >= skew && (p + 1) * kVe - skew <= n) return __ldg(aligned + p);
        union { uint4 v; T t[kVe]; } u;
#pragma unroll
        for (int j = 0; j < kVe; ++j) {
            const int i = p * kVe + j - skew;
            u.t[j] = i >= 0 && i < n ? logits[i] : from_float<T>(-INFINITY);
        }
        return u.v;
    };
    const auto piece = [&](int p, float x[kVe]) {
        union { uint4 v; T t[kVe]; } u;
        u.v = kCached ? kept_row[p - p0] : fetch(p);
#pragma unroll
        for (int j = 0; j < kVe; ++j) x[j] = to_float(u.t[j]);
    };

    cluster_arrive();                           // every CTA of the cluster runs before any store into its shared memory
    if (kCached) {                              // a warp's whole pieces by one bulk copy, those at the row's ends apart
        const int whole = (n + skew) / kVe, b0 = max(w0, skew ? 1 : 0), b1 = min(w1, whole);
        if (lane == 0) {
            mbar_init(&s_bar[warp], 1);
            fence_mbar_init();
            if (b0 < b1) {
                mbar_arrive_expect_tx(&s_bar[warp], (b1 - b0) * 16);
                bulk_g2s(kept_row + (b0 - p0), aligned + b0, (b1 - b0) * 16, &s_bar[warp], l2_policy_evict_first());
            }
        }
        if (lane == 1 && w0 == 0 && skew && w1 > 0) kept_row[0] = fetch(0);
        if (lane == 2 && w0 <= whole && whole < w1 && !(whole == 0 && skew)) kept_row[whole - p0] = fetch(whole);
        __syncwarp();
        if (b0 < b1) wait_stage(&s_bar[warp], 0, a.status);
    }

    // The largest logit, and the smallest of the threads' maxima that are above -infinity.
    for (int i = tid; i < kBins; i += kThreads) s.bins()[i] = 0;
    if (tid == 0) s.listed = 0;
    float own = -INFINITY;                      // the thread's maximum (fmaxf passes NaN over)
#pragma unroll 4
    for (int p = w0 + lane; p < w1; p += 32) {
        float x[kVe];
        piece(p, x);
#pragma unroll
        for (int j = 0; j < kVe; ++j) own = fmaxf(own, x[j]);
    }
    float top = own, low = own == -INFINITY ? INFINITY : own;
    for (int k = 16; k; k >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, k));
        low = fminf(low, __shfl_xor_sync(kFullMask, low, k));
    }
    if (lane == 0) s.warp[warp] = static_cast<u64>(__float_as_uint(top)) << 32 | __float_as_uint(low);
    __syncthreads();
    // What each CTA has to say goes to all: gather[rank][slot], and the barrier of the cluster.
    const auto tell = [&](int slot, u64 v) {
        if (tid < static_cast<int>(ctas)) cluster_store(cluster_map(&s.gather[rank][slot], tid), v);
    };
    cluster_wait();
    {
        u64 v = s.warp[lane % kWarps];
        top = __uint_as_float(static_cast<unsigned>(v >> 32));
        low = __uint_as_float(static_cast<unsigned>(v));
        for (int k = 16; k; k >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(kFullMask, top, k));
            low = fminf(low, __shfl_xor_sync(kFullMask, low, k));
        }
        tell(kTellTop, static_cast<u64>(__float_as_uint(top)) << 32 | __float_as_uint(low));
    }
    cluster_sync_all();
    {
        const u64 v = s.gather[lane % ctas][kTellTop];
        top = __uint_as_float(static_cast<unsigned>(v >> 32));
        low = __uint_as_float(static_cast<unsigned>(v));
        for (int k = kMaxCluster / 2; k; k >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(kFullMask, top, k));
            low = fminf(low, __shfl_xor_sync(kFullMask, low, k));
        }
    }
    // a value that every CTA told, summed over the cluster
    const auto told = [&](int slot) { return lanes_sum<kMaxCluster>(lane % kMaxCluster < ctas ? s.gather[lane % kMaxCluster][slot] : 0); };
    top += 0.0f;                                // -0 as 0, as the keys have it

    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    if (top == -INFINITY) {
        if (rank == 0 && tid == 0) {
            a.token[row] = -1;
            if (a.logprob) a.logprob[row] = -INFINITY;
        }
        return;
    }
    if (!(temp > 0.0f)) {                       // the first of the largest
        int first = 0x7fffffff;
        for (int p = w0 + lane; p < w1 && first == 0x7fffffff; p += 32) {
            float x[kVe];
            piece(p, x);
#pragma unroll
            for (int j = kVe - 1; j >= 0; --j)
                if (x[j] == top) first = p * kVe + j - skew;
        }
        first = __reduce_min_sync(kFullMask, first);
        if (lane == 0) s.warp[warp] = first;
        __syncthreads();
        first = __reduce_min_sync(kFullMask, static_cast<int>(s.warp[lane % kWarps]));
        tell(kTellFirst, first);
        cluster_sync_all();
        if (rank == 0 && tid == 0) {
            for (unsigned q = 0; q < ctas; ++q) first = min(first, static_cast<int>(s.gather[q][kTellFirst]));
            a.token[row] = first;
            if (a.logprob) a.logprob[row] = 0.0f;
        }
        return;
    }
    const float c = __fdiv_rn(1.44269504088896340736f, temp);
    const float min_p = a.min_p && a.min_p[row] > 0.0f ? a.min_p[row] : 0.0f;
    const auto weight = [&](float x) { return units(power(exponent(x, top, c))); };
    // where x - top and c are finite numbers, the exponent is their product, whatever x (-infinity, NaN: far below 0)
    const bool plain = top < INFINITY && c < INFINITY;
    // The passes over a row are written without branches: exponents that are far below 0 at least, their powers, and
    // masks. `is_plain` (Yes or No) says whether `plain` holds.
    const auto y_of = [&](auto is_plain, float x) {
        if constexpr (decltype(is_plain)::value) return fmaxf(__fmul_rn(__fsub_rn(x, top), c), -64.0f);
        else return fmaxf(exponent(x, top, c), -64.0f);
    };
    const auto power_of = [](float y) {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
        return e;
    };
    const int k = a.top_k && a.top_k[row] > 0 && a.top_k[row] < n ? a.top_k[row] : 0;
    const float share_p = a.top_p ? a.top_p[row] : 1.0f;
    const long long p24 = share_p < 1.0f ? __float2ll_rn(fmaxf(share_p, 0.0f) * 16777216.0f) : 1ll << kShareBits;
    const bool by_p = p24 < 1ll << kShareBits;
    const float u = a.u[row];
    const u64 share = u > 0.0f ? static_cast<u64>(fminf(u, 1.0f - 0x1p-24f) * 16777216.0f) : 0;
    const auto finish = [&](int token, float x, u64 total) {
        a.token[row] = token;
        if (a.logprob)
            a.logprob[row] = exponent(x, top, c) * 0.693147180559945309417f -
                             logf(static_cast<float>(total) * (1.0f / static_cast<float>(1ull << kUnitBits)));
    };

    // The smallest logit that can be kept, where few enough can be.
    bool listed = false;
    float floor_x = -INFINITY;
    if (k > 0 && k <= kMaxListK) {
        listed = true;
        const float scale = top > low ? (kBins - 1) / (top - low) : 0.0f;   // 0 where top - low overflows, too
        if (own != -INFINITY) {
            const int bin = own == top ? 0 : min(static_cast<int>((top - own) * scale), kBins - 1);
            atomicAdd(&s.bins()[bin], 1u);
        }
        cluster_sync_all();
        // the bin with the k-th largest maximum: its far edge, and a little for the rounding of the bins
        u64 mine[2], total;
        cluster_sum2(&s.bins()[2 * tid], ctas, mine);
        const u64 sum = mine[0] + mine[1];
        u64 before = block_scan(sum, s.warp, &total) - sum;
        if (tid == 0) s.bin = kBins;
        __syncthreads();
        if (before < static_cast<u64>(k) && static_cast<u64>(k) <= before + sum) {
            s.bin = 2 * tid + (before + mine[0] < static_cast<u64>(k));
        }
        __syncthreads();
        if (s.bin < kBins - 1 && scale > 0.0f) floor_x = top - (s.bin + 1.01f) / scale;
    } else if (k == 0 && by_p) {
        // the weight of all tokens, and of those within 2^-10 of the largest
        u64 all = 0, near = 0;
        unsigned near_count = 0;
        const auto weigh_all = [&](auto is_plain) {
#pragma unroll 2
            for (int p = w0 + lane; p < w1; p += 32) {
                float x[kVe];
                piece(p, x);
                uint32_t hi = 0, lo = 0, near_hi = 0, near_lo = 0;
#pragma unroll
                for (int j = 0; j < kVe; ++j) {
                    const float y = y_of(is_plain, x[j]);
                    uint32_t h, l;
                    split_units(power_of(y), &h, &l);
                    hi += h, lo += l;
                    const uint32_t is_near = y >= kNear ? kFullMask : 0;
                    near_hi += (h - kBase) & is_near, near_lo += (l - kBase) & is_near;
                    near_count -= is_near;
                }
                all += join_units(hi, lo, kVe);
                near += join_units(near_hi, near_lo, 0);
            }
        };
        if (plain) weigh_all(Yes()); else weigh_all(No());
        all = warp_sum(all), near = warp_sum(near);
        near_count = __reduce_add_sync(kFullMask, near_count);
        if (lane == 0) s.mass[0][warp] = all, s.mass[0][32 + warp] = near, s.mass[0][64 + warp] = near_count;
        __syncthreads();
        all = warps_total(s.mass[0]), near = warps_total(s.mass[0] + 32);
        tell(kTellAll, all), tell(kTellNear, near), tell(kTellCount, warps_total(s.mass[0] + 64));
        cluster_sync_all();
        all = told(kTellAll), near = told(kTellNear);
        s.weight = all;                         // every thread writes the same
        listed = part_up(static_cast<u64>(p24), all) <= near && told(kTellCount) <= kList;
    }
    // Tokens that `wanted` names go to this CTA's list, and from there to rank 0's; true where that holds all of them.
    // Call `turn` of a row; s.listed is 0 before it, and rank 0 has the number after it.
    u64 above = 0;                              // this thread's share of what lies above the list, from the second call on
    const auto collect = [&](int turn, auto wanted) {
        for (int p = w0 + lane; p < w1; p += 32) {
            float x[kVe];
            piece(p, x);
            unsigned take = 0;
#pragma unroll
            for (int j = 0; j < kVe; ++j)
                take |= static_cast<unsigned>(wanted(x[j])) << j;
            if (!take) continue;
            unsigned at = atomicAdd(&s.listed, static_cast<unsigned>(__popc(take)));
#pragma unroll
            for (int j = 0; j < kVe; ++j)
                if (take >> j & 1) {
                    if (at < kList) list[at] = static_cast<u64>(order_key(clean(x[j]))) << 32 | static_cast<unsigned>(p * kVe + j - skew);
                    ++at;
                }
        }
        if (turn > 0) {
            above = warp_sum(above);
            if (lane == 0) s.warp[warp] = above;
        }
        __syncthreads();
        const unsigned mine = s.listed;
        if (turn > 0) tell(kTellAbove + turn - 1, warps_total(s.warp));
        tell(kTellList + turn, mine);
        cluster_sync_all();
        const u64 upto = lanes_scan<kMaxCluster>(lane < static_cast<int>(ctas) ? s.gather[lane % kMaxCluster][kTellList + turn] : 0);
        const u64 all = __shfl_sync(kFullMask, upto, kMaxCluster - 1), before = __shfl_sync(kFullMask, upto, rank) - mine;
        if (all <= kList && rank > 0) {
            const uint32_t there = cluster_map(list, 0) + static_cast<uint32_t>(before) * 8;
            for (unsigned i = tid; i < mine; i += kThreads) cluster_store(there + i * 8, list[i]);
        }
        if (rank == 0 && tid == 0) s.listed = static_cast<unsigned>(all);
        cluster_sync_all();
        return all <= kList;
    };
    if (listed) {
        if (k > 0) listed = collect(0, [&](float x) { return (x >= floor_x) & (x != -INFINITY); });
        else if (plain) listed = collect(0, [&](float x) { return y_of(Yes(), x) >= kNear; });
        else listed = collect(0, [&](float x) { return y_of(No(), x) >= kNear; });
        if (listed && rank != 0) return;        // rank 0 does the rest, in its own memory
    }
    if (listed) {
        const int m = static_cast<int>(s.listed);
        if (m <= kFew) {
            // Each candidate against each, kThreads / wide threads to one: its rank and the weight before it, both in
            // falling order; then, of what is kept, the weight of lower indexes.
            int wide = 32;
            while (wide < m) wide *= 2;
            const int i = tid & (wide - 1), part0 = tid / wide, parts = kThreads / wide;
            const u64 e = i < m ? list[i] ^ 0xffffffffull : 0;     // the lower index is the larger number
            const float x = value_of(static_cast<uint32_t>(e >> 32)), v = power(exponent(x, top, c));
            const u64 w = i < m ? units(v) : 0;
            u64 *weights = s.mass[0], *kept = s.mass[1];
            if (tid < wide) weights[i] = w;
            __syncthreads();
            u64 before = 0, sum;
            unsigned ahead = 0;
            for (int j = part0; j < m; j += parts)
                if ((list[j] ^ 0xffffffffull) > e) ++ahead, before += weights[j];
            s.sums[tid] = before;
            s.bins()[tid] = ahead;
            __syncthreads();
            before = ahead = 0;
            for (int j = 0; j < parts; ++j) before += s.sums[j * wide + i], ahead += s.bins()[j * wide + i];
            bool keep = i < m && (k == 0 || ahead < static_cast<unsigned>(k));
            if (by_p) {
                u64 all = s.weight;
                if (k > 0) block_scan(tid < wide && keep ? w : 0, s.warp, &all);
                u64 need = part_up(static_cast<u64>(p24), all);
                if (need < 1) need = 1;
                keep = keep && before < need;
            }
            keep = keep && (v >= min_p || ahead == 0);
            const u64 mine = keep ? w : 0;
            block_scan(tid < wide ? mine : 0, s.warp, &sum);
            if (tid < wide) kept[i] = mine;
            const u64 target = part(share, sum);
            const uint32_t index = static_cast<uint32_t>(list[i < m ? i : 0]);
            __syncthreads();
            before = 0;
            for (int j = part0; j < m; j += parts)
                if (static_cast<uint32_t>(list[j]) < index) before += kept[j];
            s.sums[tid] = before;
            __syncthreads();
            if (tid < wide && mine) {
                before = 0;
                for (int j = 0; j < parts; ++j) before += s.sums[j * wide + i];
                if (before <= target && target < before + mine) finish(static_cast<int>(index), x, sum);
            }
            return;
        }
        uint32_t edge = 0;
        u64 ties = 0, total;
        if (k > 0 && k < m) {
            select_listed<true>(s, list, m, 24, k, [](u64 e, uint32_t *d) {
                *d = static_cast<uint32_t>(e >> 32);
                return 1ull;
            });
            edge = s.prefix;
            ties = s.left;
        }
        if (by_p) {
            u64 sum = 0;
            if (k > 0) {                        // of the k, the ties at the edge by their number
                for (int i = tid; i < m; i += kThreads)
                    if (static_cast<uint32_t>(list[i] >> 32) > edge) sum += weight(value_of(static_cast<uint32_t>(list[i] >> 32)));
                block_scan(sum, s.warp, &sum);
            } else {
                sum = s.weight;
            }
            u64 w_edge = 0;
            if (edge) w_edge = weight(value_of(edge)) * ties;
            u64 need = part_up(static_cast<u64>(p24), sum + w_edge);
            if (need < 1) need = 1;
            __syncthreads();
            if (tid == 0) s.prefix = 0, s.left = need;
            for (int shift = 24; shift >= 0; shift -= 8) {
                if (tid < 256) s.mass[0][tid] = 0;
                __syncthreads();
                const uint32_t prefix = s.prefix, mask = shift == 24 ? 0 : kFullMask << (shift + 8);
                for (int i = tid; i < m; i += kThreads) {
                    const uint32_t key = static_cast<uint32_t>(list[i] >> 32);
                    if (key > edge && (key & mask) == prefix) {
                        const u64 w = weight(value_of(static_cast<uint32_t>(list[i] >> 32)));
                        if (w) add_mass(&s.mass[0][key >> shift & 255], w);
                    }
                }
                if (tid == 0 && w_edge && (edge & mask) == prefix) add_mass(&s.mass[0][edge >> shift & 255], w_edge);
                __syncthreads();
                pick_bin<true>(s, s.mass[0], shift);
                __syncthreads();
            }
            edge = s.prefix;
            const u64 w = weight(value_of(edge));
            ties = (s.left + w - 1) / w;
            __syncthreads();
        }
        if (min_p > 1.0f) edge = order_key(top), ties = 1;
        // the ties' lowest indexes: up to `last`
        u64 equal = 0;
        for (int i = tid; i < m; i += kThreads) equal += static_cast<uint32_t>(list[i] >> 32) == edge;
        block_scan(equal, s.warp, &equal);
        uint32_t last = kFullMask;
        if (ties < equal) {
            select_listed<false>(s, list, m, 16, ties, [edge](u64 e, uint32_t *d) {
                *d = static_cast<uint32_t>(e);
                return static_cast<u64>(static_cast<uint32_t>(e >> 32) == edge);
            });
            last = s.prefix;
        }
        const auto kept = [&](u64 e, uint32_t *d) -> u64 {
            const uint32_t key = static_cast<uint32_t>(e >> 32);
            *d = static_cast<uint32_t>(e);
            if (key < edge || (key == edge && *d > last)) return 0;
            const float x = value_of(key), v = power(exponent(x, top, c));
            return v < min_p && x != top ? 0 : units(v);
        };
        u64 sum = 0;
        for (int i = tid; i < m; i += kThreads) {
            uint32_t d;
            sum += kept(list[i], &d);
        }
        block_scan(sum, s.warp, &total);
        __syncthreads();
        select_listed<false>(s, list, m, 16, part(share, total) + 1, kept);
        const uint32_t token = s.prefix;
        for (int i = tid; i < m; i += kThreads)
            if (static_cast<uint32_t>(list[i]) == token) finish(static_cast<int>(token), value_of(static_cast<uint32_t>(list[i] >> 32)), total);
        return;
    }

    // The whole row. What the filters keep of it: keys above `edge`, and the first `ties` at it. First by the
    // distance from the top, in kBins bins up to where a weight is 0; then among the tokens of the bin it falls in;
    // where those are too many for the list, by 8-bit digits of all keys.
    uint32_t edge = 0;
    u64 ties = 0;
    constexpr float kBinsPerOctave = kBins / 41.0f;
    const auto bin_of_y = [](float y) {         // 1023 for all that weighs nothing, NaN among it
        return static_cast<int>(__float_as_uint(__fmaf_rd(-fmaxf(y, -40.97f), kBinsPerOctave, 8388608.0f)) - kBase);
    };
    const auto bin_of = [&](float x) { return bin_of_y(exponent(x, top, c)); };
    // `left` tokens (or weight, `total` in all) are kept, of those above the present edge and edge_mass at it
    const auto cut_row = [&](u64 left, bool by_mass, u64 total, u64 edge_mass) {
        unsigned *sums = reinterpret_cast<unsigned *>(s.sums);
        for (int i = tid; i < kBins; i += kThreads) sums[i] = 0;
        if (tid == 0) s.listed = 0, s.bin = 0, s.last_bin = kBins - 2;
        __syncthreads();
        // Weights are summed in units of 2^shift, in which all of them fit 32 bits: short by less than a unit each,
        // so the cut lies in one of a few bins. Tokens so light that all of them together are less than what is given
        // up need not be summed: the sums from the top do not come to them.
        const int shift = by_mass ? max(0, 32 - __clzll(static_cast<long long>(total))) : 0;
        const unsigned light = by_mass ? max(static_cast<unsigned>((total - left) / static_cast<u64>(n) >> shift), 1u) - 1 : 0;
        const float old_x = edge ? value_of(edge) : -INFINITY;
        const uint32_t sums_at = smem_addr(sums);
        const auto sum_up = [&](auto is_plain, auto mass) {
            for (int p = w0 + lane; p < w1; p += 32) {
                float x[kVe];
                piece(p, x);
#pragma unroll
                for (int j = 0; j < kVe; ++j) {
                    const float y = y_of(is_plain, x[j]);
                    unsigned add;
                    if constexpr (decltype(mass)::value) {
                        add = static_cast<unsigned>(units(power_of(y)) >> shift);
                        add = (x[j] > old_x) & (add > light) ? add : 0;
                    } else {
                        const int i = p * kVe + j - skew;
                        add = (i >= 0) & (i < n);
                    }
                    shared_add_if(sums_at + bin_of_y(y) * 4, add, add != 0);
                }
            }
        };
        if (!by_mass) sum_up(No(), No());
        else if (plain) sum_up(Yes(), Yes());
        else sum_up(No(), Yes());
        if (rank == 0 && tid == 0 && edge_mass) atomicAdd(&sums[bin_of(value_of(edge))], static_cast<unsigned>(edge_mass >> shift));
        cluster_sync_all();
        u64 mine[2], all;
        cluster_sum2(&sums[2 * tid], ctas, mine);
        const u64 before = block_scan(mine[0] + mine[1], s.warp, &all) - mine[0] - mine[1];
        {
            const u64 half = before + mine[0], upto = half + mine[1];
            const u64 sure = left + ((1ull << shift) - 1) >> shift, slack = by_mass ? static_cast<u64>(n) + 1 : 0;
            const u64 maybe = sure > slack ? sure - slack : 0;
            if (before < maybe && maybe <= upto) s.bin = 2 * tid + (half < maybe);
            if (before < sure && sure <= upto) s.last_bin = 2 * tid + (half < sure);
        }
        __syncthreads();
        const int bin = s.bin, last_bin = s.last_bin;
        if (bin == kBins - 1) {                 // (of the counts) what follows weighs nothing
            cluster_sync_all();
            return;
        }
        u64 w = 1;
        above = edge_mass && rank == 0 && tid == 0 && bin_of(value_of(edge)) < bin ? edge_mass : 0;
        const auto near_cut = [&](auto is_plain, auto mass) {
            return collect(1 + by_mass, [&](float x) {
                const float y = y_of(is_plain, x);
                const int b = bin_of_y(y);
                if constexpr (decltype(mass)::value) {
                    const bool open = x > old_x;
                    above += units(open & (b < bin) ? power_of(y) : 0.0f);
                    return open & (b >= bin) & (b <= last_bin);
                } else {
                    above += b < bin;
                    return (b >= bin) & (b <= last_bin);
                }
            });
        };
        const bool fits = !by_mass ? near_cut(No(), No()) : plain ? near_cut(Yes(), Yes()) : near_cut(No(), Yes());
        if (fits) {
            const u64 inside = left - told(kTellAbove + by_mass);
            if (rank == 0) {
                const int m = static_cast<int>(s.listed);
                const uint32_t old = edge;
                const int old_bin = bin_of(value_of(old));
                const bool edge_here = edge_mass && old_bin >= bin && old_bin <= last_bin;
                // the keys of a bin are near each other: from the first digit in which any differs from the first
                uint32_t differ = edge_here ? old ^ static_cast<uint32_t>(list[0] >> 32) : 0;
                for (int i = tid; i < m; i += kThreads) differ |= static_cast<uint32_t>(list[i] >> 32) ^ static_cast<uint32_t>(list[0] >> 32);
                differ = __reduce_or_sync(kFullMask, differ);
                if (lane == 0) s.warp[warp] = differ;
                __syncthreads();
                for (int q = 0; q < kWarps; ++q) differ |= static_cast<uint32_t>(s.warp[q]);
                const int from = differ >> 24 ? 24 : differ >> 16 ? 16 : differ >> 8 ? 8 : 0;
                const uint32_t above = from == 24 ? 0 : kFullMask << (from + 8);
                if (tid == 0) s.prefix = static_cast<uint32_t>(list[0] >> 32) & above, s.left = inside;
                for (int shift = from; shift >= 0; shift -= 8) {
                    if (tid < 256) s.mass[0][tid] = 0;
                    __syncthreads();
                    const uint32_t prefix = s.prefix, mask = shift == 24 ? 0 : kFullMask << (shift + 8);
                    for (int i = tid; i < m; i += kThreads) {
                        const uint32_t key = static_cast<uint32_t>(list[i] >> 32);
                        if ((key & mask) == prefix) add_mass(&s.mass[0][key >> shift & 255], by_mass ? weight(value_of(key)) : 1);
                    }
                    if (tid == 0 && edge_here && (old & mask) == prefix)
                        add_mass(&s.mass[0][old >> shift & 255], edge_mass);
                    __syncthreads();
                    pick_bin<true>(s, s.mass[0], shift);
                    __syncthreads();
                }
                if (by_mass) w = weight(value_of(s.prefix));
                tell(kTellCut + by_mass, static_cast<u64>(s.prefix) << 32 | ((s.left + w - 1) / w));
            }
            cluster_sync_all();
            edge = static_cast<uint32_t>(s.gather[0][kTellCut + by_mass] >> 32);
            ties = static_cast<uint32_t>(s.gather[0][kTellCut + by_mass]);
            return;
        }
        const uint32_t old = edge;
        int turn = 0;
        if (tid == 0) s.prefix = 0, s.left = left;
        for (int shift = 24; shift >= 0; shift -= 8, turn ^= 1) {
            if (tid < 256) s.mass[turn][tid] = 0;
            __syncthreads();
            const uint32_t prefix = s.prefix, mask = shift == 24 ? 0 : kFullMask << (shift + 8);
            for (int p = w0 + lane; p < w1; p += 32) {
                float x[kVe];
                piece(p, x);
#pragma unroll
                for (int j = 0; j < kVe; ++j) {
                    const float v = clean(x[j]);
                    const uint32_t key = order_key(v);
                    const int i = p * kVe + j - skew;
                    if (i < 0 || i >= n || (key & mask) != prefix || (by_mass && key <= old)) continue;
                    const u64 add = by_mass ? weight(v) : 1;
                    if (add) add_mass(&s.mass[turn][key >> shift & 255], add);
                }
            }
            if (rank == 0 && tid == 0 && edge_mass && (old & mask) == prefix) add_mass(&s.mass[turn][old >> shift & 255], edge_mass);
            // every CTA adds up all CTAs' sums; the next pass uses the other set, so one barrier a pass is enough
            cluster_sync_all();
            if (tid < 128) cluster_sum2(&s.mass[turn][2 * tid], ctas, &s.sums[2 * tid]);
            __syncthreads();
            pick_bin<true>(s, s.sums, shift);
            __syncthreads();
        }
        edge = s.prefix;
        if (by_mass) w = weight(value_of(edge));
        ties = (s.left + w - 1) / w;
        cluster_sync_all();
    };
    if (k > 0) cut_row(k, false, 0, 0);
    if (by_p) {
        u64 sum = s.weight;                     // of all tokens, where there is no top-k
        if (k > 0) {
            sum = 0;
            const float old_x = edge ? value_of(edge) : -INFINITY;
            const auto weigh_above = [&](auto is_plain) {
                for (int p = w0 + lane; p < w1; p += 32) {
                    float x[kVe];
                    piece(p, x);
#pragma unroll
                    for (int j = 0; j < kVe; ++j) sum += units(x[j] > old_x ? power_of(y_of(is_plain, x[j])) : 0.0f);
                }
            };
            if (plain) weigh_above(Yes()); else weigh_above(No());
            block_scan(sum, s.warp, &sum);
            tell(kTellSum, sum);
            cluster_sync_all();
            sum = told(kTellSum);
        }
        const u64 at_edge = edge ? weight(value_of(edge)) * ties : 0;
        u64 need = part_up(static_cast<u64>(p24), sum + at_edge);
        if (need < 1) need = 1;
        cut_row(need, true, sum + at_edge, at_edge);
    }
    if (min_p > 1.0f) edge = order_key(top), ties = 1;

    // The kept weight of each warp's tokens, and where u falls among them.
    const float edge_x = edge ? value_of(edge) : -INFINITY;
    // ties that weigh something: all of them are summed, and those too many taken off again
    const bool tied = edge && !(power(exponent(edge_x, top, c)) < min_p && edge_x != top);
    const u64 w_edge = tied ? weight(edge_x) : 0;
    u64 sum = 0, equal = 0;
    const auto weigh_kept = [&](auto is_plain, auto is_cut) {
#pragma unroll 2
        for (int p = w0 + lane; p < w1; p += 32) {
            float x[kVe];
            piece(p, x);
            uint32_t hi = 0, lo = 0;
            int ties_here = 0;
#pragma unroll
            for (int j = 0; j < kVe; ++j) {
                float e = power_of(y_of(is_plain, x[j]));
                uint32_t h, l;
                if constexpr (decltype(is_cut)::value) {
                    e = (x[j] < edge_x) | ((e < min_p) & (x[j] != top)) ? 0.0f : e;
                    ties_here += x[j] == edge_x;
                }
                split_units(e, &h, &l);
                hi += h, lo += l;
            }
            sum += join_units(hi, lo, kVe);
            equal += ties_here;
        }
    };
    const bool cut = edge || min_p > 0.0f;
    if (plain && !cut) weigh_kept(Yes(), No());
    else if (plain) weigh_kept(Yes(), Yes());
    else weigh_kept(No(), Yes());
    sum = warp_sum(sum);
    if (cut) equal = warp_sum(equal);
    __syncthreads();
    if (lane == 0) s.warp[warp] = sum, s.warp_ties[warp] = equal;
    __syncthreads();
    tell(kTellKept, warps_total(s.warp));
    tell(kTellTies, warps_total(s.warp_ties));
    cluster_sync_all();
    // Stretches of the row, a lane to each: their ties and sums, without the ties past the last one that is kept.
    const auto stretches = [&](u64 seen, u64 eq, u64 part_sum, u64 *ties_upto) {
        *ties_upto = lanes_scan<16>(eq);
        const u64 first = seen + *ties_upto - eq;
        return lanes_scan<16>(part_sum - (tied ? eq - (first >= ties ? 0 : min(eq, ties - first)) : 0) * w_edge);
    };
    static_assert(kMaxCluster <= 16 && kWarps <= 16, "a lane to each");
    const bool here = lane < static_cast<int>(ctas);
    u64 ties_upto;
    const u64 upto = stretches(0, here ? s.gather[lane % kMaxCluster][kTellTies] : 0, here ? s.gather[lane % kMaxCluster][kTellKept] : 0, &ties_upto);
    const u64 total = __shfl_sync(kFullMask, upto, 15), target = part(share, total);
    const unsigned cta = __ffs(__ballot_sync(kFullMask, upto > target)) - 1;
    if (rank != cta) return;
    // this CTA's, then: the warp's stretch it falls in, which all threads go over, a piece each
    u64 before = __shfl_sync(kFullMask, upto, rank > 0 ? rank - 1 : 0), seen = __shfl_sync(kFullMask, ties_upto, rank > 0 ? rank - 1 : 0);
    if (rank == 0) before = seen = 0;
    const u64 warp_upto = before + stretches(seen, lane < kWarps ? s.warp_ties[lane % kWarps] : 0, lane < kWarps ? s.warp[lane % kWarps] : 0, &ties_upto);
    const int win = __ffs(__ballot_sync(kFullMask, warp_upto > target)) - 1;
    if (win > 0) {
        before = __shfl_sync(kFullMask, warp_upto, win - 1);
        seen += __shfl_sync(kFullMask, ties_upto, win - 1);
    }
    const int f0 = min(p0 + win * per_warp, p1), f1 = min(f0 + per_warp, p1);
    for (int base = f0; base < f1; base += kThreads) {
        const int p = base + tid;
        float x[kVe];
        u64 w[kVe], all = 0, weight_all;
        if (p < f1) piece(p, x);
        u64 skip = seen;
        if (tied) {
            u64 eq = 0, eq_all;
            if (p < f1)
#pragma unroll
                for (int j = 0; j < kVe; ++j) eq += x[j] == edge_x;
            skip = seen + block_scan(eq, s.mass[0], &eq_all) - eq;
            seen += eq_all;
        }
#pragma unroll
        for (int j = 0; j < kVe; ++j) {
            w[j] = 0;
            if (p >= f1) continue;
            const float e = power(exponent(x[j], top, c));
            if (!(x[j] < edge_x || (e < min_p && x[j] != top)) && !(tied && x[j] == edge_x && skip++ >= ties)) w[j] = units(e);
            all += w[j];
        }
        u64 at = before + block_scan(all, s.mass[1], &weight_all) - all;
        if (at <= target && target < at + all) {
            bool done = false;
#pragma unroll
            for (int j = 0; j < kVe; ++j) {
                at += w[j];
                if (!done && at > target) {
                    done = true;
                    finish(p * kVe + j - skew, clean(x[j]), total);
                }
            }
        }
        before += weight_all;
        if (target < before) return;
    }
}

template <typename T, bool kCached>
cudaError_t launch(const SampleArgs &a, int batch, int ctas, cudaStream_t stream) {
    const int smem = kList * 8 + (kCached ? a.slice * 16 : 0);
    if (!ensure_smem(reinterpret_cast<const void *>(sample_kernel<T, kCached>), smem)) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(batch * ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, sample_kernel<T, kCached>, a);
}

// CTAs to a row: as many as give each at least 16 KB of it and the GPU work
// (a few rows alone), or as its share must have to fit beside another CTA's.
template <typename T>
cudaError_t launch_rows(SampleArgs a, int batch, cudaStream_t stream) {
    constexpr int kVe = 16 / sizeof(T);
    constexpr int kFit = 64 * 1024, kMost = 180 * 1024;
    const int pieces = (a.n + 2 * kVe - 2) / kVe;          // wherever the row begins
    int ctas = 1;
    while (ctas < kMaxCluster && (pieces * 16 / ctas > kFit || (batch * ctas < sm_count() && pieces * 16 / ctas >= 2 * 16384))) ctas *= 2;
    a.slice = ((pieces + ctas - 1) / ctas + kWarps * 32 - 1) / (kWarps * 32) * (kWarps * 32);
    return a.slice * 16 <= kMost ? launch<T, true>(a, batch, ctas, stream) : launch<T, false>(a, batch, ctas, stream);
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
    a.status = status_word();
    if (!a.status) return cudaErrorInvalidDevice;
    if (p->dtype == B200_F32) return launch_rows<float>(a, p->batch, stream);
    if (p->dtype == B200_F16) return launch_rows<__half>(a, p->batch, stream);
    return launch_rows<__nv_bfloat16>(a, p->batch, stream);
}

}  // namespace b200
