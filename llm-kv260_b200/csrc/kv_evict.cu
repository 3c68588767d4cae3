// b200_kv_evict: a cache cut to its budget by accumulated attention weight.
//
// A cluster of CTAs takes one cache head of a sequence, each CTA a stretch of
// its slots. (1) Of every slot one 32-bit key, ordered as the slots are given
// up; the keys stay in shared memory where they fit. (2) A radix select over
// the cluster, 11 bits at a time, finds the key of the last slot to give up.
// (3) A bit per slot says whether it is kept. (4) The i-th kept slot past the
// budget moves to the i-th free one below it: the pairs are dealt out evenly
// over the cluster's CTAs, which copy the rows. Sources lie past the budget and
// targets below it, so the order of the copies does not matter.
//
// Weights and positions are read once and written once, and only the rows that
// have to move are touched: for a cache one token over its budget, one row per
// head. The size of the clusters and the shared memory of the keys go by what the
// table can hold, since the host does not know the lengths: 16 sequences of 1025
// slots, 8 heads, take 16 us from an empty L2 with a table of 1040 slots, 18 with
// one of 16384 and 49 with one of 131072.
//
// What bounds it: the chain of barriers. 8 sequences of up to 16000 slots cut to
// 1000 (63 MB to read and write) take 35 us: 5 for the keys, 3 x 2.7 for the
// digits, 6 for counting and listing, 8 for the copies (7 TB/s, from the L2 in
// part), the rest start and skew. A step of 16 sequences of 1025 slots takes 12
// us on the GPU. With one CTA per head the first takes 58 us; with 1024 threads,
// one CTA per SM, 50.
#include <cuda_runtime.h>

#include "common.cuh"
#include "serve_dev.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 4 * kThreads;   // of an 11-bit digit
constexpr int kMoves = 1024;          // pairs that a CTA takes at a time
constexpr int kMaxKeys = 36 * 1024;   // keys of a CTA's stretch kept in shared memory

struct EvictArgs {
    KvView kv;
    const float *weights;
    float *weights_out;
    const int *positions;
    int *positions_out;
    long long aux_stride;
    const int *seen;
    int *lengths_out;
    int budget, recent, sinks;
    int row_chunks;             // 16-byte pieces of a row
    int max_slice;              // slots of a CTA's stretch at most
    bool lengths_in_place;
    unsigned *ticket;
};

// Unsigned order of what is given up first: NaN, then the weights upwards (-0
// as 0), then the tokens kept for their position.
__device__ __forceinline__ uint32_t keep_key(float w, int pos, long long first_recent, int sinks) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    const uint32_t key = w != w ? 0 : u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
    return pos >= first_recent || pos < sinks ? 0xffffffffu : key;
}

__device__ __forceinline__ unsigned lanes_scan(unsigned v) {   // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
        const unsigned y = __shfl_up_sync(kFullMask, v, k);
        if (lane >= k) v += y;
    }
    return v;
}

// Inclusive prefix of one value per thread, and the total.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned *s, unsigned *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = lanes_scan(v);
    __syncthreads();
    if (lane == 31) s[warp] = v;
    __syncthreads();
    const unsigned upto = lanes_scan(s[lane % kWarps]);
    *total = __shfl_sync(kFullMask, upto, kWarps - 1);
    const unsigned before = __shfl_sync(kFullMask, upto, warp > 0 ? warp - 1 : 0);
    return warp > 0 ? v + before : v;
}

__device__ __forceinline__ void cluster_store(uint32_t a, unsigned v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

template <bool kCached>
__global__ void __launch_bounds__(kThreads, 2) kv_evict_kernel(const EvictArgs a) {
    extern __shared__ __align__(16) uint32_t dyn[];
    __shared__ __align__(16) unsigned s_hist[2][kBins];
    __shared__ unsigned s_warp[kWarps], s_gather[3][kMaxCluster];
    __shared__ int s_from[kMoves], s_to[kMoves];
    __shared__ long long s_from_row[kMoves], s_to_row[kMoves];
    __shared__ unsigned s_digit, s_left, s_equal;
    uint32_t *s_kept = dyn;                            // a bit per slot of the stretch
    uint32_t *s_key = dyn + (a.max_slice + 31) / 32;   // kCached
    unsigned ctas;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    const unsigned rank = cluster_ctarank();
    const int h = blockIdx.x / ctas, b = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = kv_length(a.kv, b), cut = min(n, a.budget);
    const long long aux = (static_cast<long long>(b) * a.kv.n_head_kv + h) * a.aux_stride;
    const float *w = a.weights + aux;
    const int *pos = a.positions + aux;
    float *w_out = a.weights_out + aux;
    int *pos_out = a.positions_out + aux;
    const long long first_recent = static_cast<long long>(a.seen[b]) - a.recent;
    // the stretch [i0, i1), of whole words of 32 slots
    const int slice = ((n + static_cast<int>(ctas) - 1) / static_cast<int>(ctas) + 31) / 32 * 32;
    const int i0 = min(static_cast<int>(rank) * slice, n), i1 = min(i0 + slice, n);
    const auto key_at = [&](int i) { return kCached ? s_key[i - i0] : keep_key(w[i], pos[i], first_recent, a.sinks); };
    // What each CTA tells all of them, and the sum of those of lower rank; every use has a row of its own.
    const auto tell = [&](int what, unsigned v) {
        if (tid < static_cast<int>(ctas)) cluster_store(cluster_map(&s_gather[what][rank], tid), v);
    };
    const auto before_me = [&](int what, unsigned *total) {
        const unsigned mine = lane < static_cast<int>(ctas) ? s_gather[what][lane % kMaxCluster] : 0, upto = lanes_scan(mine);
        *total = __shfl_sync(kFullMask, upto, 31);
        return __shfl_sync(kFullMask, upto - mine, rank);
    };

    if (n > a.budget) {
        // (1), (2)
        for (int i = tid; i < kBins; i += kThreads) s_hist[0][i] = 0;
        __syncthreads();
        uint32_t edge = 0;
        unsigned left = n - a.budget, equal = 0;
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, digits = pass == 2 ? 10 : 11;
            const uint32_t mask = pass == 0 ? 0 : kFullMask << (shift + digits);
            unsigned *hist = s_hist[pass & 1], *other = s_hist[~pass & 1];
            if (pass == 0) {
#pragma unroll 8
                for (int i = i0 + tid; i < i1; i += kThreads) {
                    const uint32_t key = keep_key(w[i], pos[i], first_recent, a.sinks);
                    if (kCached) s_key[i - i0] = key;
                    atomicAdd(&hist[key >> 21], 1u);
                }
            } else {
#pragma unroll 4
                for (int i = i0 + tid; i < i1; i += kThreads) {
                    const uint32_t key = key_at(i);
                    if ((key & mask) == edge) atomicAdd(&hist[key >> shift & ((1u << digits) - 1)], 1u);
                }
            }
            cluster_sync_all();
            // every CTA adds up the digits of all, and clears its next set
            uint4 v[kMaxCluster];
#pragma unroll
            for (unsigned q = 0; q < kMaxCluster; ++q) {
                v[q] = make_uint4(0, 0, 0, 0);
                if (q < ctas)
                    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(v[q].x), "=r"(v[q].y), "=r"(v[q].z), "=r"(v[q].w)
                                 : "r"(cluster_map(hist + 4 * tid, q))
                                 : "memory");
            }
            for (int i = tid; i < kBins; i += kThreads) other[i] = 0;
            unsigned c[4] = {0, 0, 0, 0}, total;
#pragma unroll
            for (unsigned q = 0; q < kMaxCluster; ++q) c[0] += v[q].x, c[1] += v[q].y, c[2] += v[q].z, c[3] += v[q].w;
            const unsigned sum = c[0] + c[1] + c[2] + c[3];
            unsigned before = block_scan(sum, s_warp, &total) - sum;
            if (before < left && left <= before + sum) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (before < left && left <= before + c[j]) {
                        s_digit = 4 * tid + j;
                        s_left = left - before;
                        s_equal = c[j];
                    }
                    before += c[j];
                }
            }
            __syncthreads();
            edge |= s_digit << shift;
            left = s_left;
            equal = s_equal;
            __syncthreads();
        }
        const unsigned spare = equal - left;           // slots at the edge that stay, the lowest first
        // (3) each warp takes whole words, side by side
        const int words = (i1 - i0 + 31) / 32, per_warp = (words + kWarps - 1) / kWarps;
        const int k0 = min(warp * per_warp, words), k1 = min(k0 + per_warp, words);
        unsigned ties = 0;
        for (int k = k0; k < k1; ++k) {
            const int i = i0 + k * 32 + lane;
            const uint32_t key = i < i1 ? key_at(i) : 0;
            const unsigned more = __ballot_sync(kFullMask, i < i1 && key > edge);
            if (lane == 0) s_kept[k] = more;
            ties += __popc(__ballot_sync(kFullMask, i < i1 && key == edge));
        }
        unsigned all;
        if (spare > 0) {
            unsigned seen = block_scan(lane == 0 ? ties : 0, s_warp, &all);
            seen = __shfl_sync(kFullMask, seen, 0) - ties;
            tell(0, all);
            cluster_sync_all();
            seen += before_me(0, &all);
            for (int k = k0; k < k1 && ties && seen < spare; ++k) {
                const int i = i0 + k * 32 + lane;
                const bool is = i < i1 && key_at(i) == edge;
                const unsigned eq = __ballot_sync(kFullMask, is);
                const unsigned stay = __ballot_sync(kFullMask, is && seen + __popc(eq & ((1u << lane) - 1)) < spare);
                if (lane == 0) s_kept[k] |= stay;
                seen += __popc(eq);
            }
        }
        __syncthreads();
        // (4) the free slots below the budget and the kept ones past it, numbered over the cluster
        const auto below = [&](int k) {                // the bits of word k below the budget
            const int at = i0 + k * 32;
            return at + 32 <= a.budget ? kFullMask : at >= a.budget ? 0 : (1u << (a.budget - at)) - 1;
        };
        unsigned holes = 0, movers = 0, moves;
        for (int k = k0 + lane; k < k1; k += 32) {
            holes += __popc(~s_kept[k] & below(k));
            movers += __popc(s_kept[k] & ~below(k));
        }
        holes = __reduce_add_sync(kFullMask, holes);
        movers = __reduce_add_sync(kFullMask, movers);
        unsigned hole = block_scan(lane == 0 ? holes : 0, s_warp, &all);
        hole = __shfl_sync(kFullMask, hole, 0) - holes;
        tell(1, all);
        unsigned mover = block_scan(lane == 0 ? movers : 0, s_warp, &all);
        mover = __shfl_sync(kFullMask, mover, 0) - movers;
        tell(2, all);
        cluster_sync_all();
        hole += before_me(1, &moves);
        mover += before_me(2, &moves);
        const unsigned each = min((moves + ctas - 1) / ctas, static_cast<unsigned>(kMoves));   // pairs of a CTA at a time
        for (unsigned first = 0; first < moves; first += each * ctas) {
            const auto list = [&](int *s, unsigned i, int slot) {   // pair `i` is that of CTA (i - first) / each
                const unsigned j = i - first;
                if (i >= first && j < each * ctas) cluster_store(cluster_map(s + j % each, j / each), slot);
            };
            unsigned ho = hole, mo = mover;
            for (int k = k0; k < k1; ++k) {            // a lane to a slot
                const unsigned up = s_kept[k] & ~below(k), down = ~s_kept[k] & below(k), before = (1u << lane) - 1;
                if (down >> lane & 1) list(s_to, ho + __popc(down & before), i0 + k * 32 + lane);
                if (up >> lane & 1) list(s_from, mo + __popc(up & before), i0 + k * 32 + lane);
                ho += __popc(down);
                mo += __popc(up);
            }
            cluster_sync_all();
            const int mine = static_cast<int>(min(max(static_cast<long long>(moves) - first - rank * each, 0ll), static_cast<long long>(each)));
            for (int j = tid; j < mine; j += kThreads) {
                const int from = s_from[j], to = s_to[j];
                s_from_row[j] = kv_row(a.kv, b, h, from);
                s_to_row[j] = kv_row(a.kv, b, h, to);
                w_out[to] = w[from];
                pos_out[to] = pos[from];
            }
            __syncthreads();
            const int pieces = 2 * a.row_chunks, total = mine * pieces;
            for (int u0 = tid; u0 < total; u0 += 4 * kThreads) {
                uint4 v[4];
                char *dst[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int u = u0 + x * kThreads, j = u / pieces, c = u - j * pieces;
                    dst[x] = nullptr;
                    if (u >= total || s_from_row[j] < 0 || s_to_row[j] < 0) continue;
                    char *pool = c < a.row_chunks ? a.kv.k + c * 16 : a.kv.v + (c - a.row_chunks) * 16;
                    dst[x] = pool + s_to_row[j];
                    v[x] = *reinterpret_cast<const uint4 *>(pool + s_from_row[j]);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (dst[x]) *reinterpret_cast<uint4 *>(dst[x]) = v[x];
            }
            if (first + each * ctas < moves) cluster_sync_all();   // the lists may be overwritten
        }
    }
    if (w_out != w || pos_out != pos)
#pragma unroll 4
        for (int i = i0 + tid; i < min(i1, cut); i += kThreads)
            if (n <= a.budget || (s_kept[(i - i0) >> 5] >> ((i - i0) & 31) & 1)) {
                w_out[i] = w[i];
                pos_out[i] = pos[i];
            }
    if (!a.lengths_out) return;
    if (!a.lengths_in_place) {
        if (blockIdx.x == 0 && tid == 0) a.lengths_out[b] = cut;
    } else if (last_cta(a.ticket, gridDim.x * gridDim.y)) {
        for (int i = tid; i < a.kv.batch; i += kThreads) a.lengths_out[i] = min(kv_length(a.kv, i), a.budget);
    }
}

template <bool kCached>
cudaError_t launch(const EvictArgs &a, int ctas, cudaStream_t stream) {
    const int smem = (a.max_slice + 31) / 32 * 4 + (kCached ? a.max_slice * 4 : 0);
    if (!ensure_smem(reinterpret_cast<const void *>(kv_evict_kernel<kCached>), smem)) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.kv.n_head_kv * ctas, a.kv.batch);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv_evict_kernel<kCached>, a);
}

}  // namespace

int kv_evict_validate(const b200_kv_t *kv, const b200_kv_evict_t *a, const char **why) {
    if (int rc = kv_validate(kv, why)) return rc;
    const auto bad = [why](const char *w) { *why = w; return kErrInval; };
    if (!a) return bad("null arguments");
    if (!a->weights || !a->weights_out || !a->positions || !a->positions_out || !a->seen) return bad("null address");
    if (a->weights % 4 || a->weights_out % 4 || a->positions % 4 || a->positions_out % 4 || a->seen % 4 ||
        a->lengths_out % 4)
        return bad("addresses must be 4-byte aligned");
    if (a->aux_stride < static_cast<int64_t>(kv->table_cols) * kv->page_size)
        return bad("aux_stride is below the cache's slots");
    if (a->budget < 1 || a->recent < 0 || a->sinks < 0 || static_cast<int64_t>(a->recent) + a->sinks > a->budget)
        return bad("budget must be positive and hold recent + sinks");
    return 0;
}

cudaError_t kv_evict_launch(const b200_kv_t *kv, const b200_kv_evict_t *p, void *scratch, cudaStream_t stream) {
    EvictArgs a;
    a.kv = kv_view(kv);
    a.weights = reinterpret_cast<const float *>(p->weights);
    a.weights_out = reinterpret_cast<float *>(p->weights_out);
    a.positions = reinterpret_cast<const int *>(p->positions);
    a.positions_out = reinterpret_cast<int *>(p->positions_out);
    a.aux_stride = p->aux_stride;
    a.seen = reinterpret_cast<const int *>(p->seen);
    a.lengths_out = reinterpret_cast<int *>(p->lengths_out);
    a.budget = p->budget;
    a.recent = p->recent;
    a.sinks = p->sinks;
    a.row_chunks = kv->head_dim * esize(kv->dtype) / 16;
    a.lengths_in_place = p->lengths_out == kv->lengths;
    a.ticket = static_cast<unsigned *>(scratch) + 1;
    // CTAs to a head: more where the heads alone leave SMs idle and each still has slots enough to be worth the
    // barriers (8 heads of 16000 slots: 28.7 us against 55 with one CTA each; 16 heads of 4000: 22.5 with two
    // against 38.9 with one and 32.8 with four), and where its keys would not fit
    const int slots = kv->table_cols * kv->page_size, heads = kv->n_head_kv * kv->batch;
    int ctas = 1;
    while (ctas < kMaxCluster && (slots / ctas > kMaxKeys || (heads * ctas <= sm_count() && slots / ctas >= 1536))) ctas *= 2;
    a.max_slice = ((slots + ctas - 1) / ctas + 31) / 32 * 32;
    return a.max_slice <= kMaxKeys ? launch<true>(a, ctas, stream) : launch<false>(a, ctas, stream);
}

}  // namespace b200
