// b200_kv_evict: a cache cut to its budget by accumulated attention weight.
#include <cuda_runtime.h>

#include "common.cuh"
#include "serve_dev.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMoves = 2048;   // (from, to) pairs listed at a time

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
    bool lengths_in_place;
    unsigned *ticket;
};

// Unsigned order of what is given up first: NaN, then the weights upwards (-0
// as 0), then the tokens kept for their position.
__device__ __forceinline__ uint32_t keep_key(float w, long long pos, long long first_recent, int sinks) {
    if (pos >= first_recent || pos < sinks) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    if (w != w) return 0;
    return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

// Exclusive prefix of one value per warp, and the total, in every thread.
__device__ __forceinline__ int warp_prefix(int *s, int mine, int *total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) s[warp] = mine;
    __syncthreads();
    int v = s[lane], x = v;
    for (int k = 1; k < 32; k <<= 1) {
        const int y = __shfl_up_sync(kFullMask, x, k);
        if (lane >= k) x += y;
    }
    *total = __shfl_sync(kFullMask, x, 31);
    const int before = __shfl_sync(kFullMask, x - v, warp);
    __syncthreads();
    return before;
}

__device__ __forceinline__ int lane_prefix(int v, int lane) {   // exclusive
    int x = v;
    for (int k = 1; k < 32; k <<= 1) {
        const int y = __shfl_up_sync(kFullMask, x, k);
        if (lane >= k) x += y;
    }
    return x - v;
}

// One CTA per cache head of a sequence: (1) a radix select of the e-th
// smallest key, e the slots to give up, by 8-bit digits from the top; (2) one
// bit per slot, kept or not, ties going to the lower slots; (3) the i-th kept
// slot past the budget moves to the i-th free one below it.
__global__ void __launch_bounds__(kThreads) kv_evict_kernel(const EvictArgs a) {
    extern __shared__ uint32_t s_kept[];         // a bit per slot
    __shared__ uint32_t s_hist[256];
    __shared__ int s_warp[32];
    __shared__ int s_from[kMoves], s_to[kMoves];
    __shared__ uint32_t s_prefix;
    __shared__ int s_left, s_equal;
    const int h = blockIdx.x, b = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = kv_length(a.kv, b), cut = min(n, a.budget);
    const long long aux = (static_cast<long long>(b) * a.kv.n_head_kv + h) * a.aux_stride;
    const float *w = a.weights + aux;
    const int *pos = a.positions + aux;
    float *w_out = a.weights_out + aux;
    int *pos_out = a.positions_out + aux;
    const long long first_recent = static_cast<long long>(a.seen[b]) - a.recent;

    if (n > a.budget) {
        // (1)
        if (tid == 0) s_prefix = 0, s_left = n - a.budget;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) s_hist[tid] = 0;
            __syncthreads();
            const uint32_t prefix = s_prefix, mask = shift == 24 ? 0 : 0xffffffffu << (shift + 8);
            for (int i = tid; i < n; i += kThreads) {
                const uint32_t key = keep_key(w[i], pos[i], first_recent, a.sinks);
                if ((key & mask) == prefix) atomicAdd(&s_hist[(key >> shift) & 255], 1u);
            }
            __syncthreads();
            if (warp == 0) {
                int c[8], mine = 0;
                for (int j = 0; j < 8; ++j) mine += c[j] = static_cast<int>(s_hist[lane * 8 + j]);
                const int left = s_left;
                int before = lane_prefix(mine, lane);
                const unsigned there = __ballot_sync(kFullMask, before < left && left <= before + mine);
                if (lane == __ffs(there) - 1) {
                    int j = 0;
                    while (before + c[j] < left) before += c[j++];
                    s_prefix = prefix | static_cast<uint32_t>(lane * 8 + j) << shift;
                    s_left = left - before;
                    s_equal = c[j];
                }
            }
            __syncthreads();
        }
        const uint32_t edge = s_prefix;
        const int spare = s_equal - s_left;       // slots at the edge that stay, the lowest first
        // (2) each warp takes whole words of 32 slots
        const int words = (n + 31) / 32, per_warp = (words + kWarps - 1) / kWarps;
        const int w0 = min(warp * per_warp, words), w1 = min(w0 + per_warp, words);
        int equal = 0;
        for (int k = w0; k < w1; ++k) {
            const int i = k * 32 + lane;
            const uint32_t key = i < n ? keep_key(w[i], pos[i], first_recent, a.sinks) : 0;
            const unsigned eq = __ballot_sync(kFullMask, i < n && key == edge);
            const unsigned gt = __ballot_sync(kFullMask, i < n && key > edge);
            if (lane == 0) s_kept[k] = gt;
            equal += __popc(eq);
        }
        int total;
        int rank = warp_prefix(s_warp, equal, &total);
        for (int k = w0; k < w1 && equal && rank < spare; ++k) {
            const int i = k * 32 + lane;
            const bool is = i < n && keep_key(w[i], pos[i], first_recent, a.sinks) == edge;
            const unsigned eq = __ballot_sync(kFullMask, is);
            const bool stays = is && rank + __popc(eq & ((1u << lane) - 1)) < spare;
            const unsigned more = __ballot_sync(kFullMask, stays);
            if (lane == 0) s_kept[k] |= more;
            rank += __popc(eq);
        }
        __syncthreads();
        // (3) ranks of the free slots below the budget and of the kept ones past it
        int holes = 0, movers = 0;
        for (int k = w0 + lane; k < w1; k += 32) {
            const uint32_t low = k * 32 + 32 <= a.budget ? kFullMask : k * 32 >= a.budget ? 0 : (1u << (a.budget - k * 32)) - 1;
            holes += __popc(~s_kept[k] & low);
            movers += __popc(s_kept[k] & ~low);
        }
        for (int x = 16; x; x >>= 1) {
            holes += __shfl_xor_sync(kFullMask, holes, x);
            movers += __shfl_xor_sync(kFullMask, movers, x);
        }
        int moves;
        const int hole0 = warp_prefix(s_warp, holes, &moves);
        const int mover0 = warp_prefix(s_warp, movers, &moves);
        for (int first = 0; first < moves; first += kMoves) {
            int hr = hole0, mr = mover0;
            for (int base = w0; base < w1; base += 32) {
                const int k = base + lane;
                uint32_t hole = 0, mover = 0;
                if (k < w1) {
                    const uint32_t low = k * 32 + 32 <= a.budget ? kFullMask : k * 32 >= a.budget ? 0 : (1u << (a.budget - k * 32)) - 1;
                    hole = ~s_kept[k] & low;
                    mover = s_kept[k] & ~low;
                }
                int hn = __popc(hole), mn = __popc(mover);
                int ho = hr + lane_prefix(hn, lane), mo = mr + lane_prefix(mn, lane);
                for (; hole; hole &= hole - 1, ++ho)
                    if (ho >= first && ho < first + kMoves) s_to[ho - first] = k * 32 + __ffs(hole) - 1;
                for (; mover; mover &= mover - 1, ++mo)
                    if (mo >= first && mo < first + kMoves) s_from[mo - first] = k * 32 + __ffs(mover) - 1;
                for (int x = 16; x; x >>= 1) {
                    hn += __shfl_xor_sync(kFullMask, hn, x);
                    mn += __shfl_xor_sync(kFullMask, mn, x);
                }
                hr += hn;
                mr += mn;
            }
            __syncthreads();
            const int count = min(moves - first, kMoves);
            for (int j = tid; j < count; j += kThreads) {
                w_out[s_to[j]] = w[s_from[j]];
                pos_out[s_to[j]] = pos[s_from[j]];
            }
            const int pieces = 2 * a.row_chunks;
            for (int u = tid; u < count * pieces; u += kThreads) {
                const int j = u / pieces, c = u - j * pieces;
                const long long from = kv_row(a.kv, b, h, s_from[j]), to = kv_row(a.kv, b, h, s_to[j]);
                if (from < 0 || to < 0) continue;
                char *pool = c < a.row_chunks ? a.kv.k : a.kv.v;
                const int off = (c < a.row_chunks ? c : c - a.row_chunks) * 16;
                *reinterpret_cast<uint4 *>(pool + to + off) = *reinterpret_cast<const uint4 *>(pool + from + off);
            }
            __syncthreads();
        }
    }
    if (w_out != w || pos_out != pos)
        for (int i = tid; i < cut; i += kThreads)
            if (n <= a.budget || (s_kept[i >> 5] >> (i & 31) & 1)) {
                w_out[i] = w[i];
                pos_out[i] = pos[i];
            }
    if (!a.lengths_out) return;
    if (!a.lengths_in_place) {
        if (h == 0 && tid == 0) a.lengths_out[b] = cut;
    } else if (last_cta(a.ticket, gridDim.x * gridDim.y)) {
        for (int i = tid; i < a.kv.batch; i += kThreads) a.lengths_out[i] = min(kv_length(a.kv, i), a.budget);
    }
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
    const int smem = (kv->table_cols * kv->page_size + 31) / 32 * 4;
    if (!ensure_smem(reinterpret_cast<const void *>(kv_evict_kernel), smem)) return cudaErrorInvalidValue;
    kv_evict_kernel<<<dim3(kv->n_head_kv, kv->batch), kThreads, smem, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace b200
