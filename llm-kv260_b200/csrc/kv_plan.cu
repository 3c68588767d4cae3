// b200_kv_plan: pages and slots for new tokens.
#include <cuda_runtime.h>

#include "common.cuh"
#include "q4gemv.h"
#include "serve_dev.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 1024;
constexpr int kAtOnce = 8192;          // tokens whose slots the first kernel finds itself
constexpr int kSlotThreads = 256;

struct PlanArgs {
    KvView kv;
    const int *new_tokens, *held, *free_count, *seen;
    int *held_out, *free_pages, *free_count_out, *offsets, *granted, *seen_out, *lengths_out;
    int free_capacity, n_tokens, n_slots;  // n_slots: tokens whose slots are wanted
    long long *slots;
    int *positions, *sequences;
    int *state;                        // scratch [2][batch]: a sequence's old length (-1: it got nothing), and seen
};

// A sequence's wishes.
struct Wish {
    int length, held, want;
    long long add;
    bool done, fits;
};

__device__ __forceinline__ Wish wish_of(const PlanArgs &a, int b) {
    Wish w;
    w.length = kv_length(a.kv, b);
    w.held = min(max(a.held[b], 0), a.kv.cols);
    const int n = a.new_tokens[b];
    w.done = n < 0;
    w.add = max(n, 0);
    const long long total = w.done ? 0 : w.length + w.add;
    w.fits = total <= static_cast<long long>(a.kv.cols) * a.kv.page_size;
    w.want = w.fits ? static_cast<int>((total + a.kv.page_size - 1) / a.kv.page_size) : w.held;
    return w;
}

// Inclusive sums of two numbers over the CTA; *total is theirs.
__device__ __forceinline__ void scan2(long long &x, long long &y, long long *total_x, long long *total_y) {
    __shared__ long long s[2][kThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
        const long long u = __shfl_up_sync(kFullMask, x, i), v = __shfl_up_sync(kFullMask, y, i);
        if (lane >= i) x += u, y += v;
    }
    __syncthreads();                   // the last scan's sums have been read
    if (lane == 31) s[0][warp] = x, s[1][warp] = y;
    __syncthreads();
    long long bx = lane < kThreads / 32 ? s[0][lane] : 0, by = lane < kThreads / 32 ? s[1][lane] : 0;
    const long long ox = bx, oy = by;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
        const long long u = __shfl_up_sync(kFullMask, bx, i), v = __shfl_up_sync(kFullMask, by, i);
        if (lane >= i) bx += u, by += v;
    }
    *total_x = __shfl_sync(kFullMask, bx, 31);
    *total_y = __shfl_sync(kFullMask, by, 31);
    x += __shfl_sync(kFullMask, bx - ox, warp);
    y += __shfl_sync(kFullMask, by - oy, warp);
}

// First j of `n` inclusive sums with sums[j] > i.
template <typename T>
__device__ __forceinline__ int first_above(const T *sums, int n, long long i) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > i) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// Token t's slot, from what the first kernel has left.
__device__ __forceinline__ void slot_of(const PlanArgs &a, int t, int batch, const int *offsets) {
    const bool any = t < offsets[batch];
    int b = -1, position = -1;
    long long slot = -1;
    if (any) {
        b = first_above(offsets + 1, batch, t);
        const int i = t - offsets[b], length = a.state[b];
        position = a.state[a.kv.batch + b] + i;
        if (length >= 0) {
            const int at = length + i, col = at / a.kv.page_size;
            const int page = a.kv.table[b * a.kv.table_stride + col];
            if (static_cast<unsigned>(page) < static_cast<unsigned>(a.kv.n_pages))
                slot = static_cast<long long>(page) * a.kv.page_size + (at - col * a.kv.page_size);
        }
    }
    if (a.slots) a.slots[t] = slot;
    if (a.positions) a.positions[t] = position;
    if (a.sequences) a.sequences[t] = b;
}

// One CTA moves the pages: what comes back is on the stack before anything is
// taken, and a page's place follows from two running sums over the sequences,
// so any thread can move any page (a search in the sums of up to 1024
// sequences finds its owner) and the result does not depend on timing. Nothing
// here is long enough to be bound by anything but the chain of dependent reads.
__global__ void __launch_bounds__(kThreads) kv_plan_kernel(const PlanArgs a) {
    __shared__ long long s_sum[kThreads];
    __shared__ int s_from[kThreads], s_given[kThreads];
    const int tid = threadIdx.x, batch = a.kv.batch;
    int *table = const_cast<int *>(a.kv.table);
    const long long had = min(max(*a.free_count, 0), a.free_capacity);
    long long back_all = 0;
    for (int base = 0; base < batch; base += kThreads) {
        const int b = base + tid, n = min(kThreads, batch - base);
        long long back = 0, unused = 0, total, total2;
        if (b < batch) {
            const Wish w = wish_of(a, b);
            back = max(w.held - w.want, 0);
            s_from[tid] = w.want;
        }
        const long long mine = back;
        scan2(back, unused, &total, &total2);
        s_sum[tid] = back;
        s_given[tid] = static_cast<int>(mine);
        __syncthreads();
        for (long long p = tid; p < total; p += kThreads) {
            const int j = first_above(s_sum, n, p);
            const int col = s_from[j] + static_cast<int>(p - (s_sum[j] - s_given[j]));
            const long long dst = had + back_all + p;
            if (dst < a.free_capacity) a.free_pages[dst] = table[(base + j) * a.kv.table_stride + col];
        }
        back_all += total;
        __syncthreads();
    }
    const long long count = min(had + back_all, static_cast<long long>(a.free_capacity));
    long long need_all = 0, tokens_all = 0, taken = 0;
    for (int base = 0; base < batch; base += kThreads) {
        const int b = base + tid, n = min(kThreads, batch - base);
        long long need = 0, upto, tokens, total, total_tokens;
        Wish w{};
        int seen = 0;
        if (b < batch) {
            w = wish_of(a, b);
            need = max(w.want - w.held, 0);
            seen = a.seen ? a.seen[b] : w.length;
        }
        upto = need;
        tokens = w.add;
        scan2(upto, tokens, &total, &total_tokens);
        const bool given = w.fits && (need == 0 || need_all + upto <= count);
        s_sum[tid] = upto;
        s_from[tid] = w.held - static_cast<int>(min(upto - need, 0x7fe00000ll));
        s_given[tid] = given;
        if (b < batch) {
            const int got = given ? static_cast<int>(w.add) : 0;
            if (b == 0) a.offsets[0] = 0;
            a.offsets[b + 1] = static_cast<int>(min(tokens_all + tokens, static_cast<long long>(a.n_tokens)));
            a.held_out[b] = given ? w.want : w.held;
            if (a.granted) a.granted[b] = got;
            if (a.seen_out) a.seen_out[b] = w.done ? 0 : seen + got;
            a.lengths_out[b] = w.done ? 0 : w.length + got;
            a.state[b] = given ? w.length : -1;
            a.state[batch + b] = seen;
        }
        __syncthreads();
        const long long reach = min(total, count - need_all);
        for (long long p = tid; p < reach; p += kThreads) {
            const int j = first_above(s_sum, n, p);
            if (s_given[j])
                table[(base + j) * a.kv.table_stride + s_from[j] + static_cast<int>(p)] = a.free_pages[count - 1 - need_all - p];
        }
        // those that got pages come before those that did not
        const long long mine = given && need > 0 ? upto : 0;
        long long most = mine;
#pragma unroll
        for (int i = 16; i; i >>= 1) most = max(most, __shfl_xor_sync(kFullMask, most, i));
        __syncthreads();
        if ((tid & 31) == 0) s_sum[tid >> 5] = most;
        __syncthreads();
        for (int i = 0; i < kThreads / 32; ++i) taken = max(taken, s_sum[i] > 0 ? need_all + s_sum[i] : 0ll);
        need_all += total;
        tokens_all += total_tokens;
        __syncthreads();
    }
    if (tid == 0) *a.free_count_out = static_cast<int>(count - taken);
    if (a.n_slots > kAtOnce) return;
    for (int t = tid; t < a.n_slots; t += kThreads) slot_of(a, t, batch, a.offsets);
}

__global__ void __launch_bounds__(kSlotThreads) kv_slots_kernel(const PlanArgs a) {
    pdl_wait_prior_grid();
    const int t = blockIdx.x * kSlotThreads + threadIdx.x;
    if (t < a.n_slots) slot_of(a, t, a.kv.batch, a.offsets);
}

}  // namespace

size_t kv_plan_scratch_bytes() { return 2 * 65536 * sizeof(int); }

int kv_plan_validate(const b200_kv_t *kv, const b200_kv_plan_t *a, const char **why) {
    if (int rc = kv_validate(kv, why)) return rc;
    const auto bad = [why](const char *w) { *why = w; return kErrInval; };
    if (!a) return bad("null arguments");
    if (a->n_tokens < 0 || a->free_capacity < 0) return bad("n_tokens and free_capacity must not be negative");
    if (static_cast<int64_t>(kv->n_pages) * kv->page_size > INT64_MAX / 2) return bad("too many slots");
    if (!a->new_tokens || !a->held || !a->held_out || !a->free_count || !a->free_count_out || !a->offsets ||
        !a->lengths_out || (a->free_capacity > 0 && !a->free_pages))
        return bad("null address");
    if (a->seen_out && !a->seen) return bad("seen_out without seen");
    if (a->slots % 8) return bad("slots must be 8-byte aligned");
    if (a->new_tokens % 4 || a->held % 4 || a->held_out % 4 || a->free_pages % 4 || a->free_count % 4 ||
        a->free_count_out % 4 || a->offsets % 4 || a->positions % 4 || a->sequences % 4 || a->granted % 4 || a->seen % 4 ||
        a->seen_out % 4 || a->lengths_out % 4)
        return bad("addresses must be 4-byte aligned");
    return 0;
}

cudaError_t kv_plan_launch(const b200_kv_t *kv, const b200_kv_plan_t *p, void *scratch, cudaStream_t stream) {
    const auto ints = [](uint64_t at) { return reinterpret_cast<int *>(at); };
    PlanArgs a;
    a.kv = kv_view(kv);
    a.new_tokens = ints(p->new_tokens);
    a.held = ints(p->held);
    a.free_count = ints(p->free_count);
    a.seen = ints(p->seen);
    a.held_out = ints(p->held_out);
    a.free_pages = ints(p->free_pages);
    a.free_count_out = ints(p->free_count_out);
    a.offsets = ints(p->offsets);
    a.granted = ints(p->granted);
    a.seen_out = ints(p->seen_out);
    a.lengths_out = ints(p->lengths_out);
    a.free_capacity = p->free_capacity;
    a.n_tokens = p->n_tokens;
    a.n_slots = p->slots || p->positions || p->sequences ? p->n_tokens : 0;
    a.slots = reinterpret_cast<long long *>(p->slots);
    a.positions = ints(p->positions);
    a.sequences = ints(p->sequences);
    a.state = static_cast<int *>(scratch);
    kv_plan_kernel<<<1, kThreads, 0, stream>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || a.n_slots <= kAtOnce) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((a.n_slots - 1) / kSlotThreads + 1);
    cfg.blockDim = dim3(kSlotThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv_slots_kernel, a);
}

}  // namespace b200
