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
__device__ __forceinline__ void scan2(unsigned long long &x, long long &y, unsigned long long *total_x, long long *total_y) {
    __shared__ unsigned long long sx[kThreads / 32];
    __shared__ long long sy[kThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
        const unsigned long long u = __shfl_up_sync(kFullMask, x, i);
        const long long v = __shfl_up_sync(kFullMask, y, i);
        if (lane >= i) x += u, y += v;
    }
    __syncthreads();                   // the last scan's sums have been read
    if (lane == 31) sx[warp] = x, sy[warp] = y;
    __syncthreads();
    unsigned long long bx = sx[lane];
    long long by = sy[lane];
    const unsigned long long ox = bx;
    const long long oy = by;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
        const unsigned long long u = __shfl_up_sync(kFullMask, bx, i);
        const long long v = __shfl_up_sync(kFullMask, by, i);
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

// What the slots' search needs of a sequence, in shared memory as far as it goes.
struct Ends {
    int end[kThreads];
};

// Token t's slot, from what is known of its sequence: `ends` the offsets' tail,
// `length` its old length or -1 where it got nothing.
__device__ __forceinline__ void slot_of(const PlanArgs &a, int t, const int *ends) {
    const int batch = a.kv.batch;
    int b = -1, position = -1;
    long long slot = -1;
    if (t < ends[batch - 1]) {
        b = first_above(ends, batch, t);
        const int i = t - (b ? ends[b - 1] : 0), length = a.state[b];
        position = a.state[batch + b] + i;
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
// taken, and a page's place follows from running sums over the sequences, so any
// thread can move any page (a search in the sums of up to 1024 sequences finds
// its owner) and the result does not depend on timing. Nothing here is long
// enough to be bound by anything but the chain of dependent reads: the wishes,
// the pages that move, the slots' pages (256 sequences: 9.5 us from a cold cache,
// 13 with the wishes read and summed twice and the slots' search in global
// memory; the call takes 15). Up to 1024 sequences' wishes are read and summed
// once, more of them twice. Beyond 8192 tokens, eight to a thread, a second
// kernel finds the slots (61 prompts of up to 4000 tokens: 4.5 us beside 10.5).
__global__ void __launch_bounds__(kThreads) kv_plan_kernel(const PlanArgs a) {
    __shared__ int s_sum[kThreads], s_from[kThreads];
    __shared__ bool s_given[kThreads];
    __shared__ Ends s_ends;
    __shared__ int s_most[kThreads / 32];
    const int tid = threadIdx.x, batch = a.kv.batch;
    const bool once = batch <= kThreads;
    int *table = const_cast<int *>(a.kv.table);
    const long long had = min(max(*a.free_count, 0), a.free_capacity);
    Wish w{};
    int seen = 0, back = 0, need = 0, back_all = 0, need_all = 0;      // of up to 1024 sequences: below 2^30
    unsigned long long upto = 0, total = 0;            // pages that come back, and needs above them
    long long tokens = 0, total_tokens = 0;
    const auto load = [&](int base) {
        const int b = base + tid;
        w = Wish{};
        seen = 0;
        if (b < batch) {
            w = wish_of(a, b);
            seen = a.seen ? a.seen[b] : w.length;
        }
        back = max(w.held - w.want, 0);
        need = max(w.want - w.held, 0);
        upto = static_cast<unsigned>(back) | static_cast<unsigned long long>(need) << 32;
        tokens = w.add;
        scan2(upto, tokens, &total, &total_tokens);
        back_all = static_cast<int>(total & 0xffffffffu);
        need_all = static_cast<int>(total >> 32);
    };
    long long returned = 0;
    for (int base = 0; base < batch; base += kThreads) {
        load(base);
        if (back_all) {
            s_sum[tid] = static_cast<int>(upto & 0xffffffffu);
            s_from[tid] = w.want - (static_cast<int>(upto & 0xffffffffu) - back);
            __syncthreads();
            for (int p = tid; p < back_all; p += kThreads) {
                const int j = first_above(s_sum, min(kThreads, batch - base), p);
                const long long dst = had + returned + p;
                if (dst < a.free_capacity) a.free_pages[dst] = table[(base + j) * a.kv.table_stride + s_from[j] + p];
            }
            returned += back_all;
            __syncthreads();
        }
    }
    const long long count = min(had + returned, static_cast<long long>(a.free_capacity));
    long long needed = 0, asked = 0, taken = 0;
    for (int base = 0; base < batch; base += kThreads) {
        const int b = base + tid;
        if (!once) load(base);
        const int need_upto = static_cast<int>(upto >> 32);
        const bool given = w.fits && (need == 0 || needed + need_upto <= count);
        const int got = given ? static_cast<int>(w.add) : 0;
        const int end = static_cast<int>(min(asked + tokens, static_cast<long long>(a.n_tokens)));
        s_sum[tid] = need_upto;
        s_from[tid] = w.held - (need_upto - need);
        s_given[tid] = given;
        s_ends.end[tid] = end;
        if (b < batch) {
            if (b == 0) a.offsets[0] = 0;
            a.offsets[b + 1] = end;
            a.held_out[b] = given ? w.want : w.held;
            if (a.granted) a.granted[b] = got;
            if (a.seen_out) a.seen_out[b] = w.done ? 0 : seen + got;
            a.lengths_out[b] = w.done ? 0 : w.length + got;
            a.state[b] = given ? w.length : -1;
            a.state[batch + b] = seen;
        }
        // those that got pages come before those that did not
        const int most = __reduce_max_sync(kFullMask, given && need ? need_upto : 0);
        if ((tid & 31) == 0) s_most[tid >> 5] = most;
        __syncthreads();
        const int most_of_all = __reduce_max_sync(kFullMask, s_most[tid & 31]);
        if (most_of_all) taken = needed + most_of_all;
        for (int p = tid; p < most_of_all; p += kThreads) {
            const int j = first_above(s_sum, min(kThreads, batch - base), p);
            if (s_given[j]) table[(base + j) * a.kv.table_stride + s_from[j] + p] = a.free_pages[count - 1 - needed - p];
        }
        needed += need_all;
        asked += total_tokens;
        __syncthreads();
    }
    if (tid == 0) *a.free_count_out = static_cast<int>(count - taken);
    if (a.n_slots > kAtOnce) return;
    for (int t = tid; t < a.n_slots; t += kThreads) slot_of(a, t, once ? s_ends.end : a.offsets + 1);
}

__global__ void __launch_bounds__(kSlotThreads) kv_slots_kernel(const PlanArgs a) {
    __shared__ Ends s_ends;
    pdl_wait_prior_grid();
    const bool once = a.kv.batch <= kThreads;
    if (once) {
        for (int b = threadIdx.x; b < a.kv.batch; b += kSlotThreads) s_ends.end[b] = a.offsets[b + 1];
        __syncthreads();
    }
    const int t = blockIdx.x * kSlotThreads + threadIdx.x;
    if (t < a.n_slots) slot_of(a, t, once ? s_ends.end : a.offsets + 1);
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
