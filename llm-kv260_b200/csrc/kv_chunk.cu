// b200_kv_attend_chunk: checks, workspace and choice of the kernel.
#include <cuda_runtime.h>

#include "kv_chunk.cuh"

namespace b200 {

namespace {

chunk::Shape shape_of(const b200_kv_t *kv, int dtype) {
    if (dtype != B200_F32) return chunk::mma_shape(kv->head_dim);
    return kv->dtype == B200_F32 ? chunk::f32_shape(kv->head_dim) : chunk::split_shape(kv->head_dim);
}

uint64_t workspace_bytes(const b200_kv_t *kv, int dtype) {
    const chunk::Shape s = shape_of(kv, dtype);
    return static_cast<uint64_t>(most_sms()) * s.ctas * (2 * s.part + sizeof(chunk::Joint)) + 16;
}

// What the kernels can do of types and heads, apart from the call's other arguments.
const char *unusable(const b200_kv_t *kv, int dtype, int n_head) {
    if (dtype != kv->dtype && !(dtype == B200_F32 && kv->dtype == B200_F16))
        return "q must be of the cache's type, or float32 with a float16 cache";
    if (n_head < 1 || n_head % kv->n_head_kv) return "n_head must be a multiple of n_head_kv";
    if (n_head / kv->n_head_kv > 4096) return "at most 4096 query heads read one cache head";
    return nullptr;
}

}  // namespace

int kv_chunk_validate(const b200_kv_t *kv, const b200_kv_chunk_t *a, const char **why) {
    if (int rc = kv_validate(kv, why)) return rc;
    const auto bad = [why](const char *w) { *why = w; return kErrInval; };
    if (!a) return bad("null arguments");
    if (const char *w = unusable(kv, a->dtype, a->n_head)) return bad(w);
    if (a->n_tokens < 0 || static_cast<int64_t>(a->n_tokens) * a->n_head > 1ll << 30)
        return bad("n_tokens must be in [0, 2^30 / n_head]");
    if (a->window < 0) return bad("window must not be negative");
    if (!(a->scale * chunk::kLog2e >= 1e-37f) || !(a->scale * chunk::kLog2e <= 1e37f))
        return bad("scale must be positive, in [1e-37, 1e37]");
    if (!a->offsets || (a->n_tokens > 0 && (!a->q || !a->out))) return bad("null address");
    const int es = esize(a->dtype);
    if (a->q_token_stride < 0 || a->q_head_stride < 0 || a->out_token_stride < 0 || a->out_head_stride < 0)
        return bad("strides must not be negative");
    if (a->q % 16 || a->out % 16 || a->q_token_stride * es % 16 || a->q_head_stride * es % 16 ||
        a->out_token_stride * es % 16 || a->out_head_stride * es % 16)
        return bad("addresses and strides of q and out must be multiples of 16 bytes");
    if (a->offsets % 4 || a->lse % 4) return bad("offsets and lse must be 4-byte aligned");
    if (!a->workspace || a->workspace % 16 || a->workspace_bytes < workspace_bytes(kv, a->dtype))
        return bad("needs a workspace of b200_kv_chunk_workspace() bytes, 16-byte aligned");
    return 0;
}

cudaError_t kv_chunk_launch(const b200_kv_t *kv, const b200_kv_chunk_t *p, cudaStream_t stream) {
    if (p->n_tokens == 0) return cudaSuccess;
    chunk::Args a;
    const int es = esize(p->dtype);
    a.kv = kv_view(kv);
    a.page_magic = (1ull << 40) / static_cast<unsigned>(kv->page_size) + 1;
    a.q = reinterpret_cast<const char *>(p->q);
    a.out = reinterpret_cast<char *>(p->out);
    a.lse = reinterpret_cast<float *>(p->lse);
    a.offsets = reinterpret_cast<const int *>(p->offsets);
    a.q_token = p->q_token_stride * es;
    a.q_head = p->q_head_stride * es;
    a.out_token = p->out_token_stride * es;
    a.out_head = p->out_head_stride * es;
    a.n_tokens = p->n_tokens;
    a.n_head = p->n_head;
    a.group = p->n_head / kv->n_head_kv;
    a.group_magic = static_cast<unsigned>((1ull << 32) / static_cast<unsigned>(a.group)) + 1;
    a.window = p->window < kMaxSlots ? p->window : 0;      // one that leaves nothing out
    a.scale = p->scale * chunk::kLog2e;
    const chunk::Shape s = shape_of(kv, p->dtype);
    a.parts = reinterpret_cast<float *>(p->workspace);
    a.joints = reinterpret_cast<chunk::Joint *>(p->workspace + static_cast<uint64_t>(sm_count()) * s.ctas * 2 * s.part);
    a.status = status_word();
    if (p->dtype != B200_F32) return chunk::mma_launch(a, kv->dtype, stream);
    return kv->dtype == B200_F32 ? chunk::f32_launch(a, stream) : chunk::split_launch(a, stream);
}

}  // namespace b200

extern "C" uint64_t b200_kv_chunk_workspace(const b200_kv_t *kv, int dtype, int n_head) {
    const char *why = nullptr;
    if (b200::kv_validate(kv, &why) || b200::unusable(kv, dtype, n_head)) return 0;
    return b200::workspace_bytes(kv, dtype);
}
