// Launchers of the serving operators (kv_append.cu, kv_attend.cu,
// kv_evict.cu, sample.cu, kv_plan.cu, rope.cu, rms_norm.cu, kv_chunk.cu): the
// device side of b200_kv_*, b200_sample, b200_rope and b200_rms_norm.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/b200_engine.h"

namespace b200 {

constexpr int kMaxHeadDim = 256;
constexpr int kMaxSlots = 1 << 20;     // slots of one sequence
constexpr int kMaxVocab = 1 << 22;     // keeps the sampler's sums below 2^62

inline int esize(int dtype) { return dtype == B200_F32 ? 4 : 2; }

// A b200_kv_t as the kernels take it.
struct KvView {
    char *k = nullptr, *v = nullptr;
    long long page_stride = 0, head_stride = 0, row_stride = 0;  // bytes
    const int *table = nullptr;
    long long table_stride = 0;
    const int *lengths = nullptr;
    int n_pages = 0, page_size = 0, n_head_kv = 0, head_dim = 0, cols = 0, batch = 0;
};

// Each checks a call's arguments: 0, or kErrInval with *why set.
int kv_validate(const b200_kv_t *kv, const char **why);
int kv_append_validate(const b200_kv_t *kv, const b200_kv_append_t *a, const char **why);
int kv_attend_validate(const b200_kv_t *kv, const b200_kv_attend_t *a, const char **why);
int kv_evict_validate(const b200_kv_t *kv, const b200_kv_evict_t *a, const char **why);
int sample_validate(const b200_sample_t *s, const char **why);
int kv_plan_validate(const b200_kv_t *kv, const b200_kv_plan_t *a, const char **why);
int rope_validate(const b200_kv_t *kv, const b200_rope_t *a, const char **why);
int rms_norm_validate(const b200_rms_norm_t *a, const char **why);
int kv_chunk_validate(const b200_kv_t *kv, const b200_kv_chunk_t *a, const char **why);

KvView kv_view(const b200_kv_t *kv);

// `scratch` of each: serve_scratch_bytes() on the device, zeroed once; one
// call at a time uses it (an engine's calls follow one another on a stream).
// kv_plan's, kv_plan_scratch_bytes(), needs no zeros.
size_t serve_scratch_bytes();
size_t kv_plan_scratch_bytes();

// Each launches on `stream` and returns 0 or a CUDA error.
cudaError_t kv_append_launch(const b200_kv_t *kv, const b200_kv_append_t *a, void *scratch, cudaStream_t stream);
cudaError_t kv_attend_launch(const b200_kv_t *kv, const b200_kv_attend_t *a, void *scratch, cudaStream_t stream);
cudaError_t kv_evict_launch(const b200_kv_t *kv, const b200_kv_evict_t *a, void *scratch, cudaStream_t stream);
cudaError_t sample_launch(const b200_sample_t *s, cudaStream_t stream);
cudaError_t kv_plan_launch(const b200_kv_t *kv, const b200_kv_plan_t *a, void *scratch, cudaStream_t stream);
cudaError_t rope_launch(const b200_kv_t *kv, const b200_rope_t *a, cudaStream_t stream);
cudaError_t rms_norm_launch(const b200_rms_norm_t *a, int round_mode, cudaStream_t stream);
cudaError_t kv_chunk_launch(const b200_kv_t *kv, const b200_kv_chunk_t *a, cudaStream_t stream);

// b200_rope_freqs: 0, or kErrInval with *why set.
int rope_freqs(uint64_t *freqs, int rot_dim, double base, const float *factors, int scaling, double factor,
               double context, double low, double high, const char **why);

}  // namespace b200
