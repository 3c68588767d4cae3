// Device helpers of the serving operators.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx.cuh"
#include "serve.h"

namespace b200 {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Slots of sequence b in use, whatever the caller left in lengths[b].
__device__ __forceinline__ int kv_length(const KvView &kv, int b) {
    return min(max(kv.lengths[b], 0), kv.cols * kv.page_size);
}

// Byte offset of head h's row for slot `slot` of sequence b, or -1 where the
// table names no page of the pool.
__device__ __forceinline__ long long kv_row(const KvView &kv, int b, int h, int slot) {
    const int col = slot / kv.page_size;
    const int page = kv.table[b * kv.table_stride + col];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(kv.n_pages)) return -1;
    return page * kv.page_stride + h * kv.head_stride + (slot - col * kv.page_size) * kv.row_stride;
}

// True in every thread of the CTA that is the last of `ctas` to come here. All
// the CTA's earlier reads and writes are done before any CTA sees true; the
// counter is left at 0 for the next call.
__device__ __forceinline__ bool last_cta(unsigned *counter, unsigned ctas) {
    __shared__ bool last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(counter, 1u) == ctas - 1;
        if (last) *counter = 0;
        __threadfence();
    }
    __syncthreads();
    return last;
}

}  // namespace b200
