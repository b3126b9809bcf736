// Attention with a decaying state: what its kernels share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace fb {

using LinArgs = functs_b200_linear_attention_args;

constexpr int kLinMaxDim = 128;

// kernels_linattn_tc.cu
int64_t linattn_chunk_scratch_bytes(const LinArgs& a);
int launch_linattn_chunk(const LinArgs& a, void* scratch, cudaStream_t st);

#ifdef __CUDACC__

__device__ __forceinline__ float lin_float(float x) { return x; }
__device__ __forceinline__ float lin_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float lin_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T lin_from(float x);
template <>
__device__ __forceinline__ float lin_from<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half lin_from<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 lin_from<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// A head's log decay.  One of -inf forgets at once, but not what it just saw: -1e30 * 0 is 0 where -inf * 0 is not.  A NaN stays one.
__device__ __forceinline__ float lin_log_decay(const LinArgs& a, int h) { return max_nan(a.log_decay[h], -1e30f); }

__device__ __forceinline__ int lin_length(const LinArgs& a, int b) {
    return a.lengths == nullptr ? a.tokens : min(max(a.lengths[b], 0), a.tokens);
}

// Zeros in rows [first, last) of a head's output, `cols` of them adjacent; the whole block, a warp's lanes along a row (or along several,
// 16 bytes each, where they lie on such boundaries).
template <typename T>
__device__ __forceinline__ void lin_clear(T* out, int64_t stride, int first, int last, int cols) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    constexpr int N = 16 / sizeof(T);
    if (cols % N == 0 && stride % N == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0) {
        const int pieces = cols / N, rows = 32 / pieces, row = lane / pieces;  // (up to 32 pieces: 128 channels of 4 bytes)
        if (row >= rows) return;
        for (int t = first + warp * rows + row; t < last; t += warps * rows)
            *reinterpret_cast<uint4*>(out + t * stride + (lane - row * pieces) * N) = make_uint4(0, 0, 0, 0);
    } else {
        for (int t = first + warp; t < last; t += warps)
            for (int c = lane; c < cols; c += 32) out[t * stride + c] = lin_from<T>(0.0f);
    }
}

// The state that sequence b uses, or -1 for none; `bits` gets the status bit that says why.  Called by a whole warp.
__device__ __forceinline__ int lin_slot(const LinArgs& a, int b, int lane, int& bits) {
    bits = 0;
    if (a.slots == nullptr) return b;
    const int slot = a.slots[b];
    if (slot < 0) return -1;
    if (slot >= a.num_slots) {
        bits = FB_STATUS_INDEX_RANGE;
        return -1;
    }
    bool twice = false;
    for (int i = lane; i < b; i += 32) twice |= a.slots[i] == slot;
    if (__any_sync(kFullMask, twice)) {
        bits = FB_STATUS_INDEX_TWICE;
        return -1;
    }
    return slot;
}

#endif

}  // namespace fb
