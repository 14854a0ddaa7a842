// Tensors read and written through buffer resources: an access past a window's end reads 0, or is not made.
#pragma once

#include "ramnet_device.hpp"

namespace ramnet {

// A window of rows in memory: loads past it give 0, stores past it are dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t window(const void *base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, static_cast<int>(bytes), kBufWord3);
}

constexpr int kNowhere = 1 << 30;  // past every window, with any row's offset on top

template<typename T>
__device__ __forceinline__ uint32_t buffer_bits(__amdgpu_buffer_rsrc_t from, int at) {
    if constexpr (sizeof(T) == 4)
        return __builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0);
    else
        return __builtin_amdgcn_raw_buffer_load_b16(from, at, 0, 0);
}

template<typename T>
__device__ __forceinline__ void buffer_store(float v, __amdgpu_buffer_rsrc_t to, int at) {
    if constexpr (sizeof(T) == 4)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), to, at, 0, 0);
    else if constexpr (__is_same(T, bf16_t))
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, static_cast<__bf16>(v)), to, at, 0, 0);
    else
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, static_cast<_Float16>(v)), to, at, 0, 0);
}

}  // namespace ramnet
