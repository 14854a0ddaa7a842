// Rows read and written 16 bytes at a time at an element's alignment: a row of odd
// length begins anywhere, and gfx950 takes such accesses whole.
#pragma once

#include "ramnet_device.hpp"

namespace ramnet {

// N adjacent elements as they are stored (16 bytes, or one element).
template<typename Scalar, int N>
struct Vec {
    static constexpr int kBytes = N * static_cast<int>(sizeof(Scalar)), kWords = kBytes >= 4 ? kBytes / 4 : 1;
    uint32_t w[kWords];

    __device__ __forceinline__ float operator[](int e) const {
        if constexpr (sizeof(Scalar) == 4)
            return __uint_as_float(w[e]);
        else
            return bits_f32<Scalar>((w[e / 2] >> (e % 2 * 16)) & 0xFFFFu);
    }
};

template<typename Scalar, int N>
__device__ __forceinline__ Vec<Scalar, N> load_vec(const Scalar *p) {
    if constexpr (N == 1) {
        return {{load_bits(p)}};
    } else {
        struct __attribute__((packed, aligned(sizeof(Scalar)))) Raw {
            uint32_t w[Vec<Scalar, N>::kWords];
        };
        const Raw r = *reinterpret_cast<const Raw *>(p);
        Vec<Scalar, N> out;
#pragma unroll
        for (int i = 0; i < Vec<Scalar, N>::kWords; ++i)
            out.w[i] = r.w[i];
        return out;
    }
}

template<typename Scalar, int N>
__device__ __forceinline__ void store_vec(Scalar *p, const Vec<Scalar, N> &v) {
    if constexpr (N == 1) {
        if constexpr (sizeof(Scalar) == 4)
            *reinterpret_cast<uint32_t *>(p) = v.w[0];
        else
            *reinterpret_cast<uint16_t *>(p) = static_cast<uint16_t>(v.w[0]);
    } else {
        struct __attribute__((packed, aligned(sizeof(Scalar)))) Raw {
            uint32_t w[Vec<Scalar, N>::kWords];
        };
        Raw r;
#pragma unroll
        for (int i = 0; i < Vec<Scalar, N>::kWords; ++i)
            r.w[i] = v.w[i];
        *reinterpret_cast<Raw *>(p) = r;
    }
}

// Rounded to Scalar, to nearest even.
template<typename Scalar>
__device__ __forceinline__ uint32_t round_bits(float x) {
    if constexpr (sizeof(Scalar) == 4) {
        return __float_as_uint(x);
    } else if constexpr (__is_same(Scalar, bf16_t)) {
        return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
    } else {
        return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
    }
}

template<typename Scalar, int N>
__device__ __forceinline__ Vec<Scalar, N> round_vec(const float (&x)[N]) {
    Vec<Scalar, N> out;
    if constexpr (sizeof(Scalar) == 4 || N == 1) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            out.w[i] = round_bits<Scalar>(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2)
            out.w[i / 2] = round_bits<Scalar>(x[i]) | round_bits<Scalar>(x[i + 1]) << 16;
    }
    return out;
}

// 1 / (1 + e^-x), on the hardware's exponential and reciprocal (1 ulp each).
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}

}  // namespace ramnet
