// Shared pieces of the kernels on rows of per-pixel features (layernorm.cu,
// activations.cu): element types, 16-byte loads and stores that convert to
// and from fp32, and the sums and maxima over the lanes that hold one row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace mg {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// VEC elements at p as fp32; VEC * sizeof(T) is 16 bytes (p aligned to it) or
// VEC is 1. Read-once data: past L1.
template <typename T, int VEC>
__device__ __forceinline__ void load_row(const T* __restrict__ p, float* v) {
    if constexpr (VEC == 1) {
        v[0] = to_f32<T>(__ldg(p));
    } else {
        static_assert(VEC * sizeof(T) == 16, "16-byte vectors");
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
        T e[VEC];
        memcpy(e, &r, 16);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = to_f32<T>(e[i]);
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_row(T* __restrict__ p, const float* v) {
    if constexpr (VEC == 1) {
        p[0] = from_f32<T>(v[0]);
    } else {
        T e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(v[i]);
        uint4 r;
        memcpy(&r, e, 16);
        *reinterpret_cast<uint4*>(p) = r;
    }
}

// The same without the conversion: 16-bit rows wait in half the registers.
template <typename T, int VEC>
__device__ __forceinline__ void load_raw(const T* __restrict__ p, T* v) {
    if constexpr (VEC == 1) {
        v[0] = __ldg(p);
    } else {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
        memcpy(v, &r, 16);
    }
}

// VEC codes (VEC 1, 4 or 8; p aligned to VEC bytes).
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* __restrict__ p, const int* q) {
    if constexpr (VEC == 1) {
        p[0] = (int8_t)q[0];
    } else {
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) {
            const uint32_t w = (uint32_t)(uint8_t)q[4 * k] | (uint32_t)(uint8_t)q[4 * k + 1] << 8 |
                               (uint32_t)(uint8_t)q[4 * k + 2] << 16 |
                               (uint32_t)(uint8_t)q[4 * k + 3] << 24;
            if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(p) = w;
            else reinterpret_cast<uint32_t*>(p)[k] = w;
        }
    }
}

template <int VEC>
__device__ __forceinline__ void load_codes(const int8_t* __restrict__ p, float* v) {
    if constexpr (VEC == 1) {
        v[0] = (float)__ldg(p);
    } else {
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) {
            const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(p) + k);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * k + i] = (float)(int8_t)(w >> (8 * i));
        }
    }
}

template <int VEC>
__device__ __forceinline__ void load_codes_raw(const int8_t* __restrict__ p, int8_t* v) {
    if constexpr (VEC == 1) {
        v[0] = __ldg(p);
    } else {
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) {
            const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(p) + k);
            memcpy(v + 4 * k, &w, 4);
        }
    }
}

// Sum over groups of L lanes (a power of two); every lane gets it. Lanes of a
// group take the same steps, so the order of the sum is fixed.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// ------------------------------------------------------------ the 8-bit form
//
// kBlock8 consecutive channels of a row (fewer at its end) share one fp32
// scale: a the largest magnitude, inv = 127 / a, scale = a / 127, code =
// round-half-even(x * inv), value = code * scale. Every operation is a
// correctly rounded fp32 one, so the codes are the same wherever they are
// computed. |x * inv| <= 127 (1 + 2^-23) rounds to at most 127. A block below
// kTiny8 (127 / a would overflow) is held as zeros; a block with an infinity
// or a NaN gets a NaN scale, so all of it reads back as NaN.
constexpr int kBlock8 = 128;
constexpr float kTiny8 = 1e-30f;

struct Scale8 {
    float inv, scale;
};

// fmaxf drops NaNs, so the caller's maximum is over |x| with NaN mapped to
// infinity (mag8).
__device__ __forceinline__ float mag8(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : __int_as_float(0x7f800000);
}

__device__ __forceinline__ Scale8 scale8(float a) {
    Scale8 s;
    if (!(a <= 3.402823466e38f)) {
        s.inv = 0.0f;
        s.scale = __int_as_float(0x7fc00000);
    } else if (a < kTiny8) {
        s.inv = 0.0f;
        s.scale = 0.0f;
    } else {
        s.inv = __fdiv_rn(127.0f, a);
        s.scale = __fdiv_rn(a, 127.0f);
        // next to the largest float, 127 * scale may round past it: one step down
        if (__fmul_rn(127.0f, s.scale) > 3.402823466e38f)
            s.scale = __int_as_float(__float_as_int(s.scale) - 1);
    }
    return s;
}

// A NaN or infinite x times inv = 0 is NaN, which converts to code 0.
__device__ __forceinline__ int code8(float x, float inv) { return __float2int_rn(__fmul_rn(x, inv)); }

inline int blocks8(int64_t channels) { return (int)((channels + kBlock8 - 1) / kBlock8); }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0u; }

// SMs of the current device (cached per device).
int sm_count();

}  // namespace mg
