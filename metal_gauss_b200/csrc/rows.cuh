// Shared pieces of the kernels on rows of per-pixel features (layernorm.cu,
// activations.cu): element types, 16-byte loads and stores that convert to
// and from fp32, and the sums and maxima over the lanes that hold one row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>

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

// VEC elements at p from fp32; VEC * sizeof(T) is 16 bytes (p aligned to it) or
// VEC is 1.
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

// VEC elements at p as they are: 16-bit rows wait in half the registers.
// Read-once data: past L1.
template <typename T, int VEC>
__device__ __forceinline__ void load_raw(const T* __restrict__ p, T* v) {
    if constexpr (VEC == 1) {
        v[0] = __ldg(p);
    } else {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
        memcpy(v, &r, 16);
    }
}

// VEC codes, the low bytes of q (VEC 1, 4 or 8; p aligned to VEC bytes).
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* __restrict__ p, const uint32_t* q) {
    if constexpr (VEC == 1) {
        p[0] = (int8_t)q[0];
    } else {
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k)
            reinterpret_cast<uint32_t*>(p)[k] =
                __byte_perm(__byte_perm(q[4 * k], q[4 * k + 1], 0x0040),
                            __byte_perm(q[4 * k + 2], q[4 * k + 3], 0x0040), 0x5410);
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
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    if constexpr (L == 32) return __reduce_max_sync(0xffffffffu, v);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
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

// |x| as an integer, whose order is that of the magnitudes with infinity and
// then NaN above them: the maximum of these misses no NaN, as fmaxf would.
__device__ __forceinline__ uint32_t mag8(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The largest of N elements' magnitudes; 16-bit types two at a time.
template <typename T, int N>
__device__ __forceinline__ uint32_t largest8(const T* v) {
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
        uint32_t a = 0u;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            uint32_t w;
            memcpy(&w, v + i, 4);
            a = __vmaxu2(a, w & 0x7fff7fffu);
        }
        const uint16_t top = (uint16_t)max(a & 0xffffu, a >> 16);
        T t;
        memcpy(&t, &top, 2);
        return __float_as_uint(to_f32<T>(t));
    } else {
        uint32_t a = 0u;
#pragma unroll
        for (int i = 0; i < N; ++i) a = max(a, mag8(to_f32<T>(v[i])));
        return a;
    }
}

__device__ __forceinline__ Scale8 scale8(uint32_t magnitude) {
    const float a = __uint_as_float(magnitude);
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

// The code in the low byte: adding 1.5 * 2^23 rounds a product of at most 127
// to an integer, half to even, in the sum's last bits. (In a block with a NaN
// or an infinity the byte means nothing: its scale is NaN.)
__device__ __forceinline__ uint32_t code8(float x, float inv) {
    return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.0f));
}

// ------------------------------------------------- rows of any length, staged
//
// Rows whose length is no multiple of 16 bytes start anywhere, but a chunk of
// rows is one stretch of memory: a block copies it to shared memory in 16-byte
// pieces (asynchronous, the next chunk while this one is worked on), works on
// it there by rows or columns, and writes the result back the same way. Chunks
// of stage_rows rows start on 16-byte boundaries when the tensor does.

constexpr int kStageMaxChannels = 1024;

// Rows of a chunk: about 16 KB, a multiple of 16 rows while that allows (so
// that rows of single bytes keep the boundary too), at least 8.
__host__ __device__ inline int stage_rows(int channels, int elem_bytes) {
    const int fit = 16384 / (channels * elem_bytes);
    return fit >= 16 ? fit / 16 * 16 : 8;
}

// The pieces (16, 8, 4 bytes or single ones) that a tensor's chunks of
// chunk_bytes allow.
inline int stage_width(const void* base, int64_t chunk_bytes) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(base) | (uintptr_t)chunk_bytes;
    return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 1;
}

// `bytes` from global to 16-byte aligned shared memory by a whole block, in
// pieces of `width` (asynchronous from 4 up). The caller commits the group.
__device__ __forceinline__ void stage_in(uint8_t* dst, const uint8_t* __restrict__ src, int bytes,
                                         int width) {
    const int whole = width > 1 ? bytes / width * width : 0;
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    if (width == 16) {
        for (int i = threadIdx.x * 16; i < whole; i += blockDim.x * 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + i), "l"(src + i) : "memory");
    } else if (width == 8) {
        for (int i = threadIdx.x * 8; i < whole; i += blockDim.x * 8)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d + i), "l"(src + i) : "memory");
    } else if (width == 4) {
        for (int i = threadIdx.x * 4; i < whole; i += blockDim.x * 4)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d + i), "l"(src + i) : "memory");
    }
    for (int i = whole + threadIdx.x; i < bytes; i += blockDim.x) dst[i] = __ldg(src + i);
}
__device__ __forceinline__ void stage_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void stage_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

__device__ __forceinline__ void stage_out(uint8_t* __restrict__ dst, const uint8_t* src, int bytes,
                                          int width) {
    const int whole = width > 1 ? bytes / width * width : 0;
    if (width == 16) {
        for (int i = threadIdx.x * 16; i < whole; i += blockDim.x * 16)
            *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<const uint4*>(src + i);
    } else if (width == 8) {
        for (int i = threadIdx.x * 8; i < whole; i += blockDim.x * 8)
            *reinterpret_cast<uint2*>(dst + i) = *reinterpret_cast<const uint2*>(src + i);
    } else if (width == 4) {
        for (int i = threadIdx.x * 4; i < whole; i += blockDim.x * 4)
            *reinterpret_cast<uint32_t*>(dst + i) = *reinterpret_cast<const uint32_t*>(src + i);
    }
    for (int i = whole + threadIdx.x; i < bytes; i += blockDim.x) dst[i] = src[i];
}

__host__ __device__ inline int align16(int bytes) { return (bytes + 15) & ~15; }

inline int blocks8(int64_t channels) { return (int)((channels + kBlock8 - 1) / kBlock8); }

// The 8-bit form of n staged rows by the whole block (kThreads of it, LPR lanes
// to a row): maxima, then one thread for each block's two quotients, then codes.
// work: n * blocks floats. Ends with a barrier.
template <typename T, int LPR>
__device__ __forceinline__ void staged_codes(const T* rows, int n, int channels, float* work,
                                             int8_t* codes, float* __restrict__ scales) {
    const int nb = (channels + kBlock8 - 1) / kBlock8, lane = threadIdx.x % LPR;
    const int teams = blockDim.x / LPR, team = threadIdx.x / LPR;
    for (int r0 = 0; r0 < n; r0 += teams) {
        const int r = r0 + team;
        for (int q = 0; q < nb; ++q) {
            uint32_t a = 0u;
            if (r < n)
                for (int c = q * kBlock8 + lane; c < min(channels, (q + 1) * kBlock8); c += LPR)
                    a = max(a, mag8(to_f32<T>(rows[r * channels + c])));
            a = lanes_max<LPR>(a);
            if (lane == 0 && r < n) work[r * nb + q] = __uint_as_float(a);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * nb; i += blockDim.x) {
        const Scale8 s = scale8(__float_as_uint(work[i]));
        scales[i] = s.scale;
        work[i] = s.inv;
    }
    __syncthreads();
    for (int r = team; r < n; r += teams)
        for (int c = lane; c < channels; c += LPR)
            codes[r * channels + c] = (int8_t)code8(to_f32<T>(rows[r * channels + c]), work[r * nb + c / kBlock8]);
    __syncthreads();
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0u; }

inline int elem_bytes(int32_t dtype) { return dtype == MG_F32 ? 4 : 2; }

// Whether all of these are on a boundary of `bytes` (NULL is). An address off its
// element's boundary would fault on the device.
inline bool on_boundary(int bytes, std::initializer_list<const void*> pointers) {
    uintptr_t all = 0;
    for (const void* p : pointers) all |= reinterpret_cast<uintptr_t>(p);
    return all % (uintptr_t)bytes == 0;
}

// SMs of the current device (cached per device).
int sm_count();

// Readies a staged kernel for `smem` bytes of dynamic shared memory and gives
// the blocks of one wave on an SM (by shared memory: 227 KB, 1 KB a block kept
// back, and 2048 threads).
constexpr int kStageMaxShared = 160 * 1024;
template <typename K>
mg_status staged_launch(K kernel, int threads, int smem, int (&known)[64], int* per_sm, const char* what) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
    if (known[dev] == 0) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kStageMaxShared) !=
            cudaSuccess)
            return check_launch(what);
        known[dev] = 1;
    }
    *per_sm = std::max(1, std::min(2048 / threads, 227 * 1024 / (smem + 1024)));
    return MG_OK;
}

}  // namespace mg
