// The label loss's row bookkeeping, shared by its kernels.
#pragma once

#include "rows.cuh"
#include "tensor.cuh"

namespace mg {

// A row's class: its label, kIgnored for the ignored value, kBadLabel for one
// outside [0, classes).
constexpr int kIgnored = -1;
constexpr int kBadLabel = -2;

struct LabelSource {
    const void* labels;
    int bytes;  // 1 (uint8), 4 (int32) or 8 (int64)
    int64_t ignore_index;
    int classes;

    __device__ __forceinline__ int at(int64_t row) const {
        int64_t v;
        if (bytes == 1) v = static_cast<const uint8_t*>(labels)[row];
        else if (bytes == 4) v = static_cast<const int32_t*>(labels)[row];
        else v = static_cast<const int64_t*>(labels)[row];
        if (v == ignore_index) return kIgnored;
        return v >= 0 && v < classes ? (int)v : kBadLabel;
    }
};

// A row's factor on its gradient: the upstream gradient, over the live count
// for a mean; 0 for a row that is ignored or has no valid label.
struct RowGrad {
    const float* grad;
    const float* live;  // live count, for a mean only
    int per_row;

    __device__ __forceinline__ float at(int64_t row, int label) const {
        if (label < 0) return 0.0f;
        const float g = per_row ? grad[row] : grad[0];
        return live != nullptr ? g / fmaxf(live[0], 1.0f) : g;
    }
};

// What the backward pass's scores need of a row: minus log2 of its sum, r, G at
// its label, its label (an int), each kRowBlock in a row per block of rows.
constexpr int kRowValues = 4;
constexpr int kRowBlock = 64;
constexpr int kClassPad = 256;  // class_bias is padded to a multiple of this

constexpr float kInf = __builtin_huge_valf();
constexpr float kNaN = __builtin_nanf("");
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Within 2^-22 of the value; below fp32's smallest normal number (2^-126) 0, so
// smaller entries of a softmax count as none.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 operations in one instruction, each rounded as its scalar form.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
        "fma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\n"
        "add.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\n"
        "mul.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// The largest of three; NaNs drop out as with fmaxf.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// --------------------------------------------------------------------- parts

// The number of bf16 parts of a type.
template <typename T>
constexpr int kPartsOf = sizeof(T) == 4 ? 3 : 2;
template <>
constexpr int kPartsOf<__nv_bfloat16> = 1;

// An fp32 value past bf16's largest (by less than half a step of it, the type's
// lowest among them) takes that as its first part; rounded, it would be infinite.
template <int PARTS>
__device__ __forceinline__ void split_parts(float v, __nv_bfloat16 (&p)[PARTS]) {
    constexpr float kMost = 3.38953138925153547e38f;
    p[0] = __float2bfloat16_rn(PARTS == 3 && fabsf(v) < kInf ? fminf(fmaxf(v, -kMost), kMost) : v);
#pragma unroll
    for (int i = 1; i < PARTS; ++i) {
        v -= __bfloat162float(p[i - 1]);
        p[i] = __float2bfloat16_rn(v);
    }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    uint32_t r;
    memcpy(&r, &v, 4);
    return r;
}

// One part of (lo, hi) as a word; lo and hi keep what it leaves over.
__device__ __forceinline__ uint32_t take_part(float& lo, float& hi) {
    const uint32_t w = pack_bf16(lo, hi);
    const float2 rest = fma2(make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)), both(-1.0f),
                             make_float2(lo, hi));
    lo = rest.x;
    hi = rest.y;
    return w;
}

// Parts of the logits' gradient: two also for bf16 features, whose gradients
// then carry no other rounding than their own (one part alone brings their
// error from 0.0017 to 0.0028 of the norm).
// A part below 2^-126 counts as none, so an entry of G under 2^-118 keeps fewer bits.
template <int PARTS>
constexpr int kGParts = PARTS == 1 ? 2 : PARTS;

// Products of parts (a, b), smallest first: of the 1, 3, 4 or 6 pairs that
// matter at PARTS parts, the i-th.
template <int PARTS>
__device__ constexpr int pair_a(int pairs, int i) {
    if (PARTS == 1) return 0;
    if (PARTS == 2) return (i + 4 - pairs) == 0 || (i + 4 - pairs) == 1 ? 1 : 0;
    return i == 0 ? 2 : i == 1 || i == 3 ? 1 : 0;
}
template <int PARTS>
__device__ constexpr int pair_b(int pairs, int i) {
    if (PARTS == 1) return 0;
    if (PARTS == 2) return (i + 4 - pairs) == 0 || (i + 4 - pairs) == 2 ? 1 : 0;
    return i == 2 ? 2 : i == 1 || i == 4 ? 1 : 0;
}

// The same for products of G's parts with a side's.
template <int PARTS>
constexpr int kGPairs = PARTS == 1 ? 2 : PARTS == 2 ? 3 : 6;
template <int PARTS>
__device__ constexpr int g_pair_a(int i) {
    return PARTS == 1 ? 1 - i : pair_a<PARTS>(kGPairs<PARTS>, i);
}
template <int PARTS>
__device__ constexpr int g_pair_b(int i) {
    return PARTS == 1 ? 0 : pair_b<PARTS>(kGPairs<PARTS>, i);
}

// What a wait that gave up leaves of n results.
template <typename T>
__device__ __forceinline__ void store_nan(T* dst, int n) {
#pragma unroll 1
    for (int i = 0; i < n; ++i) dst[i] = from_f32<T>(kNaN);
}

// The features' type, by its parts.
template <int PARTS>
struct PartsType;
template <>
struct PartsType<1> { using type = __nv_bfloat16; };
template <>
struct PartsType<2> { using type = __half; };
template <>
struct PartsType<3> { using type = float; };
template <int PARTS>
using TypeOf = typename PartsType<PARTS>::type;

}  // namespace mg
