// Activation checkpoints in 8 bits: rows of features to codes with one fp32
// scale per 128 channels, and back (the form is defined in rows.cuh).
//
// Memory bounds both: pack reads 4 (or 2) bytes and writes 1 per element,
// unpack the reverse. One team of LPR lanes takes one block of up to 128
// channels of a row: the whole block is in its registers when the maximum is
// known, so the input is read once. kUnits blocks are in flight per team to
// cover the latency of HBM.
#include "rows.cuh"

namespace mg {

namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;

// Unit u is block u % nb of row u / nb. Lane `lane` holds NV groups of VEC
// channels, group k at channel (k * LPR + lane) * VEC of the block.
template <typename T, int VEC, int LPR, int NV>
__global__ void __launch_bounds__(kThreads)
pack8_kernel(const T* __restrict__ x, int64_t units, int nb, int channels,
             int8_t* __restrict__ codes, float* __restrict__ scales) {
    constexpr int kTeams = kThreads / LPR;
    const int lane = threadIdx.x % LPR;
    const int64_t u0 = (int64_t)blockIdx.x * kTeams * kUnits + threadIdx.x / LPR;
    float v[kUnits][NV * VEC];
    int64_t base[kUnits];
    int len[kUnits];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int64_t u = u0 + j * kTeams;
        const int64_t row = nb == 1 ? u : u / nb;
        const int c0 = nb == 1 ? 0 : (int)(u - row * nb) * kBlock8;
        base[j] = row * channels + c0;
        len[j] = u < units ? min(kBlock8, channels - c0) : 0;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * LPR + lane) * VEC;
            if (c < len[j]) {
                load_row<T, VEC>(x + base[j] + c, &v[j][k * VEC]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[j][k * VEC + i] = 0.0f;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i) a = fmaxf(a, mag8(v[j][i]));
        a = lanes_max<LPR>(a);
        const Scale8 s = scale8(a);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * LPR + lane) * VEC;
            if (c < len[j]) {
                int q[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) q[i] = code8(v[j][k * VEC + i], s.inv);
                store_codes<VEC>(codes + base[j] + c, q);
            }
        }
        if (lane == 0 && len[j] > 0) scales[u0 + j * kTeams] = s.scale;
    }
}

template <typename T, int VEC, int LPR, int NV>
__global__ void __launch_bounds__(kThreads)
unpack8_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, int64_t units,
               int nb, int channels, T* __restrict__ x) {
    constexpr int kTeams = kThreads / LPR;
    const int lane = threadIdx.x % LPR;
    const int64_t u0 = (int64_t)blockIdx.x * kTeams * kUnits + threadIdx.x / LPR;
    float v[kUnits][NV * VEC], s[kUnits];
    int64_t base[kUnits];
    int len[kUnits];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int64_t u = u0 + j * kTeams;
        const int64_t row = nb == 1 ? u : u / nb;
        const int c0 = nb == 1 ? 0 : (int)(u - row * nb) * kBlock8;
        base[j] = row * channels + c0;
        len[j] = u < units ? min(kBlock8, channels - c0) : 0;
        s[j] = len[j] > 0 ? __ldg(scales + u) : 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * LPR + lane) * VEC;
            if (c < len[j]) load_codes<VEC>(codes + base[j] + c, &v[j][k * VEC]);
        }
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * LPR + lane) * VEC;
            if (c < len[j]) {
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = __fmul_rn(v[j][k * VEC + i], s[j]);
                store_row<T, VEC>(x + base[j] + c, o);
            }
        }
    }
}

struct Pack {
    const void* x;
    int64_t rows;
    int channels;
    int8_t* codes;
    float* scales;
    cudaStream_t st;

    template <typename T, int VEC, int LPR, int NV>
    mg_status run() const {
        const int nb = blocks8(channels);
        const int64_t units = rows * nb;
        pack8_kernel<T, VEC, LPR, NV>
            <<<ceil_div(units, kThreads / LPR * kUnits), kThreads, 0, st>>>(
                static_cast<const T*>(x), units, nb, channels, codes, scales);
        return check_launch("pack8");
    }
};

struct Unpack {
    const int8_t* codes;
    const float* scales;
    int64_t rows;
    int channels;
    void* x;
    cudaStream_t st;

    template <typename T, int VEC, int LPR, int NV>
    mg_status run() const {
        const int nb = blocks8(channels);
        const int64_t units = rows * nb;
        unpack8_kernel<T, VEC, LPR, NV>
            <<<ceil_div(units, kThreads / LPR * kUnits), kThreads, 0, st>>>(
                codes, scales, units, nb, channels, static_cast<T*>(x));
        return check_launch("unpack8");
    }
};

// The fewest lanes that hold a block (the whole row when it is shorter).
template <typename T, int VEC, typename Op>
mg_status pick_team(const Op& op, int channels) {
    const int vecs = (std::min(channels, kBlock8) + VEC - 1) / VEC;
    if (vecs <= 4) return op.template run<T, VEC, 4, 1>();
    if (vecs <= 8) return op.template run<T, VEC, 8, 1>();
    if (vecs <= 16) return op.template run<T, VEC, 16, 1>();
    if constexpr (VEC < 8) {
        if (vecs <= 32) return op.template run<T, VEC, 32, 1>();
    }
    if constexpr (VEC == 1) {
        if (vecs <= 64) return op.template run<T, VEC, 32, 2>();
        return op.template run<T, VEC, 32, 4>();
    }
    return MG_ERR_INVALID_ARGUMENT;  // not reached: 128 channels are 32 or 16 vectors
}

template <typename Op>
mg_status pick_type(const Op& op, int dtype, int channels, bool aligned) {
    if (dtype == MG_F32)
        return aligned && channels % 4 == 0 ? pick_team<float, 4>(op, channels)
                                            : pick_team<float, 1>(op, channels);
    if (dtype == MG_BF16)
        return aligned && channels % 8 == 0 ? pick_team<__nv_bfloat16, 8>(op, channels)
                                            : pick_team<__nv_bfloat16, 1>(op, channels);
    return aligned && channels % 8 == 0 ? pick_team<__half, 8>(op, channels)
                                        : pick_team<__half, 1>(op, channels);
}

mg_status check_sizes(int32_t dtype, int64_t rows, int64_t channels, const int8_t* codes,
                      const char* who) {
    const std::string w(who);
    MG_REQUIRE(dtype == MG_F32 || dtype == MG_BF16 || dtype == MG_F16, w + ": unknown dtype");
    MG_REQUIRE(rows >= 0 && channels >= 1, w + ": rows must be >= 0 and channels >= 1");
    MG_REQUIRE((reinterpret_cast<uintptr_t>(codes) & 7u) == 0u, w + ": codes must be 8-byte aligned");
    // grid of 32-bit blocks: at most 2^31 - 1 of at least 32 units
    if (channels > (int64_t)1 << 30 || rows > ((int64_t)1 << 36) / blocks8(channels))
        return fail(MG_ERR_CAPACITY, w + ": too many elements");
    return MG_OK;
}

}  // namespace

}  // namespace mg

using namespace mg;

extern "C" mg_status mg_pack8(const void* x, int32_t dtype, int64_t rows, int64_t channels,
                              int8_t* codes, float* scales, mg_stream_t stream) {
    MG_TRY(check_sizes(dtype, rows, channels, codes, "pack8"));
    if (rows == 0) return MG_OK;
    MG_REQUIRE(x && codes && scales, "pack8: null pointer");
    const Pack op{x, rows, (int)channels, codes, scales, reinterpret_cast<cudaStream_t>(stream)};
    return pick_type(op, dtype, (int)channels, aligned16(x));
}

extern "C" mg_status mg_unpack8(const int8_t* codes, const float* scales, int64_t rows,
                                int64_t channels, int32_t dtype, void* x, mg_stream_t stream) {
    MG_TRY(check_sizes(dtype, rows, channels, codes, "unpack8"));
    if (rows == 0) return MG_OK;
    MG_REQUIRE(x && codes && scales, "unpack8: null pointer");
    const Unpack op{codes, scales, rows, (int)channels, x, reinterpret_cast<cudaStream_t>(stream)};
    return pick_type(op, dtype, (int)channels, aligned16(x));
}
