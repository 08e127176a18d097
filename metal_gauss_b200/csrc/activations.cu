// Activation checkpoints in 8 bits: rows of features to codes with one fp32
// scale per 128 channels, and back (the form is defined in rows.cuh).
//
// Memory bounds both: pack reads 4 (or 2) bytes and writes 1 per element,
// unpack the reverse. 1440000 x 32 fp32: pack 40 us (5.9 TB/s), unpack 47 (5.0);
// 262144 x 512 bf16: 80 (5.1) and 84 (4.8). pack: one team of LPR lanes takes one block of up to 128
// channels of a row; the whole block is in its registers when the maximum is
// known, so the input is read once, and kUnits blocks are in flight per team to
// cover the latency of HBM. unpack needs no row: it runs over the flat tensor.
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
    T v[kUnits][NV * VEC];
    int64_t base[kUnits];
    int len[kUnits];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int64_t u = u0 + j * kTeams;
        int64_t row = u;
        int c0 = 0;
        if (nb > 1) {  // 32-bit division where it does: the 64-bit one costs more than the block
            row = u <= 0xffffffffll ? (int64_t)((uint32_t)u / (uint32_t)nb) : u / nb;
            c0 = (int)(u - row * nb) * kBlock8;
        }
        base[j] = row * channels + c0;
        len[j] = u < units ? min(kBlock8, channels - c0) : 0;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * LPR + lane) * VEC;
            if (c < len[j]) {
                load_raw<T, VEC>(x + base[j] + c, &v[j][k * VEC]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[j][k * VEC + i] = from_f32<T>(0.0f);
            }
        }
    }
    // The two quotients of unit j are lane j's to compute: two divisions for all
    // kUnits blocks, where each lane doing them for its own cost more than all else.
    static_assert(kUnits <= LPR, "a lane for each unit");
    uint32_t mine = 0u;
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const uint32_t a = lanes_max<LPR>(largest8<T, NV * VEC>(v[j]));
        if (lane == j) mine = a;
    }
    const Scale8 s = scale8(mine);
    if (lane < kUnits && u0 + lane * kTeams < units) scales[u0 + lane * kTeams] = s.scale;
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const float inv = __shfl_sync(0xffffffffu, s.inv, j, LPR);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * LPR + lane) * VEC;
            if (c < len[j]) {
                uint32_t q[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) q[i] = code8(to_f32<T>(v[j][k * VEC + i]), inv);
                store_codes<VEC>(codes + base[j] + c, q);
            }
        }
    }
}

// Rows of a length that is no multiple of 16 bytes, a staged chunk at a time.
template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads)
pack8_staged_kernel(const T* __restrict__ x, int64_t rows, int channels, int chunk, int width,
                    int codes_width, int8_t* __restrict__ codes, float* __restrict__ scales) {
    extern __shared__ __align__(16) uint8_t staged[];
    const int row_bytes = channels * (int)sizeof(T), nb = (channels + kBlock8 - 1) / kBlock8;
    const int buffer = align16(chunk * row_bytes);
    int8_t* out = reinterpret_cast<int8_t*>(staged + 2 * buffer);
    float* work = reinterpret_cast<float*>(staged + 2 * buffer + align16(chunk * channels));
    const int64_t chunks = (rows + chunk - 1) / chunk;
    const auto rows_of = [&](int64_t i) { return (int)min((int64_t)chunk, rows - i * chunk); };
    const auto fetch = [&](int64_t i, int b) {
        stage_in(staged + b * buffer, reinterpret_cast<const uint8_t*>(x + i * chunk * channels),
                 rows_of(i) * row_bytes, width);
        stage_commit();
    };
    int b = 0;
    if (blockIdx.x < chunks) fetch(blockIdx.x, 0);
    for (int64_t i = blockIdx.x; i < chunks; i += gridDim.x, b ^= 1) {
        if (i + gridDim.x < chunks) {
            fetch(i + gridDim.x, b ^ 1);
            stage_wait<1>();
        } else {
            stage_wait<0>();
        }
        __syncthreads();
        const int n = rows_of(i);
        staged_codes<T, LPR>(reinterpret_cast<const T*>(staged + b * buffer), n, channels, work, out,
                             scales + i * chunk * nb);
        stage_out(reinterpret_cast<uint8_t*>(codes + i * chunk * channels), reinterpret_cast<uint8_t*>(out),
                  n * channels, codes_width);
        __syncthreads();
    }
}

// x = code * scale over the flat tensor, kFlat groups of VEC elements to a
// thread wherever rows and blocks end (VEC 1 for what is left, or tensors off
// the boundaries).
constexpr int kFlat = 2;
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
unpack8_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, int64_t first,
               int64_t count, int nb, int channels, T* __restrict__ x) {
    const int64_t v0 = (int64_t)blockIdx.x * (kThreads * kFlat) + threadIdx.x;
    int8_t q[kFlat][VEC];
    const float* s[kFlat];
    float scale[kFlat];
    int c[kFlat];
#pragma unroll
    for (int j = 0; j < kFlat; ++j) {
        const int64_t v = v0 + j * kThreads, e = first + v * VEC;
        if (v >= count) continue;
        if constexpr (VEC == 8) {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(codes + e));
            memcpy(q[j], &w, 8);
        } else {
            q[j][0] = __ldg(codes + e);
        }
        int64_t row;
        if (e <= 0xffffffffll) {
            const uint32_t r = (uint32_t)e / (uint32_t)channels;
            row = r;
            c[j] = (int)((uint32_t)e - r * (uint32_t)channels);
        } else {
            row = e / channels;
            c[j] = (int)(e - row * channels);
        }
        s[j] = scales + row * nb + c[j] / kBlock8;
        scale[j] = __ldg(s[j]);
    }
#pragma unroll
    for (int j = 0; j < kFlat; ++j) {
        const int64_t v = v0 + j * kThreads, e = first + v * VEC;
        if (v >= count) continue;
        T o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            o[i] = from_f32<T>(__fmul_rn((float)q[j][i], scale[j]));
            ++c[j];
            if (i + 1 < VEC && (c[j] == channels || c[j] % kBlock8 == 0)) {
                if (c[j] == channels) c[j] = 0;
                scale[j] = __ldg(++s[j]);  // the next block, of this row or the next
            }
        }
        if constexpr (VEC == 8) {
            uint4 w[sizeof(o) / 16];
            memcpy(w, o, sizeof(o));
#pragma unroll
            for (int i = 0; i < (int)(sizeof(o) / 16); ++i) reinterpret_cast<uint4*>(x + e)[i] = w[i];
        } else {
            x[e] = o[0];
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

template <typename T, int LPR>
mg_status pack_staged(const Pack& p) {
    const int chunk = stage_rows(p.channels, (int)sizeof(T)), nb = blocks8(p.channels);
    const int bytes = chunk * p.channels * (int)sizeof(T);
    const int smem = 2 * align16(bytes) + align16(chunk * p.channels) + 4 * chunk * nb;
    static int known[64] = {};
    int per_sm = 0;
    MG_TRY(staged_launch(pack8_staged_kernel<T, LPR>, kThreads, smem, known, &per_sm, "pack8"));
    const int64_t chunks = (p.rows + chunk - 1) / chunk;
    const int grid = (int)std::min<int64_t>(chunks, per_sm * (int64_t)sm_count());
    pack8_staged_kernel<T, LPR><<<grid, kThreads, smem, p.st>>>(
        static_cast<const T*>(p.x), p.rows, p.channels, chunk, stage_width(p.x, bytes),
        stage_width(p.codes, chunk * p.channels), p.codes, p.scales);
    return check_launch("pack8");
}

// Whole 16-byte vectors by row where the length allows; where not, staged chunks
// of short rows and single elements of longer ones. In us, staged and by elements:
//   1766022 x 19 fp32 92 and 96, fp16 88 and 94; 400000 x 61 55 and 35, 53 and 35
//   435771 x 77 fp32 68 and 47; 260111 x 129 76 and 70; 111476 x 301 72 and 49
//   5000 x 19 8 and 6, 110000 x 19 12 and 10, 160000 x 19 14 and 14
// So the border of 64 channels is too high (61 channels lose), by up to 20 us.
template <typename T, int VEC>
mg_status pack(const Pack& p) {
    if (aligned16(p.x) && p.channels % VEC == 0) return pick_team<T, VEC>(p, p.channels);
    const bool many = p.rows * p.channels >= 1 << 21;  // (5000 x 19 fp16: 2.5 us by elements, 7.9 staged)
    if (many && p.channels <= 64) return p.channels <= 32 ? pack_staged<T, 8>(p) : pack_staged<T, 16>(p);
    return pick_team<T, 1>(p, p.channels);
}

template <typename T>
mg_status unpack(const int8_t* codes, const float* scales, int64_t rows, int channels, T* x,
                 cudaStream_t st) {
    const int64_t n = rows * channels;
    const int nb = blocks8(channels);
    const int64_t vectors = aligned16(x) ? n / 8 : 0, left = n - 8 * vectors;
    if (vectors > 0) {
        unpack8_kernel<T, 8><<<(unsigned)((vectors + kThreads * kFlat - 1) / (kThreads * kFlat)), kThreads, 0, st>>>(
            codes, scales, 0, vectors, nb, channels, x);
        MG_TRY(check_launch("unpack8"));
    }
    if (left == 0) return MG_OK;
    unpack8_kernel<T, 1><<<(unsigned)((left + kThreads * kFlat - 1) / (kThreads * kFlat)), kThreads, 0, st>>>(
        codes, scales, 8 * vectors, left, nb, channels, x);
    return check_launch("unpack8");
}

mg_status check_sizes(int32_t dtype, int64_t rows, int64_t channels, const int8_t* codes,
                      const char* who) {
    const std::string w(who);
    MG_REQUIRE(dtype == MG_F32 || dtype == MG_BF16 || dtype == MG_F16, w + ": unknown dtype");
    MG_REQUIRE(rows >= 0 && channels >= 1, w + ": rows must be >= 0 and channels >= 1");
    MG_REQUIRE((reinterpret_cast<uintptr_t>(codes) & 7u) == 0u, w + ": codes must be 8-byte aligned");
    // grids are 32-bit: at most 2^31 - 1 blocks of 2048 elements or 32 units
    if (channels > (int64_t)1 << 30 || rows > ((int64_t)1 << 36) / blocks8(channels) ||
        rows > ((int64_t)1 << 38) / channels)
        return fail(MG_ERR_CAPACITY, w + ": too many elements");
    return MG_OK;
}

}  // namespace

}  // namespace mg

using namespace mg;

extern "C" mg_status mg_pack8(const void* x, int32_t dtype, int64_t rows, int64_t channels,
                              int8_t* codes, float* scales, mg_stream_t stream) try {
    MG_TRY(check_sizes(dtype, rows, channels, codes, "pack8"));
    if (rows == 0) return MG_OK;
    MG_REQUIRE(x && codes && scales, "pack8: null pointer");
    MG_REQUIRE(on_boundary(elem_bytes(dtype), {x}) && on_boundary(4, {scales}),
               "pack8: a pointer off its element's boundary");
    const Pack op{x, rows, (int)channels, codes, scales, reinterpret_cast<cudaStream_t>(stream)};
    if (dtype == MG_F32) return pack<float, 4>(op);
    if (dtype == MG_BF16) return pack<__nv_bfloat16, 8>(op);
    return pack<__half, 8>(op);
} catch (...) {
    return caught("pack8");
}

extern "C" mg_status mg_unpack8(const int8_t* codes, const float* scales, int64_t rows,
                                int64_t channels, int32_t dtype, void* x, mg_stream_t stream) try {
    MG_TRY(check_sizes(dtype, rows, channels, codes, "unpack8"));
    if (rows == 0) return MG_OK;
    MG_REQUIRE(x && codes && scales, "unpack8: null pointer");
    MG_REQUIRE(on_boundary(elem_bytes(dtype), {x}) && on_boundary(4, {scales}),
               "unpack8: a pointer off its element's boundary");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == MG_F32) return unpack(codes, scales, rows, (int)channels, static_cast<float*>(x), st);
    if (dtype == MG_BF16) return unpack(codes, scales, rows, (int)channels, static_cast<__nv_bfloat16*>(x), st);
    return unpack(codes, scales, rows, (int)channels, static_cast<__half*>(x), st);
} catch (...) {
    return caught("unpack8");
}
