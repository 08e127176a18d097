// Layer normalisation of rows of channels, forward and adjoint.
//
//   mean, var over the row; rstd = 1 / sqrt(var + eps); h = (x - mean) rstd
//   y  = h w + b
//   dx = rstd (g - mean(g) - h mean(g h)),  g = dy w
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// Memory bounds it: forward reads x and writes y, the adjoint reads dy and x
// (or x's 8-bit form) and writes dx. A row is held in the registers of a team
// of lanes between its reductions, so each tensor crosses HBM once: LPR lanes
// of a warp for rows up to 1024 channels (several rows to a warp when they are
// short), the 8 warps of a block above that. The variance is the mean of
// (x - mean)^2 from those registers, never E[x^2] - mean^2.
// Measured (of 6.55 TB/s copied): 640000 x 64 fp32 58 us forward (86 %), 77 us
// adjoint (98 %); with the 8-bit form 80 and 75 us (73, 74 %); 262144 x 512 bf16
// 103 and 160 us (80, 77 %: a lane's 32 sums for dw and db leave room for 20
// warps on an SM). Odd lengths: 500000 x 77 fp32 94 and 149 us (50, 47 %).
// dw and db: a lane owns the same channels of every row its team takes, so
// the sums over rows stay in its registers; teams of a block join in shared
// memory, blocks through one fp32 row each in scratch, summed in a fixed order
// by a second kernel (no atomics: equal calls give equal bits).
#include "rows.cuh"

namespace mg {

namespace {

constexpr int kThreads = 256;

// The channel of register group k (VEC channels) of this lane. A warp's 32
// lanes cover 128 consecutive channels (4 groups at VEC 1, one at VEC 4, half
// of one at VEC 8), so the channels that share an 8-bit scale are in one warp.
template <int VEC, int LPR, int WARPS>
__device__ __forceinline__ int channel_of(int k, int warp, int lane) {
    if constexpr (WARPS == 1) return (k * LPR + lane) * VEC;
    if constexpr (VEC == 1) return ((k / 4) * WARPS + warp) * 128 + (k % 4) * 32 + lane;
    return ((k * WARPS + warp) * 32 + lane) * VEC;
}

// weight or bias of a register group's channels: in shared memory (rows up to
// 1024 channels, where registers hold rows in flight instead) or registers. At
// 8 channels to a lane the two halves of each 8 are apart, so that the lanes'
// 16-byte reads follow one another.
template <int N, int VEC, int WARPS>
struct Params {
    float v[WARPS > 1 ? N : 1];
    const float* sh;
    int channels;

    __device__ __forceinline__ static int place(int c, int channels) {
        if constexpr (VEC == 8) return (c & 4 ? channels / 2 : 0) + (c >> 3) * 4 + (c & 3);
        return c;
    }
    // the VEC values of group k, which starts at channel c
    __device__ __forceinline__ void get(int k, int c, float (&o)[VEC]) const {
        if constexpr (WARPS > 1) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] = v[k * VEC + i];
        } else if constexpr (VEC == 1) {
            o[0] = sh[c];
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                const float4 q = *reinterpret_cast<const float4*>(sh + place(c + i, channels));
                o[i] = q.x;
                o[i + 1] = q.y;
                o[i + 2] = q.z;
                o[i + 3] = q.w;
            }
        }
    }
};

// Rows a team takes at once: enough loads in flight to cover HBM's latency
// (about 40 KB an SM), 64 bytes a lane at most, and their reductions overlap.
__host__ __device__ constexpr int rows_at_once(int bytes) {
    return bytes >= 64 ? 1 : bytes >= 32 ? 2 : 4;
}

// Sum over the team that holds a row.
template <int LPR, int WARPS>
__device__ __forceinline__ float2 team_sum(float a, float b, float2* sh, int warp, int lane) {
    a = lanes_sum<LPR>(a);
    b = lanes_sum<LPR>(b);
    if constexpr (WARPS > 1) {
        __syncthreads();  // the previous sum's readers are done
        if (lane == 0) sh[warp] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            a += sh[w].x;
            b += sh[w].y;
        }
    }
    return make_float2(a, b);
}

__device__ __forceinline__ float param_at(const void* p, int dtype, int c) {
    if (dtype == MG_F32) return static_cast<const float*>(p)[c];
    if (dtype == MG_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[c]);
    return to_f32(static_cast<const __half*>(p)[c]);
}

template <typename T, int VEC, int LPR, int NV, int WARPS>
__global__ void __launch_bounds__(kThreads)
norm_forward_kernel(const T* __restrict__ x, const void* __restrict__ weight,
                    const void* __restrict__ bias, int param_dtype, int64_t rows, int channels,
                    float eps, T* __restrict__ y, float* __restrict__ mean_out,
                    float* __restrict__ rstd_out, int8_t* __restrict__ codes,
                    float* __restrict__ scales) {
    __shared__ float2 sh[WARPS > 1 ? WARPS : 1];
    constexpr int kTeams = WARPS > 1 ? 1 : kThreads / LPR;
    const int lane = WARPS > 1 ? threadIdx.x % 32 : threadIdx.x % LPR;
    const int warp = WARPS > 1 ? threadIdx.x / 32 : 0;
    const int team = WARPS > 1 ? 0 : threadIdx.x / LPR;
    const float inv_n = 1.0f / (float)channels;
    const int nb = (channels + kBlock8 - 1) / kBlock8;

    extern __shared__ float dynamic[];
    using P = Params<NV * VEC, VEC, WARPS>;
    P w, b;
    w.sh = dynamic;
    b.sh = dynamic + channels;
    w.channels = b.channels = channels;
    if constexpr (WARPS > 1) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = channel_of<VEC, LPR, WARPS>(k, warp, lane);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                w.v[k * VEC + i] = (weight != nullptr && c < channels) ? param_at(weight, param_dtype, c + i) : 1.0f;
                b.v[k * VEC + i] = (bias != nullptr && c < channels) ? param_at(bias, param_dtype, c + i) : 0.0f;
            }
        }
    } else {
        for (int c = threadIdx.x; c < channels; c += kThreads) {
            dynamic[P::place(c, channels)] = weight != nullptr ? param_at(weight, param_dtype, c) : 1.0f;
            dynamic[channels + P::place(c, channels)] = bias != nullptr ? param_at(bias, param_dtype, c) : 0.0f;
        }
        __syncthreads();
    }

    // every lane of a warp takes every round: the reductions are warp-wide
    constexpr int R = rows_at_once(NV * VEC * (int)sizeof(T));
    const int64_t step = (int64_t)gridDim.x * kTeams * R;
    const int64_t rounds = (rows + step - 1) / step;
    for (int64_t it = 0; it < rounds; ++it) {
        const int64_t row0 = (it * gridDim.x + blockIdx.x) * (kTeams * R) + team;
        T v[R][NV * VEC];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + r * kTeams;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = channel_of<VEC, LPR, WARPS>(k, warp, lane);
                if (row < rows && c < channels) {
                    load_raw<T, VEC>(x + row * channels + c, v[r] + k * VEC);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[r][k * VEC + i] = from_f32<T>(0.0f);
                }
            }
        }
        float mean[R], rstd[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < NV * VEC; ++i) s += to_f32<T>(v[r][i]);
            mean[r] = team_sum<LPR, WARPS>(s, 0.0f, sh, warp, lane).x * inv_n;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float q = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (channel_of<VEC, LPR, WARPS>(k, warp, lane) < channels) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float d = to_f32<T>(v[r][k * VEC + i]) - mean[r];
                        q = fmaf(d, d, q);
                    }
                }
            }
            rstd[r] = 1.0f / sqrtf(team_sum<LPR, WARPS>(q, 0.0f, sh, warp, lane).x * inv_n + eps);
        }
        if (codes != nullptr) {
            // one scale per 128 channels, the maximum over the kGroup lanes that hold
            // them; the quotients of block q (of a row and kStep register groups)
            // are lane q's to compute
            constexpr int kGroup = VEC == 8 ? (LPR < 16 ? LPR : 16) : LPR;
            constexpr int kStep = VEC == 1 ? (NV < 4 ? NV : 4) : 1;
            constexpr int kBlocks = R * (NV / kStep);
            static_assert(kBlocks <= kGroup, "a lane for each block");
            const int member = lane % kGroup;
            uint32_t mine = 0u;
#pragma unroll
            for (int q = 0; q < kBlocks; ++q) {
                const uint32_t a = lanes_max<kGroup>(
                    largest8<T, kStep * VEC>(v[q / (NV / kStep)] + q % (NV / kStep) * kStep * VEC));
                if (member == q) mine = a;
            }
            const Scale8 s8 = scale8(mine);
#pragma unroll
            for (int q = 0; q < kBlocks; ++q) {
                const int r = q / (NV / kStep), k0 = q % (NV / kStep) * kStep;
                const int64_t row = row0 + r * kTeams;
                const float inv = __shfl_sync(0xffffffffu, s8.inv, q, kGroup);
                if (row >= rows) continue;
                const int block = channel_of<VEC, LPR, WARPS>(k0, warp, lane) / kBlock8;
                if (member == q && block < nb) scales[row * nb + block] = s8.scale;
#pragma unroll
                for (int k = k0; k < k0 + kStep; ++k) {
                    const int c = channel_of<VEC, LPR, WARPS>(k, warp, lane);
                    if (c < channels) {
                        uint32_t qv[VEC];
#pragma unroll
                        for (int i = 0; i < VEC; ++i) qv[i] = code8(to_f32<T>(v[r][k * VEC + i]), inv);
                        store_codes<VEC>(codes + row * channels + c, qv);
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + r * kTeams;
            const bool live = row < rows;
            if (!live) continue;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = channel_of<VEC, LPR, WARPS>(k, warp, lane);
                if (c < channels) {
                    float o[VEC], wk[VEC], bk[VEC];
                    w.get(k, c, wk);
                    b.get(k, c, bk);
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        o[i] = fmaf((to_f32<T>(v[r][k * VEC + i]) - mean[r]) * rstd[r], wk[i], bk[i]);
                    store_row<T, VEC>(y + row * channels + c, o);
                }
            }
            if (mean_out != nullptr && lane == 0 && warp == 0) {
                mean_out[row] = mean[r];
                rstd_out[row] = rstd[r];
            }
        }
    }
}

template <typename T, bool HELD8>
struct HeldType { using type = T; };
template <typename T>
struct HeldType<T, true> { using type = int8_t; };

// Threads of the adjoint's block: half as many where a row has one warp, so that
// blocks of 92 registers a thread (16 channels a lane) leave fewer registers over.
template <int WARPS>
constexpr int kBackThreads = WARPS > 1 ? kThreads : 128;

template <typename T, int VEC, int LPR, int NV, int WARPS, bool HELD8>
__global__ void __launch_bounds__(kBackThreads<WARPS>)
norm_backward_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                     const int8_t* __restrict__ codes, const float* __restrict__ scales,
                     const void* __restrict__ weight, int param_dtype,
                     const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                     int64_t rows, int channels, T* __restrict__ dx,
                     float* __restrict__ partial) {
    constexpr int kThreads = kBackThreads<WARPS>;
    __shared__ float2 sh[WARPS > 1 ? WARPS : 1];
    constexpr int kTeams = WARPS > 1 ? 1 : kThreads / LPR;
    const int lane = WARPS > 1 ? threadIdx.x % 32 : threadIdx.x % LPR;
    const int warp = WARPS > 1 ? threadIdx.x / 32 : 0;
    const int team = WARPS > 1 ? 0 : threadIdx.x / LPR;
    const float inv_n = 1.0f / (float)channels;
    const int nb = (channels + kBlock8 - 1) / kBlock8;

    extern __shared__ float dynamic[];  // weight, later a row of sums per warp
    using P = Params<NV * VEC, VEC, WARPS>;
    P w;
    w.sh = dynamic;
    w.channels = channels;
    float dw[NV * VEC], db[NV * VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = channel_of<VEC, LPR, WARPS>(k, warp, lane);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if constexpr (WARPS > 1)
                w.v[k * VEC + i] = (weight != nullptr && c < channels) ? param_at(weight, param_dtype, c + i) : 1.0f;
            dw[k * VEC + i] = db[k * VEC + i] = 0.0f;
        }
    }
    if constexpr (WARPS == 1) {
        for (int c = threadIdx.x; c < channels; c += kThreads)
            dynamic[P::place(c, channels)] = weight != nullptr ? param_at(weight, param_dtype, c) : 1.0f;
        __syncthreads();
    }

    using Held = typename HeldType<T, HELD8>::type;
    constexpr int R = rows_at_once(2 * NV * VEC * (int)sizeof(T));
    const int64_t step = (int64_t)gridDim.x * kTeams * R;
    const int64_t rounds = (rows + step - 1) / step;
    for (int64_t it = 0; it < rounds; ++it) {
        const int64_t row0 = (it * gridDim.x + blockIdx.x) * (kTeams * R) + team;
        T g[R][NV * VEC];
        Held x_raw[R][NV * VEC];
        float mean[R], rstd[R], scale[R][HELD8 ? NV : 1];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + r * kTeams;
            const bool live = row < rows;
            mean[r] = live ? __ldg(mean_in + row) : 0.0f;
            rstd[r] = live ? __ldg(rstd_in + row) : 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = channel_of<VEC, LPR, WARPS>(k, warp, lane);
                if (HELD8) scale[r][HELD8 ? k : 0] = 0.0f;
                if (live && c < channels) {
                    load_raw<T, VEC>(dy + row * channels + c, g[r] + k * VEC);
                    if constexpr (HELD8) {
                        load_codes_raw<VEC>(codes + row * channels + c, x_raw[r] + k * VEC);
                        scale[r][k] = __ldg(scales + row * nb + c / kBlock8);
                    } else {
                        load_raw<T, VEC>(x + row * channels + c, x_raw[r] + k * VEC);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        g[r][k * VEC + i] = from_f32<T>(0.0f);
                        x_raw[r][k * VEC + i] = Held(0.0f);
                    }
                }
            }
        }
        // h of register i (of group k): only used where the row and channel exist
        const auto hat = [&](int r, int k, int i) {
            float v;
            if constexpr (HELD8) v = __fmul_rn((float)x_raw[r][i], scale[r][k]);
            else v = to_f32<T>(x_raw[r][i]);
            return (v - mean[r]) * rstd[r];
        };
        float2 sums[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float sg = 0.0f, sgh = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = channel_of<VEC, LPR, WARPS>(k, warp, lane);
                if (row0 + r * kTeams < rows && c < channels) {
                    float wk[VEC];
                    w.get(k, c, wk);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int i = k * VEC + j;
                        const float h = hat(r, k, i), d = to_f32<T>(g[r][i]);
                        dw[i] = fmaf(d, h, dw[i]);
                        db[i] += d;
                        const float wg = d * wk[j];
                        sg += wg;
                        sgh = fmaf(wg, h, sgh);
                    }
                }
            }
            sums[r] = make_float2(sg, sgh);
        }
        if (dx != nullptr) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t row = row0 + r * kTeams;
                const float2 m = team_sum<LPR, WARPS>(sums[r].x, sums[r].y, sh, warp, lane);
                const float c1 = m.x * inv_n, c2 = m.y * inv_n;
                if (row >= rows) continue;
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int c = channel_of<VEC, LPR, WARPS>(k, warp, lane);
                    if (c < channels) {
                        float o[VEC], wk[VEC];
                        w.get(k, c, wk);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            const int i = k * VEC + j;
                            o[j] = rstd[r] * (to_f32<T>(g[r][i]) * wk[j] - c1 - hat(r, k, i) * c2);
                        }
                        store_row<T, VEC>(dx + row * channels + c, o);
                    }
                }
            }
        }
    }

    if (partial == nullptr) return;
    // lanes of a warp that hold the same channels, then the block's warps
    float* out = partial + (int64_t)blockIdx.x * 2 * channels;
    if constexpr (WARPS == 1) {
        float* join = dynamic;
        const int wid = threadIdx.x / 32;
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i) {
#pragma unroll
            for (int o = LPR; o < 32; o <<= 1) {
                dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
                db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
            }
        }
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
            __syncthreads();
            if (threadIdx.x % 32 < LPR) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int c = channel_of<VEC, LPR, WARPS>(k, warp, lane);
                    if (c < channels) {
#pragma unroll
                        for (int i = 0; i < VEC; ++i)
                            join[wid * channels + c + i] = pass == 0 ? dw[k * VEC + i] : db[k * VEC + i];
                    }
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < channels; c += kThreads) {
                float s = 0.0f;
#pragma unroll
                for (int q = 0; q < kThreads / 32; ++q) s += join[q * channels + c];
                out[pass * channels + c] = s;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = channel_of<VEC, LPR, WARPS>(k, warp, lane);
            if (c < channels) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    out[c + i] = dw[k * VEC + i];
                    out[channels + c + i] = db[k * VEC + i];
                }
            }
        }
    }
}

// ------------------------------------------------------ rows of any length
//
// Rows that do not come in 16-byte vectors (or start off their boundary): where
// it pays (staged() below), chunks of rows staged in shared memory (rows.cuh),
// a team of LPR lanes to a row, and for dw and db a thread to a column.

template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads)
norm_forward_staged_kernel(const T* __restrict__ x, const void* __restrict__ weight,
                           const void* __restrict__ bias, int param_dtype, int64_t rows,
                           int channels, float eps, int chunk, int width, int width_y, int width_codes,
                           T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                           int8_t* __restrict__ codes, float* __restrict__ scales) {
    extern __shared__ __align__(16) uint8_t staged[];
    const int row_bytes = channels * (int)sizeof(T), nb = (channels + kBlock8 - 1) / kBlock8;
    const int buffer = align16(chunk * row_bytes);
    float* w = reinterpret_cast<float*>(staged + 2 * buffer);
    float* b = w + channels;
    float* work = b + channels;  // with codes: chunk * nb floats, then the codes
    int8_t* out8 = reinterpret_cast<int8_t*>(staged + 2 * buffer + align16(4 * (2 * channels + chunk * nb)));
    for (int c = threadIdx.x; c < channels; c += kThreads) {
        w[c] = weight != nullptr ? param_at(weight, param_dtype, c) : 1.0f;
        b[c] = bias != nullptr ? param_at(bias, param_dtype, c) : 0.0f;
    }
    const float inv_n = 1.0f / (float)channels;
    const int64_t chunks = (rows + chunk - 1) / chunk;
    const auto rows_of = [&](int64_t i) { return (int)min((int64_t)chunk, rows - i * chunk); };
    const auto fetch = [&](int64_t i, int q) {
        stage_in(staged + q * buffer, reinterpret_cast<const uint8_t*>(x + i * chunk * channels),
                 rows_of(i) * row_bytes, width);
        stage_commit();
    };
    const int lane = threadIdx.x % LPR, team = threadIdx.x / LPR;
    constexpr int kTeams = kThreads / LPR;
    int q = 0;
    if (blockIdx.x < chunks) fetch(blockIdx.x, 0);
    for (int64_t i = blockIdx.x; i < chunks; i += gridDim.x, q ^= 1) {
        if (i + gridDim.x < chunks) {
            fetch(i + gridDim.x, q ^ 1);
            stage_wait<1>();
        } else {
            stage_wait<0>();
        }
        __syncthreads();
        const int n = rows_of(i);
        T* in = reinterpret_cast<T*>(staged + q * buffer);
        if (codes != nullptr) {
            staged_codes<T, LPR>(in, n, channels, work, out8, scales + i * chunk * nb);
            stage_out(reinterpret_cast<uint8_t*>(codes + i * chunk * channels), reinterpret_cast<uint8_t*>(out8),
                      n * channels, width_codes);
        }
        for (int r0 = 0; r0 < n; r0 += kTeams) {
            const int r = r0 + team, length = r < n ? channels : 0;
            T* row = in + r * channels;
            float s = 0.0f;
            for (int c = lane; c < length; c += LPR) s += to_f32<T>(row[c]);
            const float mean = lanes_sum<LPR>(s) * inv_n;
            float v = 0.0f;
            for (int c = lane; c < length; c += LPR) {
                const float d = to_f32<T>(row[c]) - mean;
                v = fmaf(d, d, v);
            }
            const float rstd = 1.0f / sqrtf(lanes_sum<LPR>(v) * inv_n + eps);
            if (r < n) {
                for (int c = lane; c < channels; c += LPR)
                    row[c] = from_f32<T>(fmaf((to_f32<T>(row[c]) - mean) * rstd, w[c], b[c]));
                if (mean_out != nullptr && lane == 0) {
                    mean_out[i * chunk + r] = mean;
                    rstd_out[i * chunk + r] = rstd;
                }
            }
        }
        __syncthreads();
        stage_out(reinterpret_cast<uint8_t*>(y + i * chunk * channels), staged + q * buffer, n * row_bytes, width_y);
        __syncthreads();
    }
}

constexpr int kColumns = kStageMaxChannels / kThreads;  // of a thread, at most

template <typename T, int LPR, bool HELD8>
__global__ void __launch_bounds__(kThreads)
norm_backward_staged_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                            const int8_t* __restrict__ codes, const float* __restrict__ scales,
                            const void* __restrict__ weight, int param_dtype,
                            const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                            int64_t rows, int channels, int chunk, int width_dy, int width_x, int width_dx,
                            T* __restrict__ dx, float* __restrict__ partial) {
    using Held = typename HeldType<T, HELD8>::type;
    extern __shared__ __align__(16) uint8_t staged[];
    const int row_bytes = channels * (int)sizeof(T), held_bytes = channels * (int)sizeof(Held);
    const int nb = (channels + kBlock8 - 1) / kBlock8;
    const int size_g = align16(chunk * row_bytes), size_x = align16(chunk * held_bytes);
    const int buffer = size_g + size_x;
    float* w = reinterpret_cast<float*>(staged + 2 * buffer);
    float2* stat = reinterpret_cast<float2*>(w + (channels + 1) / 2 * 2);  // mean, rstd of the chunk
    for (int c = threadIdx.x; c < channels; c += kThreads)
        w[c] = weight != nullptr ? param_at(weight, param_dtype, c) : 1.0f;
    const float inv_n = 1.0f / (float)channels;
    const int64_t chunks = (rows + chunk - 1) / chunk;
    const auto rows_of = [&](int64_t i) { return (int)min((int64_t)chunk, rows - i * chunk); };
    const auto fetch = [&](int64_t i, int q) {
        stage_in(staged + q * buffer, reinterpret_cast<const uint8_t*>(dy + i * chunk * channels),
                 rows_of(i) * row_bytes, width_dy);
        const uint8_t* held = HELD8 ? reinterpret_cast<const uint8_t*>(codes + i * chunk * channels)
                                    : reinterpret_cast<const uint8_t*>(x + i * chunk * channels);
        stage_in(staged + q * buffer + size_g, held, rows_of(i) * held_bytes, width_x);
        stage_commit();
    };
    const int lane = threadIdx.x % LPR, team = threadIdx.x / LPR;
    constexpr int kTeams = kThreads / LPR;
    float dw[kColumns] = {}, db[kColumns] = {};
    int q = 0;
    if (blockIdx.x < chunks) fetch(blockIdx.x, 0);
    for (int64_t i = blockIdx.x; i < chunks; i += gridDim.x, q ^= 1) {
        const int n = rows_of(i);
        for (int r = threadIdx.x; r < n; r += kThreads)
            stat[r] = make_float2(__ldg(mean_in + i * chunk + r), __ldg(rstd_in + i * chunk + r));
        if (i + gridDim.x < chunks) {
            fetch(i + gridDim.x, q ^ 1);
            stage_wait<1>();
        } else {
            stage_wait<0>();
        }
        __syncthreads();
        T* g = reinterpret_cast<T*>(staged + q * buffer);
        const Held* h = reinterpret_cast<const Held*>(staged + q * buffer + size_g);
        const float* sc = HELD8 ? scales + i * chunk * nb : nullptr;
        const auto hat = [&](int r, int c, float2 st) {
            float v;
            if constexpr (HELD8) v = __fmul_rn((float)h[r * channels + c], __ldg(sc + r * nb + c / kBlock8));
            else v = to_f32<T>(h[r * channels + c]);
            return (v - st.x) * st.y;
        };
        if (partial != nullptr) {
#pragma unroll 4
            for (int r = 0; r < n; ++r) {
                const float2 st = stat[r];
#pragma unroll
                for (int k = 0; k < kColumns; ++k) {
                    const int c = threadIdx.x + k * kThreads;
                    if (c < channels) {
                        const float d = to_f32<T>(g[r * channels + c]);
                        dw[k] = fmaf(d, hat(r, c, st), dw[k]);
                        db[k] += d;
                    }
                }
            }
        }
        __syncthreads();
        if (dx != nullptr) {
            for (int r0 = 0; r0 < n; r0 += kTeams) {
                const int r = r0 + team;
                float sg = 0.0f, sgh = 0.0f;
                if (r < n) {
                    const float2 st = stat[r];
                    for (int c = lane; c < channels; c += LPR) {
                        const float wg = to_f32<T>(g[r * channels + c]) * w[c];
                        sg += wg;
                        sgh = fmaf(wg, hat(r, c, st), sgh);
                    }
                }
                const float c1 = lanes_sum<LPR>(sg) * inv_n, c2 = lanes_sum<LPR>(sgh) * inv_n;
                if (r < n) {
                    const float2 st = stat[r];
                    for (int c = lane; c < channels; c += LPR)
                        g[r * channels + c] = from_f32<T>(
                            st.y * (to_f32<T>(g[r * channels + c]) * w[c] - c1 - hat(r, c, st) * c2));
                }
            }
            __syncthreads();
            stage_out(reinterpret_cast<uint8_t*>(dx + i * chunk * channels), staged + q * buffer, n * row_bytes,
                      width_dx);
        }
        __syncthreads();
    }
    if (partial == nullptr) return;
    float* out = partial + (int64_t)blockIdx.x * 2 * channels;
#pragma unroll
    for (int k = 0; k < kColumns; ++k) {
        const int c = threadIdx.x + k * kThreads;
        if (c < channels) {
            out[c] = dw[k];
            out[channels + c] = db[k];
        }
    }
}

// Column sums of the blocks' partial rows: 32 columns and 32 row groups to a
// block; columns [0, channels) are dw, the rest db.
__global__ void __launch_bounds__(1024)
norm_join_kernel(const float* __restrict__ partial, int blocks, int channels, int param_dtype,
                 void* __restrict__ dweight, void* __restrict__ dbias) {
    __shared__ float sh[32][33];
    const int col = blockIdx.x * 32 + threadIdx.x;
    float s = 0.0f;
    if (col < 2 * channels) {
#pragma unroll 4
        for (int r = threadIdx.y; r < blocks; r += 32) s += partial[(int64_t)r * 2 * channels + col];
    }
    sh[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = lanes_sum<32>(sh[threadIdx.x][threadIdx.y]);
    const int c = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x != 0 || c >= 2 * channels) return;
    void* dst = c < channels ? dweight : dbias;
    if (dst == nullptr) return;
    const int i = c < channels ? c : c - channels;
    if (param_dtype == MG_F32) static_cast<float*>(dst)[i] = s;
    else if (param_dtype == MG_BF16) static_cast<__nv_bfloat16*>(dst)[i] = from_f32<__nv_bfloat16>(s);
    else static_cast<__half*>(dst)[i] = from_f32<__half>(s);
}

// Blocks of the adjoint: enough to fill the device, few enough that the join
// stays short. Depends on the sizes only, so scratch and launch agree.
int64_t backward_blocks(int64_t rows, int64_t channels) {
    const int64_t teams = channels > 1024 ? 1 : std::max<int64_t>(4, 128 / std::max<int64_t>(1, channels));
    const int64_t want = (rows + teams - 1) / teams;
    return std::max<int64_t>(1, std::min<int64_t>(want, (channels > 1024 ? 4 : 8) * (int64_t)sm_count()));
}

// Blocks of a kernel that an SM holds, asked once per device, with the shared
// memory of the kernel's longest rows: the grid, and with it the order of the
// adjoint's sums, depends on a call's own sizes and not on those of the first.
template <typename K>
int blocks_per_sm(K kernel, size_t smem, int (&known)[64], int threads = kThreads) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 2;
    if (known[dev] == 0) {
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) n = 1;
        known[dev] = n;
    }
    return known[dev];
}

struct Forward {
    const void *x, *weight, *bias;
    int param_dtype;
    int64_t rows;
    int channels;
    float eps;
    void* y;
    float *mean, *rstd;
    int8_t* codes;
    float* scales;
    cudaStream_t st;

    template <typename T, int VEC, int LPR, int NV, int WARPS>
    mg_status run() const {
        constexpr int kTeams = WARPS > 1 ? 1 : kThreads / LPR;
        // one wave of blocks that stay: each reads the parameters once
        const int64_t want = (rows + kTeams - 1) / kTeams;
        const size_t smem = WARPS == 1 ? sizeof(float) * 2 * (size_t)channels : 0;
        constexpr size_t most = WARPS == 1 ? sizeof(float) * 2 * VEC * LPR * NV : 0;
        static int known[64] = {};
        const int per_sm = blocks_per_sm(norm_forward_kernel<T, VEC, LPR, NV, WARPS>, most, known);
        const int grid = (int)std::min<int64_t>(want, per_sm * (int64_t)sm_count());
        norm_forward_kernel<T, VEC, LPR, NV, WARPS><<<grid, kThreads, smem, st>>>(
            static_cast<const T*>(x), weight, bias, param_dtype, rows, channels, eps,
            static_cast<T*>(y), mean, rstd, codes, scales);
        return check_launch("layer_norm_forward");
    }
};

struct Backward {
    const void *dy, *x;
    const int8_t* codes;
    const float* scales;
    const void* weight;
    int param_dtype;
    const float *mean, *rstd;
    int64_t rows;
    int channels;
    void* dx;
    float* partial;
    int max_grid;
    int* used;  // the grid that ran: rows of partial
    cudaStream_t st;

    template <typename T, int VEC, int LPR, int NV, int WARPS>
    mg_status run() const {
        const size_t smem = WARPS == 1 ? sizeof(float) * (kBackThreads<1> / 32) * (size_t)channels : 0;
        constexpr size_t most = WARPS == 1 ? sizeof(float) * (kBackThreads<1> / 32) * VEC * LPR * NV : 0;
        constexpr int threads = kBackThreads<WARPS>;
        static int known[2][64] = {};
        const int per_sm = codes != nullptr
                               ? blocks_per_sm(norm_backward_kernel<T, VEC, LPR, NV, WARPS, true>, most, known[0], threads)
                               : blocks_per_sm(norm_backward_kernel<T, VEC, LPR, NV, WARPS, false>, most, known[1], threads);
        const int grid = std::min(max_grid, per_sm * sm_count());
        *used = grid;
        if (codes != nullptr)
            norm_backward_kernel<T, VEC, LPR, NV, WARPS, true><<<grid, threads, smem, st>>>(
                static_cast<const T*>(dy), nullptr, codes, scales, weight, param_dtype, mean, rstd,
                rows, channels, static_cast<T*>(dx), partial);
        else
            norm_backward_kernel<T, VEC, LPR, NV, WARPS, false><<<grid, threads, smem, st>>>(
                static_cast<const T*>(dy), static_cast<const T*>(x), nullptr, nullptr, weight,
                param_dtype, mean, rstd, rows, channels, static_cast<T*>(dx), partial);
        return check_launch("layer_norm_backward");
    }
};

template <typename T, int LPR>
mg_status forward_staged(const Forward& f) {
    const int chunk = stage_rows(f.channels, (int)sizeof(T)), nb = blocks8(f.channels);
    const int bytes = chunk * f.channels * (int)sizeof(T);
    int smem = 2 * align16(bytes) + align16(4 * (2 * f.channels + chunk * nb));
    if (f.codes != nullptr) smem += align16(chunk * f.channels);
    static int known[64] = {};
    int per_sm = 0;
    MG_TRY(staged_launch(norm_forward_staged_kernel<T, LPR>, kThreads, smem, known, &per_sm, "layer_norm_forward"));
    const int grid = (int)std::min<int64_t>((f.rows + chunk - 1) / chunk, per_sm * (int64_t)sm_count());
    norm_forward_staged_kernel<T, LPR><<<grid, kThreads, smem, f.st>>>(
        static_cast<const T*>(f.x), f.weight, f.bias, f.param_dtype, f.rows, f.channels, f.eps, chunk,
        stage_width(f.x, bytes), stage_width(f.y, bytes), stage_width(f.codes, chunk * f.channels),
        static_cast<T*>(f.y), f.mean, f.rstd, f.codes, f.scales);
    return check_launch("layer_norm_forward");
}

template <typename T, int LPR, bool HELD8>
mg_status backward_staged(const Backward& f) {
    const int chunk = stage_rows(f.channels, (int)sizeof(T));
    const int bytes = chunk * f.channels * (int)sizeof(T);
    const int held = HELD8 ? chunk * f.channels : bytes;
    const int smem = 2 * (align16(bytes) + align16(held)) + 4 * (f.channels + 1) + 8 * chunk;
    static int known[64] = {};
    int per_sm = 0;
    MG_TRY(staged_launch(norm_backward_staged_kernel<T, LPR, HELD8>, kThreads, smem, known, &per_sm, "layer_norm_backward"));
    const int grid = (int)std::min<int64_t>((f.rows + chunk - 1) / chunk,
                                            std::min(f.max_grid, per_sm * sm_count()));
    *f.used = grid;
    norm_backward_staged_kernel<T, LPR, HELD8><<<grid, kThreads, smem, f.st>>>(
        static_cast<const T*>(f.dy), static_cast<const T*>(f.x), f.codes, f.scales, f.weight, f.param_dtype,
        f.mean, f.rstd, f.rows, f.channels, chunk, stage_width(f.dy, bytes),
        HELD8 ? stage_width(f.codes, held) : stage_width(f.x, bytes), stage_width(f.dx, bytes),
        static_cast<T*>(f.dx), f.partial);
    return check_launch("layer_norm_backward");
}

// Staged chunks or single elements by row: us staged/by elements, 2^25 elements
// in all, fp32 and fp16 ("8": with the 8-bit form):
//   channels  forward           forward 8          adjoint           adjoint 8
//   19        117/285  115/305  195/354  197/371
//   77         84/82    76/156  135/139  127/180
//   129        98/74    86/131  168/113  156/180
//   201        78/59    70/115  129/80   125/147
//   301        74/59    66/127  125/82   113/150   130/108  114/98   170/173  156/163
//   511        68/49    61/119  111/57   100/133   119/100  106/88   149/139  141/140
//   601        63/59    55/135  104/78   100/154   129/118   98/119  141/440  137/313
//   1001       63/49    57/135  115/61    98/147   176/102   96/106  178/322  131/264
// Forward: staged up to 128 channels and above 512. 16-bit rows would gain from
// it between those too; fp32 rows above 512 would do without. The adjoint: staged
// above 512, for the rows held in 8 bits and the 16-bit ones; fp32 rows held in
// full lose up to 70 us by it.
template <typename T>
bool staged(const Forward& f, mg_status* s) {
    if (f.channels > kStageMaxChannels || (f.channels > kBlock8 && f.channels <= 512)) return false;
    *s = f.channels <= 32 ? forward_staged<T, 8>(f)
         : f.channels <= kBlock8 ? forward_staged<T, 16>(f) : forward_staged<T, 32>(f);
    return true;
}
template <typename T>
bool staged(const Backward& f, mg_status* s) {
    if (f.channels <= 512 || f.channels > kStageMaxChannels) return false;
    *s = f.codes != nullptr ? backward_staged<T, 32, true>(f) : backward_staged<T, 32, false>(f);
    return true;
}

// The team for a row length: the fewest lanes that hold the row with one
// vector each, then more vectors per lane, then a block.
template <typename T, int VEC, typename Op>
mg_status pick_team(const Op& op, int channels) {
    const int vecs = (channels + VEC - 1) / VEC;
    if (vecs <= 4) return op.template run<T, VEC, 4, 1, 1>();
    if (vecs <= 8) return op.template run<T, VEC, 8, 1, 1>();
    if (vecs <= 16) return op.template run<T, VEC, 16, 1, 1>();
    if (vecs <= 32) return op.template run<T, VEC, 32, 1, 1>();
    if (vecs <= 64) return op.template run<T, VEC, 32, 2, 1>();
    if (vecs <= 128) return op.template run<T, VEC, 32, 4, 1>();
    if constexpr (VEC <= 4) {
        if (vecs <= 256) return op.template run<T, VEC, 32, 8, 1>();
    }
    if constexpr (VEC == 1) {
        if (vecs <= 512) return op.template run<T, VEC, 32, 16, 1>();
        if (vecs <= 1024) return op.template run<T, VEC, 32, 32, 1>();
        if (vecs <= 4096) return op.template run<T, VEC, 32, 16, 8>();
        return op.template run<T, VEC, 32, 32, 8>();
    } else {
        if (vecs <= 512) return op.template run<T, VEC, 32, 2, 8>();
        if (VEC == 8 || vecs <= 1024) return op.template run<T, VEC, 32, 4, 8>();
        return op.template run<T, VEC, 32, VEC == 8 ? 4 : 8, 8>();
    }
}

// Whole vectors, staged chunks, or single elements.
template <typename T, int VEC, typename Op>
mg_status pick_path(const Op& op, int channels, bool aligned) {
    if (aligned && channels % VEC == 0) return pick_team<T, VEC>(op, channels);
    mg_status s = MG_OK;
    return staged<T>(op, &s) ? s : pick_team<T, 1>(op, channels);
}

template <typename Op>
mg_status pick_type(const Op& op, int dtype, int channels, bool aligned) {
    if (dtype == MG_F32) return pick_path<float, 4>(op, channels, aligned);
    if (dtype == MG_BF16) return pick_path<__nv_bfloat16, 8>(op, channels, aligned);
    return pick_path<__half, 8>(op, channels, aligned);
}

bool known_dtype(int d) { return d == MG_F32 || d == MG_BF16 || d == MG_F16; }

}  // namespace

int sm_count() {
    static int cached[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (cached[dev] == 0) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1)
            n = 148;
        cached[dev] = n;
    }
    return cached[dev];
}

}  // namespace mg

using namespace mg;

extern "C" mg_status mg_layer_norm_forward(const void* x, int32_t dtype, const void* weight,
                                           const void* bias, int32_t param_dtype, int64_t rows,
                                           int64_t channels, float eps, void* y, float* mean,
                                           float* rstd, int8_t* codes, float* scales,
                                           mg_stream_t stream) try {
    MG_REQUIRE(known_dtype(dtype) && known_dtype(param_dtype), "layer_norm_forward: unknown dtype");
    MG_REQUIRE(rows >= 0, "layer_norm_forward: negative row count");
    MG_REQUIRE(channels >= 1 && channels <= MG_LAYER_NORM_MAX_CHANNELS,
               "layer_norm_forward: channels must be 1..8192");
    MG_REQUIRE(eps >= 0.0f, "layer_norm_forward: eps must not be negative");
    MG_REQUIRE((mean == nullptr) == (rstd == nullptr) && (codes == nullptr) == (scales == nullptr),
               "layer_norm_forward: mean comes with rstd, codes with scales");
    if (rows == 0) return MG_OK;
    MG_REQUIRE(x && y, "layer_norm_forward: null pointer");
    MG_REQUIRE(codes == nullptr || (reinterpret_cast<uintptr_t>(codes) & 7u) == 0u,
               "layer_norm_forward: codes must be 8-byte aligned");
    MG_REQUIRE(on_boundary(elem_bytes(dtype), {x, y}) && on_boundary(elem_bytes(param_dtype), {weight, bias}) &&
                   on_boundary(4, {mean, rstd, scales}),
               "layer_norm_forward: a pointer off its element's boundary");
    const Forward op{x, weight, bias, param_dtype, rows, (int)channels, eps, y, mean, rstd,
                     codes, scales, reinterpret_cast<cudaStream_t>(stream)};
    return pick_type(op, dtype, (int)channels, aligned16(x) && aligned16(y));
} catch (...) {
    return caught("layer_norm_forward");
}

extern "C" size_t mg_layer_norm_backward_scratch_bytes(int64_t rows, int64_t channels) {
    if (rows <= 0 || channels <= 0 || channels > MG_LAYER_NORM_MAX_CHANNELS) return 0;
    return sizeof(float) * 2 * (size_t)channels * (size_t)backward_blocks(rows, channels);
}

extern "C" mg_status mg_layer_norm_backward(const void* dy, const void* x, const int8_t* codes,
                                            const float* scales, int32_t dtype, const void* weight,
                                            int32_t param_dtype, const float* mean,
                                            const float* rstd, int64_t rows, int64_t channels,
                                            void* dx, void* dweight, void* dbias, void* scratch,
                                            size_t scratch_bytes, mg_stream_t stream) try {
    MG_REQUIRE(known_dtype(dtype) && known_dtype(param_dtype), "layer_norm_backward: unknown dtype");
    MG_REQUIRE(rows >= 0, "layer_norm_backward: negative row count");
    MG_REQUIRE(channels >= 1 && channels <= MG_LAYER_NORM_MAX_CHANNELS,
               "layer_norm_backward: channels must be 1..8192");
    MG_REQUIRE((x == nullptr) != (codes == nullptr) || rows == 0,
               "layer_norm_backward: give x or its 8-bit form");
    MG_REQUIRE((codes == nullptr) == (scales == nullptr),
               "layer_norm_backward: codes come with scales");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool params = dweight != nullptr || dbias != nullptr;
    if (rows == 0) {
        const size_t bytes = (size_t)channels * (param_dtype == MG_F32 ? 4 : 2);
        if (dweight && cudaMemsetAsync(dweight, 0, bytes, st) != cudaSuccess)
            return check_launch("layer_norm_backward memset");
        if (dbias && cudaMemsetAsync(dbias, 0, bytes, st) != cudaSuccess)
            return check_launch("layer_norm_backward memset");
        return MG_OK;
    }
    if (!params && dx == nullptr) return MG_OK;
    MG_REQUIRE(dy && mean && rstd, "layer_norm_backward: null pointer");
    MG_REQUIRE(codes == nullptr || (reinterpret_cast<uintptr_t>(codes) & 7u) == 0u,
               "layer_norm_backward: codes must be 8-byte aligned");
    MG_REQUIRE(on_boundary(elem_bytes(dtype), {dy, x, dx}) && on_boundary(4, {mean, rstd, scales, scratch}) &&
                   on_boundary(elem_bytes(param_dtype), {weight, dweight, dbias}),
               "layer_norm_backward: a pointer off its element's boundary");
    MG_REQUIRE(!params || (scratch != nullptr &&
                           scratch_bytes >= mg_layer_norm_backward_scratch_bytes(rows, channels)),
               "layer_norm_backward: scratch too small");
    int grid = 0;
    const Backward op{dy, x, codes, scales, weight, param_dtype, mean, rstd, rows, (int)channels,
                      dx, params ? static_cast<float*>(scratch) : nullptr, (int)backward_blocks(rows, channels), &grid, st};
    MG_TRY(pick_type(op, dtype, (int)channels,
                     aligned16(dy) && (x == nullptr || aligned16(x)) && (dx == nullptr || aligned16(dx))));
    if (!params) return MG_OK;
    norm_join_kernel<<<ceil_div(2 * channels, 32), dim3(32, 32), 0, st>>>(
        static_cast<const float*>(scratch), grid, (int)channels, param_dtype, dweight, dbias);
    return check_launch("layer_norm_backward join");
} catch (...) {
    return caught("layer_norm_backward");
}
