// The label loss's gradients with the logits' gradient never leaving the SM.
//
// A unit owns 128 items of one side (rows for dx, classes for dw) and a share
// of the other side, which streams past in tiles of 64:
//   S = own . stream^T       128 x 64, fp32 in tensor memory
//   G = r (softmax - onehot) from S by one of four groups of four warps, back
//       into tensor memory as bf16 parts
//   acc += G stream          128 x channels, G the A operand from tensor memory
// One streamed tile in shared memory serves both products: its channels are
// the contraction of the first and the columns of the second.
//
// Its floors: one exponential per logit (16 a clock and SM, 512 cycles a tile)
// while there are few channels, the tensor cores above (a product of 128 x 64 x 16
// takes 48 cycles with both operands in shared memory, which is what reading them
// takes; 32 with one in tensor memory). It reaches neither: a group's turn
// (scores, G, hand-over, next scores) is a chain that is waited for. Measured, in
// cycles a tile at 18944 x 4096 (rows, classes): bf16 1230 and 1290 (dx, dw) at
// 16 channels, 1360 and 1630 at 64; fp32 1730 and 1830 at 16 (exponentials 34 and
// 37 % of their rate, tensor cores 25 and 28 %), 2750 and 3040 at 64, 6000 and 6790
// at 128 (tensor cores 56 %), where only two streamed tiles fit. The logits are
// computed twice in all (dx and dw), which costs less than 2 x PARTS bytes a
// logit of G written and read twice: loss and gradients of 640000 x 16 x 256 fp32
// take 430 us in all (153 + 117 of them here) against 990 with G through scratch,
// 100003 x 77 x 4099 2240 against 2900, 640000 x 32 x 128 with its head 645 against
// 875.
// acc leaves tensor memory for the registers of eight more warps every
// `per_segment` tiles: the tensor cores' fp32 additions truncate, and fp32
// results keep their precision only over short runs of them.
#pragma once

#include "labels.cuh"

namespace mg {

namespace {

constexpr int kOwn = 128;
constexpr int kStream = 64;
constexpr int kGroups = 4;          // of four warps that turn scores into G
// copy, issue scores, issue G products, (none); the groups; 8 warps for acc
constexpr int kFusedThreads = 128 * (1 + kGroups + 2);
// Registers a thread: 72 at launch, and the issuing warps keep them; the groups
// give up 8 each for the acc warps' 16 more: 72 + 4 * 64 + 2 * 88 = 7 * 72. (Other
// splits, 40 to 120 for the issuing warps, measured level or worse.)
constexpr int kIssueRegs = 72, kScoreRegs = 64, kAccRegs = 88;
constexpr int kFusedStages = 8;     // at most
constexpr int kFusedShared = 226 * 1024;  // of it 1 KB to align

struct FusedArgs {         // counts below 2^31: at most 2^30 rows
    int units;
    int copied;            // units whose tiles are copied in: all, but for the self-test
    int rounds;            // of the issuing and copying warps' waits, at most
    int own;               // items of the owning side
    int streamed;          // items of the streaming side
    int per_split;         // tiles of a share
    int splits;
    int per_segment;
    int channels;
    int chunks;            // of 64 channels
    int stages, own_buffers, acc_buffers;
    int resident;          // the streamed tiles, all the same for every unit, stay: one stage each
    float scale;
    const float* row_values;   // kRowValues per row, in blocks of 64 rows
    const float* class_bias;   // bias times log2 e, -infinity past the last class
    float* part_bias;      // by class: (splits, kGroups, classes), or NULL
    float* part;           // fp32 shares (splits, own, part_ld), or NULL
    int part_ld;
    void* out;             // the result itself
    int32_t* error_word;
};

static_assert(kStream == kRowBlock, "a streamed tile is a block of row values");
constexpr int kColumnBytes = kRowValues * kStream * 4;  // of a streamed tile, beside its parts

struct FusedWalk {
    int own0, t0, t1, split;
};

template <int N>
__device__ __forceinline__ void registers_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// Tensor memory of a group: 64 columns of scores, in which G's first two parts
// take the place of the scores they came from (16 entries of a part are 8
// columns: part i of entries [16 s, 16 s + 16) at 16 s + 8 i), and 32 columns
// for a third part.
template <int PARTS>
constexpr int kGroupColumns = kStream + (PARTS == 3 ? kStream / 2 : 0);
__device__ __forceinline__ constexpr int g_column(int part, int entry) {
    return part < 2 ? entry + 8 * part : kStream + entry / 2;
}

__device__ __forceinline__ FusedWalk fused_unit(const FusedArgs& p, int u) {
    FusedWalk w;
    w.own0 = u / p.splits * kOwn;
    w.split = u % p.splits;
    w.t0 = w.split * p.per_split;
    w.t1 = min((p.streamed + kStream - 1) / kStream, w.t0 + p.per_split);
    return w;
}

__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
        : "memory");
}
__device__ __forceinline__ void tmem_store_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// `bytes` (a multiple of 16) from global to shared memory.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar, uint32_t on) {
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.u32 q, %4, 0;\n"
        "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n}" ::"r"(dst),
        "l"(src), "r"(bytes), "r"(bar), "r"(on)
        : "memory");
}
__device__ __forceinline__ float4 shared_float4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr));
    return v;
}
__device__ __forceinline__ int shared_int(uint32_t addr) {
    int v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

// kStep values as GP parts, two to a word.
constexpr int kStep = 16;
template <int GP>
__device__ __forceinline__ void store_parts(uint32_t group, int k, float (&z)[kStep]) {
#pragma unroll
    for (int i = 0; i < GP; ++i) {
        uint32_t r[kStep / 2];
#pragma unroll
        for (int j = 0; j < kStep / 2; ++j) {
            if (i + 1 < GP) r[j] = take_part(z[2 * j], z[2 * j + 1]);
            else r[j] = pack_bf16(z[2 * j], z[2 * j + 1]);
        }
        tmem_store(group + g_column(i, k), r);
    }
}

// Four sums of products to r softmax: logits in base 2 (scale, bias), minus the
// log of the row's sum, exponential, times r.
__device__ __forceinline__ void gradients(float* z, float c2, float2 bias0, float2 bias1, float2 minus_lse0,
                                          float2 minus_lse1, float2 r0, float2 r1) {
    const float2 a = add2(fma2(make_float2(z[0], z[1]), both(c2), bias0), minus_lse0);
    const float2 b = add2(fma2(make_float2(z[2], z[3]), both(c2), bias1), minus_lse1);
    const float2 e = mul2(make_float2(exp2_fast(a.x), exp2_fast(a.y)), r0);
    const float2 f = mul2(make_float2(exp2_fast(b.x), exp2_fast(b.y)), r1);
    z[0] = e.x;
    z[1] = e.y;
    z[2] = f.x;
    z[3] = f.y;
}

template <bool BY_CLASS, int PARTS>
__global__ void __launch_bounds__(kFusedThreads, 1)
fused_kernel(const __grid_constant__ FusedArgs p, const __grid_constant__ CUtensorMap map_own,
             const __grid_constant__ CUtensorMap map_stream) {
    constexpr int GP = kGParts<PARTS>;
    constexpr int kScorePairs = PARTS == 1 ? 1 : PARTS == 2 ? 4 : 6;
    constexpr int kOwnChunk = kOwn * 128, kStreamChunk = kStream * 128;  // 64 channels, bytes
    constexpr uint32_t kAccBase = kGroups * kGroupColumns<PARTS>;
    extern __shared__ uint8_t dynamic[];
    __shared__ uint64_t bars[2 * kFusedStages + 3 * kGroups + 10];
    __shared__ uint32_t tmem_s;
    __shared__ volatile int stop;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t base = (smem_u32(dynamic) + 1023u) & ~1023u;
    const uint32_t own_bytes = PARTS * p.chunks * kOwnChunk;
    const uint32_t tile_bytes = PARTS * p.chunks * kStreamChunk;
    const uint32_t stage_bytes = tile_bytes + kColumnBytes;  // parts, then the columns' values
    constexpr uint32_t column_bytes = BY_CLASS ? kColumnBytes : kStream * 4;
    const uint32_t stream0 = base + p.own_buffers * own_bytes;
    const uint32_t full = smem_u32(bars), empty = full + 8 * kFusedStages;
    const uint32_t own_full = empty + 8 * kFusedStages, own_empty = own_full + 16;
    const uint32_t s_full = own_empty + 16, g_full = s_full + 8 * kGroups;
    const uint32_t g_empty = g_full + 8 * kGroups;
    const uint32_t acc_full = g_empty + 8 * kGroups, acc_empty = acc_full + 16;
    const uint32_t drain = acc_empty + 16;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kFusedStages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(own_full + 8 * i, 1);
            mbar_init(own_empty + 8 * i, 1);
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, 8);
        }
        for (int i = 0; i < kGroups; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(g_full + 8 * i, 4);
            mbar_init(g_empty + 8 * i, 1);
        }
        mbar_init(drain, 1);
        mbar_init(drain + 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_shared();
        stop = 0;
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_s), kTmemColumns);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    constexpr uint32_t tmem = kTmemBase;
    // tiles that stay are waited for in their one and only phase
    const uint32_t flip = p.resident ? 0 : 1;
    const auto wait = [&](uint32_t bar, uint32_t parity) {
        return mbar_wait(bar, parity, kMbarRounds, &stop, p.error_word, DEV_ERR_TILE_WAIT);
    };

    const auto wait_warp = [&](uint32_t bar, uint32_t parity) {
        return mbar_wait_warp(bar, parity, p.rounds, &stop, p.error_word, DEV_ERR_TILE_WAIT);
    };

    // For the end of every warp: once all are past their last wait `stop` changes
    // no more, and what is in flight then is drained or has been waited for.
    const auto gave_up = [&] {
        named_sync(1, kFusedThreads);
        return stop != 0;
    };

    if (warp >= 4 + 4 * kGroups) registers_up<kAccRegs>();
    else if (warp >= 4) registers_down<kScoreRegs>();

    if (warp == 0) {
        // copies tiles in
        const uint32_t on = elect_lane();
        int stage = 0, ob = 0;
        uint32_t phase = 0, ob_phase = 0;
        int issued = 0, owns = 0;  // of the last ring, for a stop
        bool ok = true;
        for (int u = blockIdx.x; ok && u < p.copied; u += gridDim.x) {
            const FusedWalk w = fused_unit(p, u);
            ok = wait_warp(own_empty + 8 * ob, ob_phase ^ 1);
            if (!ok) break;
            mbar_expect(own_full + 8 * ob, own_bytes, on);
            for (int i = 0; i < PARTS; ++i)
                for (int c = 0; c < p.chunks; ++c)
                    tma_load(base + ob * own_bytes + (i * p.chunks + c) * kOwnChunk, &map_own,
                             c * 64, w.own0, i, own_full + 8 * ob, on);
            owns = min(owns + 1, p.own_buffers);
            if (++ob == p.own_buffers) {
                ob = 0;
                ob_phase ^= 1;
            }
            if (p.resident && u != (int)blockIdx.x) continue;
            for (int t = w.t0; t < w.t1; ++t) {
                ok = wait_warp(empty + 8 * stage, phase ^ 1);
                if (!ok) break;
                mbar_expect(full + 8 * stage, tile_bytes + column_bytes, on);
                bulk_load(stream0 + stage * stage_bytes + tile_bytes,
                          (BY_CLASS ? p.row_values : p.class_bias) + (int64_t)t * (column_bytes / 4), column_bytes,
                          full + 8 * stage, on);
                for (int i = 0; i < PARTS; ++i)
                    for (int c = 0; c < p.chunks; ++c)
                        tma_load(stream0 + stage * stage_bytes + (i * p.chunks + c) * kStreamChunk,
                                 &map_stream, c * 64, t * kStream, i, full + 8 * stage, on);
                issued = min(issued + 1, p.stages);
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        if (gave_up()) {  // its copies in flight land before the block ends
            for (int j = issued; j > 0; --j) {
                if (--stage < 0) {
                    stage = p.stages - 1;
                    phase ^= 1;
                }
                for (int i = 0; i < kMbarRounds; ++i)
                    if (mbar_try(full + 8 * stage, phase)) break;
            }
            for (int j = owns; j > 0; --j) {
                if (--ob < 0) {
                    ob = p.own_buffers - 1;
                    ob_phase ^= 1;
                }
                for (int i = 0; i < kMbarRounds; ++i)
                    if (mbar_try(own_full + 8 * ob, ob_phase)) break;
            }
        }
    } else if (warp == 1) {
        // Issues the scores. They run ahead of the G products, which have a warp
        // of their own: one issuing warp for both was what a tile of few channels
        // took (1750 cycles a tile, bf16).
        const uint32_t on = elect_lane();
        const uint32_t idesc = mma_idesc(kStream, false, false);
        const uint32_t a_part = uniform(p.chunks * kOwnChunk / 16);
        const uint32_t b_part = uniform(p.chunks * kStreamChunk / 16);
        const int steps = (int)uniform((uint32_t)(p.channels + 15) / 16);
        int stage = 0, ob = 0, g = 0;
        uint32_t phase = 0, ob_phase = 0, g_phase = 0;
        bool ok = true;
        for (int u = blockIdx.x; ok && u < p.units; u += gridDim.x) {
            const FusedWalk w = fused_unit(p, u);
            const int tiles = (int)uniform((uint32_t)(w.t1 - w.t0));
            ok = wait_warp(own_full + 8 * ob, ob_phase);
            const uint32_t a0 = uniform(k_major_lo(base + ob * own_bytes));
            for (int t = 0; ok && t < tiles; ++t) {
                ok = wait_warp(full + 8 * stage, phase) && wait_warp(g_empty + 8 * g, g_phase ^ 1);
                if (!ok) break;
                tmem_fence_after();
                const uint32_t b0 = uniform(k_major_lo(stream0 + stage * stage_bytes));
                const uint32_t d = uniform(tmem + g * kGroupColumns<PARTS>);
                // the small products first: the tensor cores truncate the running
                // sum at each step, and only the large ones' steps weigh
                if (steps <= 4) {  // 16 channels each, of one chunk: no loop to run
#pragma unroll
                    for (int q = 0; q < kScorePairs; ++q) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k < steps)
                                mma_bf16<k_major_hi(128), k_major_hi(128)>(
                                    d, a0 + pair_a<PARTS>(kScorePairs, q) * a_part + 2 * k,
                                    b0 + pair_b<PARTS>(kScorePairs, q) * b_part + 2 * k, idesc,
                                    q > 0 || k > 0, on);
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < kScorePairs; ++q) {
                        uint32_t a = uniform(a0 + pair_a<PARTS>(kScorePairs, q) * a_part);
                        uint32_t b = uniform(b0 + pair_b<PARTS>(kScorePairs, q) * b_part);
                        for (int k = 0; k < steps; ++k) {
                            mma_bf16<k_major_hi(128), k_major_hi(128)>(d, a, b, idesc, q > 0 ? true : k > 0, on);
                            a += (k & 3) == 3 ? kOwnChunk / 16 - 6 : 2;
                            b += (k & 3) == 3 ? kStreamChunk / 16 - 6 : 2;
                        }
                    }
                }
                mma_commit(s_full + 8 * g, on);
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= flip;
                }
                if (++g == kGroups) {
                    g = 0;
                    g_phase ^= 1;
                }
            }
            mma_commit(own_empty + 8 * ob, on);
            if (++ob == p.own_buffers) {
                ob = 0;
                ob_phase ^= 1;
            }
        }
        if (gave_up()) {
            mma_commit(drain, on);
            for (int k = 0; k < kMbarRounds; ++k)
                if (mbar_try(drain, 0)) break;
        }
    } else if (warp == 2) {
        // issues the G products
        const uint32_t on = elect_lane();
        const int n = (p.channels + 15) / 16 * 16;
        const uint32_t idesc = uniform(mma_idesc(n, false, true));
        const uint32_t part = uniform(p.chunks * kStreamChunk / 16);
        int stage = 0, ab = 0, g = 0;
        uint32_t g_phase = 0, ab_phase = 0;
        bool ok = true;
        for (int u = blockIdx.x; ok && u < p.units; u += gridDim.x) {
            const FusedWalk w = fused_unit(p, u);
            const int tiles = (int)uniform((uint32_t)(w.t1 - w.t0));
            int in_segment = 0;  // G products in acc
            for (int t = 0; ok && t < tiles; ++t) {
                ok = wait_warp(g_full + 8 * g, g_phase);
                if (ok && in_segment == 0) ok = wait_warp(acc_empty + 8 * ab, ab_phase ^ 1);
                if (!ok) break;
                tmem_fence_after();
                const uint32_t d = uniform(tmem + kAccBase + ab * n);
                const uint32_t a0 = uniform(tmem + g * kGroupColumns<PARTS>);
                const uint32_t b0 = uniform(mn_major_lo(stream0 + stage * stage_bytes, kStreamChunk));
#pragma unroll
                for (int q = 0; q < kGPairs<PARTS>; ++q) {
#pragma unroll
                    for (int s = 0; s < kStream / 16; ++s)
                        mma_bf16_ta<kMnMajorHi>(d, a0 + g_column(g_pair_a<PARTS>(q), 16 * s),
                                                b0 + g_pair_b<PARTS>(q) * part + 128 * s, idesc,
                                                q > 0 || s > 0 ? true : in_segment > 0, on);
                }
                mma_commit(g_empty + 8 * g, on);
                mma_commit(empty + 8 * stage, on);
                if (++in_segment == p.per_segment || t + 1 == tiles) {
                    mma_commit(acc_full + 8 * ab, on);
                    in_segment = 0;
                    if (++ab == p.acc_buffers) {
                        ab = 0;
                        ab_phase ^= 1;
                    }
                }
                if (++stage == p.stages) stage = 0;
                if (++g == kGroups) {
                    g = 0;
                    g_phase ^= 1;
                }
            }
        }
        if (gave_up()) {
            mma_commit(drain + 8, on);
            for (int k = 0; k < kMbarRounds; ++k)
                if (mbar_try(drain + 8, 0)) break;
        }
    } else if (warp >= 4 && warp < 4 + 4 * kGroups) {
        // Scores to G: group g takes every kGroups-th tile. After a wait that
        // gave up the rest fail at once and the block runs out on what is there,
        // storing NaN (`stop`).
        const int g = (warp - 4) / 4, quarter = warp & 3, in_tile = quarter * 32 + lane;
        const uint32_t group = tmem + ((uint32_t)(quarter * 32) << 16) + g * kGroupColumns<PARTS>;
        const float c2 = p.scale * kLog2e;
        int stage = 0, turn = 0;
        uint32_t phase = 0, stage_phase = 0;
        for (int u = blockIdx.x; u < p.units; u += gridDim.x) {
            const FusedWalk w = fused_unit(p, u);
            const int own = w.own0 + in_tile;
            int lab = kIgnored;
            float minus_lse = -kInf, r = 0.0f, at_label = 0.0f, own_bias = 0.0f, bias_sum = 0.0f;
            if (own < p.own) {
                if constexpr (BY_CLASS) {
                    own_bias = p.class_bias[own];
                } else {
                    const float* v = p.row_values + (int64_t)(own / kStream) * (kRowValues * kStream) + own % kStream;
                    minus_lse = v[0];
                    r = v[kStream];
                    at_label = v[2 * kStream];
                    lab = __float_as_int(v[3 * kStream]);
                }
            }
            for (int t = w.t0; t < w.t1; ++t) {
                const int at = stage;
                const uint32_t at_phase = stage_phase;
                if (++stage == p.stages) {
                    stage = 0;
                    stage_phase ^= flip;
                }
                if (turn++ != g) {
                    if (turn == kGroups) turn = 0;
                    continue;
                }
                if (turn == kGroups) turn = 0;
                const uint32_t col = stream0 + at * stage_bytes + tile_bytes;
                wait(full + 8 * at, at_phase);  // the columns' values
                wait(s_full + 8 * g, phase);
                tmem_fence_after();
                // 16 columns at a time in a loop that is not unrolled: its code has
                // to stay in the instruction cache of eight warps out of step
                // (both halves of 32 unrolled: 38 % of the stalls were fetches)
#pragma unroll 1
                for (int k = 0; k < kStream; k += kStep) {
                    float z[kStep];
                    tmem_load(group + k, z);
                    if constexpr (BY_CLASS) {
#pragma unroll
                        for (int j = 0; j < kStep; j += 4) {
                            const float4 a = shared_float4(col + 4 * (k + j));
                            const float4 b = shared_float4(col + 4 * (kStream + k + j));
                            gradients(z + j, c2, both(own_bias), both(own_bias), make_float2(a.x, a.y),
                                      make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w));
                        }
                        // rows labelled with one of this warp's classes
                        const int mine = shared_int(col + 4 * (3 * kStream + k + (lane & (kStep - 1)))) - w.own0 - quarter * 32;
                        if (__any_sync(0xffffffffu, (unsigned)mine < 32u)) {
#pragma unroll
                            for (int j = 0; j < kStep; ++j)
                                if (shared_int(col + 4 * (3 * kStream + k + j)) == own)
                                    z[j] = __int_as_float(shared_int(col + 4 * (2 * kStream + k + j)));
                        }
                        if (p.part_bias != nullptr) {
                            float q[4] = {bias_sum, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int j = 0; j < kStep; ++j) q[j % 4] += z[j];
                            bias_sum = (q[0] + q[1]) + (q[2] + q[3]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < kStep; j += 4) {
                            const float4 b = shared_float4(col + 4 * (k + j));
                            gradients(z + j, c2, make_float2(b.x, b.y), make_float2(b.z, b.w), both(minus_lse), both(minus_lse),
                                      both(r), both(r));
                        }
                        const int rel = lab - t * kStream - k;
                        if (__any_sync(0xffffffffu, (unsigned)rel < (unsigned)kStep)) {
#pragma unroll
                            for (int j = 0; j < kStep; ++j)
                                if (j == rel) z[j] = at_label;
                        }
                    }
                    store_parts<GP>(group, k, z);
                }
                tmem_store_wait();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(g_full + 8 * g);
                phase ^= 1;
            }
            if (BY_CLASS && p.part_bias != nullptr && own < p.own)
                p.part_bias[(int64_t)(w.split * kGroups + g) * p.own + own] = stop ? kNaN : bias_sum;
        }
    } else if (warp != 3) {
        // acc: quarter of the rows, and every other 32 channels
        const int quarter = warp & 3, half = (warp - 4 - 4 * kGroups) / 4;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + kAccBase;
        const int n = (p.channels + 15) / 16 * 16;
        constexpr int kKept = PARTS == 3 ? 2 : 1;  // fp32: all (<= 128 channels) stay here
        int ab = 0;
        uint32_t ab_phase = 0;
        for (int u = blockIdx.x; u < p.units; u += gridDim.x) {
            const FusedWalk w = fused_unit(p, u);
            const int own = w.own0 + quarter * 32 + lane;
            float kept[kKept][32];
            if constexpr (PARTS == 3) {
#pragma unroll
                for (int q = 0; q < kKept; ++q)
#pragma unroll
                    for (int j = 0; j < 32; ++j) kept[q][j] = 0.0f;
            }
            const auto write = [&](const float (&v)[32], int c, bool add) {
                if (own >= p.own) return;
                if (p.part != nullptr) {
                    float* dst = p.part + ((int64_t)w.split * p.own + own) * p.part_ld + c;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        if (c + j >= p.part_ld) continue;
                        float4* d4 = reinterpret_cast<float4*>(dst + j);
                        float4 o = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                        if (add) {
                            const float4 e = *d4;
                            o.x += e.x;
                            o.y += e.y;
                            o.z += e.z;
                            o.w += e.w;
                        }
                        *d4 = o;
                    }
                    return;
                }
                // 16 bytes at a time: the channels are a multiple of that here
                constexpr int kVec = 16 / sizeof(TypeOf<PARTS>);
                TypeOf<PARTS>* dst = static_cast<TypeOf<PARTS>*>(p.out) + (int64_t)own * p.channels + c;
#pragma unroll
                for (int j = 0; j < 32; j += kVec) {
                    if (c + j >= p.channels) continue;
                    float o[kVec];
#pragma unroll
                    for (int i = 0; i < kVec; ++i) o[i] = v[j + i] * p.scale;
                    store_row<TypeOf<PARTS>, kVec>(dst + j, o);
                }
            };
            bool first = true;
            for (int t = w.t0; t < w.t1; t += p.per_segment) {
                wait(acc_full + 8 * ab, ab_phase);
                tmem_fence_after();
                if constexpr (PARTS == 3) {
#pragma unroll
                    for (int q = 0; q < kKept; ++q) {
                        const int c = (2 * q + half) * 32;
                        if (c < n) {
#pragma unroll
                            for (int h = 0; h < 32; h += 16) {  // 16 at a time, for the registers' sake
                                if (c + h >= n) break;
                                float v[16];
                                tmem_load(lanes + ab * n + c + h, v);
#pragma unroll
                                for (int j = 0; j < 16; ++j) kept[q][h + j] += v[j];
                            }
                        }
                    }
                } else {
                    for (int c = half * 32; c < n; c += 64) {
                        tmem_load(lanes + ab * n + c, kept[0]);
                        if (c + 64 >= n) break;
                        write(kept[0], c, !first);
                    }
                }
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty + 8 * ab);
                if constexpr (PARTS < 3) {
                    // the last chunk is written after the buffer is given back
                    const int chunks = (n + 31) / 32;
                    const int mine = (chunks - half + 1) / 2;
                    if (mine > 0) write(kept[0], (2 * (mine - 1) + half) * 32, !first);
                }
                first = false;
                if (++ab == p.acc_buffers) {
                    ab = 0;
                    ab_phase ^= 1;
                }
            }
            if constexpr (PARTS == 3) {
#pragma unroll
                for (int q = 0; q < kKept; ++q) {
                    const int c = (2 * q + half) * 32;
                    if (c < n) write(kept[q], c, false);
                }
            }
            if (stop && own < p.own) {
                if (p.part != nullptr)
                    store_nan(p.part + ((int64_t)w.split * p.own + own) * p.part_ld, p.part_ld);
                else
                    store_nan(static_cast<TypeOf<PARTS>*>(p.out) + (int64_t)own * p.channels, p.channels);
            }
        }
    }
    if (warp > 2) gave_up();
    tmem_fence_before();
    __syncthreads();
    if (warp == 1) {
        tmem_fence_after();
        tmem_free(tmem_s, kTmemColumns);
    }
}

inline int group_columns(int parts) { return kGroups * (kStream + (parts == 3 ? kStream / 2 : 0)); }

// Whether the owning side, two streamed tiles and acc fit an SM: up to 128
// channels of fp32, 192 of fp16, 256 of bf16.
inline bool fused_fits(int parts, int channels) {
    const int chunks = (channels + 63) / 64, n = (channels + 15) / 16 * 16;
    return parts * chunks * (kOwn * 128 + 2 * kStream * 128) + 2 * kColumnBytes <= kFusedShared - 1024 &&
           group_columns(parts) + n <= 512;
}

// Buffers for what is left: a second one for the owning side if four streamed
// tiles fit beside it, then streamed tiles.
inline void fused_buffers(FusedArgs& p, int parts) {
    const int own = parts * p.chunks * kOwn * 128;
    const int stage = parts * p.chunks * kStream * 128 + kColumnBytes;
    const int room = kFusedShared - 1024, n = (p.channels + 15) / 16 * 16;
    p.own_buffers = 2 * own + 4 * stage <= room ? 2 : 1;
    p.stages = std::min(kFusedStages, (room - p.own_buffers * own) / stage);
    p.acc_buffers = group_columns(parts) + 2 * n <= 512 ? 2 : 1;
    // few streamed items and no shares of them: each unit streams the same tiles
    const int tiles = (p.streamed + kStream - 1) / kStream;
    p.resident = p.splits == 1 && tiles <= p.stages;
    if (p.resident) p.stages = tiles;
}

}  // namespace

}  // namespace mg
