// The tile kernel of the label loss (labels.cu): one pipeline of TMA copies,
// tcgen05 products and epilogue warps with four uses.
//
// Tiles are 128 x 256, the most one product takes, in two buffers of tensor
// memory, so that one is taken out while the next is computed. Measured:
//   kStats         1440000 x 64 x 1203 bf16 597 us (2.9 T exponentials a second,
//                  of 4.65 at 16 a clock and SM: the bound), 65536 x 512 x 8192
//                  bf16 370 us (1.49 PFLOP/s, 89 % of cuBLAS)
//   kLogitGrad     the same 623 us: two parts of G written out, 2.1 GB
//   kProductRow    767 us, kProductClass 836 us: 2 x 550 GFLOP each for G's two
//                  parts, 1.43 and 1.32 PFLOP/s
#pragma once

#include "labels.cuh"

namespace mg {

namespace {

constexpr int kM = 128;        // rows of a tile
constexpr int kN = 256;        // columns of a tile, at most

enum Mode { kStats, kLogitGrad, kProductRow, kProductClass };

template <int MODE, int PARTS>
struct Shape {
    static constexpr bool kProduct = MODE >= kProductRow;
    // Sets of four warps that take tiles out, 32 columns at a time in turn: the
    // exponentials of kStats wait on one another's latency and want many.
    static constexpr int kSets = MODE == kStats || (MODE == kLogitGrad && PARTS < 3) ? 4 : 2;
    static constexpr int kThreads = 64 + 128 * kSets;  // and a copying and an issuing warp
    static constexpr bool kAmn = MODE == kProductClass;  // A's row index runs fastest
    static constexpr bool kBmn = kProduct;
    static constexpr int kChunk = PARTS == 1 ? 64 : 32;  // contraction entries per stage
    static constexpr int kA = kM * kChunk * 2;           // bytes of one part
    static constexpr int kB = kN * kChunk * 2;
    static constexpr int kPartsA = kProduct ? kGParts<PARTS> : PARTS;
    static constexpr int kPartsG = kGParts<PARTS>;
    static constexpr int kStage = kPartsA * kA + PARTS * kB;
    static constexpr int kStages = PARTS == 3 ? (MODE == kLogitGrad ? 2 : 3) : (MODE == kStats ? 4 : 3);
    // G on its way out: 128 x 32 bf16 for each set of the taking warps and part
    static constexpr int kOut = MODE == kLogitGrad ? kSets * kPartsG * kM * 64 : 0;
    static constexpr int kDynamic = 1024 + kStages * kStage + kOut;
    // Scores of more than one chunk go over them twice: the small products of all
    // of them, then the large one (with its parts fetched again). The tensor
    // cores truncate the running sum at each step, and only steps that come when
    // it is large weigh: 32 of 192 at 512 fp32 channels.
    static constexpr bool kTwice = !kProduct && PARTS > 1;
    static constexpr int kBars = MODE == kStats ? 8 : kStages;  // stages at most
    // Products of parts (a, b), smallest first.
    static constexpr int kPairs = kProduct ? kGPairs<PARTS> : PARTS == 1 ? 1 : PARTS == 2 ? 4 : 6;
    __device__ static constexpr int part_a(int i) { return kProduct ? g_pair_a<PARTS>(i) : pair_a<PARTS>(kPairs, i); }
    __device__ static constexpr int part_b(int i) { return kProduct ? g_pair_b<PARTS>(i) : pair_b<PARTS>(kPairs, i); }
};

struct TileArgs {           // counts below 2^31: at most 2^30 rows
    int units;
    int copied;             // units whose tiles are copied in: all, but for the self-test
    int rounds;             // of the issuing and copying warps' waits, at most
    int a_rows;             // rows of the A side (of the piece, or classes)
    int depth;              // contraction entries
    int columns;            // columns of the B side in all (classes, or channels)
    int splits;             // shares of the classes (kStats) or of the contraction
    int per_split;          // column tiles, or chunks, per share
    int per_segment;        // chunks between visits to the registers
    int64_t row0;           // the piece's first row
    int64_t rows;           // rows in all
    float scale;
    const float* class_bias;   // bias times log2 e, -infinity past the last class
    const int32_t* row_labels; // kStats
    const float* row_values;   // kLogitGrad
    float *part_m, *part_s, *label_z;  // kStats
    int resident;           // kStats: B chunks that stay in shared memory for good, or 0
    int resident_stages;    // and the stages, of A alone, beside them
    float* part_bias;       // kLogitGrad: sums of 32 rows of G, or NULL
    float* part;            // products: fp32 shares (splits, a_rows, part_ld), or NULL
    int part_ld;
    int add;                // to what the share holds
    void* out;              // products: the result itself
    int32_t* error_word;
};

// The tiles of a unit. Scores: a unit is a row tile and a share of the column
// tiles (kStats) or one column tile (kLogitGrad). Products: a unit is a row
// tile, a column tile and a share of the contraction, in segments.
struct Walk {
    int a_row, c0, c1, split, tiles, first;
};

template <int MODE, int PARTS>
__device__ __forceinline__ Walk walk_unit(const TileArgs& p, int u) {
    Walk w;
    const int col_tiles = (p.columns + kN - 1) / kN;
    const int chunks = (p.depth + Shape<MODE, PARTS>::kChunk - 1) / Shape<MODE, PARTS>::kChunk;
    if (MODE == kStats) {
        w.a_row = p.splits == 1 ? u * kM : u / p.splits * kM;
        w.split = p.splits == 1 ? 0 : u % p.splits;
        w.first = w.split * p.per_split;
        w.tiles = min(col_tiles, w.first + p.per_split) - w.first;
        w.c0 = 0;
        w.c1 = chunks;
    } else if (MODE == kLogitGrad) {
        w.a_row = u / col_tiles * kM;
        w.first = u % col_tiles;
        w.tiles = 1;
        w.split = 0;
        w.c0 = 0;
        w.c1 = chunks;
    } else {
        w.split = u % p.splits;
        const int t = u / p.splits;
        w.first = t % col_tiles;
        w.a_row = t / col_tiles * kM;
        w.c0 = w.split * p.per_split;
        w.c1 = min(chunks, w.c0 + p.per_split);
        w.tiles = (w.c1 - w.c0 + p.per_segment - 1) / p.per_segment;
    }
    return w;
}

// What a row's scores need.
struct RowIn {
    int lab = kIgnored;
    float minus_lse = -kInf, r = 0.0f, at_label = 0.0f;
};

template <int MODE>
__device__ __forceinline__ RowIn row_in(const TileArgs& p, int a_row) {
    RowIn in;
    if (a_row >= p.a_rows) return in;
    const int64_t row = p.row0 + a_row;
    if constexpr (MODE == kStats) {
        in.lab = p.row_labels[row];
    } else {
        const float* v = p.row_values + row / kRowBlock * (kRowValues * kRowBlock) + row % kRowBlock;
        in.minus_lse = v[0];
        in.r = v[kRowBlock];
        in.at_label = v[2 * kRowBlock];
        in.lab = __float_as_int(v[3 * kRowBlock]);
    }
    return in;
}

// Sums of products to logits in base 2; `bias`, the same for all lanes, is
// read through L1 (no barrier between the warps of a tile).
template <int N>
__device__ __forceinline__ void scores(float (&z)[N], float c2, const float* __restrict__ bias) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(bias + j));
        const float2 lo = fma2(make_float2(z[j], z[j + 1]), both(c2), make_float2(b.x, b.y));
        const float2 hi = fma2(make_float2(z[j + 2], z[j + 3]), both(c2), make_float2(b.z, b.w));
        z[j] = lo.x;
        z[j + 1] = lo.y;
        z[j + 2] = hi.x;
        z[j + 3] = hi.y;
    }
}

template <int MODE, int PARTS>
__global__ void __launch_bounds__((Shape<MODE, PARTS>::kThreads), 1)
tile_kernel(const __grid_constant__ TileArgs p, const __grid_constant__ CUtensorMap map_a,
            const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_out) {
    using S = Shape<MODE, PARTS>;
    extern __shared__ uint8_t dynamic[];
    __shared__ uint64_t bars[2 * S::kBars + 6];
    __shared__ uint32_t tmem_s;
    __shared__ volatile int stop;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t base = (smem_u32(dynamic) + 1023u) & ~1023u;
    const uint32_t full = smem_u32(bars), empty = full + 8 * S::kBars;
    const uint32_t taken_full = empty + 8 * S::kBars, taken_empty = taken_full + 16;
    const uint32_t drain = taken_empty + 16, resident_full = drain + 8;
    // Few classes: every unit's B side is the same, and stays. (Each SM
    // fetching it for each tile, 24 KB at 256 classes of 16 channels, made the
    // copies the bound: 7200 cycles a tile.)
    const int resident = MODE == kStats ? p.resident : 0;
    const int stages = resident > 0 ? p.resident_stages : S::kStages;
    const uint32_t stage_bytes = resident > 0 ? S::kPartsA * S::kA : S::kStage;
    const uint32_t ring = base + resident * (PARTS * S::kB);

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kBars; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(taken_full + 8 * i, 1);
            mbar_init(taken_empty + 8 * i, 4 * S::kSets);
        }
        mbar_init(drain, 1);
        mbar_init(resident_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_shared();
        stop = 0;
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_s), kTmemColumns);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    constexpr uint32_t tmem = kTmemBase;
    // For the end of every warp: once all are past their last wait `stop` changes
    // no more, and what is in flight then is drained or has been waited for.
    const auto gave_up = [&] {
        named_sync(1, S::kThreads);
        return stop != 0;
    };

    if (warp == 0) {
        // copies tiles in
        const uint32_t on = elect_lane();
        int stage = 0;
        uint32_t phase = 0;
        int issued = 0;
        bool ok = true;
        if (MODE == kStats && resident > 0) {
            const int chunks = (int)((p.depth + S::kChunk - 1) / S::kChunk);
            mbar_expect(resident_full, resident * PARTS * S::kB, on);
            for (int c = 0; c < resident; ++c)
                for (int i = 0; i < PARTS; ++i)
                    tma_load(base + (c * PARTS + i) * S::kB, &map_b, c % chunks * S::kChunk, c / chunks * kN, i,
                             resident_full, on);
        }
        for (int u = blockIdx.x; ok && u < p.copied; u += gridDim.x) {
            const Walk w = walk_unit<MODE, PARTS>(p, u);
            for (int t = 0; ok && t < w.tiles; ++t) {
                const int b0 = (S::kProduct ? w.first : w.first + t) * kN;
                const int c0 = S::kProduct ? w.c0 + t * p.per_segment : w.c0;
                const int c1 = S::kProduct ? min(w.c1, c0 + p.per_segment) : w.c1;
                const int blocks = S::kProduct ? (min(kN, p.columns - b0) + 63) / 64 : 0;
                const uint32_t bytes =
                    S::kPartsA * S::kA +
                    (resident > 0 ? 0 : PARTS * (S::kProduct ? blocks * S::kChunk * 128 : S::kB));
                const int passes = S::kTwice && c1 - c0 > 1 ? 2 : 1;
                for (int i = 0; i < passes * (c1 - c0); ++i) {
                    const bool again = i >= c1 - c0;  // the first part alone
                    const int c = again ? i - (c1 - c0) + c0 : i + c0;
                    ok = mbar_wait_warp(empty + 8 * stage, phase ^ 1, p.rounds, &stop, p.error_word, DEV_ERR_TILE_WAIT);
                    if (!ok) break;
                    const uint32_t bar = full + 8 * stage;
                    mbar_expect(bar, again ? S::kA + (resident > 0 ? 0 : S::kB) : bytes, on);
                    const int k = c * S::kChunk;
                    const uint32_t a = ring + stage * stage_bytes, b = a + S::kPartsA * S::kA;
#pragma unroll
                    for (int j = 0; j < S::kPartsA; ++j) {
                        if (again && j > 0) break;
                        if (S::kAmn) {
                            for (int q = 0; q < 2; ++q)
                                tma_load(a + j * S::kA + q * S::kChunk * 128, &map_a, w.a_row + 64 * q, k, j, bar, on);
                        } else {
                            tma_load(a + j * S::kA, &map_a, k, w.a_row, j, bar, on);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < PARTS; ++j) {
                        if (resident > 0 || (again && j > 0)) break;
                        if (S::kBmn) {
                            for (int q = 0; q < blocks; ++q)
                                tma_load(b + j * S::kB + q * S::kChunk * 128, &map_b, b0 + 64 * q, k, j, bar, on);
                        } else {
                            tma_load(b + j * S::kB, &map_b, k, b0, j, bar, on);
                        }
                    }
                    issued = min(issued + 1, stages);
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        if (gave_up()) {  // its copies in flight land before the block ends
            if (MODE == kStats && resident > 0)
                for (int i = 0; i < kMbarRounds; ++i)
                    if (mbar_try(resident_full, 0)) break;
            for (int j = 0; j < issued; ++j) {
                if (--stage < 0) {
                    stage = stages - 1;
                    phase ^= 1;
                }
                for (int i = 0; i < kMbarRounds; ++i)
                    if (mbar_try(full + 8 * stage, phase)) break;
            }
        }
    } else if (warp == 1) {
        // issues products
        const uint32_t on = elect_lane();
        int stage = 0, buf = 0;
        uint32_t phase = 0, buf_phase = 0;
        bool ok = resident == 0 || mbar_wait_warp(resident_full, 0, p.rounds, &stop, p.error_word, DEV_ERR_TILE_WAIT);
        for (int u = blockIdx.x; ok && u < p.units; u += gridDim.x) {
            const Walk w = walk_unit<MODE, PARTS>(p, u);
            for (int t = 0; ok && t < w.tiles; ++t) {
                const int b0 = (S::kProduct ? w.first : w.first + t) * kN;
                const int c0 = S::kProduct ? w.c0 + t * p.per_segment : w.c0;
                const int c1 = S::kProduct ? min(w.c1, c0 + p.per_segment) : w.c1;
                // scores: every column that is read (32 at a time) has been written,
                // past the last class with zeros; tensor memory may hold NaNs
                constexpr int kRound = S::kProduct ? 16 : 32;
                const int n = min(kN, (p.columns - b0 + kRound - 1) / kRound * kRound);
                const uint32_t idesc = uniform(mma_idesc(n, S::kAmn, S::kBmn));
                const int chunks = (int)uniform((uint32_t)(c1 - c0));
                // 16-entry steps of the last chunk
                const int tail = (int)uniform((uint32_t)min(S::kChunk / 16, (p.depth - (c1 - 1) * S::kChunk + 15) / 16));
                ok = mbar_wait_warp(taken_empty + 8 * buf, buf_phase ^ 1, p.rounds, &stop, p.error_word, DEV_ERR_TILE_WAIT);
                if (!ok) break;
                tmem_fence_after();
                const uint32_t d = uniform(tmem + buf * kN);
                const int passes = S::kTwice && chunks > 1 ? 2 : 1;
                for (int v = 0; v < passes * chunks; ++v) {
                    ok = mbar_wait_warp(full + 8 * stage, phase, p.rounds, &stop, p.error_word, DEV_ERR_TILE_WAIT);
                    if (!ok) break;
                    tmem_fence_after();
                    const int c = v < chunks ? v : v - chunks;
                    const int steps = c + 1 < chunks ? S::kChunk / 16 : tail;
                    const uint32_t a_at = ring + stage * stage_bytes;
                    const uint32_t b_at = resident > 0 ? base + (t * chunks + c) * (PARTS * S::kB) : a_at + S::kPartsA * S::kA;
                    const uint32_t a = uniform(S::kAmn ? mn_major_lo(a_at, S::kChunk * 128) : k_major_lo(a_at));
                    const uint32_t b = uniform(S::kBmn ? mn_major_lo(b_at, S::kChunk * 128) : k_major_lo(b_at));
                    constexpr uint32_t a_hi = S::kAmn ? kMnMajorHi : k_major_hi(S::kChunk * 2);
                    constexpr uint32_t b_hi = S::kBmn ? kMnMajorHi : k_major_hi(S::kChunk * 2);
#pragma unroll
                    for (int i = 0; i < S::kPairs; ++i) {
                        // of two passes the first leaves the last, large product out
                        if (S::kTwice && passes == 2 && (i + 1 < S::kPairs) != (v < chunks)) continue;
#pragma unroll
                        for (int s = 0; s < S::kChunk / 16; ++s) {
                            // 16 entries on: 32 bytes along a row, or 16 rows of 128 bytes
                            if (s < steps)
                                mma_bf16<a_hi, b_hi>(
                                    d, a + S::part_a(i) * (S::kA / 16) + s * (S::kAmn ? 128 : 2),
                                    b + S::part_b(i) * (S::kB / 16) + s * (S::kBmn ? 128 : 2), idesc,
                                    i > 0 || s > 0 ? true : v > 0, on);
                        }
                    }
                    mma_commit(empty + 8 * stage, on);
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                mma_commit(taken_full + 8 * buf, on);
                buf ^= 1;
                if (buf == 0) buf_phase ^= 1;
            }
        }
        if (gave_up()) {
            mma_commit(drain, on);
            for (int i = 0; i < kMbarRounds; ++i)
                if (mbar_try(drain, 0)) break;
        }
    } else {
        // Takes tiles out: warp % 4 is the quarter of the rows it can reach,
        // `set` the 32-column chunks it takes (every kSets-th). After a wait
        // that gave up the remaining waits fail at once and the block runs to
        // its end on whatever is there, storing NaN (`stop`).
        const int quarter = warp & 3, set = (warp - 2) / 4;
        const int in_tile = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const bool speaks = quarter == 0 && lane == 0;  // for its set's stores
        const float c2 = p.scale * kLog2e;
        int buf = 0;
        uint32_t buf_phase = 0;
        RowIn next_row;
        if constexpr (!S::kProduct)
            next_row = row_in<MODE>(p, walk_unit<MODE, PARTS>(p, blockIdx.x).a_row + in_tile);
        for (int u = blockIdx.x; u < p.units; u += gridDim.x) {
            const Walk w = walk_unit<MODE, PARTS>(p, u);
            const int a_row = w.a_row + in_tile;
            const bool mine = a_row < p.a_rows;
            if constexpr (!S::kProduct) {
                const int64_t row = p.row0 + a_row;
                const int lab = next_row.lab;
                const float minus_lse = next_row.minus_lse, r = next_row.r, at_label = next_row.at_label;
                float m = -kInf, s = 0.0f;
                for (int t = 0; t < w.tiles; ++t) {
                    const int v0 = (w.first + t) * kN;
                    const int n = min(kN, p.columns - v0);
                    if (t + 1 == w.tiles && u + (int)gridDim.x < p.units)  // while this tile is taken
                        next_row = row_in<MODE>(p, walk_unit<MODE, PARTS>(p, u + (int)gridDim.x).a_row + in_tile);
                    mbar_wait(taken_full + 8 * buf, buf_phase, kMbarRounds, &stop, p.error_word, DEV_ERR_TILE_WAIT);
                    tmem_fence_after();
                    for (int k = set; k * 32 < n; k += S::kSets) {
                        const uint32_t at = lanes + buf * kN + k * 32;
                        const int rel = lab - v0 - k * 32;
                        if constexpr (MODE == kStats) {
                            float z[32];
                            tmem_load(at, z);
                            scores<32>(z, c2, p.class_bias + v0 + k * 32);
                            // the label's logit goes apart, 8 columns at a time: most
                            // have no row's label
#pragma unroll
                            for (int h = 0; h < 32; h += 8) {
                                const bool here = (unsigned)(rel - h) < 8u;
                                if (__any_sync(0xffffffffu, here)) {
                                    float zl = 0.0f;
#pragma unroll
                                    for (int j = h; j < h + 8; ++j) {
                                        if (j == rel) {
                                            zl = z[j];
                                            z[j] = -kInf;
                                        }
                                    }
                                    if (here) p.label_z[row] = zl;
                                }
                            }
                            float t0 = m, t1 = -kInf;
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                t0 = max3(t0, z[j], z[j + 1]);
                                t1 = max3(t1, z[j + 2], z[j + 3]);
                            }
                            const float top = fmaxf(t0, t1);
                            const float ref = top == -kInf ? 0.0f : top;
                            float2 q0 = make_float2(s * exp2_fast(m - ref), 0.0f), q1 = make_float2(0.0f, 0.0f);
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                const float2 a = add2(make_float2(z[j], z[j + 1]), both(-ref));
                                const float2 b = add2(make_float2(z[j + 2], z[j + 3]), both(-ref));
                                q0 = add2(q0, make_float2(exp2_fast(a.x), exp2_fast(a.y)));
                                q1 = add2(q1, make_float2(exp2_fast(b.x), exp2_fast(b.y)));
                            }
                            s = (q0.x + q0.y) + (q1.x + q1.y);
                            m = top;
                        } else {
                            // staging is free again once the store before has read it
                            const uint32_t stage0 = base + S::kStages * S::kStage + set * (S::kPartsG * kM * 64);
                            if (speaks) tma_store_wait_read();
                            named_sync(2 + set, 128);
                            // 16 columns at a time, the loop not unrolled: its code
                            // has to stay in the instruction cache
#pragma unroll 1
                            for (int h = 0; h < 32; h += 16) {
                                float z[16];
                                tmem_load(at + h, z);
                                scores<16>(z, c2, p.class_bias + v0 + k * 32 + h);
#pragma unroll
                                for (int j = 0; j < 16; j += 2) {
                                    const float2 d = add2(make_float2(z[j], z[j + 1]), both(minus_lse));
                                    const float2 e = mul2(make_float2(exp2_fast(d.x), exp2_fast(d.y)), both(r));
                                    z[j] = e.x;
                                    z[j + 1] = e.y;
                                }
                                if (__any_sync(0xffffffffu, (unsigned)(rel - h) < 16u)) {
#pragma unroll
                                    for (int j = 0; j < 16; ++j)
                                        if (j == rel - h) z[j] = at_label;
                                }
                                if (stop) {
#pragma unroll
                                    for (int j = 0; j < 16; ++j) z[j] = kNaN;
                                }
                                if (p.part_bias != nullptr) {
                                    // lanes c and c + 16 end with the sums of column c over
                                    // half of the warp's 32 rows each
                                    float q[16];
#pragma unroll
                                    for (int j = 0; j < 16; ++j) q[j] = z[j];
#pragma unroll
                                    for (int o = 8; o > 0; o >>= 1) {
#pragma unroll
                                        for (int j = 0; j < o; ++j) {
                                            const bool up = (lane & o) != 0;
                                            const float send = up ? q[j] : q[j + o];
                                            const float keep = up ? q[j + o] : q[j];
                                            q[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
                                        }
                                    }
                                    q[0] += __shfl_xor_sync(0xffffffffu, q[0], 16);
                                    const int v = v0 + k * 32 + h + lane;
                                    if (lane < 16 && v < p.columns)
                                        p.part_bias[(int64_t)(w.a_row / 32 + quarter) * p.columns + v] = q[0];
                                }
                                // part i of 8 columns: 16 bytes of this row's 64, swizzled
#pragma unroll
                                for (int i = 0; i < S::kPartsG; ++i) {
#pragma unroll
                                    for (int g = 0; g < 2; ++g) {
                                        uint32_t word[4];
#pragma unroll
                                        for (int j = 0; j < 4; ++j) {
                                            word[j] = take_part(z[8 * g + 2 * j], z[8 * g + 2 * j + 1]);
                                        }
                                        const int piece = (h / 8 + g) ^ ((in_tile >> 1) & 3);
                                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                                                         stage0 + i * kM * 64 + in_tile * 64 + piece * 16),
                                                     "r"(word[0]), "r"(word[1]), "r"(word[2]), "r"(word[3])
                                                     : "memory");
                                    }
                                }
                            }
                            fence_async_shared();
                            named_sync(2 + set, 128);
                            if (speaks) {
#pragma unroll
                                for (int i = 0; i < S::kPartsG; ++i)
                                    tma_store(&map_out, v0 + k * 32, w.a_row, i, stage0 + i * kM * 64);
                                tma_store_commit();
                            }
                        }
                    }
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(taken_empty + 8 * buf);
                    buf ^= 1;
                    if (buf == 0) buf_phase ^= 1;
                }
                if (MODE == kStats && mine) {
                    const int64_t at = (int64_t)(w.split * S::kSets + set) * p.rows + row;
                    p.part_m[at] = m;
                    p.part_s[at] = stop ? kNaN : s;
                }
            } else {
                const int d0 = w.first * kN;
                const int n = min(kN, p.columns - d0);
                float acc[4][32];
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[q][j] = 0.0f;
                for (int t = 0; t < w.tiles; ++t) {
                    mbar_wait(taken_full + 8 * buf, buf_phase, kMbarRounds, &stop, p.error_word, DEV_ERR_TILE_WAIT);
                    tmem_fence_after();
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if ((2 * q + set) * 32 < n) {
                            float v[32];
                            tmem_load(lanes + buf * kN + (2 * q + set) * 32, v);
#pragma unroll
                            for (int j = 0; j < 32; ++j) acc[q][j] += v[j];
                        }
                    }
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(taken_empty + 8 * buf);
                    buf ^= 1;
                    if (buf == 0) buf_phase ^= 1;
                }
                if (mine) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int c = d0 + (2 * q + set) * 32;
                        if (c >= p.columns) continue;
                        if (p.part != nullptr) {
                            float* dst = p.part + ((int64_t)w.split * p.a_rows + a_row) * p.part_ld + c;
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                if (c + j >= p.part_ld) continue;
                                float4* d4 = reinterpret_cast<float4*>(dst + j);
                                float4 o = make_float4(acc[q][j], acc[q][j + 1], acc[q][j + 2], acc[q][j + 3]);
                                if (p.add) {
                                    const float4 e = *d4;
                                    o.x += e.x;
                                    o.y += e.y;
                                    o.z += e.z;
                                    o.w += e.w;
                                }
                                *d4 = o;
                            }
                        } else {
                            // 16 bytes at a time: the channels are a multiple of that here
                            using T = TypeOf<PARTS>;
                            constexpr int kVec = 16 / sizeof(T);
                            T* dst = static_cast<T*>(p.out) + (p.row0 + a_row) * p.columns + c;
#pragma unroll
                            for (int j = 0; j < 32; j += kVec) {
                                if (c + j >= p.columns) continue;
                                float o[kVec];
#pragma unroll
                                for (int i = 0; i < kVec; ++i) o[i] = acc[q][j + i] * p.scale;
                                store_row<T, kVec>(dst + j, o);
                            }
                        }
                    }
                    if (stop) {
                        if (p.part != nullptr)
                            store_nan(p.part + ((int64_t)w.split * p.a_rows + a_row) * p.part_ld + d0, min(n, p.part_ld - d0));
                        else
                            store_nan(static_cast<TypeOf<PARTS>*>(p.out) + (p.row0 + a_row) * p.columns + d0, n);
                    }
                }
            }
        }
        if (MODE == kLogitGrad && speaks) tma_store_wait_all();
        gave_up();
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 1) {
        tmem_fence_after();
        tmem_free(tmem_s, kTmemColumns);
    }
}

}  // namespace

}  // namespace mg
