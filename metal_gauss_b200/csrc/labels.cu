// Softmax cross entropy of rows of features against class embeddings, without
// the logits ever being stored, and its gradients.
//
//   z[p, v] = scale x[p] . w[v] + b[v]
//   loss[p] = log sum_v exp(z[p, v]) - z[p, label]
//   G[p, v] = r[p] (softmax(z[p])[v] - [v == label])
//   dx = scale G w,  dw = scale G^T x,  db = column sums of G
//
// All four products run on the tensor cores as bf16 tiles of 128 x up to 256
// with fp32 sums. A feature or embedding becomes PARTS bf16 numbers that add up
// to it: one for bf16 (exact), two for fp16 (exact: 11 bits), three for fp32
// (24 bits); a product is the sum of the products of its parts, smallest first,
// down to those of 2^-24 of it (fp32) or all (fp16). So fp32 features keep
// fp32 logits, which a single tf32 or bf16 product would not.
//
//   split_kernel   x and w as parts; rows that are ignored become zeros, so
//                  whatever they hold meets nothing
//   kStats         a block takes 128 rows and walks its share of the classes,
//                  keeping per row the running maximum and the sum of
//                  exponentials of every class but the label's, and the
//                  label's logit. The label's own share is kept apart so that
//                  1 - softmax(label) of a confident row is not a difference
//                  of two numbers near 1.
//   fused_kernel   the backward pass for features of up to 128 fp32, 192 fp16 or
//                  256 bf16 channels: G stays on the SM (label_fused.cuh)
//   kLogitGrad     for wider ones: the logits again, turned into G, which goes to
//                  scratch as bf16 parts, a piece of rows at a time
//   kProductRow    dx = G w of the piece
//   kProductClass  dw += G^T x of the piece
//
// The tensor cores truncate each addition to an fp32 sum, which costs a sum of
// many terms 2^-25 of itself at every step. fp32 therefore issues a tile's small
// products before its large ones, and takes sums over rows or classes out to
// registers after every 64 entries (32 through scratch): 640000 x 32 x 128 has
// dclasses off by 3.4e-7 of its norm where runs of 256 entries gave 1.2e-6 and a
// plain fp32 product 4.9e-7.
// Classes or rows are split over blocks when there are few of the others; shares
// are joined in a fixed order.
#include "label_fused.cuh"
#include "label_tiles.cuh"

namespace mg {

namespace {

// What the scores need beside the parts: labels (forward) or the row values
// (backward), and the bias.
struct ColumnValues {
    RowGrad rg;
    const float* stats;
    const float* bias;
    int32_t* row_labels;
    float* row_values;
    float* class_bias;
};

// Features (live rows) and embeddings as (row, part, depth) bf16, depth the
// channels rounded up to 8 with zeros. One thread: 8 channels of one row.
template <typename T>
__global__ void __launch_bounds__(256)
split_kernel(const T* __restrict__ x, const T* __restrict__ w, LabelSource labels, int64_t rows,
             int classes, int channels, int depth, ColumnValues cv, __nv_bfloat16* __restrict__ xs,
             __nv_bfloat16* __restrict__ ws) {
    constexpr int PARTS = kPartsOf<T>;
    const int groups = depth / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t all = i / groups;
    const int c = (int)(i - all * groups) * 8;
    if (cv.row_labels != nullptr && i < rows) cv.row_labels[i] = labels.at(i);
    if (cv.row_values != nullptr && i < (rows + kRowBlock - 1) / kRowBlock * kRowBlock) {
        float v[kRowValues] = {-kInf, 0.0f, 0.0f, __int_as_float(kIgnored)};
        if (i < rows) {
            const int lab = labels.at(i);
            if (lab >= 0) {
                v[0] = -cv.stats[i];
                v[1] = cv.rg.at(i, lab);
                v[2] = -cv.stats[rows + i] * v[1];
                v[3] = __int_as_float(lab);
            }
        }
#pragma unroll
        for (int k = 0; k < kRowValues; ++k)
            cv.row_values[i / kRowBlock * (kRowValues * kRowBlock) + k * kRowBlock + i % kRowBlock] = v[k];
    }
    if (i < (classes + kClassPad - 1) / kClassPad * kClassPad)
        cv.class_bias[i] = i < classes ? (cv.bias != nullptr ? cv.bias[i] * kLog2e : 0.0f) : -kInf;
    if (all >= rows + classes) return;
    const bool feature = all < rows;
    const int64_t row = feature ? all : all - rows;
    const T* src = (feature ? x : w) + row * channels + c;
    const bool live = !feature || labels.at(row) >= 0;
    __nv_bfloat16 out[PARTS][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float v = live && c + k < channels ? to_f32<T>(src[k]) : 0.0f;
        __nv_bfloat16 p[PARTS];
        split_parts<PARTS>(v, p);
        // an infinity is its first part alone: the rest would be inf - inf
#pragma unroll
        for (int j = 0; j < PARTS; ++j)
            out[j][k] = j > 0 && fabsf(v) == kInf ? __float2bfloat16_rn(0.0f) : p[j];
    }
    __nv_bfloat16* dst = (feature ? xs : ws) + row * PARTS * depth + c;
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
        uint4 r;
        memcpy(&r, out[j], 16);
        *reinterpret_cast<uint4*>(dst + j * depth) = r;
    }
}

// ------------------------------------------------------------- rows and joins

// (m, s) of two shares of one row: maximum and sum of exp2(z - m).
__device__ __forceinline__ void join_stats(float& m, float& s, float m2, float s2) {
    const float t = fmaxf(m, m2);
    if (t == -kInf) {  // neither share has a finite logit; a NaN stays
        s += s2;
        return;
    }
    s = s * exp2f(m - t) + s2 * exp2f(m2 - t);
    m = t;
}

// Per row: the shares' join, the loss, and what the backward pass needs
// (stats: log2 of the sum, then 1 - softmax(label)); per block the sum of the losses and
// the count of live rows.
template <int L>
__global__ void __launch_bounds__(256)
label_rows_kernel(const float* __restrict__ part_m, const float* __restrict__ part_s,
                  const float* __restrict__ label_z, LabelSource labels, int splits, int64_t rows,
                  float* __restrict__ stats, float* __restrict__ row_loss,
                  double* __restrict__ block_sum, float* __restrict__ total, int mean,
                  float* __restrict__ live_out, int32_t* __restrict__ error_word) {
    const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int lane = threadIdx.x % L;
    const uint32_t lanes = L == 32 ? 0xffffffffu : 1u << (threadIdx.x & 31);
    float loss = 0.0f;
    int live = 0;
    if (row < rows) {
        const int lab = labels.at(row);
        float lse = kInf, miss = 0.0f;
        if (lab >= 0) {
            live = 1;
            float m = -kInf, s = 0.0f;
            for (int k = lane; k < splits; k += L) {
                const float m2 = part_m[(int64_t)k * rows + row];
                const float s2 = part_s[(int64_t)k * rows + row];
                join_stats(m, s, m2, s2);
            }
#pragma unroll
            for (int o = 1; o < L; o <<= 1) {  // the row's lanes are in step: all have its label
                const float m2 = __shfl_xor_sync(lanes, m, o), s2 = __shfl_xor_sync(lanes, s, o);
                join_stats(m, s, m2, s2);
            }
            const float z = label_z[row];
            // all in base 2; others = sum over the other classes of exp2(z_v - top)
            const float top = fmaxf(m, z);
            // no finite logit, an infinite one (inf - inf) or a NaN
            if (fabsf(top) == kInf || z != z || s != s) {
                lse = loss = miss = __int_as_float(0x7fc00000);
            } else {
                const float others = m == -kInf ? 0.0f : s * exp2f(m - top);
                const float own = exp2f(z - top);
                const float total = others + own;
                lse = top + log2f(total);
                miss = others / total;
                loss = z == top ? log1pf(others) : (top - z) * kLn2 + logf(total);
            }
        } else if (lab == kBadLabel) {
            live = 1;
            loss = __int_as_float(0x7fc00000);
            if (lane == 0) record_device_error(error_word, DEV_ERR_LABEL);
        }
        if (lane != 0) {
            loss = 0.0f;
            live = 0;
        } else if (stats != nullptr) {
            stats[row] = lse;
            stats[rows + row] = miss;
        }
        if (row_loss != nullptr && lane == 0) row_loss[row] = loss;
    }
    if (block_sum == nullptr && total == nullptr) return;
    __shared__ double sh[256];
    sh[threadIdx.x] = (double)loss;
    const int count = __syncthreads_count(live);
    for (int o = 128; o > 0; o >>= 1) {
        if (threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x != 0) return;
    if (total != nullptr) {  // the only block
        total[0] = (float)(mean ? sh[0] / fmax((double)count, 1.0) : sh[0]);
        if (live_out != nullptr) live_out[0] = (float)count;
    } else {
        block_sum[2 * blockIdx.x] = sh[0];
        block_sum[2 * blockIdx.x + 1] = (double)count;
    }
}

__global__ void __launch_bounds__(1024)
label_total_kernel(const double* __restrict__ block_sum, int blocks, int mean,
                   float* __restrict__ loss, float* __restrict__ live) {
    __shared__ double sh[1024], cn[1024];
    double s = 0.0, c = 0.0;
    for (int i = threadIdx.x; i < blocks; i += 1024) {
        s += block_sum[2 * i];
        c += block_sum[2 * i + 1];
    }
    sh[threadIdx.x] = s;
    cn[threadIdx.x] = c;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if (threadIdx.x < o) {
            sh[threadIdx.x] += sh[threadIdx.x + o];
            cn[threadIdx.x] += cn[threadIdx.x + o];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        loss[0] = (float)(mean ? sh[0] / fmax(cn[0], 1.0) : sh[0]);
        if (live != nullptr) live[0] = (float)cn[0];
    }
}

// out = scale times the sum of the shares (splits, n, ld), columns of each row.
template <typename T>
__global__ void __launch_bounds__(256)
join_kernel(const float* __restrict__ part, int splits, int64_t n, int ld, int columns, float scale,
            T* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n * columns) return;
    const int64_t row = i / columns;
    const int c = (int)(i - row * columns);
    float s = 0.0f;
    for (int k = 0; k < splits; ++k) s += part[((int64_t)k * n + row) * ld + c];
    out[i] = from_f32<T>(s * scale);
}

// Column sums of (lines, columns): block (x, y) takes 32 columns and the y-th
// share of the lines.
__global__ void __launch_bounds__(1024)
column_sum_kernel(const float* __restrict__ in, int64_t lines, int64_t per_block, int columns,
                  float* __restrict__ out) {
    __shared__ float sh[32][33];
    const int col = blockIdx.x * 32 + threadIdx.x;
    const int64_t end = min(lines, (int64_t)(blockIdx.y + 1) * per_block);
    float s = 0.0f;
    if (col < columns) {
#pragma unroll 4
        for (int64_t r = (int64_t)blockIdx.y * per_block + threadIdx.y; r < end; r += 32) s += in[r * columns + col];
    }
    sh[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = lanes_sum<32>(sh[threadIdx.x][threadIdx.y]);
    const int c = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && c < columns) out[(int64_t)blockIdx.y * columns + c] = s;
}

// ------------------------------------------------------------------- the host

struct Shares {
    int splits;
    int64_t per_split;
};

// Splits `tiles` over blocks when `others` blocks alone would not fill the
// device (one block to an SM).
Shares split(int64_t tiles, int64_t others) {
    const int64_t want = std::max<int64_t>(1, sm_count() / std::max<int64_t>(1, others));
    const int64_t per = (tiles + std::min(tiles, want) - 1) / std::min(tiles, want);
    return {(int)((tiles + per - 1) / per), per};
}

inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// G of a piece of rows is kept to about this much scratch: small beside the
// features, large enough that a piece's three launches each fill the device.
constexpr int64_t kPieceBytes = (int64_t)256 << 20;
constexpr int64_t kPieceRows = 1024;  // and to at least this many rows
constexpr int64_t kBiasLines = 1024;

struct Sizes {
    int64_t rows;
    int channels, classes, parts;

    int chunk() const { return parts == 1 ? 64 : 32; }
    // fp32: 32 entries between visits to the registers; the others round their
    // result to 11 bits or fewer and go 4096
    int segment() const { return (parts == 3 ? 32 : 4096) / chunk(); }
    int depth() const { return (int)up(channels, 8) * 8; }
    int part_ld() const { return (int)up(channels, 4) * 4; }
    int64_t row_tiles() const { return up(rows, kM); }
    int64_t class_columns() const { return up(classes, kN); }
    int64_t channel_columns() const { return up(channels, kN); }
    int64_t g_ld() const { return up(classes, 64) * 64; }
    int g_parts() const { return parts == 1 ? 2 : parts; }
    // dx and dw straight from the product: one share, in rows of whole 16-byte stores
    bool whole_stores() const { return channels % (parts == 3 ? 4 : 8) == 0; }
    bool direct() const { return by_row().splits == 1 && whole_stores(); }
    bool class_direct() const { return pieces() == 1 && by_class().splits == 1 && whole_stores(); }
    int64_t piece() const {
        const int64_t fit = kPieceBytes / (2 * g_parts() * g_ld()) / kM * kM;
        return std::min(up(rows, kM) * kM, std::max(kPieceRows, fit));
    }
    Shares stats() const { return split(class_columns(), row_tiles()); }
    Shares by_row() const {
        return split(up(classes, chunk()), up(piece(), kM) * channel_columns());
    }
    Shares by_class() const {
        return split(up(piece(), chunk()), up(classes, kM) * channel_columns());
    }
    // The backward pass that keeps G on the SM, and its shares.
    bool fused() const { return fused_fits(parts, channels); }
    int fused_segment() const { return parts == 3 ? 1 : 4096 / kStream; }
    Shares fused_by_row() const { return split(up(classes, kStream), up(rows, kOwn)); }
    Shares fused_by_class() const { return split(up(rows, kStream), up(classes, kOwn)); }
    // dx in one visit, in rows of whole 16-byte stores: no shares to join.
    // (Single elements, 32 rows apart in a warp, took 2 us of a unit.)
    bool fused_direct() const {
        const Shares s = fused_by_row();
        return s.splits == 1 && (parts == 3 || s.per_split <= fused_segment()) && whole_stores();
    }
    int64_t class_pad() const { return up(classes, kClassPad) * kClassPad; }
    // the forward's join: a warp to a row where the classes are in many shares
    bool wide_rows() const { return stats().splits >= 8; }
    int64_t row_blocks() const { return up(rows, wide_rows() ? 8 : 256); }
    // the bias's gradient: sums of 32 rows, then of up to kBiasLines of those; the
    // pieces' shares follow one another, and those of the last, short one are fewer
    int64_t pieces() const { return up(rows, piece()); }
    int64_t bias_lines() const { return piece() / 32; }
    int64_t bias_shares(int64_t piece_rows) const { return up(up(piece_rows, kM) * 4, kBiasLines); }
    int64_t all_bias_shares() const {
        const int64_t whole = pieces() - 1;
        return whole * bias_shares(piece()) + bias_shares(rows - whole * piece());
    }
};

struct Scratch {
    char* p;
    template <typename T>
    T* take(size_t n) {
        T* r = reinterpret_cast<T*>(p);
        p += align256(n * sizeof(T));
        return r;
    }
};

struct ForwardScratch {
    __nv_bfloat16 *xs, *ws;
    int32_t* row_labels;
    float *class_bias, *m, *s, *z;
    double* sums;
    size_t bytes;
    ForwardScratch(void* base, const Sizes& n) {
        Scratch a{static_cast<char*>(base)};
        xs = a.take<__nv_bfloat16>((size_t)n.rows * n.parts * n.depth());
        ws = a.take<__nv_bfloat16>((size_t)n.classes * n.parts * n.depth());
        row_labels = a.take<int32_t>((size_t)n.rows);
        class_bias = a.take<float>((size_t)n.class_pad());
        m = a.take<float>((size_t)n.stats().splits * Shape<kStats, 1>::kSets * n.rows);
        s = a.take<float>((size_t)n.stats().splits * Shape<kStats, 1>::kSets * n.rows);
        z = a.take<float>((size_t)n.rows);
        sums = a.take<double>(2 * (size_t)n.row_blocks());
        bytes = (size_t)(a.p - static_cast<char*>(base));
    }
};

struct BackwardScratch {
    __nv_bfloat16 *xs, *ws, *g;
    float *row_values, *class_bias, *row_part, *class_part, *bias_part, *bias_part2;
    size_t bytes;
    BackwardScratch(void* base, const Sizes& n) {
        Scratch a{static_cast<char*>(base)};
        xs = a.take<__nv_bfloat16>((size_t)n.rows * n.parts * n.depth());
        ws = a.take<__nv_bfloat16>((size_t)n.classes * n.parts * n.depth());
        row_values = a.take<float>((size_t)up(n.rows, kRowBlock) * kRowBlock * kRowValues);
        class_bias = a.take<float>((size_t)n.class_pad());
        if (n.fused()) {
            const Shares rs = n.fused_by_row(), cs = n.fused_by_class();
            g = nullptr;
            row_part = a.take<float>(n.fused_direct() ? 0 : (size_t)rs.splits * n.rows * n.part_ld());
            class_part = a.take<float>((size_t)cs.splits * n.classes * n.part_ld());
            bias_part = a.take<float>((size_t)cs.splits * kGroups * n.classes);
            bias_part2 = nullptr;
        } else {
            g = a.take<__nv_bfloat16>((size_t)n.piece() * n.g_parts() * n.g_ld());
            row_part = a.take<float>(n.direct() ? 0 : (size_t)n.by_row().splits * n.piece() * n.part_ld());
            class_part = a.take<float>((size_t)n.by_class().splits * n.classes * n.part_ld());
            bias_part = a.take<float>((size_t)n.bias_lines() * n.classes);
            bias_part2 = a.take<float>((size_t)n.all_bias_shares() * n.classes);
        }
        bytes = (size_t)(a.p - static_cast<char*>(base));
    }
};

// What the tile kernels' waits are held to.
struct Waits {
    int rounds = kMbarRounds;
    int units = INT32_MAX;  // that are copied in; the self-test starves the others
};

struct Args {
    const void *x, *w;
    int dtype;
    const float* bias;
    LabelSource labels;
    Sizes n;
    float scale;
    cudaStream_t st;
    Waits waits = {};
};

template <int MODE, int PARTS>
mg_status launch_tiles(TileArgs& p, const CUtensorMap& a, const CUtensorMap& b,
                       const CUtensorMap& out, const Args& args, const char* what) {
    constexpr int bytes = Shape<MODE, PARTS>::kDynamic;
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(tile_kernel<MODE, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 bytes) != cudaSuccess)
            return check_launch(what);
        ready[dev] = true;
    }
    const int grid = std::min(p.units, sm_count());
    p.copied = std::min(p.units, args.waits.units);
    p.rounds = args.waits.rounds;
    tile_kernel<MODE, PARTS><<<grid, Shape<MODE, PARTS>::kThreads, bytes, args.st>>>(p, a, b, out);
    return check_launch(what);
}

template <typename T>
mg_status split_inputs(const Args& a, __nv_bfloat16* xs, __nv_bfloat16* ws,
                       const ColumnValues& cv) {
    // a thread for each 8 channels, and for each of the padded rows and classes
    const int64_t threads = std::max({(a.n.rows + a.n.classes) * (a.n.depth() / 8),
                                      up(a.n.rows, kRowBlock) * kRowBlock, a.n.class_pad()});
    split_kernel<T><<<(unsigned)up(threads, 256), 256, 0, a.st>>>(
        static_cast<const T*>(a.x), static_cast<const T*>(a.w), a.labels, a.n.rows, a.n.classes,
        a.n.channels, a.n.depth(), cv, xs, ws);
    return check_launch("label_loss split");
}

// Maps of the parts of features or embeddings: contraction along the channels
// (box_rows rows of a tile) or along the rows (box_rows 0).
mg_status parts_map(CUtensorMap* m, const __nv_bfloat16* base, const Sizes& n, int64_t rows,
                    int box_rows) {
    const int64_t part = 2 * (int64_t)n.depth(), row = n.parts * part;
    if (box_rows > 0)
        return make_tensor_map(m, base, n.depth(), rows, n.parts, row, part, n.chunk(), box_rows,
                               n.chunk() == 64, "label_loss parts");
    return make_tensor_map(m, base, n.depth(), rows, n.parts, row, part, 64, n.chunk(), true,
                           "label_loss parts");
}

template <typename T>
mg_status forward(const Args& a, int reduction, float* loss, float* stats, float* live,
                  void* scratch) {
    constexpr int PARTS = kPartsOf<T>;
    const ForwardScratch f(scratch, a.n);
    MG_TRY((split_inputs<T>(a, f.xs, f.ws, ColumnValues{{}, nullptr, a.bias, f.row_labels, nullptr, f.class_bias})));
    CUtensorMap mx, mw;
    MG_TRY(parts_map(&mx, f.xs, a.n, a.n.rows, kM));
    MG_TRY(parts_map(&mw, f.ws, a.n, a.n.classes, kN));
    const Shares sh = a.n.stats();
    TileArgs p{};
    p.units = (int)(a.n.row_tiles() * sh.splits);
    p.a_rows = (int)a.n.rows;
    p.rows = a.n.rows;
    p.depth = a.n.depth();
    p.columns = a.n.classes;
    p.splits = sh.splits;
    p.per_split = (int)sh.per_split;
    p.scale = a.scale;
    p.class_bias = f.class_bias;
    p.row_labels = f.row_labels;
    p.part_m = f.m;
    p.part_s = f.s;
    p.label_z = f.z;
    p.error_word = device_error_word();
    // every class's chunks stay in shared memory where they leave two stages
    using S = Shape<kStats, PARTS>;
    const int64_t chunks = a.n.class_columns() * up(p.depth, S::kChunk);
    const int64_t room = S::kStages * S::kStage - chunks * PARTS * S::kB;
    if (sh.splits == 1 && room >= 2 * PARTS * S::kA) {
        p.resident = (int)chunks;
        p.resident_stages = (int)std::min<int64_t>(S::kBars, room / (PARTS * S::kA));
    }
    MG_TRY((launch_tiles<kStats, PARTS>(p, mx, mw, mw, a, "label_loss_forward")));
    const int shares = sh.splits * S::kSets, mean = reduction == MG_REDUCE_MEAN;
    const bool none = reduction == MG_REDUCE_NONE, single = a.n.row_blocks() == 1;
    const auto rows_kernel = a.n.wide_rows() ? label_rows_kernel<32> : label_rows_kernel<1>;
    rows_kernel<<<(unsigned)a.n.row_blocks(), 256, 0, a.st>>>(
        f.m, f.s, f.z, a.labels, shares, a.n.rows, stats, none ? loss : nullptr,
        none || single ? nullptr : f.sums, none || !single ? nullptr : loss, mean, live, p.error_word);
    MG_TRY(check_launch("label_loss_forward rows"));
    if (none || single) return MG_OK;
    label_total_kernel<<<1, 1024, 0, a.st>>>(f.sums, (int)a.n.row_blocks(), mean, loss, live);
    return check_launch("label_loss_forward total");
}

template <typename T>
mg_status join(const float* part, int splits, int64_t n, int ld, int columns, float scale, T* out,
               cudaStream_t st) {
    join_kernel<T><<<(unsigned)up(n * columns, 256), 256, 0, st>>>(part, splits, n, ld, columns, scale, out);
    return check_launch("label_loss_backward join");
}

// Sums of shares of per_block lines each.
mg_status column_sum(const float* in, int64_t lines, int64_t per_block, int columns, float* out,
                     cudaStream_t st) {
    const dim3 grid((unsigned)up(columns, 32), (unsigned)up(lines, per_block));
    column_sum_kernel<<<grid, dim3(32, 32), 0, st>>>(in, lines, per_block, columns, out);
    return check_launch("label_loss_backward bias");
}

template <bool BY_CLASS, int PARTS>
mg_status launch_fused(FusedArgs& p, const Sizes& n, const CUtensorMap& own,
                       const CUtensorMap& stream, const Args& args, const char* what) {
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(fused_kernel<BY_CLASS, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kFusedShared) != cudaSuccess)
            return check_launch(what);
        // the registers that its warps hand on are those it is launched with
        cudaFuncAttributes at{};
        if (cudaFuncGetAttributes(&at, fused_kernel<BY_CLASS, PARTS>) != cudaSuccess)
            return check_launch(what);
        if ((at.numRegs + 7) / 8 * 8 * (kFusedThreads / 128) < kIssueRegs + kGroups * kScoreRegs + 2 * kAccRegs)
            return fail(MG_ERR_CUDA, std::string(what) + ": built with too few registers");
        ready[dev] = true;
    }
    fused_buffers(p, PARTS);
    const int grid = std::min(p.units, sm_count());
    p.copied = std::min(p.units, args.waits.units);
    p.rounds = args.waits.rounds;
    fused_kernel<BY_CLASS, PARTS><<<grid, kFusedThreads, kFusedShared, args.st>>>(p, own, stream);
    return check_launch(what);
}

template <typename T>
mg_status backward_fused(const Args& a, const RowGrad& rg, const float* stats, T* dx, T* dw,
                         float* db, void* scratch) {
    constexpr int PARTS = kPartsOf<T>;
    const Sizes& n = a.n;
    const BackwardScratch f(scratch, n);
    MG_TRY((split_inputs<T>(a, f.xs, f.ws, ColumnValues{rg, stats, a.bias, nullptr, f.row_values, f.class_bias})));
    const int64_t part = 2 * (int64_t)n.depth(), row = n.parts * part;
    const auto map = [&](CUtensorMap* m, const __nv_bfloat16* b, int64_t rows, int box) {
        return make_tensor_map(m, b, n.depth(), rows, PARTS, row, part, 64, box, true, "label_loss parts");
    };
    FusedArgs p{};
    p.channels = n.channels;
    p.chunks = (int)up(n.channels, 64);
    p.per_segment = n.fused_segment();
    p.scale = a.scale;
    p.row_values = f.row_values;
    p.class_bias = f.class_bias;
    p.part_ld = n.part_ld();
    p.error_word = device_error_word();
    CUtensorMap own, stream;
    if (dx != nullptr) {
        const Shares sh = n.fused_by_row();
        MG_TRY(map(&own, f.xs, n.rows, kOwn));
        MG_TRY(map(&stream, f.ws, n.classes, kStream));
        p.units = (int)(up(n.rows, kOwn) * sh.splits);
        p.own = (int)n.rows;
        p.streamed = n.classes;
        p.splits = sh.splits;
        p.per_split = (int)sh.per_split;
        p.part = n.fused_direct() ? nullptr : f.row_part;
        p.out = dx;
        MG_TRY((launch_fused<false, PARTS>(p, n, own, stream, a, "label_loss_backward rows")));
        if (!n.fused_direct())
            MG_TRY(join(f.row_part, sh.splits, n.rows, n.part_ld(), n.channels, a.scale, dx, a.st));
    }
    if (dw != nullptr || db != nullptr) {
        const Shares sh = n.fused_by_class();
        MG_TRY(map(&own, f.ws, n.classes, kOwn));
        MG_TRY(map(&stream, f.xs, n.rows, kStream));
        p.units = (int)(up(n.classes, kOwn) * sh.splits);
        p.own = n.classes;
        p.streamed = (int)n.rows;
        p.splits = sh.splits;
        p.per_split = (int)sh.per_split;
        p.part = f.class_part;
        p.part_bias = db != nullptr ? f.bias_part : nullptr;
        MG_TRY((launch_fused<true, PARTS>(p, n, own, stream, a, "label_loss_backward classes")));
        if (dw != nullptr)
            MG_TRY(join(f.class_part, sh.splits, n.classes, n.part_ld(), n.channels, a.scale, dw, a.st));
        if (db != nullptr)
            MG_TRY(column_sum(f.bias_part, kGroups * sh.splits, kGroups * sh.splits, n.classes, db, a.st));
    }
    return MG_OK;
}

template <typename T>
mg_status backward(const Args& a, const RowGrad& rg, const float* stats, T* dx, T* dw, float* db,
                   void* scratch) {
    constexpr int PARTS = kPartsOf<T>;
    const Sizes& n = a.n;
    if (n.fused()) return backward_fused<T>(a, rg, stats, dx, dw, db, scratch);
    const BackwardScratch f(scratch, n);
    MG_TRY((split_inputs<T>(a, f.xs, f.ws, ColumnValues{rg, stats, a.bias, nullptr, f.row_values, f.class_bias})));
    CUtensorMap mw_score, mw_prod;
    MG_TRY(parts_map(&mw_score, f.ws, n, n.classes, kN));
    MG_TRY(parts_map(&mw_prod, f.ws, n, n.classes, 0));
    const int64_t g_part = n.piece() * n.g_ld() * 2;
    for (int64_t row0 = 0; row0 < n.rows; row0 += n.piece()) {
        const int64_t rows = std::min(n.piece(), n.rows - row0);
        const __nv_bfloat16* xs = f.xs + row0 * PARTS * n.depth();
        CUtensorMap mx, mg_out;
        MG_TRY(parts_map(&mx, xs, n, rows, kM));
        MG_TRY(make_tensor_map(&mg_out, f.g, n.classes, rows, kGParts<PARTS>, n.g_ld() * 2, g_part, 32, kM,
                               false, "label_loss G"));
        TileArgs p{};
        p.units = (int)(up(rows, kM) * n.class_columns());
        p.a_rows = (int)rows;
        p.rows = n.rows;
        p.row0 = row0;
        p.depth = n.depth();
        p.columns = n.classes;
        p.splits = 1;
        p.scale = a.scale;
        p.class_bias = f.class_bias;
        p.row_values = f.row_values;
        p.part_bias = db != nullptr ? f.bias_part : nullptr;
        p.error_word = device_error_word();
        MG_TRY((launch_tiles<kLogitGrad, PARTS>(p, mx, mw_score, mg_out, a, "label_loss_backward logits")));
        if (db != nullptr) {
            float* sums = f.bias_part2 + row0 / n.piece() * n.bias_shares(n.piece()) * n.classes;
            MG_TRY(column_sum(f.bias_part, up(rows, kM) * 4, kBiasLines, n.classes,
                              n.all_bias_shares() > 1 ? sums : db, a.st));
        }
        p.part_bias = nullptr;
        p.per_segment = n.segment();
        p.columns = n.channels;
        if (dx != nullptr) {
            CUtensorMap mg_in;
            MG_TRY(make_tensor_map(&mg_in, f.g, n.classes, rows, kGParts<PARTS>, n.g_ld() * 2, g_part, n.chunk(),
                                   kM, n.chunk() == 64, "label_loss G"));
            const Shares sh = n.by_row();
            p.units = (int)(up(rows, kM) * n.channel_columns() * sh.splits);
            p.depth = n.classes;
            p.splits = sh.splits;
            p.per_split = (int)sh.per_split;
            p.part = n.direct() ? nullptr : f.row_part;
            p.part_ld = n.part_ld();
            p.out = dx;
            MG_TRY((launch_tiles<kProductRow, PARTS>(p, mg_in, mw_prod, mw_prod, a, "label_loss_backward rows")));
            if (!n.direct())
                MG_TRY(join(f.row_part, sh.splits, rows, n.part_ld(), n.channels, a.scale,
                            dx + row0 * n.channels, a.st));
        }
        if (dw != nullptr) {
            CUtensorMap mg_in, mx_prod;
            MG_TRY(make_tensor_map(&mg_in, f.g, n.classes, rows, kGParts<PARTS>, n.g_ld() * 2, g_part, 64,
                                   n.chunk(), true, "label_loss G"));
            MG_TRY(parts_map(&mx_prod, xs, n, rows, 0));
            const Shares sh = n.by_class();
            p.units = (int)(up(n.classes, kM) * n.channel_columns() * sh.splits);
            p.a_rows = n.classes;
            p.depth = (int)rows;
            p.splits = sh.splits;
            p.per_split = (int)sh.per_split;
            p.part = n.class_direct() ? nullptr : f.class_part;
            p.part_ld = n.part_ld();
            p.add = row0 > 0;
            p.row0 = 0;
            p.out = dw;
            MG_TRY((launch_tiles<kProductClass, PARTS>(p, mg_in, mx_prod, mx_prod, a, "label_loss_backward classes")));
        }
    }
    if (dw != nullptr && !n.class_direct())
        MG_TRY(join(f.class_part, n.by_class().splits, n.classes, n.part_ld(), n.channels, a.scale, dw, a.st));
    if (db != nullptr && n.all_bias_shares() > 1) {
        const int64_t shares = n.all_bias_shares();
        MG_TRY(column_sum(f.bias_part2, shares, shares, n.classes, db, a.st));
    }
    return MG_OK;
}

int parts_of_dtype(int32_t dtype) { return dtype == MG_F32 ? 3 : dtype == MG_F16 ? 2 : 1; }

mg_status check_args(const char* who, const void* x, const void* w, int32_t dtype,
                     const void* labels, int32_t label_bytes, int64_t rows, int64_t channels,
                     int64_t classes, int32_t reduction) {
    const std::string n(who);
    MG_REQUIRE(dtype == MG_F32 || dtype == MG_BF16 || dtype == MG_F16, n + ": unknown dtype");
    MG_REQUIRE(label_bytes == 1 || label_bytes == 4 || label_bytes == 8,
               n + ": labels must be 1, 4 or 8 bytes");
    MG_REQUIRE(reduction >= MG_REDUCE_NONE && reduction <= MG_REDUCE_SUM, n + ": unknown reduction");
    MG_REQUIRE(rows >= 0, n + ": negative row count");
    MG_REQUIRE(channels >= 1 && channels <= MG_LABEL_MAX_CHANNELS, n + ": channels must be 1..512");
    MG_REQUIRE(classes >= 1 && classes <= MG_LABEL_MAX_CLASSES, n + ": classes must be 1..2^20");
    MG_REQUIRE(rows == 0 || (x && labels), n + ": null pointer");
    MG_REQUIRE(w != nullptr, n + ": null pointer");
    if (rows > MG_LABEL_MAX_ROWS) return fail(MG_ERR_CAPACITY, n + ": at most 2^30 rows");
    return MG_OK;
}

}  // namespace

mg_status make_tensor_map(CUtensorMap* map, const void* base, int64_t columns, int64_t rows,
                          int64_t parts, int64_t row_bytes, int64_t part_bytes, int box_columns,
                          int box_rows, bool swizzle128, const char* what) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = [] {
        void* f = nullptr;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault) == cudaSuccess
                   ? reinterpret_cast<Encode>(f)
                   : nullptr;
    }();
    if (encode == nullptr) return fail(MG_ERR_CUDA, std::string(what) + ": the driver has no tensor maps");
    const cuuint64_t dims[3] = {(cuuint64_t)columns, (cuuint64_t)rows, (cuuint64_t)parts};
    const cuuint64_t strides[2] = {(cuuint64_t)row_bytes, (cuuint64_t)part_bytes};
    const cuuint32_t box[3] = {(cuuint32_t)box_columns, (cuuint32_t)box_rows, 1};
    const cuuint32_t step[3] = {1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims,
                              strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              swizzle128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(MG_ERR_CUDA, std::string(what) + ": cuTensorMapEncodeTiled returned " + std::to_string((int)r));
    return MG_OK;
}

}  // namespace mg

using namespace mg;

extern "C" size_t mg_label_loss_scratch_bytes(int64_t rows, int64_t channels, int64_t classes,
                                              int32_t dtype, int32_t backward) {
    if (rows <= 0 || rows > MG_LABEL_MAX_ROWS || channels < 1 || channels > MG_LABEL_MAX_CHANNELS ||
        classes < 1 || classes > MG_LABEL_MAX_CLASSES)
        return 0;
    const Sizes n{rows, (int)channels, (int)classes, parts_of_dtype(dtype)};
    return backward ? BackwardScratch(nullptr, n).bytes : ForwardScratch(nullptr, n).bytes;
}

namespace {

mg_status run_forward(const Args& a, int reduction, float* loss, float* stats, float* live, void* scratch) {
    if (a.dtype == MG_F32) return forward<float>(a, reduction, loss, stats, live, scratch);
    if (a.dtype == MG_BF16) return forward<__nv_bfloat16>(a, reduction, loss, stats, live, scratch);
    return forward<__half>(a, reduction, loss, stats, live, scratch);
}

mg_status run_backward(const Args& a, const RowGrad& rg, const float* stats, void* dx, void* dw, float* db,
                       void* scratch) {
    if (a.dtype == MG_F32)
        return backward(a, rg, stats, static_cast<float*>(dx), static_cast<float*>(dw), db, scratch);
    if (a.dtype == MG_BF16)
        return backward(a, rg, stats, static_cast<__nv_bfloat16*>(dx), static_cast<__nv_bfloat16*>(dw), db, scratch);
    return backward(a, rg, stats, static_cast<__half*>(dx), static_cast<__half*>(dw), db, scratch);
}

}  // namespace

extern "C" mg_status mg_label_loss_forward(const void* features, const void* classes, int32_t dtype,
                                           const float* class_bias, const void* labels,
                                           int32_t label_bytes, int64_t ignore_index, int64_t rows,
                                           int64_t channels, int64_t n_classes, float scale,
                                           int32_t reduction, float* loss, float* stats,
                                           float* live, void* scratch, size_t scratch_bytes,
                                           mg_stream_t stream) try {
    MG_TRY(check_args("label_loss_forward", features, classes, dtype, labels, label_bytes, rows,
                      channels, n_classes, reduction));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (rows == 0) {
        if (reduction == MG_REDUCE_NONE) return MG_OK;
        MG_REQUIRE(loss != nullptr, "label_loss_forward: null pointer");
        if (cudaMemsetAsync(loss, 0, sizeof(float), st) != cudaSuccess ||
            (live && cudaMemsetAsync(live, 0, sizeof(float), st) != cudaSuccess))
            return check_launch("label_loss_forward memset");
        return MG_OK;
    }
    MG_REQUIRE(loss != nullptr, "label_loss_forward: null pointer");
    MG_REQUIRE(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 255u) == 0u &&
                   scratch_bytes >=
                       mg_label_loss_scratch_bytes(rows, channels, n_classes, dtype, 0),
               "label_loss_forward: scratch too small or not 256-byte aligned");
    MG_REQUIRE(on_boundary(elem_bytes(dtype), {features, classes}) && on_boundary(label_bytes, {labels}) &&
                   on_boundary(4, {class_bias, loss, stats, live}),
               "label_loss_forward: a pointer off its element's boundary");
    const Args a{features, classes, dtype, class_bias,
                 LabelSource{labels, label_bytes, ignore_index, (int)n_classes},
                 Sizes{rows, (int)channels, (int)n_classes, parts_of_dtype(dtype)}, scale, st};
    return run_forward(a, reduction, loss, stats, live, scratch);
} catch (...) {
    return caught("label_loss_forward");
}

extern "C" mg_status mg_label_loss_backward(
    const void* features, const void* classes, int32_t dtype, const float* class_bias,
    const void* labels, int32_t label_bytes, int64_t ignore_index, int64_t rows, int64_t channels,
    int64_t n_classes, float scale, int32_t reduction, const float* grad_loss, const float* stats,
    const float* live, void* d_features, void* d_classes, float* d_bias, void* scratch,
    size_t scratch_bytes, mg_stream_t stream) try {
    MG_TRY(check_args("label_loss_backward", features, classes, dtype, labels, label_bytes, rows,
                      channels, n_classes, reduction));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (rows == 0) {
        const size_t b = (size_t)n_classes * channels * (dtype == MG_F32 ? 4 : 2);
        if ((d_classes && cudaMemsetAsync(d_classes, 0, b, st) != cudaSuccess) ||
            (d_bias && cudaMemsetAsync(d_bias, 0, sizeof(float) * n_classes, st) != cudaSuccess))
            return check_launch("label_loss_backward memset");
        return MG_OK;
    }
    if (d_features == nullptr && d_classes == nullptr && d_bias == nullptr) return MG_OK;
    MG_REQUIRE(aligned16(d_features) && aligned16(d_classes),
               "label_loss_backward: d_features and d_classes must be 16-byte aligned");
    MG_REQUIRE(grad_loss && stats && (reduction != MG_REDUCE_MEAN || live),
               "label_loss_backward: null pointer");
    MG_REQUIRE(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 255u) == 0u &&
                   scratch_bytes >=
                       mg_label_loss_scratch_bytes(rows, channels, n_classes, dtype, 1),
               "label_loss_backward: scratch too small or not 256-byte aligned");
    MG_REQUIRE(on_boundary(elem_bytes(dtype), {features, classes}) && on_boundary(label_bytes, {labels}) &&
                   on_boundary(4, {class_bias, grad_loss, stats, live, d_bias}),
               "label_loss_backward: a pointer off its element's boundary");
    const Args a{features, classes, dtype, class_bias,
                 LabelSource{labels, label_bytes, ignore_index, (int)n_classes},
                 Sizes{rows, (int)channels, (int)n_classes, parts_of_dtype(dtype)}, scale, st};
    const RowGrad rg{grad_loss, reduction == MG_REDUCE_MEAN ? live : nullptr,
                     reduction == MG_REDUCE_NONE};
    return run_backward(a, rg, stats, d_features, d_classes, d_bias, scratch);
} catch (...) {
    return caught("label_loss_backward");
}

extern "C" mg_status mg_label_loss_wait_selftest(
    int32_t rounds, int32_t units, const void* features, const void* classes, int32_t dtype,
    const int64_t* labels, int64_t rows, int64_t channels, int64_t n_classes, float* loss,
    float* stats, const float* grad_loss, void* d_features, void* d_classes, float* d_bias,
    void* scratch, size_t scratch_bytes, mg_stream_t stream) try {
    const bool back = grad_loss != nullptr;
    MG_TRY(check_args("label_loss_wait_selftest", features, classes, dtype, labels, 8, rows, channels,
                      n_classes, MG_REDUCE_NONE));
    MG_REQUIRE(rounds >= 1 && rounds <= 1 << 12, "label_loss_wait_selftest: rounds must be 1..4096");
    MG_REQUIRE(units >= 0, "label_loss_wait_selftest: units must not be negative");
    MG_REQUIRE(rows >= 1 && rows <= 1 << 20, "label_loss_wait_selftest: rows must be 1..2^20");
    MG_REQUIRE(stats && (back ? d_features && d_classes && d_bias : loss != nullptr),
               "label_loss_wait_selftest: null pointer");
    MG_REQUIRE(aligned16(d_features) && aligned16(d_classes),
               "label_loss_wait_selftest: d_features and d_classes must be 16-byte aligned");
    MG_REQUIRE(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 255u) == 0u &&
                   scratch_bytes >= mg_label_loss_scratch_bytes(rows, channels, n_classes, dtype, back),
               "label_loss_wait_selftest: scratch too small or not 256-byte aligned");
    MG_REQUIRE(on_boundary(elem_bytes(dtype), {features, classes}) && on_boundary(8, {labels}) &&
                   on_boundary(4, {loss, stats, grad_loss, d_bias}),
               "label_loss_wait_selftest: a pointer off its element's boundary");
    const Args a{features, classes, dtype, nullptr, LabelSource{labels, 8, -100, (int)n_classes},
                 Sizes{rows, (int)channels, (int)n_classes, parts_of_dtype(dtype)}, 1.0f,
                 reinterpret_cast<cudaStream_t>(stream), Waits{rounds, units}};
    if (!back) return run_forward(a, MG_REDUCE_NONE, loss, stats, nullptr, scratch);
    return run_backward(a, RowGrad{grad_loss, nullptr, 1}, stats, d_features, d_classes, d_bias, scratch);
} catch (...) {
    return caught("label_loss_wait_selftest");
}
