// Softmax cross entropy of rows of features against class embeddings, without
// the logits ever being stored, and its gradients.
//
//   z[p, v] = scale x[p] . w[v] + b[v]
//   loss[p] = log sum_v exp(z[p, v]) - z[p, label]
//   G[p, v] = r[p] (softmax(z[p])[v] - [v == label])
//   dx = scale G w,  dw = scale G^T x,  db = column sums of G
//
// Forward: a block owns 64 rows and walks its share of the classes in tiles,
// keeping per row the running maximum, the sum of exponentials of every class
// but the label's, and the label's logit. The label's own share is kept apart
// so that 1 - softmax(label) of a confident row is not a difference of two
// numbers near 1. The backward kernels compute each tile of z again.
// The classes (forward, dx) or the rows (dw) are split over blocks when there
// are few of the others, and the shares joined in a fixed order.
#include "labels.cuh"

namespace mg {

namespace {

constexpr int kTile = 64;    // rows x classes of a score tile
constexpr int kDepth = 16;   // channels per step
constexpr int kThreads = 256;  // 16 x 16 threads, 4 x 4 scores each
constexpr float kInf = __builtin_huge_valf();

// acc[i][j] += a[ty * 4 + i] . b[tx * 4 + j] over the channels; a and b are
// 64 rows of row-major (n, channels) tensors, rows at or past n read as 0.
template <typename T>
__device__ __forceinline__ void score_tile(const T* __restrict__ a, int64_t a0, int64_t an,
                                           const T* __restrict__ b, int64_t b0, int64_t bn,
                                           int channels, float (*sa)[kTile + 4],
                                           float (*sb)[kTile + 4], float acc[4][4]) {
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (int k0 = 0; k0 < channels; k0 += kDepth) {
        __syncthreads();
        for (int i = threadIdx.x; i < kTile * kDepth; i += kThreads) {
            const int r = i / kDepth, k = i % kDepth;
            const bool in = k0 + k < channels;
            sa[k][r] = in && a0 + r < an ? to_f32<T>(a[(a0 + r) * channels + k0 + k]) : 0.0f;
            sb[k][r] = in && b0 + r < bn ? to_f32<T>(b[(b0 + r) * channels + k0 + k]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; ++k) {
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = sa[k][ty * 4 + i];
                y[i] = sb[k][tx * 4 + i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
        }
    }
}

// (m, s) of two shares of one row: maximum and sum of exp(z - m).
__device__ __forceinline__ void join_stats(float& m, float& s, float m2, float s2) {
    const float t = fmaxf(m, m2);
    if (t == -kInf) return;  // neither share has a finite logit
    s = s * expf(m - t) + s2 * expf(m2 - t);
    m = t;
}

// NaN logits: m stays a number, s becomes NaN and the row's loss with it.
template <typename T>
__global__ void __launch_bounds__(kThreads)
label_stats_kernel(const T* __restrict__ x, const T* __restrict__ w,
                   const float* __restrict__ bias, LabelSource labels, int64_t rows, int channels,
                   int classes, float scale, int tiles_per_split, float* __restrict__ part_m,
                   float* __restrict__ part_s, float* __restrict__ label_z) {
    __shared__ float sa[kDepth][kTile + 4], sb[kDepth][kTile + 4];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int64_t row0 = (int64_t)blockIdx.x * kTile;
    int lab[4];
    float m[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + ty * 4 + i;
        lab[i] = row < rows ? labels.at(row) : kIgnored;
        m[i] = -kInf;
        s[i] = 0.0f;
    }
    const int first = blockIdx.y * tiles_per_split;
    const int last = min((classes + kTile - 1) / kTile, first + tiles_per_split);
    for (int t = first; t < last; ++t) {
        float acc[4][4] = {};
        score_tile<T>(x, row0, rows, w, (int64_t)t * kTile, classes, channels, sa, sb, acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int v = t * kTile + tx * 4 + j;
                if (v >= classes) continue;
                const float z = fmaf(acc[i][j], scale, bias != nullptr ? bias[v] : 0.0f);
                if (v == lab[i]) {
                    label_z[row0 + ty * 4 + i] = z;
                } else if (z > m[i]) {
                    s[i] = fmaf(s[i], expf(m[i] - z), 1.0f);
                    m[i] = z;
                } else if (z > -kInf || z != z) {
                    s[i] += expf(z - m[i]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m[i], o);
            const float s2 = __shfl_xor_sync(0xffffffffu, s[i], o);
            join_stats(m[i], s[i], m2, s2);
            if (m[i] == -kInf) s[i] += s2;  // carries a NaN
        }
        const int64_t row = row0 + ty * 4 + i;
        if (tx == 0 && row < rows) {
            part_m[(int64_t)blockIdx.y * rows + row] = m[i];
            part_s[(int64_t)blockIdx.y * rows + row] = s[i];
        }
    }
}

// Per row: the shares' join, the loss, and what the backward pass needs
// (stats: lse, then 1 - softmax(label)); per block the sum of the losses and
// the count of live rows.
__global__ void __launch_bounds__(256)
label_rows_kernel(const float* __restrict__ part_m, const float* __restrict__ part_s,
                  const float* __restrict__ label_z, LabelSource labels, int splits, int64_t rows,
                  float* __restrict__ stats, float* __restrict__ row_loss,
                  double* __restrict__ block_sum, int32_t* __restrict__ error_word) {
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    float loss = 0.0f;
    int live = 0;
    if (row < rows) {
        const int lab = labels.at(row);
        float lse = kInf, miss = 0.0f;
        if (lab >= 0) {
            live = 1;
            float m = -kInf, s = 0.0f;
            for (int k = 0; k < splits; ++k) {
                const float m2 = part_m[(int64_t)k * rows + row];
                const float s2 = part_s[(int64_t)k * rows + row];
                join_stats(m, s, m2, s2);
                if (m == -kInf) s += s2;
            }
            const float z = label_z[row];
            // others = sum over the other classes of exp(z_v - top)
            const float top = fmaxf(m, z);
            if (top == -kInf || z != z || s != s) {
                lse = loss = miss = __int_as_float(0x7fc00000);
            } else {
                const float others = m == -kInf ? 0.0f : s * expf(m - top);
                const float own = expf(z - top);
                const float total = others + own;
                lse = top + logf(total);
                miss = others / total;
                loss = z == top ? log1pf(others) : (top - z) + logf(total);
            }
        } else if (lab == kBadLabel) {
            live = 1;
            loss = __int_as_float(0x7fc00000);
            record_device_error(error_word, DEV_ERR_LABEL);
        }
        if (stats != nullptr) {
            stats[row] = lse;
            stats[rows + row] = miss;
        }
        if (row_loss != nullptr) row_loss[row] = loss;
    }
    if (block_sum == nullptr) return;
    __shared__ double sh[256];
    sh[threadIdx.x] = (double)loss;
    const int count = __syncthreads_count(live);
    for (int o = 128; o > 0; o >>= 1) {
        if (threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
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

// One side's gradient for 64 of its items (BY_CLASS: classes, else rows) and
// 64 of its channels, over a share of the other side's items:
//   out[i, c] = scale sum_j G[i, j] other[j, c].
// A row that is ignored counts as zeros on both sides, whatever its features.
template <typename T, bool BY_CLASS>
__global__ void __launch_bounds__(kThreads)
label_grad_kernel(const T* __restrict__ x, const T* __restrict__ w,
                  const float* __restrict__ bias, LabelSource labels, RowGrad rg,
                  const float* __restrict__ stats, int64_t rows, int channels, int classes,
                  float scale, int64_t tiles_per_split, float* __restrict__ part,
                  float* __restrict__ part_bias) {
    __shared__ float sa[kDepth][kTile + 4], sb[kDepth][kTile + 4];
    __shared__ float g[kTile][kTile + 1], other[kTile][kTile + 1];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int64_t mine_n = BY_CLASS ? classes : rows, other_n = BY_CLASS ? rows : classes;
    const int64_t i0 = (int64_t)blockIdx.x * kTile;
    const int c0 = blockIdx.y * kTile;
    const int64_t first = blockIdx.z * tiles_per_split;
    const int64_t last = min((other_n + kTile - 1) / kTile, first + tiles_per_split);
    float out[4][4] = {};
    float bsum = 0.0f;
    for (int64_t t = first; t < last; ++t) {
        const int64_t j0 = t * kTile;
        float acc[4][4] = {};
        if constexpr (BY_CLASS) score_tile<T>(w, i0, classes, x, j0, rows, channels, sa, sb, acc);
        else score_tile<T>(x, i0, rows, w, j0, classes, channels, sa, sb, acc);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t mi = i0 + ty * 4 + i, oj = j0 + tx * 4 + j;
                const int64_t p = BY_CLASS ? oj : mi, v = BY_CLASS ? mi : oj;
                float e = 0.0f;
                if (p < rows && v < classes) {
                    const int lab = labels.at(p);
                    if (lab >= 0) {
                        const float z = fmaf(acc[i][j], scale, bias != nullptr ? bias[v] : 0.0f);
                        e = (v == lab ? -stats[rows + p] : expf(z - stats[p])) * rg.at(p, lab);
                    }
                }
                g[ty * 4 + i][tx * 4 + j] = e;
            }
        }
        for (int i = threadIdx.x; i < kTile * kTile; i += kThreads) {
            const int r = i / kTile, c = i % kTile;
            const int64_t j = j0 + r;
            float v = 0.0f;
            if (j < other_n && c0 + c < channels && (!BY_CLASS || labels.at(j) >= 0))
                v = to_f32<T>((BY_CLASS ? x : w)[j * channels + c0 + c]);
            other[r][c] = v;
        }
        __syncthreads();
        for (int r = 0; r < kTile; ++r) {
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = g[ty * 4 + i][r];
                b[i] = other[r][tx * 4 + i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) out[i][j] = fmaf(a[i], b[j], out[i][j]);
        }
        if (part_bias != nullptr && blockIdx.y == 0 && threadIdx.x < kTile) {
            for (int r = 0; r < kTile; ++r) bsum += g[threadIdx.x][r];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t mi = i0 + ty * 4 + i;
            const int c = c0 + tx * 4 + j;
            if (mi < mine_n && c < channels)
                part[((int64_t)blockIdx.z * mine_n + mi) * channels + c] = out[i][j] * scale;
        }
    }
    if (part_bias != nullptr && blockIdx.y == 0 && threadIdx.x < kTile && i0 + threadIdx.x < mine_n)
        part_bias[(int64_t)blockIdx.z * mine_n + i0 + threadIdx.x] = bsum;
}

template <typename T>
__global__ void __launch_bounds__(256)
label_join_kernel(const float* __restrict__ part, int splits, int64_t n, T* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.0f;
    for (int k = 0; k < splits; ++k) s += part[(int64_t)k * n + i];
    out[i] = from_f32<T>(s);
}

struct Shares {
    int splits;
    int64_t per_split;
};

// Splits `tiles` over blocks when `blocks` others alone would not fill the device.
Shares split(int64_t tiles, int64_t blocks) {
    const int64_t want = std::max<int64_t>(1, 2 * (int64_t)sm_count() / std::max<int64_t>(1, blocks));
    const int64_t per = (tiles + std::min(tiles, want) - 1) / std::min(tiles, want);
    return {(int)((tiles + per - 1) / per), per};
}

struct Sizes {
    int64_t rows;
    int channels, classes;

    int64_t row_tiles() const { return (rows + kTile - 1) / kTile; }
    int64_t class_tiles() const { return (classes + kTile - 1) / kTile; }
    int64_t depth_tiles() const { return (channels + kTile - 1) / kTile; }
    Shares stats() const { return split(class_tiles(), row_tiles()); }
    Shares by_row() const { return split(class_tiles(), row_tiles() * depth_tiles()); }
    Shares by_class() const { return split(row_tiles(), class_tiles() * depth_tiles()); }
    int64_t row_blocks() const { return (rows + 255) / 256; }

    size_t forward_bytes() const {
        return 16 * (size_t)row_blocks() +
               sizeof(float) * (size_t)rows * (2 * (size_t)stats().splits + 1);
    }
    size_t backward_bytes() const {
        const size_t a = (size_t)by_row().splits * rows * channels;
        const size_t b = (size_t)by_class().splits * classes * (channels + 1);
        return sizeof(float) * std::max(a, b);
    }
};

struct Args {
    const void *x, *w;
    int dtype;
    const float* bias;
    LabelSource labels;
    Sizes n;
    float scale;
    cudaStream_t st;
};

template <typename T>
mg_status forward(const Args& a, int reduction, float* loss, float* stats, float* live,
                  void* scratch) {
    const Shares sh = a.n.stats();
    double* sums = static_cast<double*>(scratch);
    float* m = reinterpret_cast<float*>(sums + 2 * a.n.row_blocks());
    float* s = m + sh.splits * a.n.rows;
    float* z = s + sh.splits * a.n.rows;
    label_stats_kernel<T><<<dim3((unsigned)a.n.row_tiles(), sh.splits), kThreads, 0, a.st>>>(
        static_cast<const T*>(a.x), static_cast<const T*>(a.w), a.bias, a.labels, a.n.rows,
        a.n.channels, a.n.classes, a.scale, (int)sh.per_split, m, s, z);
    MG_TRY(check_launch("label_loss_forward"));
    label_rows_kernel<<<(unsigned)a.n.row_blocks(), 256, 0, a.st>>>(
        m, s, z, a.labels, sh.splits, a.n.rows, stats, reduction == MG_REDUCE_NONE ? loss : nullptr,
        reduction == MG_REDUCE_NONE ? nullptr : sums, device_error_word());
    MG_TRY(check_launch("label_loss_forward rows"));
    if (reduction == MG_REDUCE_NONE) return MG_OK;
    label_total_kernel<<<1, 1024, 0, a.st>>>(sums, (int)a.n.row_blocks(),
                                             reduction == MG_REDUCE_MEAN, loss, live);
    return check_launch("label_loss_forward total");
}

template <typename T, bool BY_CLASS>
mg_status grad(const Args& a, const RowGrad& rg, const float* stats, void* out, float* out_bias,
               float* scratch) {
    const Shares sh = BY_CLASS ? a.n.by_class() : a.n.by_row();
    const int64_t n = BY_CLASS ? a.n.classes : a.n.rows;
    float* part_bias = out_bias != nullptr ? scratch + (int64_t)sh.splits * n * a.n.channels : nullptr;
    const dim3 grid((unsigned)((n + kTile - 1) / kTile), (unsigned)a.n.depth_tiles(), sh.splits);
    label_grad_kernel<T, BY_CLASS><<<grid, kThreads, 0, a.st>>>(
        static_cast<const T*>(a.x), static_cast<const T*>(a.w), a.bias, a.labels, rg, stats,
        a.n.rows, a.n.channels, a.n.classes, a.scale, sh.per_split, scratch, part_bias);
    MG_TRY(check_launch("label_loss_backward"));
    if (out != nullptr) {
        const int64_t e = n * a.n.channels;
        label_join_kernel<T><<<ceil_div(e, 256), 256, 0, a.st>>>(scratch, sh.splits, e,
                                                                 static_cast<T*>(out));
        MG_TRY(check_launch("label_loss_backward join"));
    }
    if (out_bias == nullptr) return MG_OK;
    label_join_kernel<float><<<ceil_div(n, 256), 256, 0, a.st>>>(part_bias, sh.splits, n, out_bias);
    return check_launch("label_loss_backward bias");
}

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

}  // namespace mg

using namespace mg;

extern "C" size_t mg_label_loss_scratch_bytes(int64_t rows, int64_t channels, int64_t classes,
                                              int32_t dtype, int32_t backward) {
    (void)dtype;
    if (rows <= 0 || rows > MG_LABEL_MAX_ROWS || channels < 1 || channels > MG_LABEL_MAX_CHANNELS ||
        classes < 1 || classes > MG_LABEL_MAX_CLASSES)
        return 0;
    const Sizes n{rows, (int)channels, (int)classes};
    return backward ? n.backward_bytes() : n.forward_bytes();
}

extern "C" mg_status mg_label_loss_forward(const void* features, const void* classes, int32_t dtype,
                                           const float* class_bias, const void* labels,
                                           int32_t label_bytes, int64_t ignore_index, int64_t rows,
                                           int64_t channels, int64_t n_classes, float scale,
                                           int32_t reduction, float* loss, float* stats,
                                           float* live, void* scratch, size_t scratch_bytes,
                                           mg_stream_t stream) {
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
    const Args a{features, classes, dtype, class_bias,
                 LabelSource{labels, label_bytes, ignore_index, (int)n_classes},
                 Sizes{rows, (int)channels, (int)n_classes}, scale, st};
    if (dtype == MG_F32) return forward<float>(a, reduction, loss, stats, live, scratch);
    if (dtype == MG_BF16) return forward<__nv_bfloat16>(a, reduction, loss, stats, live, scratch);
    return forward<__half>(a, reduction, loss, stats, live, scratch);
}

extern "C" mg_status mg_label_loss_backward(
    const void* features, const void* classes, int32_t dtype, const float* class_bias,
    const void* labels, int32_t label_bytes, int64_t ignore_index, int64_t rows, int64_t channels,
    int64_t n_classes, float scale, int32_t reduction, const float* grad_loss, const float* stats,
    const float* live, void* d_features, void* d_classes, float* d_bias, void* scratch,
    size_t scratch_bytes, mg_stream_t stream) {
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
    MG_REQUIRE(grad_loss && stats && (reduction != MG_REDUCE_MEAN || live),
               "label_loss_backward: null pointer");
    MG_REQUIRE(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 255u) == 0u &&
                   scratch_bytes >=
                       mg_label_loss_scratch_bytes(rows, channels, n_classes, dtype, 1),
               "label_loss_backward: scratch too small or not 256-byte aligned");
    const Args a{features, classes, dtype, class_bias,
                 LabelSource{labels, label_bytes, ignore_index, (int)n_classes},
                 Sizes{rows, (int)channels, (int)n_classes}, scale, st};
    const RowGrad rg{grad_loss, reduction == MG_REDUCE_MEAN ? live : nullptr,
                     reduction == MG_REDUCE_NONE};
    float* f = static_cast<float*>(scratch);
    if (d_features != nullptr) {
        if (dtype == MG_F32) MG_TRY((grad<float, false>(a, rg, stats, d_features, nullptr, f)));
        else if (dtype == MG_BF16) MG_TRY((grad<__nv_bfloat16, false>(a, rg, stats, d_features, nullptr, f)));
        else MG_TRY((grad<__half, false>(a, rg, stats, d_features, nullptr, f)));
    }
    if (d_classes != nullptr || d_bias != nullptr) {
        if (dtype == MG_F32) MG_TRY((grad<float, true>(a, rg, stats, d_classes, d_bias, f)));
        else if (dtype == MG_BF16) MG_TRY((grad<__nv_bfloat16, true>(a, rg, stats, d_classes, d_bias, f)));
        else MG_TRY((grad<__half, true>(a, rg, stats, d_classes, d_bias, f)));
    }
    return MG_OK;
}
