// The label loss's row bookkeeping, shared by its kernels.
#pragma once

#include "rows.cuh"

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

}  // namespace mg
