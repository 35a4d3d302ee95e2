// The gated residual of a branch and the modulated norm of the sum, in one pass
// (gated_norm.hip), behind mh_gated_norm of include/moebius_hip.h. No counterpart
// in the reference, whose LayerNorms stand alone (src/engine/norm.rs:151-173).
#pragma once

#include <cstdint>

#include "common.hpp"
#include "kernels.hpp"

namespace mh {

enum class NormKind : int { None = 0, Rms = 1, Layer = 2 };

// (v - mean) / sqrt(var + eps) * gamma + beta over a row (Rms: v / sqrt(mean(v^2) + eps)).
struct NormSpec {
    NormKind kind = NormKind::None;
    float eps = 0;
    const float *gamma = nullptr, *beta = nullptr;  // [c] or NULL
};

// A vector of c f32 for every item, ld apart; NULL: none.
struct ItemVectors {
    const float *p = nullptr;
    int64_t ld = 0;
};

constexpr int kGatedNormMaxC = 32768;

// s = keep x + gate post(branch) (branch NULL: s = x), x_out = s, y = pre(s) (1 + scale) + shift,
// for `rows` rows of c <= kGatedNormMaxC channels; row r takes the vectors of item r / rows_per_item.
struct GatedNorm {
    const void *x = nullptr, *branch = nullptr;
    void *x_out = nullptr, *y = nullptr;  // either may be NULL
    int64_t ld_x = 0, ld_branch = 0, ld_x_out = 0, ld_y = 0;
    WeightType x_type = kF32, branch_type = kF32;  // of x and x_out, of branch and y
    int64_t rows = 0, rows_per_item = 1;
    int c = 0;
    float keep = 1.0f;
    NormSpec post, pre;
    ItemVectors gate, scale, shift;
};
void gated_norm(Context &ctx, const GatedNorm &g);

}  // namespace mh
