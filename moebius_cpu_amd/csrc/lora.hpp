// Shared by the adapter kernels (lora.hip, lora_gemm.hip): see lora.hip for the mathematics.
#pragma once

#include "attention.hpp"

namespace mh {
namespace lora {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));

struct LoraArgs {
    const float *x;
    const void *a, *b;
    const float *scale;
    const int32_t *slot;
    float *t, *out;
    int64_t rows, rows_per_slot;
    int ci, co, rank, slots, rank_pad;  // rank_pad: rank rounded up to 16
};

// N values at p + k of a run of n, zeros behind it, in one load: behind n - N the last N are
// loaded instead and shifted, so that no load waits for a branch. VEC: n is a multiple of N
// and every run aligned; else the load is of the element's alignment (the same instruction),
// but for runs shorter than N.
template <int N, bool VEC, typename T>
__device__ __forceinline__ auto load_run(const T *p, int k, int n) {
    typedef T V __attribute__((ext_vector_type(N)));
    typedef T U __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    V v = T(0);
    if constexpr (VEC) {
        const V r = *reinterpret_cast<const V *>(p + min(k, n - N));
        v = k < n ? r : v;
    } else if (n >= N) {
        const int at = min(k, n - N), d = k - at;  // values that the run's end is short of
        const U r = *reinterpret_cast<const U *>(p + at);
        if constexpr (N * sizeof(T) == 16) {
            const unsigned __int128 bits = __builtin_bit_cast(unsigned __int128, V(r));
            v = d < N ? __builtin_bit_cast(V, bits >> (min(d, N - 1) * int(8 * sizeof(T)))) : v;
        } else {
            const uint64_t bits = __builtin_bit_cast(uint64_t, V(r));
            v = d < N ? __builtin_bit_cast(V, bits >> (min(d, N - 1) * int(8 * sizeof(T)))) : v;
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = k + e < n ? p[min(k + e, n - 1)] : T(0);
    }
    return v;
}
template <bool VEC>
__device__ __forceinline__ floatx4 load4(const float *p, int k, int n) {
    return load_run<4, VEC>(p, k, n);
}
template <bool VEC>
__device__ __forceinline__ floatx4 load4(const _Float16 *p, int k, int n) {
    const halfx4 r = load_run<4, VEC>(p, k, n);
    floatx4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = float(r[e]);
    return v;
}

__device__ __forceinline__ floatx4 mfma(float a, float b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ int slot_of(const LoraArgs &p, int64_t row) {
    if (row >= p.rows) return -1;
    const int s = p.slot[uint32_t(row) / uint32_t(p.rows_per_slot)];  // both below 2^31
    return s < p.slots ? s : -1;
}

// f32 values as two f16 parts, x 2^e = hi + lo to 2^-24 of it (2^-40 of the largest value
// of what e was taken from, scaled to 2^14 .. 2^15); one that is not finite is all in hi.
constexpr int kSplitExp = 14;
__device__ __forceinline__ void split2(float x, int e, _Float16 &hi, _Float16 &lo) {
    const float y = ldexpf(x, e);
    hi = static_cast<_Float16>(y);
    const float r = y - float(hi);
    lo = static_cast<_Float16>(__builtin_fabsf(y) < __builtin_huge_valf() ? r : 0.0f);
}
__device__ __forceinline__ int top_exp(float mx) { return mx == 0.0f ? 0 : __builtin_amdgcn_frexp_expf(mx) - 1; }

// The projection with the adapters' second product in its epilogue (lora_gemm.hip).
struct GemmArgs {
    LoraArgs l;
    const void *w;           // [co][ci], or its parts [co][nparts][cip]
    const int *w_exp;        // [co] where w is in parts
    const _Float16 *xp;      // [rows][nparts][cip]
    const int *x_exp;        // [rows]
    const float *bias, *residual;
    int cip;                 // ci padded (padded_channels)
    int tiles_m, tiles_n;    // of columns, of rows
};
// Channels and rows that the parts have room for: whole stages and tiles of the product.
inline int padded_channels(int ci) { return int(ceil_div(ci, 256) * 256); }
inline int64_t padded_rows(int64_t rows) { return ceil_div(rows, 128) * 128; }
// Rows [ci] -> parts [nparts][cip] (zeros behind ci) and each row's exponent, of one or two sets.
struct SplitRows {
    const float *x = nullptr;
    int64_t rows = 0;
    _Float16 *parts = nullptr;
    int *exps = nullptr;
};
void split_rows(Context &ctx, const SplitRows &a, const SplitRows &b, int ci, int cip, int nparts);
// The same of p.x and, for f16 adapters, p.t of every row that has one.
void split_shrink(Context &ctx, const LoraArgs &p, int cip, int nparts, _Float16 *parts, int *exps);
// nparts: 2, or 1 where operands are rounded to f16. An f32 weight is in parts.
void gemm(Context &ctx, const GemmArgs &g, int nparts, WeightType wt, WeightType at);

}  // namespace lora
}  // namespace mh
