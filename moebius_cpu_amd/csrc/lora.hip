// Low-rank adapters of many requests beside a shared 1x1 projection:
//   y = x W^T + bias + residual + scale_s (x A_s^T) B_s^T,  s the row's adapter.
//
// The projection is the library's GEMM. The adapters take two passes of f32 products
// (v_mfma_f32_16x16x4_f32, f16 adapters widened exactly) in EXACT and FAST contexts
// alike: at rank r they are r (c_in + c_out) of the projection's c_in c_out operations,
// so memory bounds them, x read once more and out read and written once.
//   shrink: t = x A_s^T [rows][rank], the long axis split over the waves of a workgroup,
//           joined in LDS, and over workgroups where rows are few (partials side by side);
//   expand: out += scale_s t B_s^T, the partials added up as t is read.
//
// A tile of 16 rows takes the adapters its rows name one after another, each product
// over all 16 rows and kept for its own: rows of one image share one, single tokens of
// 16 requests read 16 adapters, which each has to be read anyway. Rows of other adapters
// are selected away, not multiplied by zero, so values that are not finite stay with
// their own requests.
#include <algorithm>

#include "attention.hpp"

namespace mh {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));

struct LoraArgs {
    const float *x;
    const void *a, *b;
    const float *scale;
    const int32_t *slot;
    float *t, *out;
    int64_t rows, rows_per_slot;
    int ci, co, rank, slots, splits, rank_pad;  // rank_pad: rank rounded up to 16
    int chunk;                                  // of the long axis per split, a multiple of 64
};

// Four values at p + k of a run of n, zeros behind it; VEC: n and p keep every run of four aligned.
template <bool VEC>
__device__ __forceinline__ floatx4 load4(const float *p, int k, int n) {
    if constexpr (VEC) {
        return k < n ? *reinterpret_cast<const floatx4 *>(p + k) : floatx4{0, 0, 0, 0};
    } else {
        floatx4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = k + e < n ? p[k + e] : 0.0f;
        return v;
    }
}
template <bool VEC>
__device__ __forceinline__ floatx4 load4(const _Float16 *p, int k, int n) {
    floatx4 v = {0, 0, 0, 0};
    if constexpr (VEC) {
        if (k < n) {
            const halfx4 r = *reinterpret_cast<const halfx4 *>(p + k);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = float(r[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k + e < n) v[e] = float(p[k + e]);
    }
    return v;
}

__device__ __forceinline__ floatx4 mfma(float a, float b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ int slot_of(const LoraArgs &p, int64_t row) {
    if (row >= p.rows) return -1;
    const int s = p.slot[row / p.rows_per_slot];
    return s < p.slots ? s : -1;
}

constexpr int kRankTiles = 4;  // 16 ranks each per pass over x

// Workgroup (16 rows, split of the long axis); wave w takes every fourth 16 of its share.
// Lane l holds row (rank) l % 16 and four values of the long axis at 4 (l / 16).
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraArgs p) {
    __shared__ float part[4][kRankTiles][4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, kg = lane >> 4;
    const int64_t r0 = int64_t(blockIdx.x) * 16;
    const int k0 = int(blockIdx.y) * p.chunk, k1 = min(k0 + p.chunk, p.ci);
    const int mine = slot_of(p, r0 + r16);
    const float *x = p.x + min(r0 + r16, p.rows - 1) * p.ci;
    uint32_t todo = uint32_t(__ballot(mine >= 0)) & 0xFFFFu;
    while (todo) {
        const int s = __shfl(mine, __builtin_ctz(todo));
        const bool own = mine == s;
        todo &= ~uint32_t(__ballot(own));
        for (int q0 = 0; q0 < p.rank; q0 += 16 * kRankTiles) {
            floatx4 acc[kRankTiles];
            const T *a[kRankTiles];
#pragma unroll
            for (int j = 0; j < kRankTiles; ++j) {
                acc[j] = floatx4{0, 0, 0, 0};
                a[j] = static_cast<const T *>(p.a) + (int64_t(s) * p.rank + min(q0 + j * 16 + r16, p.rank - 1)) * p.ci;
            }
            for (int k = k0 + wave * 16; k < k1; k += 64) {
                const floatx4 xv = load4<VEC>(x, k + kg * 4, k1);
#pragma unroll
                for (int j = 0; j < kRankTiles; ++j) {
                    if (q0 + j * 16 < p.rank) {
                        const floatx4 av = load4<VEC>(a[j], k + kg * 4, k1);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[j] = mfma(av[e], xv[e], acc[j]);
                    }
                }
            }
            __syncthreads();  // the sums before have been read
#pragma unroll
            for (int j = 0; j < kRankTiles; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[wave][j][e][lane] = acc[j][e];
            __syncthreads();
            // wave w joins rank tile w; register e is rank 4 (l / 16) + e of row l % 16
            const int q = q0 + wave * 16 + kg * 4;
            if (q0 + wave * 16 < p.rank && own && r0 + r16 < p.rows) {
                floatx4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = (part[0][wave][e][lane] + part[1][wave][e][lane]) +
                           (part[2][wave][e][lane] + part[3][wave][e][lane]);
                *reinterpret_cast<floatx4 *>(p.t + (int64_t(blockIdx.y) * p.rows + r0 + r16) * p.rank_pad + q) = v;
            }
        }
    }
}

// A wave takes 16 rows and 64 columns; register e of a 16-column tile is column
// 4 (l / 16) + e of row l % 16, so a lane reads and writes runs of four columns.
template <typename T, bool VEC, bool VOUT>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs p) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, kg = lane >> 4;
    const int64_t r0 = int64_t(blockIdx.x) * 16;
    const int c0 = (int(blockIdx.y) * 4 + wave) * 64;
    if (c0 >= p.co) return;
    const int mine = slot_of(p, r0 + r16);
    uint32_t todo = uint32_t(__ballot(mine >= 0)) & 0xFFFFu;
    if (!todo) return;
    const int64_t row = min(r0 + r16, p.rows - 1);
    float *out = p.out + row * p.co;
    while (todo) {
        const int s = __shfl(mine, __builtin_ctz(todo));
        const bool own = mine == s;
        todo &= ~uint32_t(__ballot(own));
        floatx4 acc[4];
        const T *b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[j] = floatx4{0, 0, 0, 0};
            b[j] = static_cast<const T *>(p.b) + (int64_t(s) * p.co + min(c0 + j * 16 + r16, p.co - 1)) * p.rank;
        }
        for (int k = 0; k < p.rank; k += 16) {
            // rows of other adapters: whatever lies there, selected away below
            floatx4 tv = {0, 0, 0, 0};
            if (own)
                for (int i = 0; i < p.splits; ++i)
                    tv += *reinterpret_cast<const floatx4 *>(p.t + (int64_t(i) * p.rows + row) * p.rank_pad + k + kg * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const floatx4 bv = load4<VEC>(b[j], k + kg * 4, p.rank);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[j] = mfma(bv[e], k + kg * 4 + e < p.rank ? tv[e] : 0.0f, acc[j]);
            }
        }
        if (!own) continue;
        const float scale = p.scale[s];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + j * 16 + kg * 4;
            if constexpr (VOUT) {
                if (c < p.co) {
                    floatx4 v = *reinterpret_cast<const floatx4 *>(out + c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(scale, acc[j][e], v[e]);
                    *reinterpret_cast<floatx4 *>(out + c) = v;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < p.co) out[c + e] = __builtin_fmaf(scale, acc[j][e], out[c + e]);
            }
        }
    }
}

// Splits of the long axis: two workgroups per CU, at least 128 values each.
int lora_splits(const Context &ctx, int64_t rows, int c_in) {
    const int64_t tiles = ceil_div(rows, 16);
    const int64_t s = std::min<int64_t>(2 * ctx.cu_count / std::max<int64_t>(tiles, 1), c_in / 128);
    return int(std::max<int64_t>(1, std::min<int64_t>(s, 16)));
}

template <typename T>
void run(Context &ctx, const LoraArgs &p) {
    const int64_t tiles = ceil_div(p.rows, 16);
    MH_REQUIRE(tiles < (int64_t(1) << 31), "lora: too many rows");
    const dim3 tb{256};
    const bool vx = p.ci % 4 == 0 && aligned16(p.x) && reinterpret_cast<uintptr_t>(p.a) % (4 * sizeof(T)) == 0;
    const dim3 sg{uint32_t(tiles), uint32_t(p.splits)};
    if (vx) lora_shrink_kernel<T, true><<<sg, tb, 0, ctx.stream>>>(p);
    else lora_shrink_kernel<T, false><<<sg, tb, 0, ctx.stream>>>(p);
    MH_LAUNCH_CHECK();
    const bool vb = p.rank % 4 == 0 && reinterpret_cast<uintptr_t>(p.b) % (4 * sizeof(T)) == 0;
    const bool vo = p.co % 4 == 0 && aligned16(p.out);
    const dim3 eg{uint32_t(tiles), uint32_t(ceil_div(p.co, 256))};
    if (vb && vo) lora_expand_kernel<T, true, true><<<eg, tb, 0, ctx.stream>>>(p);
    else if (vb) lora_expand_kernel<T, true, false><<<eg, tb, 0, ctx.stream>>>(p);
    else if (vo) lora_expand_kernel<T, false, true><<<eg, tb, 0, ctx.stream>>>(p);
    else lora_expand_kernel<T, false, false><<<eg, tb, 0, ctx.stream>>>(p);
    MH_LAUNCH_CHECK();
}

}  // namespace

size_t lora_scratch(const Context &ctx, int64_t rows, int c_in, int rank) {
    return size_t(lora_splits(ctx, rows, c_in)) * size_t(rows) * size_t(ceil_div(rank, 16) * 16) * sizeof(float);
}

void conv1x1_lora(Context &ctx, const float *x, int64_t rows, int c_in, const void *weight, WeightType wt, int c_out,
                  const float *bias, const float *residual, const Lora &l, float *out, void *scratch) {
    conv1x1(ctx, x, rows, c_in, weight, wt, c_out, bias, residual, out);
    if (!rows) return;
    LoraArgs p{};
    p.x = x, p.a = l.a, p.b = l.b, p.scale = l.scale, p.slot = l.slot, p.out = out;
    // behind the projection on the stream: its split sums in the workspace are done with
    p.t = static_cast<float *>(scratch ? scratch : ctx.ws.get(lora_scratch(ctx, rows, c_in, l.rank), ctx.stream));
    p.rows = rows, p.rows_per_slot = l.rows_per_slot;
    p.ci = c_in, p.co = c_out, p.rank = l.rank, p.slots = l.slots;
    p.rank_pad = int(ceil_div(l.rank, 16) * 16);
    p.splits = lora_splits(ctx, rows, c_in);
    p.chunk = int(ceil_div(ceil_div(c_in, p.splits), 64) * 64);
    if (l.type == kF16) run<_Float16>(ctx, p);
    else run<float>(ctx, p);
}

}  // namespace mh
