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

#include "lora.hpp"

namespace mh {
namespace lora {
namespace {

constexpr int kRankTiles = 4;     // 16 ranks each per pass over x
constexpr int kShrinkUnroll = 5;  // steps of the long axis whose loads are in flight together

constexpr int kShrinkWaves = 8;

// Workgroup (16 rows, split of the long axis); wave w takes an eighth of its share.
// Lane l holds row (rank) l % 16 and four values of the long axis at 4 (l / 16).
template <typename T, bool VEC>
__global__ __launch_bounds__(64 * kShrinkWaves) void lora_shrink_kernel(LoraArgs p) {
    __shared__ float part[kShrinkWaves][kRankTiles][4][64];
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
            const int share = ((k1 - k0 + 15) / 16 + kShrinkWaves - 1) / kShrinkWaves * 16, kw = k0 + wave * share;
            const int ke = min(kw + share, k1);
            for (int k = kw; k < ke; k += 16 * kShrinkUnroll) {
                floatx4 xv[kShrinkUnroll];
#pragma unroll
                for (int u = 0; u < kShrinkUnroll; ++u) xv[u] = load4<VEC>(x, k + u * 16 + kg * 4, ke);
#pragma unroll
                for (int j = 0; j < kRankTiles; ++j) {
                    if (q0 + j * 16 < p.rank) {
                        floatx4 av[kShrinkUnroll];
#pragma unroll
                        for (int u = 0; u < kShrinkUnroll; ++u) av[u] = load4<VEC>(a[j], k + u * 16 + kg * 4, ke);
#pragma unroll
                        for (int u = 0; u < kShrinkUnroll; ++u)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[j] = mfma(av[u][e], xv[u][e], acc[j]);
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
            if (wave < kRankTiles && q0 + wave * 16 < p.rank && own && r0 + r16 < p.rows) {
                floatx4 v = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < kShrinkWaves; ++w)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += part[w][wave][e][lane];
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

// Few rows (single tokens): each row reads its own adapter anyway, so a wave takes one rank
// of one row, lanes over the long axis; t [rows][rank_pad].
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void lora_row_shrink_kernel(LoraArgs p) {
    const int lane = threadIdx.x & 63, q = int(blockIdx.y) * 4 + (threadIdx.x >> 6);
    const int64_t row = blockIdx.x;
    const int s = slot_of(p, row);
    if (s < 0 || q >= p.rank) return;
    const float *x = p.x + row * p.ci;
    const T *a = static_cast<const T *>(p.a) + (int64_t(s) * p.rank + q) * p.ci;
    float sum[4] = {0, 0, 0, 0};
#pragma unroll 4
    for (int k = lane * 4; k < p.ci; k += 256) {
        const floatx4 xv = load4<VEC>(x, k, p.ci), av = load4<VEC>(a, k, p.ci);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(xv[e], av[e], sum[e]);
    }
    float v = (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    if (lane == 0) p.t[row * p.rank_pad + q] = v;
}

// The projection and the adapters' second product of 16 rows and 16 columns: eight waves
// split the long axis (f32 products, eight values of it per lane and step: column or row
// l % 16, values 8 (l / 16) ..), join in LDS, and 256 threads finish one value each.
// Bound: the weight, read once per 16 rows.
constexpr int kRowUnroll = 5;  // steps of 256 values in flight: 1280 at once

template <typename W, typename T, bool VEC>
__global__ __launch_bounds__(512) void lora_row_project_kernel(LoraArgs p, const W *w, const float *bias,
                                                               const float *residual) {
    __shared__ float part[8][4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, kg = lane >> 4;
    const int c0 = int(blockIdx.x) * 16;
    const int64_t r0 = int64_t(blockIdx.y) * 16;
    const W *wr = w + int64_t(min(c0 + r16, p.co - 1)) * p.ci;
    const float *x = p.x + min(r0 + r16, p.rows - 1) * p.ci;
    const int s = slot_of(p, r0 + (tid >> 4));  // of the row that this thread finishes
    const float scale = s >= 0 ? p.scale[s] : 0.0f;
    floatx4 acc = {0, 0, 0, 0};
    for (int k0 = __builtin_amdgcn_readfirstlane(wave) * 32; k0 < p.ci; k0 += 256 * kRowUnroll) {
        floatx4 wv[kRowUnroll][2], xv[kRowUnroll][2];
#pragma unroll
        for (int u = 0; u < kRowUnroll; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int k = k0 + u * 256 + kg * 8 + 4 * i;
                wv[u][i] = load4<VEC>(wr, k, p.ci);
                xv[u][i] = load4<VEC>(x, k, p.ci);
            }
#pragma unroll
        for (int u = 0; u < kRowUnroll; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc = mfma(wv[u][i][e], xv[u][i][e], acc);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][e][lane] = acc[e];
    __syncthreads();
    if (tid >= 256) return;
    // thread: column tid % 16 (register e = % 4 of lane group / 4) of row tid / 16
    const int c = c0 + (tid & 15);
    const int64_t row = r0 + (tid >> 4);
    if (c >= p.co || row >= p.rows) return;
    const int e = tid & 3, l = ((tid & 15) >> 2) * 16 + (tid >> 4);
    float v = bias ? bias[c] : 0.0f;
    if (residual) v += residual[row * p.co + c];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += part[i][e][l];
    v += sum;
    if (s >= 0) {
        const T *b = static_cast<const T *>(p.b) + (int64_t(s) * p.co + c) * p.rank;
        const float *t = p.t + row * p.rank_pad;
        float y = 0.0f;
        if (p.rank % 4 == 0 && reinterpret_cast<uintptr_t>(p.b) % (4 * sizeof(T)) == 0) {
            for (int k = 0; k < p.rank; k += 16) {
                floatx4 bv[4], tv[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    bv[u] = load4<true>(b, k + 4 * u, p.rank);
                    tv[u] = load4<true>(t, k + 4 * u, p.rank);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) y = __builtin_fmaf(tv[u][i], bv[u][i], y);
            }
        } else {
            for (int k = 0; k < p.rank; ++k) y = __builtin_fmaf(t[k], float(b[k]), y);
        }
        v = __builtin_fmaf(scale, y, v);
    }
    p.out[row * p.co + c] = v;
}

// Rows up to which the projection is worth forming beside the adapters (few_rows): both
// of its passes over 16 rows against the general product's split sums and the two
// adapter passes over its output.
constexpr int kFewRows = 64;
bool few_rows(int64_t rows) { return rows <= kFewRows; }

// Splits of the long axis: two workgroups per CU, at least 128 values each.
int lora_splits(const Context &ctx, int64_t rows, int c_in, bool own) {
    if (few_rows(rows) || own) return 1;  // their second products read t as it is
    const int64_t tiles = ceil_div(rows, 16);
    const int64_t s = std::min<int64_t>(2 * ctx.cu_count / std::max<int64_t>(tiles, 1), c_in / 128);
    return int(std::max<int64_t>(1, std::min<int64_t>(s, 16)));
}

template <typename T>
void run_shrink(Context &ctx, const LoraArgs &p) {
    const int64_t tiles = ceil_div(p.rows, 16);
    MH_REQUIRE(tiles < (int64_t(1) << 31), "lora: too many rows");
    const dim3 tb{64 * kShrinkWaves};
    const bool vx = p.ci % 4 == 0 && aligned16(p.x) && reinterpret_cast<uintptr_t>(p.a) % (4 * sizeof(T)) == 0;
    const dim3 sg{uint32_t(tiles), uint32_t(p.splits)};
    if (vx) lora_shrink_kernel<T, true><<<sg, tb, 0, ctx.stream>>>(p);
    else lora_shrink_kernel<T, false><<<sg, tb, 0, ctx.stream>>>(p);
    MH_LAUNCH_CHECK();
}

template <typename T>
void run_expand(Context &ctx, const LoraArgs &p) {
    const int64_t tiles = ceil_div(p.rows, 16);
    const dim3 tb{256};
    const bool vb = p.rank % 4 == 0 && reinterpret_cast<uintptr_t>(p.b) % (4 * sizeof(T)) == 0;
    const bool vo = p.co % 4 == 0 && aligned16(p.out);
    const dim3 eg{uint32_t(tiles), uint32_t(ceil_div(p.co, 256))};
    if (vb && vo) lora_expand_kernel<T, true, true><<<eg, tb, 0, ctx.stream>>>(p);
    else if (vb) lora_expand_kernel<T, true, false><<<eg, tb, 0, ctx.stream>>>(p);
    else if (vo) lora_expand_kernel<T, false, true><<<eg, tb, 0, ctx.stream>>>(p);
    else lora_expand_kernel<T, false, false><<<eg, tb, 0, ctx.stream>>>(p);
    MH_LAUNCH_CHECK();
}

template <typename W, typename T>
void run_few(Context &ctx, const LoraArgs &p, const void *weight, const float *bias, const float *residual) {
    const bool va = p.ci % 4 == 0 && aligned16(p.x) && reinterpret_cast<uintptr_t>(p.a) % (4 * sizeof(T)) == 0;
    const dim3 sg{uint32_t(p.rows), uint32_t(ceil_div(p.rank, 4))};
    if (va) lora_row_shrink_kernel<T, true><<<sg, dim3{256}, 0, ctx.stream>>>(p);
    else lora_row_shrink_kernel<T, false><<<sg, dim3{256}, 0, ctx.stream>>>(p);
    MH_LAUNCH_CHECK();
    const bool vw = p.ci % 4 == 0 && aligned16(p.x) && reinterpret_cast<uintptr_t>(weight) % (4 * sizeof(W)) == 0;
    const dim3 pg{uint32_t(ceil_div(p.co, 16)), uint32_t(ceil_div(p.rows, 16))};
    const W *w = static_cast<const W *>(weight);
    if (vw) lora_row_project_kernel<W, T, true><<<pg, dim3{512}, 0, ctx.stream>>>(p, w, bias, residual);
    else lora_row_project_kernel<W, T, false><<<pg, dim3{512}, 0, ctx.stream>>>(p, w, bias, residual);
    MH_LAUNCH_CHECK();
}

// Scratch: t, then the parts of x and their exponents, then those of an f32 weight.
struct Layout {
    size_t t = 0, x = 0, x_exp = 0, w = 0, w_exp = 0;
    size_t total() const { return t + x + x_exp + w + w_exp; }
};

bool use_gemm(const Context &ctx, int64_t rows, int c_in, int c_out) {
    return !few_rows(rows) && ctx.precision == Precision::Exact && gemm_fits(ctx, rows, c_out, c_in);
}

Layout layout(const Context &ctx, int64_t rows, int c_in, int c_out, WeightType wt, int rank) {
    auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
    const size_t cip = size_t(ceil_div(c_in, 64) * 64);
    Layout l;
    const bool own = use_gemm(ctx, rows, c_in, c_out);
    l.t = up(size_t(lora_splits(ctx, rows, c_in, own)) * size_t(rows) * size_t(ceil_div(rank, 16) * 16) * sizeof(float));
    if (own) {
        l.x = up(size_t(padded_rows(rows)) * 2 * cip * 2);
        l.x_exp = up(size_t(rows) * 4);
        if (wt == kF32) {
            l.w = up(size_t(c_out) * 2 * cip * 2);
            l.w_exp = up(size_t(c_out) * 4);
        }
    }
    return l;
}

}  // namespace
}  // namespace lora

size_t lora_scratch(const Context &ctx, int64_t rows, int c_in, int c_out, WeightType wt, int rank) {
    return rows ? lora::layout(ctx, rows, c_in, c_out, wt, rank).total() : 0;
}

void conv1x1_lora(Context &ctx, const float *x, int64_t rows, int c_in, const void *weight, WeightType wt, int c_out,
                  const float *bias, const float *residual, const Lora &l, float *out, void *scratch) {
    if (!rows) return;
    const bool few = lora::few_rows(rows), own = lora::use_gemm(ctx, rows, c_in, c_out);
    if (!few && !own) conv1x1(ctx, x, rows, c_in, weight, wt, c_out, bias, residual, out);
    const lora::Layout mem = lora::layout(ctx, rows, c_in, c_out, wt, l.rank);
    // behind the projection on the stream: its split sums in the workspace are done with
    char *at = static_cast<char *>(scratch ? scratch : ctx.ws.get(mem.total(), ctx.stream));
    lora::LoraArgs p{};
    p.x = x, p.a = l.a, p.b = l.b, p.scale = l.scale, p.slot = l.slot, p.out = out;
    p.t = reinterpret_cast<float *>(at);
    p.rows = rows, p.rows_per_slot = l.rows_per_slot;
    p.ci = c_in, p.co = c_out, p.rank = l.rank, p.slots = l.slots;
    p.rank_pad = int(ceil_div(l.rank, 16) * 16);
    p.splits = lora::lora_splits(ctx, rows, c_in, own);
    p.chunk = int(ceil_div(ceil_div(c_in, p.splits), 64) * 64);
    const bool ah = l.type == kF16;
    if (few) {
        if (wt == kF16 && ah) lora::run_few<_Float16, _Float16>(ctx, p, weight, bias, residual);
        else if (wt == kF16) lora::run_few<_Float16, float>(ctx, p, weight, bias, residual);
        else if (ah) lora::run_few<float, _Float16>(ctx, p, weight, bias, residual);
        else lora::run_few<float, float>(ctx, p, weight, bias, residual);
        return;
    }
    if (!own) {
        if (ah) lora::run_shrink<_Float16>(ctx, p);
        else lora::run_shrink<float>(ctx, p);
        if (ah) lora::run_expand<_Float16>(ctx, p);
        else lora::run_expand<float>(ctx, p);
        return;
    }
    lora::GemmArgs g{};
    g.l = p;
    g.cip = int(ceil_div(c_in, 64) * 64);
    auto *xp = reinterpret_cast<_Float16 *>(at + mem.t);
    auto *xe = reinterpret_cast<int *>(at + mem.t + mem.x);
    if (ah) {
        lora::split_shrink(ctx, p, g.cip, xp, xe);
    } else {
        lora::run_shrink<float>(ctx, p);
        lora::split_rows(ctx, x, rows, c_in, g.cip, xp, xe);
    }
    g.xp = xp, g.x_exp = xe, g.w = weight, g.bias = bias, g.residual = residual;
    if (wt == kF32) {
        auto *wp = reinterpret_cast<_Float16 *>(at + mem.t + mem.x + mem.x_exp);
        auto *we = reinterpret_cast<int *>(at + mem.t + mem.x + mem.x_exp + mem.w);
        lora::split_rows(ctx, static_cast<const float *>(weight), c_out, c_in, g.cip, wp, we);
        g.w = wp, g.w_exp = we;
    }
    lora::gemm(ctx, g, wt, l.type);
}

}  // namespace mh
