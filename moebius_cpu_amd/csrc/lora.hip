// Low-rank adapters of many requests beside a shared 1x1 projection:
//   y = x W^T + bias + residual + scale_s (x A_s^T) B_s^T,  s the row's adapter.
//
// The adapters' products keep f32's accuracy in EXACT and FAST contexts alike: at rank r they
// are r (c_in + c_out) of the projection's c_in c_out operations. Few rows take two passes of
// f32 products:
//   row shrink: t = x A_s^T [rows][rank], a wave per rank of a row;
//   row project: x W^T in tiles of 16 x 16, finished with bias, residual and scale_s t B_s^T.
// More rows take the product of lora_gemm.hip behind one pass over x, which forms t as well:
// with adapters stored in f16 by f16 products of x and t in two parts, with f32 ones by f32
// products (and x split in a pass of its own).
//
// A tile of 16 rows takes the adapters its rows name one after another, each product
// over all 16 rows and kept for its own: rows of one image share one, single tokens of
// 16 requests read 16 adapters, which each has to be read anyway. Rows of other adapters
// are selected away, not multiplied by zero, so values that are not finite stay with
// their own requests.
#include <algorithm>
#include <type_traits>

#include "lora.hpp"

namespace mh {
namespace lora {
namespace {

constexpr int kRankTiles = 4;     // 16 ranks each per pass over x
constexpr int kShrinkUnroll = 5;  // steps of the long axis whose loads are in flight together
constexpr int kShrinkWaves = 8;

// Adapters stored in f32: a workgroup takes 16 rows, wave w an eighth of the long axis.
// Lane l holds row (rank) l % 16 and four values of the long axis at 4 (l / 16).
template <bool VEC>
__global__ __launch_bounds__(64 * kShrinkWaves) void lora_shrink_kernel(LoraArgs p) {
    __shared__ float part[kShrinkWaves][kRankTiles][4][64];
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t r0 = int64_t(blockIdx.x) * 16;
    const int share = ((p.ci + 15) / 16 + kShrinkWaves - 1) / kShrinkWaves * 16;
    const int k0 = wave * share, ke = min(k0 + share, p.ci);
    const int mine = slot_of(p, r0 + r16);
    const float *x = p.x + min(r0 + r16, p.rows - 1) * p.ci;
    uint32_t todo = uint32_t(__ballot(mine >= 0)) & 0xFFFFu;
    while (todo) {
        const int s = __shfl(mine, __builtin_ctz(todo));
        const bool own = mine == s;
        todo &= ~uint32_t(__ballot(own));
        for (int q0 = 0; q0 < p.rank; q0 += 16 * kRankTiles) {
            floatx4 acc[kRankTiles];
            const float *a[kRankTiles];
#pragma unroll
            for (int j = 0; j < kRankTiles; ++j) {
                acc[j] = floatx4{0, 0, 0, 0};
                a[j] = static_cast<const float *>(p.a) + (int64_t(s) * p.rank + min(q0 + j * 16 + r16, p.rank - 1)) * p.ci;
            }
            for (int k = k0; k < ke; k += 16 * kShrinkUnroll) {
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
                *reinterpret_cast<floatx4 *>(p.t + (r0 + r16) * p.rank_pad + q) = v;
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
        auto second = [&](auto vec) {
            constexpr bool V = decltype(vec)::value;
            for (int k = 0; k < p.rank; k += 16) {
                floatx4 bv[4], tv[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    bv[u] = load4<V>(b, k + 4 * u, p.rank);
                    tv[u] = load4<V>(t, k + 4 * u, p.rank);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) y = __builtin_fmaf(tv[u][i], bv[u][i], y);
            }
        };
        if (p.rank % 4 == 0 && reinterpret_cast<uintptr_t>(p.b) % (4 * sizeof(T)) == 0) second(std::true_type{});
        else second(std::false_type{});
        v = __builtin_fmaf(scale, y, v);
    }
    p.out[row * p.co + c] = v;
}

// Whether the two passes over few rows are taken: they cost 10 us and 4.7 us more for every
// 256 tiles of 16 x 16 behind the first (at c_in 1280), the other way two thirds more to
// begin with. 1280 x 1280, f16 / f32 weight, us against that: 16 rows 9.8 / 9.8 (22 / 30),
// 96 rows 14.8 / 14.7 (23 / 33), 128 rows 19.5 / 19.7 (23 / 34), 256 rows 30 / 30 (23 / 35);
// 320 x 320, 256 rows 14.6 / 14.6 (15.8 / 17.8), 512 rows 20.7 / 20.1 (15.8 / 17.9). The first
// pass reads an adapter per row: rank 256, 640 x 64, 256 rows 31 us (67), 512 rows 48 (50).
bool few_rows(const Context &ctx, int64_t rows, int c_out, WeightType wt, int rank) {
    return rows * rank <= 1 << 16 && ceil_div(rows, 16) * ceil_div(c_out, 16) <= (wt == kF32 ? 3 : 2) * ctx.cu_count;
}

void run_shrink(Context &ctx, const LoraArgs &p) {
    const dim3 grid{uint32_t(ceil_div(p.rows, 16))}, tb{64 * kShrinkWaves};
    if (p.ci % 4 == 0 && aligned16(p.x) && aligned16(p.a)) lora_shrink_kernel<true><<<grid, tb, 0, ctx.stream>>>(p);
    else lora_shrink_kernel<false><<<grid, tb, 0, ctx.stream>>>(p);
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

// FAST rounds the projection's operands to f16.
int parts_of(const Context &ctx) { return ctx.precision == Precision::Fast ? 1 : 2; }

// Scratch: t, then the parts of x and their exponents, then those of an f32 weight.
struct Layout {
    size_t t = 0, x = 0, x_exp = 0, w = 0, w_exp = 0;
    size_t total() const { return t + x + x_exp + w + w_exp; }
};

Layout layout(const Context &ctx, int64_t rows, int c_in, int c_out, WeightType wt, int rank) {
    auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
    Layout l;
    l.t = up(size_t(rows) * size_t(ceil_div(rank, 16) * 16) * sizeof(float));
    if (few_rows(ctx, rows, c_out, wt, rank)) return l;
    const size_t row = size_t(parts_of(ctx)) * padded_channels(c_in) * sizeof(_Float16);
    l.x = up(size_t(padded_rows(rows)) * row);
    l.x_exp = up(size_t(rows) * sizeof(int));
    if (wt == kF32) {
        l.w = up(size_t(c_out) * row);
        l.w_exp = up(size_t(c_out) * sizeof(int));
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
    const lora::Layout mem = lora::layout(ctx, rows, c_in, c_out, wt, l.rank);
    char *at = static_cast<char *>(scratch ? scratch : ctx.ws.get(mem.total(), ctx.stream));
    lora::LoraArgs p{};
    p.x = x, p.a = l.a, p.b = l.b, p.scale = l.scale, p.slot = l.slot, p.out = out;
    p.t = reinterpret_cast<float *>(at);
    p.rows = rows, p.rows_per_slot = l.rows_per_slot;
    p.ci = c_in, p.co = c_out, p.rank = l.rank, p.slots = l.slots;
    p.rank_pad = int(ceil_div(l.rank, 16) * 16);
    const bool ah = l.type == kF16;
    if (lora::few_rows(ctx, rows, c_out, wt, l.rank)) {
        if (wt == kF16 && ah) lora::run_few<_Float16, _Float16>(ctx, p, weight, bias, residual);
        else if (wt == kF16) lora::run_few<_Float16, float>(ctx, p, weight, bias, residual);
        else if (ah) lora::run_few<float, _Float16>(ctx, p, weight, bias, residual);
        else lora::run_few<float, float>(ctx, p, weight, bias, residual);
        return;
    }
    const int nparts = lora::parts_of(ctx);
    lora::GemmArgs g{};
    g.l = p;
    g.cip = lora::padded_channels(c_in);
    auto *xp = reinterpret_cast<_Float16 *>(at + mem.t);
    auto *xe = reinterpret_cast<int *>(at + mem.t + mem.x);
    g.xp = xp, g.x_exp = xe, g.w = weight, g.bias = bias, g.residual = residual;
    lora::SplitRows xs, ws;
    if (ah) {
        lora::split_shrink(ctx, p, g.cip, nparts, xp, xe);
    } else {
        lora::run_shrink(ctx, p);
        xs = {x, rows, xp, xe};
    }
    if (wt == kF32) {
        auto *wp = reinterpret_cast<_Float16 *>(at + mem.t + mem.x + mem.x_exp);
        auto *we = reinterpret_cast<int *>(at + mem.t + mem.x + mem.x_exp + mem.w);
        ws = {static_cast<const float *>(weight), c_out, wp, we};
        g.w = wp, g.w_exp = we;
    }
    if (xs.rows || ws.rows) lora::split_rows(ctx, xs, ws, c_in, g.cip, nparts);
    lora::gemm(ctx, g, nparts, wt, l.type);
}

}  // namespace mh
