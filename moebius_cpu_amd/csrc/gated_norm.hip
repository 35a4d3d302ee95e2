// The gated residual of a branch and the modulated norm of the sum.
//
// s = keep x + gate post(branch), y = pre(s) (1 + scale) + shift, where a norm is
// (v - mean) / sqrt(mean((v - mean)^2) + eps) gamma + beta, or without the mean. The sums are
// f32 over values that stay in registers, the mean taken first and the squares of what is left
// after it, so that a large mean costs no bits; x_out and y are each rounded once, y from the
// sum as it is before x_out is rounded.
//
// Bound: memory; every array is read or written once, the vectors of the norms and of the item
// from the caches. 16384 rows of 2048, f32 with f16 branches: 79 us (5.1 TB/s) without vectors,
// 87 with the norms' two, 97 with the item's three more; two rows to a group, which reads them
// half as often, 106.
#include <type_traits>

#include "gated_norm.hpp"

namespace mh {
namespace {

template <typename T, bool VEC>
struct Four {
    typedef T V __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ void load(const void *row, int ch, int c, float (&x)[4]) {
        const T *p = static_cast<const T *>(row) + ch;
        if constexpr (VEC) {
            const V v = *reinterpret_cast<const V *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = float(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = ch + i < c ? float(p[i]) : 0.0f;
        }
    }
    static __device__ __forceinline__ void store(void *row, int ch, int c, const float (&x)[4]) {
        T *p = static_cast<T *>(row) + ch;
        if constexpr (VEC) {
            V v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = static_cast<T>(x[i]);
            *reinterpret_cast<V *>(p) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (ch + i < c) p[i] = static_cast<T>(x[i]);
        }
    }
};

// The sum over the threads of a row, in the same order on all of them.
template <int NT>
__device__ __forceinline__ float row_sum(float v, float *red) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) v += __shfl_xor(v, o);
    if constexpr (NT > 64) {
        __syncthreads();  // the sum before has been read
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) v += red[i];
    }
    return v;
}

template <int NT, int R, bool VEC>
__device__ __forceinline__ void norm_row(float (&v)[R][4], const NormSpec &n, int c, int tid, float *red) {
    const float size = float(c);
    if (n.kind == NormKind::None) return;
    if (n.kind == NormKind::Layer) {
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += v[r][i];
        const float mean = row_sum<NT>(sum, red) / size;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[r][i] = (r * NT + tid) * 4 + i < c ? v[r][i] - mean : 0.0f;
    }
    float sq = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) sq = __builtin_fmaf(v[r][i], v[r][i], sq);
    const float inv = 1.0f / __builtin_sqrtf(row_sum<NT>(sq, red) / size + n.eps);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int ch = (r * NT + tid) * 4;
        if (ch >= c) continue;
        float g[4] = {1.0f, 1.0f, 1.0f, 1.0f}, b[4] = {};
        if (n.gamma) Four<float, VEC>::load(n.gamma, ch, c, g);
        if (n.beta) Four<float, VEC>::load(n.beta, ch, c, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[r][i] = __builtin_fmaf(v[r][i] * inv, g[i], b[i]);
    }
}

// NT threads per row (64: four rows per workgroup), R runs of 4 channels each.
template <typename TX, typename TH, bool VEC, int NT, int R>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void gated_norm_kernel(GatedNorm a) {
    __shared__ float red[NT > 64 ? NT / 64 : 1];
    const int tid = NT == 64 ? int(threadIdx.x & 63) : int(threadIdx.x);
    const int64_t row = NT == 64 ? int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6) : int64_t(blockIdx.x);
    if (row >= a.rows) return;
    const int64_t item = uint32_t(row) / uint32_t(a.rows_per_item);
    const TX *x = static_cast<const TX *>(a.x) + row * a.ld_x;
    float s[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int ch = (r * NT + tid) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[r][i] = 0.0f;
        if (ch < a.c) Four<TX, VEC>::load(x, ch, a.c, s[r]);
    }
    if (a.branch) {
        const TH *h = static_cast<const TH *>(a.branch) + row * a.ld_branch;
        float v[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int ch = (r * NT + tid) * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[r][i] = 0.0f;
            if (ch < a.c) Four<TH, VEC>::load(h, ch, a.c, v[r]);
        }
        norm_row<NT, R, VEC>(v, a.post, a.c, tid, red);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int ch = (r * NT + tid) * 4;
            if (ch >= a.c) continue;
            float g[4] = {1.0f, 1.0f, 1.0f, 1.0f};
            if (a.gate.p) Four<float, VEC>::load(a.gate.p + item * a.gate.ld, ch, a.c, g);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[r][i] = __builtin_fmaf(g[i], v[r][i], a.keep * s[r][i]);
        }
    }
    if constexpr (!VEC) {  // (a run that the row ends in adds nothing to the sums)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if ((r * NT + tid) * 4 + i >= a.c) s[r][i] = 0.0f;
    }
    if (a.x_out) {
        TX *o = static_cast<TX *>(a.x_out) + row * a.ld_x_out;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int ch = (r * NT + tid) * 4;
            if (ch < a.c) Four<TX, VEC>::store(o, ch, a.c, s[r]);
        }
    }
    if (!a.y) return;
    norm_row<NT, R, VEC>(s, a.pre, a.c, tid, red);
    TH *y = static_cast<TH *>(a.y) + row * a.ld_y;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int ch = (r * NT + tid) * 4;
        if (ch >= a.c) continue;
        float m[4] = {}, b[4] = {};
        if (a.scale.p) Four<float, VEC>::load(a.scale.p + item * a.scale.ld, ch, a.c, m);
        if (a.shift.p) Four<float, VEC>::load(a.shift.p + item * a.shift.ld, ch, a.c, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[r][i] = __builtin_fmaf(s[r][i], 1.0f + m[i], b[i]);
        Four<TH, VEC>::store(y, ch, a.c, s[r]);
    }
}

// Threads per row, up to 16 values of each: a wave up to 768 channels, two to 2048, four to 4096,
// eight to 8192, sixteen beyond. 16384 rows of 2048, f32 with f16 branches, both norms and all
// vectors: one wave 113 us, two 97, four 99, eight 107; 65536 of 512: 88, 90, 129, 215; 8192 of 1280,
// f32, LayerNorm: 28.3, 29.2, 30.7, 31.8 (16384 with f16 branches 50.8, 48.2, 49.0, 59.6).
template <typename TX, typename TH, bool VEC>
void launch(Context &ctx, const GatedNorm &a) {
    using std::integral_constant;
    auto go = [&](auto nt, auto r) {
        constexpr int NT = decltype(nt)::value, R = decltype(r)::value, kGroups = NT == 64 ? 4 : 1;
        const dim3 grid{uint32_t(ceil_div(a.rows, kGroups))};
        gated_norm_kernel<TX, TH, VEC, NT, R><<<grid, dim3{uint32_t(NT * kGroups)}, 0, ctx.stream>>>(a);
    };
    auto by_runs = [&](auto nt) {
        const int64_t runs = ceil_div(a.c, 4 * decltype(nt)::value);
        if (runs <= 1) go(nt, integral_constant<int, 1>{});
        else if (runs <= 2) go(nt, integral_constant<int, 2>{});
        else if (runs <= 3) go(nt, integral_constant<int, 3>{});
        else go(nt, integral_constant<int, 4>{});
    };
    if (a.c <= 768) by_runs(integral_constant<int, 64>{});
    else if (a.c <= 2048) by_runs(integral_constant<int, 128>{});
    else if (a.c <= 4096) by_runs(integral_constant<int, 256>{});
    else if (a.c <= 8192) by_runs(integral_constant<int, 512>{});
    else if (a.c <= 16384) by_runs(integral_constant<int, 1024>{});
    else go(integral_constant<int, 1024>{}, integral_constant<int, 8>{});
    MH_LAUNCH_CHECK();
}

bool wide(const void *p, int64_t ld, int size) { return !p || (reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && ld % 4 == 0); }

}  // namespace

void gated_norm(Context &ctx, const GatedNorm &a) {
    if (!a.rows) return;
    const int xs = a.x_type == kF16 ? 2 : 4, hs = a.branch_type == kF16 ? 2 : 4;
    const bool vec = a.c % 4 == 0 && wide(a.x, a.ld_x, xs) && wide(a.x_out, a.ld_x_out, xs) &&
                     wide(a.branch, a.ld_branch, hs) && wide(a.y, a.ld_y, hs) && wide(a.gate.p, a.gate.ld, 4) &&
                     wide(a.scale.p, a.scale.ld, 4) && wide(a.shift.p, a.shift.ld, 4) && aligned16(a.post.gamma) &&
                     aligned16(a.post.beta) && aligned16(a.pre.gamma) && aligned16(a.pre.beta);
    auto by_type = [&](auto v) {
        constexpr bool V = decltype(v)::value;
        if (a.x_type == kF16) {
            if (a.branch_type == kF16) launch<_Float16, _Float16, V>(ctx, a);
            else launch<_Float16, float, V>(ctx, a);
        } else {
            if (a.branch_type == kF16) launch<float, _Float16, V>(ctx, a);
            else launch<float, float, V>(ctx, a);
        }
    };
    if (vec) by_type(std::true_type{});
    else by_type(std::false_type{});
}

}  // namespace mh
