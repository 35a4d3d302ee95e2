// Rotary positions over several axes, alone and behind the RMS norm of query and
// key heads. Pair (x0, x1) of a head at position p of its axis:
//   (y0, y1) = (x0 cos a - x1 sin a, x0 sin a + x1 cos a),  a = p . freq,
// with x replaced by x . rsqrt(mean x^2 + eps) . gamma first where there is a norm.
//
// Bound: memory, each value read and written once. A lane holds one unit of a head
// (16 bytes of pairs, two runs of 16 bytes where the pairs are the head's halves),
// a group of lanes the head, and the group takes several heads of one token, so the
// unit's cosines and sines are computed once for all of them.
//
// The angle in turns is reduced to an eighth of a turn in f64 (a position of 10^5
// times a frequency in f32 would be off by 10^-3 turns) and only the remainder's
// sine and cosine are f32. The sum of squares is f32 for f16 values, whose squares
// f32 holds, and f64 for f32 values, whose squares it may not.
//
// Measured on a card that copies at 5.1 TB/s: 16384 rows of 16 heads of 128, f16, 27.1 us
// (4.95 TB/s); with norms, 8192 rows of 8 + 8 heads of 160, f32, 37.3 us (4.5 TB/s); 64
// rows of 8 heads of 40 4.9 us, 8 rows of 32 + 8 heads with norms 6.2, both of a launch.
#include <algorithm>
#include <cmath>

#include "attention.hpp"

namespace mh {
namespace {

struct RopeArgs {
    const void *x[2];  // q (or x), k
    void *y[2];
    int64_t ldx[2], ldy[2];
    const float *gamma[2];
    int heads[2];   // heads[1] is 0 where there is one tensor
    int chunks[2];  // groups of `per` heads
    int per;        // heads per lane group
    const int32_t *pos;
    const double *freq;
    float eps;
    uint32_t rows, pos_rows;
    int d, axes, pairs;
    int e0, e1, e2;  // pair_end of the first three axes
    float sign;      // -1: the inverse rotation
    int rot_units, units;
};

// sin and cos of 2 pi turns: the quarter is taken off in f64, the remainder of at
// most an eighth by its Taylor series (next terms 2e-9 and 2e-10), in f32.
__device__ __forceinline__ void sincos_turns(double turns, float &s, float &c) {
    const double t = turns - __builtin_rint(turns);
    const double k = __builtin_rint(4.0 * t);
    const float r = float(__builtin_fma(-0.25, k, t));
    const float z = r * r;
    float p = 42.0586939449f;
    p = __builtin_fmaf(p, z, -76.7058597531f);
    p = __builtin_fmaf(p, z, 81.6052492761f);
    p = __builtin_fmaf(p, z, -41.3417022404f);
    const float sr = r * __builtin_fmaf(p, z, 6.28318530718f);
    float q = -26.4262567834f;
    q = __builtin_fmaf(q, z, 60.2446413719f);
    q = __builtin_fmaf(q, z, -85.4568172067f);
    q = __builtin_fmaf(q, z, 64.9393940227f);
    q = __builtin_fmaf(q, z, -19.7392088022f);
    const float cr = __builtin_fmaf(q, z, 1.0f);
    const int n = int(k) & 3;  // -2 .. 2
    const float a = (n & 1) ? cr : sr, b = (n & 1) ? sr : cr;
    s = (n & 2) ? -a : a;
    c = (n == 1 || n == 2) ? -b : b;
}

template <typename T, int W>
struct Vec {
    typedef T V __attribute__((ext_vector_type(W)));
    static __device__ __forceinline__ void load(const T *p, float (&v)[W]) {
        const V r = *reinterpret_cast<const V *>(p);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = float(r[i]);
    }
    static __device__ __forceinline__ void store(T *p, const float (&v)[W]) {
        V r;
#pragma unroll
        for (int i = 0; i < W; ++i) r[i] = static_cast<T>(v[i]);
        *reinterpret_cast<V *>(p) = r;
    }
};

template <typename T>
struct Vec<T, 1> {
    static __device__ __forceinline__ void load(const T *p, float (&v)[1]) { v[0] = float(*p); }
    static __device__ __forceinline__ void store(T *p, const float (&v)[1]) { *p = static_cast<T>(v[0]); }
};

// A unit's values: W channels at `lo` and W at `hi`. Halves: pair i is (a[i], b[i]),
// channels apart by the number of pairs. Interleaved: 2 W consecutive channels for
// W = 1, else the pairs lie within each run of W and only `lo` is there. Channels
// behind the pairs: one run of W, no rotation.
template <int W, bool HALVES>
struct Unit {
    static constexpr bool kTwo = HALVES || W == 1;   // runs of a rotated unit
    static constexpr int kPairs = kTwo ? W : W / 2;  // pairs of a rotated unit
    int lo, hi;                                      // channels of the runs, hi -1: none
    int pair;                                        // first pair, -1: no rotation
    __device__ __forceinline__ void at(int u, const RopeArgs &a) {
        if (u < a.rot_units) {
            pair = u * kPairs;
            lo = HALVES ? pair : 2 * pair;
            hi = !kTwo ? -1 : HALVES ? a.pairs + pair : lo + 1;
        } else {
            pair = -1;
            lo = 2 * a.pairs + (u - a.rot_units) * W;
            hi = -1;
        }
    }
};

template <int N>
__device__ __forceinline__ void angles(const RopeArgs &a, uint32_t row, int pair, float (&s)[N], float (&c)[N]) {
    const int32_t *p = a.pos + int64_t(row % a.pos_rows) * a.axes;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int pi = pair + i;
        const int axis = (pi >= a.e0) + (pi >= a.e1) + (pi >= a.e2);
        sincos_turns(double(p[axis]) * (a.freq[pi] * 0.15915494309189533577), s[i], c[i]);
        s[i] *= a.sign;
    }
}

template <int W, bool HALVES, int N>
__device__ __forceinline__ void turn(float (&x)[W], float (&y)[W], const float (&s)[N], const float (&c)[N]) {
    if constexpr (Unit<W, HALVES>::kTwo) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float u = x[i], v = y[i];
            x[i] = __builtin_fmaf(u, c[i], -(v * s[i]));
            y[i] = __builtin_fmaf(u, s[i], v * c[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
            const float u = x[2 * i], v = x[2 * i + 1];
            x[2 * i] = __builtin_fmaf(u, c[i], -(v * s[i]));
            x[2 * i + 1] = __builtin_fmaf(u, s[i], v * c[i]);
        }
    }
}

// Sum of squares: f16 values in f32, f32 values in f64.
template <typename T>
struct Sum {
    typedef double S;
};
template <>
struct Sum<_Float16> {
    typedef float S;
};

template <typename S>
__device__ __forceinline__ S group_sum(S v, int lanes) {
    for (int m = lanes / 2; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

__device__ __forceinline__ float norm_scale(float sum, float eps, int d) {
    return 1.0f / sqrtf(sum / float(d) + eps);
}
__device__ __forceinline__ double norm_scale(double sum, float eps, int d) {
    return 1.0 / sqrt(sum / double(d) + double(eps));
}

// One lane group of GL lanes per (row, chunk of `per` heads). ONE: a lane's unit is
// its only one (units <= GL), its values, cosines and sines stay in registers and
// HU heads are in flight; else the units of a head are walked, twice where there is
// a norm.
template <typename T, int W, bool HALVES, bool NORM, bool ONE, int GL>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    using U = Unit<W, HALVES>;
    using L = Vec<T, W>;
    using S = typename Sum<T>::S;
    const uint32_t lane = threadIdx.x % GL;
    const uint64_t group = uint64_t(blockIdx.x) * (256 / GL) + threadIdx.x / GL;
    const uint32_t chunks = uint32_t(a.chunks[0] + a.chunks[1]);
    const uint64_t row64 = group / chunks;
    if (row64 >= a.rows) return;
    const uint32_t row = uint32_t(row64);
    const int chunk = int(group - row64 * chunks);
    const int side = NORM && chunk >= a.chunks[0];
    const int h0 = (side ? chunk - a.chunks[0] : chunk) * a.per;
    const int h1 = min(h0 + a.per, a.heads[side]);
    const T *x = static_cast<const T *>(a.x[side]) + int64_t(row) * a.ldx[side];
    T *y = static_cast<T *>(a.y[side]) + int64_t(row) * a.ldy[side];
    const float *gamma = a.gamma[side];
    if constexpr (ONE) {
        constexpr int HU = 4;
        U u;
        const bool live = int(lane) < a.units;
        u.at(live ? int(lane) : a.units - 1, a);
        float s[U::kPairs], c[U::kPairs];
        const bool rotated = u.pair >= 0;
        if (rotated) angles<U::kPairs>(a, row, u.pair, s, c);
        float ga[W], gb[W];
        if constexpr (NORM) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                ga[i] = gamma ? gamma[u.lo + i] : 1.0f;
                gb[i] = gamma && u.hi >= 0 ? gamma[u.hi + i] : 1.0f;
            }
        }
        for (int h = h0; h < h1; h += HU) {
            float p[HU][W], q[HU][W];
#pragma unroll
            for (int j = 0; j < HU; ++j) {
                const T *xh = x + int64_t(min(h + j, h1 - 1)) * a.d;
                L::load(xh + u.lo, p[j]);
                if constexpr (U::kTwo)
                    if (u.hi >= 0) L::load(xh + u.hi, q[j]);
            }
            if constexpr (NORM) {
                S sum[HU];
#pragma unroll
                for (int j = 0; j < HU; ++j) {
                    sum[j] = 0;
                    if (live) {
#pragma unroll
                        for (int i = 0; i < W; ++i) {
                            sum[j] += S(p[j][i]) * S(p[j][i]);
                            if constexpr (U::kTwo)
                                if (u.hi >= 0) sum[j] += S(q[j][i]) * S(q[j][i]);
                        }
                    }
                }
#pragma unroll
                for (int m = GL / 2; m; m >>= 1)
#pragma unroll
                    for (int j = 0; j < HU; ++j) sum[j] += __shfl_xor(sum[j], m);
#pragma unroll
                for (int j = 0; j < HU; ++j) {
                    const S r = norm_scale(sum[j], a.eps, a.d);
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        p[j][i] = float(S(p[j][i]) * r) * ga[i];
                        if constexpr (U::kTwo) q[j][i] = float(S(q[j][i]) * r) * gb[i];
                    }
                }
            }
            if (!live) continue;
#pragma unroll
            for (int j = 0; j < HU; ++j) {
                if (h + j >= h1) break;
                T *yh = y + int64_t(h + j) * a.d;
                if (rotated) turn<W, HALVES>(p[j], q[j], s, c);
                L::store(yh + u.lo, p[j]);
                if constexpr (U::kTwo)
                    if (u.hi >= 0) L::store(yh + u.hi, q[j]);
            }
        }
    } else {
        for (int h = h0; h < h1; ++h) {
            const T *xh = x + int64_t(h) * a.d;
            T *yh = y + int64_t(h) * a.d;
            S r = 1;
            if constexpr (NORM) {
                S sum = 0;
                for (int ch = int(lane); ch < a.d; ch += GL) {
                    const S v = S(float(xh[ch]));
                    sum += v * v;
                }
                r = norm_scale(group_sum(sum, GL), a.eps, a.d);
            }
            for (int n = int(lane); n < a.units; n += GL) {
                U u;
                u.at(n, a);
                float p[W], q[W] = {};
                L::load(xh + u.lo, p);
                if constexpr (U::kTwo)
                    if (u.hi >= 0) L::load(xh + u.hi, q);
                if constexpr (NORM) {
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        p[i] = float(S(p[i]) * r) * (gamma ? gamma[u.lo + i] : 1.0f);
                        if (u.hi >= 0) q[i] = float(S(q[i]) * r) * (gamma ? gamma[u.hi + i] : 1.0f);
                    }
                }
                if (u.pair >= 0) {
                    float s[U::kPairs], c[U::kPairs];
                    angles<U::kPairs>(a, row, u.pair, s, c);
                    turn<W, HALVES>(p, q, s, c);
                }
                L::store(yh + u.lo, p);
                if constexpr (U::kTwo)
                    if (u.hi >= 0) L::store(yh + u.hi, q);
            }
        }
    }
}

template <typename T, int W, bool HALVES, bool NORM>
void launch_w(Context &ctx, RopeArgs &a) {
    using U = Unit<W, HALVES>;
    a.rot_units = a.pairs / U::kPairs;
    a.units = a.rot_units + (a.d - 2 * a.pairs) / W;
    const int gl = a.units <= 8 ? 8 : a.units <= 16 ? 16 : a.units <= 32 ? 32 : 64;
    // Heads per lane group: all of them share the unit's cosines, but the card wants
    // about 16 waves on every CU first. 24 heads of 128, 16384 rows, f16: 1 56.9 us, 2 35.5,
    // 4 or more 32; 8 heads, 64 rows: 5 us each way.
    const int most = std::max(a.heads[0], a.heads[1]);
    const int64_t want = int64_t(ctx.cu_count) * 16 * 64;
    a.per = int(std::max<int64_t>(1, std::min<int64_t>(most, int64_t(a.rows) * (a.heads[0] + a.heads[1]) * gl / want)));
    for (int i = 0; i < 2; ++i) a.chunks[i] = int(ceil_div(a.heads[i], a.per));
    const int64_t groups = int64_t(a.rows) * (a.chunks[0] + a.chunks[1]);
    const int64_t blocks = ceil_div(groups, 256 / gl);
    MH_REQUIRE(blocks < (int64_t(1) << 31), "rope: too many heads");
    const dim3 grid{uint32_t(blocks)}, block{256};
    if (a.units > 64) {
        if constexpr (W == 1) rope_kernel<T, W, HALVES, NORM, false, 64><<<grid, block, 0, ctx.stream>>>(a);
    } else if (gl == 8) {
        rope_kernel<T, W, HALVES, NORM, true, 8><<<grid, block, 0, ctx.stream>>>(a);
    } else if (gl == 16) {
        rope_kernel<T, W, HALVES, NORM, true, 16><<<grid, block, 0, ctx.stream>>>(a);
    } else if (gl == 32) {
        rope_kernel<T, W, HALVES, NORM, true, 32><<<grid, block, 0, ctx.stream>>>(a);
    } else {
        rope_kernel<T, W, HALVES, NORM, true, 64><<<grid, block, 0, ctx.stream>>>(a);
    }
    MH_LAUNCH_CHECK();
}

template <typename T, bool HALVES, bool NORM>
void launch(Context &ctx, RopeArgs &a) {
    constexpr int V = 16 / int(sizeof(T));
    // The widest run that every unit, row and base keeps aligned, if a head is then one
    // unit per lane; single channels otherwise.
    auto fits = [&](int w) {
        const int64_t bytes = int64_t(w) * int64_t(sizeof(T));
        const int rest = a.d - 2 * a.pairs;
        if ((HALVES ? a.pairs % w : 2 * a.pairs % w) || rest % w || a.d % w) return false;
        if (a.pairs / (HALVES ? w : w / 2) + rest / w > 64) return false;
        for (int i = 0; i < 2; ++i) {
            if (!a.heads[i]) continue;
            if (a.ldx[i] % w || a.ldy[i] % w) return false;
            if (reinterpret_cast<uintptr_t>(a.x[i]) % bytes || reinterpret_cast<uintptr_t>(a.y[i]) % bytes) return false;
        }
        return true;
    };
    if (fits(V)) launch_w<T, V, HALVES, NORM>(ctx, a);
    else if (fits(V / 2)) launch_w<T, V / 2, HALVES, NORM>(ctx, a);
    else launch_w<T, 1, HALVES, NORM>(ctx, a);
}

template <bool NORM>
void dispatch(Context &ctx, WeightType type, const RopeTable &t, RopeArgs &a) {
    const bool halves = t.pairing == RopePairing::Halves;
    if (type == kF16) {
        if (halves) launch<_Float16, true, NORM>(ctx, a);
        else launch<_Float16, false, NORM>(ctx, a);
    } else {
        if (halves) launch<float, true, NORM>(ctx, a);
        else launch<float, false, NORM>(ctx, a);
    }
}

RopeArgs base_args(int64_t rows, int d, const RopeTable &t) {
    RopeArgs a{};
    a.pos = t.pos;
    a.freq = t.freq;
    a.rows = uint32_t(rows);
    a.pos_rows = uint32_t(std::min<int64_t>(t.pos_rows, 0xFFFFFFFFll));
    a.d = d;
    a.axes = t.axes;
    a.pairs = t.pair_end[t.axes - 1];
    a.e0 = t.pair_end[0];
    a.e1 = t.axes > 1 ? t.pair_end[1] : a.pairs;
    a.e2 = t.axes > 2 ? t.pair_end[2] : a.pairs;
    a.sign = t.inverse ? -1.0f : 1.0f;
    return a;
}

}  // namespace

void rope_frequencies(double theta, int axes, const uint32_t *axis_dims, double *freq) {
    for (int a = 0; a < axes; ++a)
        for (uint32_t i = 0; i < axis_dims[a] / 2; ++i)
            *freq++ = std::pow(theta, -2.0 * double(i) / double(axis_dims[a]));
}

void rope_axes(Context &ctx, HeadRows x, WeightType type, int64_t rows, int d, const RopeTable &t, void *out,
               int64_t ld_out) {
    if (!rows) return;
    RopeArgs a = base_args(rows, d, t);
    a.x[0] = x.p, a.y[0] = out, a.ldx[0] = x.ld, a.ldy[0] = ld_out, a.heads[0] = x.heads;
    dispatch<false>(ctx, type, t, a);
}

void qk_norm_rope(Context &ctx, HeadRows q, HeadRows k, WeightType type, int64_t rows, int d, const float *gamma_q,
                  const float *gamma_k, float eps, const RopeTable &t, void *q_out, int64_t ld_qo, void *k_out,
                  int64_t ld_ko) {
    if (!rows) return;
    RopeArgs a = base_args(rows, d, t);
    a.x[0] = q.p, a.y[0] = q_out, a.ldx[0] = q.ld, a.ldy[0] = ld_qo, a.heads[0] = q.heads, a.gamma[0] = gamma_q;
    a.x[1] = k.p, a.y[1] = k_out, a.ldx[1] = k.ld, a.ldy[1] = ld_ko, a.heads[1] = k.heads, a.gamma[1] = gamma_k;
    a.eps = eps;
    dispatch<true>(ctx, type, t, a);
}

}  // namespace mh
