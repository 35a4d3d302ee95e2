// The projection of many rows with the adapters' second product in its epilogue.
//
// f32 products at the f16 matrix rate: x = hi + lo, two f16 parts that hold 24 bits of
// values down to 2^-18 of their row's largest (split_rows scales each row by a power of
// two), so x W^T takes two f16 products where W is stored in f16 and three where it is f32
// and split alike (lo . lo is below 2^-24 of its product). Sums are f32. An eighth of the
// f32 instructions' time and a third of six bf16 products'.
//
// An infinite value is all in its first part. Its products with the second parts of others are
// NaN (of zeros) or of either sign, those with first parts what the whole products are: sums
// that are NaN are formed again from first parts alone. 4096 rows, 1280 x 1280, NaN in every row
// 154 us against 64, infinities in every row and an f32 weight 230 against 86.
//
// FAST contexts take one part (operands rounded to f16 after their row's scale).
//
// A workgroup forms BM columns x BN rows, four waves the 2 x 2 quarters, as W . X^T: a lane
// of a 32x32 result holds one row and four runs of four columns, so a row's scale and its
// adapter are the lane's own. 64 of the long axis are staged in LDS at a time while the
// next are loaded; where the tiles are too few to hide those loads in each other, two or
// four such groups of waves share the long axis. Bound: the matrix instructions; the parts
// of x are written and read once more than x itself.
//
// Measured: 8192 rows, 1280 x 1280, f16 weight, rank 32, residual: 118 us, of it 88 the
// product (54 GFLOP in two f16 products: 611 TFLOP/s; 75 us without residual and adapters)
// and 24 the pass over x.
#include <algorithm>

#include "lora.hpp"

namespace mh {
namespace lora {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

// A wave per row, its values in registers up to kHold runs of 8 per lane.
constexpr int kHold = 4;
template <bool VEC, int P>
__global__ __launch_bounds__(256) void split_rows_kernel(SplitRows s0, SplitRows s1, int ci, int cip) {
    const int lane = threadIdx.x & 63;
    const int64_t at = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6), row = at < s0.rows ? at : at - s0.rows;
    const SplitRows &s = at < s0.rows ? s0 : s1;
    if (row >= s.rows) return;
    const float *x = s.x;
    _Float16 *parts = s.parts;
    int *exps = s.exps;
    const float *src = x + row * ci;
    _Float16 *dst = parts + row * P * cip;
    floatx4 v[kHold][2];
    float mx = 0.0f;
    auto scan = [&](const floatx4 &a) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float f = __builtin_fabsf(a[e]);
            mx = f < __builtin_huge_valf() ? __builtin_fmaxf(mx, f) : mx;
        }
    };
    const int runs = cip / 8;
#pragma unroll
    for (int i = 0; i < kHold; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            v[i][j] = load4<VEC>(src, (i * 64 + lane) * 8 + j * 4, ci);
            scan(v[i][j]);
        }
    for (int r = kHold * 64 + lane; r < runs; r += 64)
#pragma unroll
        for (int j = 0; j < 2; ++j) scan(load4<VEC>(src, r * 8 + j * 4, ci));
#pragma unroll
    for (int m = 32; m; m >>= 1) mx = __builtin_fmaxf(mx, __shfl_xor(mx, m));
    const int e = top_exp(mx);
    auto put = [&](int r, const floatx4 &a, const floatx4 &b) {
        halfx8 hi, lo;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            _Float16 p, q;
            split2(c < 4 ? a[c] : b[c - 4], kSplitExp - e, p, q);
            hi[c] = p, lo[c] = q;
        }
        *reinterpret_cast<halfx8 *>(dst + r * 8) = hi;
        if constexpr (P == 2) *reinterpret_cast<halfx8 *>(dst + cip + r * 8) = lo;
    };
#pragma unroll
    for (int i = 0; i < kHold; ++i)
        if (i * 64 + lane < runs) put(i * 64 + lane, v[i][0], v[i][1]);
    for (int r = kHold * 64 + lane; r < runs; r += 64) put(r, load4<VEC>(src, r * 8, ci), load4<VEC>(src, r * 8 + 4, ci));
    if (lane == 0) exps[row] = e;
}

template <bool VEC>
__device__ __forceinline__ halfx8 load8(const _Float16 *p, int k, int n) {
    return load_run<8, VEC>(p, k, n);
}

__device__ __forceinline__ floatx16 mfma16(halfx8 a, halfx8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

typedef floatx4 accx4;

// The sums of a 32 x 32 result that are NaN, from `again` where the row counts (want).
template <typename F>
__device__ __forceinline__ void redo_nan(floatx16 &acc, bool want, F again) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) any = any || acc[i] != acc[i];
    if (!__any(any && want)) return;
    floatx16 sum;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.0f;
    again(sum);
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = acc[i] == acc[i] ? acc[i] : sum[i];
}

// split_rows and the adapters' first product of 16 rows in one pass over x, for adapters
// stored in f16: t = 2^-e (hi A^T + lo A^T) on v_mfma_f32_16x16x32_f16. Eight waves share
// the long axis, 32 values of 16 rows per step (lane: row l % 16, values 8 (l / 16) ..),
// kUnits steps in registers between the row's maximum and its parts; longer rows are read
// again. Bound: memory, x read and its parts written.
constexpr int kUnits = 5, kPassWaves = 8, kPass = kUnits * kPassWaves * 32;
constexpr int kTiles = 2;  // of 16 ranks per round: rank 256 of 512 rows 62 -> 47 us against one

template <bool VEC, int P>
__global__ __launch_bounds__(64 * kPassWaves) void split_shrink_kernel(LoraArgs p, int cip, _Float16 *parts, int *exps) {
    __shared__ float wave_max[kPassWaves][16];
    __shared__ float part[kPassWaves][kTiles][4][64];
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t r0 = int64_t(blockIdx.x) * 16, row = r0 + r16;
    const int mine = slot_of(p, row);
    const float *x = p.x + min(row, p.rows - 1) * p.ci;
    const int passes = (cip + kPass - 1) / kPass;
    floatx4 v[kUnits][2];
    auto load = [&](int pass) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                v[u][j] = load4<VEC>(x, pass * kPass + (wave * kUnits + u) * 32 + kg * 8 + j * 4, p.ci);
    };
    float mx = 0.0f;
    for (int pass = passes - 1; pass >= 0; --pass) {
        load(pass);
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float f = __builtin_fabsf(v[u][i / 4][i % 4]);
                mx = f < __builtin_huge_valf() ? __builtin_fmaxf(mx, f) : mx;
            }
    }
    mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
    mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
    if (lane < 16) wave_max[wave][lane] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPassWaves; ++w) mx = __builtin_fmaxf(mx, wave_max[w][r16]);
    const int e = top_exp(mx);
    if (tid < 16 && row < p.rows) exps[row] = e;

    // The values' parts take their place; those of a row longer than a pass are loaded for every round.
    halfx8 hi[kUnits], lo[kUnits];
    auto part_values = [&] {
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                _Float16 h, l;
                split2(v[u][i / 4][i % 4], kSplitExp - e, h, l);
                hi[u][i] = h, lo[u][i] = l;
            }
    };
    if (passes == 1) part_values();
    // Adapters one after another, ranks kTiles x 16 at a time, the next round's loaded before
    // this one's sums are joined; the parts are written by the first round.
    halfx8 av[kTiles][kUnits];
    auto fetch = [&](int s, int q0, int pass) {
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
            const _Float16 *a = static_cast<const _Float16 *>(p.a) +
                                (int64_t(s) * p.rank + min(q0 + j * 16 + r16, p.rank - 1)) * p.ci;
#pragma unroll
            for (int u = 0; u < kUnits; ++u)
                av[j][u] = load8<VEC>(a, pass * kPass + (wave * kUnits + u) * 32 + kg * 8, p.ci);
        }
    };
    uint32_t todo = uint32_t(__ballot(mine >= 0)) & 0xFFFFu;
    bool first = true;
    do {
        const int s = todo ? __builtin_amdgcn_readfirstlane(__shfl(mine, __builtin_ctz(todo))) : -1;
        const bool own = s >= 0 && mine == s;
        todo &= ~uint32_t(__ballot(own));
        if (s >= 0) fetch(s, 0, 0);
        for (int q0 = 0; q0 < p.rank; q0 += 16 * kTiles) {
            accx4 acc[kTiles], low[kTiles];
#pragma unroll
            for (int j = 0; j < kTiles; ++j) acc[j] = low[j] = accx4{0, 0, 0, 0};
            for (int pass = 0; pass < passes; ++pass) {
                if (passes > 1) {
                    load(pass);
                    part_values();
                }
                if (first && row < p.rows)
#pragma unroll
                    for (int u = 0; u < kUnits; ++u) {
                        const int k = pass * kPass + (wave * kUnits + u) * 32 + kg * 8;
                        if (k >= cip) continue;
                        _Float16 *dst = parts + row * P * cip + k;
                        *reinterpret_cast<halfx8 *>(dst) = hi[u];
                        if constexpr (P == 2) *reinterpret_cast<halfx8 *>(dst + cip) = lo[u];
                    }
                if (s < 0) continue;
#pragma unroll
                for (int u = 0; u < kUnits; ++u)
#pragma unroll
                    for (int j = 0; j < kTiles; ++j) {
                        low[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[j][u], lo[u], low[j], 0, 0, 0);
                        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[j][u], hi[u], acc[j], 0, 0, 0);
                    }
                if (pass + 1 < passes) fetch(s, q0, pass + 1);
                else if (q0 + 16 * kTiles < p.rank) fetch(s, q0 + 16 * kTiles, 0);
            }
            first = false;
            if (s < 0) break;
            __syncthreads();  // the sums before have been read
#pragma unroll
            for (int j = 0; j < kTiles; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float both = acc[j][i] + low[j][i];
                    part[wave][j][i][lane] = both == both ? both : acc[j][i];
                }
            __syncthreads();
            // wave j joins rank tile j; register i is rank 4 (l / 16) + i of row l % 16
            if (wave < kTiles && own && q0 + wave * 16 < p.rank) {
                floatx4 t = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < kPassWaves; ++w)
#pragma unroll
                    for (int i = 0; i < 4; ++i) t[i] += part[w][wave][i][lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) t[i] = ldexpf(t[i], e - kSplitExp);
                *reinterpret_cast<floatx4 *>(p.t + row * p.rank_pad + q0 + wave * 16 + kg * 4) = t;
            }
        }
    } while (todo);
}

// Eight ranks of a row of t (padded to sixteens), zeros behind the last and where not wanted.
__device__ __forceinline__ void read_t(const float *t, int k, int rank, bool want, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const floatx4 r = *reinterpret_cast<const floatx4 *>(t + k + 4 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * j + e] = want && k + 4 * j + e < rank ? r[e] : 0.0f;
    }
}

// P: parts of x; WPARTS: the weight is in as many, rows of P cip (else f16 as stored, rows
// of ci); VW: its rows allow 16-byte loads; T: the adapters' storage; KG: groups of four waves that share the
// long axis.
template <int BM, int BN, int KG, int P, bool WPARTS, bool VW, typename T>
__global__ __launch_bounds__(256 * KG, KG == 4 ? 4 : WPARTS || BM > 128 ? 2 : 3) void lora_gemm_kernel(GemmArgs g) {
    constexpr int NT = 256 * KG, GK = 64 * KG;  // GK: of the long axis per stage
    constexpr int WP = WPARTS ? P : 1;
    constexpr int SM = BM / 64, SN = BN / 64;       // 32-tiles of a wave: of columns, of rows
    constexpr int XS = P * GK + 8, WS = WP * GK + 8;  // staged rows (halves), on distinct banks
    constexpr int R = GK / 8, XU = BN * P * R / NT, WU = BM * WP * R / NT;  // runs of 8 per part, per thread
    __shared__ __align__(16) _Float16 xs[BN * XS], ws[BM * WS];
    const LoraArgs &p = g.l;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave & 1, wn = wave >> 1 & 1, kg = wave >> 2, l32 = lane & 31, h = lane >> 5;
    // Tiles of columns within tiles of rows, a contiguous eighth per XCD: a tile's rows are
    // read from memory once.
    const int tiles = g.tiles_m * g.tiles_n, per_xcd = (tiles + 7) / 8;
    const int w = int(blockIdx.x % 8) * per_xcd + int(blockIdx.x / 8);
    if (int(blockIdx.x / 8) >= per_xcd || w >= tiles) return;
    const int c0 = (w % g.tiles_m) * BM;
    const int64_t r0 = int64_t(w / g.tiles_m) * BN;

    // A thread's runs: the same place of rows NT / (P R) (columns NT / (WP R)) apart, as
    // offsets from the tile's first, which the step moves on. The runs of hi, then of lo.
    static_assert(NT % (P * R) == 0, "runs");
    halfx8 xr[XU], wv[WU];
    uint32_t wo[WU];
    const int xrun = tid % (P * R), wrun = tid % (WP * R);
    // (the parts of x hold whole tiles of rows)
    const uint32_t xo = uint32_t((tid / (P * R) * P + xrun / R) * g.cip + xrun % R * 8) * 2;
    const uint32_t xstep = uint32_t(NT / (P * R)) * P * uint32_t(g.cip) * 2;
#pragma unroll
    for (int u = 0; u < WU; ++u) {
        const int c = min(tid / (WP * R) + u * (NT / (WP * R)), p.co - 1 - c0);
        wo[u] = uint32_t(WPARTS ? (c * P + wrun / R) * g.cip + wrun % R * 8 : c * p.ci) * 2;
    }
    const char *xb = reinterpret_cast<const char *>(g.xp + r0 * P * g.cip);
    const char *wb = static_cast<const char *>(g.w) + int64_t(c0) * (WPARTS ? P * g.cip : p.ci) * 2;
    auto fetch = [&](int k) {
#pragma unroll
        for (int u = 0; u < XU; ++u) xr[u] = *reinterpret_cast<const halfx8 *>(xb + k * 2 + u * xstep + xo);
#pragma unroll
        for (int u = 0; u < WU; ++u) {
            if constexpr (WPARTS) wv[u] = *reinterpret_cast<const halfx8 *>(wb + k * 2 + wo[u]);
            else wv[u] = load8<VW>(reinterpret_cast<const _Float16 *>(wb + wo[u]), k + wrun * 8, p.ci);
        }
    };
    // The adapters of this lane's rows and the exponents of their parts.
    int slot[SN], xe[SN];
#pragma unroll
    for (int n = 0; n < SN; ++n) {
        const int64_t row = r0 + (wn * SN + n) * 32 + l32;
        slot[n] = slot_of(p, row);
        xe[n] = g.x_exp[min(row, p.rows - 1)] - kSplitExp;
    }
    floatx16 acc[SM][SN];
#pragma unroll
    for (int m = 0; m < SM; ++m)
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[m][n][i] = 0.0f;
    fetch(0);
    for (int k = 0; k < p.ci; k += GK) {  // (cip is a whole number of stages)
        if (k) __syncthreads();
#pragma unroll
        for (int u = 0; u < XU; ++u) {
            const int i = tid + u * NT;
            *reinterpret_cast<halfx8 *>(xs + i / (P * R) * XS + i % (P * R) * 8) = xr[u];
        }
#pragma unroll
        for (int u = 0; u < WU; ++u) {
            const int i = tid + u * NT;
            *reinterpret_cast<halfx8 *>(ws + i / (WP * R) * WS + i % (WP * R) * 8) = wv[u];
        }
        __syncthreads();
        if (k + GK < p.ci) fetch(k + GK);
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
            const int c = kg * 4 + c4;
            halfx8 xh[SN], xl[SN];
#pragma unroll
            for (int n = 0; n < SN; ++n) {
                const _Float16 *q = xs + (wn * SN * 32 + n * 32 + l32) * XS + c * 16 + h * 8;
                xh[n] = *reinterpret_cast<const halfx8 *>(q);
                if constexpr (P == 2) xl[n] = *reinterpret_cast<const halfx8 *>(q + GK);
            }
#pragma unroll
            for (int m = 0; m < SM; ++m) {
                const _Float16 *q = ws + (wm * SM * 32 + m * 32 + l32) * WS + c * 16 + h * 8;
                const halfx8 wh = *reinterpret_cast<const halfx8 *>(q);
                if constexpr (WP == 2) {
                    const halfx8 wl = *reinterpret_cast<const halfx8 *>(q + GK);
#pragma unroll
                    for (int n = 0; n < SN; ++n) acc[m][n] = mfma16(wl, xh[n], acc[m][n]);
                }
                if constexpr (P == 2)
#pragma unroll
                    for (int n = 0; n < SN; ++n) acc[m][n] = mfma16(wh, xl[n], acc[m][n]);
#pragma unroll
                for (int n = 0; n < SN; ++n) acc[m][n] = mfma16(wh, xh[n], acc[m][n]);
            }
        }
    }

    if constexpr (KG > 1) {  // the groups' sums, one after another
        static_assert(sizeof(xs) >= 4 * SM * SN * 16 * 64 * sizeof(float), "sums");
        float *sum = reinterpret_cast<float *>(xs) + (wave & 3) * SM * SN * 16 * 64 + lane;
        for (int q = 1; q < KG; ++q) {
            __syncthreads();
            if (kg == q)
#pragma unroll
                for (int i = 0; i < SM * SN * 16; ++i) sum[i * 64] = acc[i / 16 / SN][i / 16 % SN][i % 16];
            __syncthreads();
            if (kg == 0)
#pragma unroll
                for (int i = 0; i < SM * SN * 16; ++i) acc[i / 16 / SN][i / 16 % SN][i % 16] += sum[i * 64];
        }
        if (kg) return;
    }

    // Columns 8 f + 4 h + e of a 32-tile are register 4 f + e; the row is lane % 32.
    const bool vb = p.rank % 8 == 0 && reinterpret_cast<uintptr_t>(p.b) % 16 == 0;
    typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (int n = 0; n < SN; ++n) {
        const int64_t row = r0 + (wn * SN + n) * 32 + l32, row_in = min(row, p.rows - 1);
        if constexpr (P == 2)
#pragma unroll
            for (int m = 0; m < SM; ++m)
                redo_nan(acc[m][n], row < p.rows, [&](floatx16 &sum) {
                    constexpr int U = 2;
                    const int c = min((wm * SM + m) * 32 + l32, p.co - 1 - c0);
                    const _Float16 *x = g.xp + row_in * P * g.cip + h * 8;
                    const _Float16 *w = reinterpret_cast<const _Float16 *>(wb) + int64_t(c) * (WPARTS ? P * g.cip : p.ci);
#pragma nounroll
                    for (int k = 0; k < p.ci; k += 16 * U) {
                        halfx8 a[U], b[U];
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            b[u] = *reinterpret_cast<const halfx8 *>(x + k + 16 * u);
                            if constexpr (WPARTS) a[u] = *reinterpret_cast<const halfx8 *>(w + k + 16 * u + h * 8);
                            else a[u] = load8<VW>(w, k + 16 * u + h * 8, p.ci);
                        }
#pragma unroll
                        for (int u = 0; u < U; ++u) sum = mfma16(a[u], b[u], sum);
                    }
                });
#pragma unroll
        for (int m = 0; m < SM; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                int e = xe[n];
                if constexpr (WPARTS)
                    e += g.w_exp[min(c0 + (wm * SM + m) * 32 + 8 * (i / 4) + 4 * h + i % 4, p.co - 1)] - kSplitExp;
                acc[m][n][i] = ldexpf(acc[m][n][i], e);
            }
        const int mine = slot[n];
        uint32_t todo = uint32_t(__ballot(mine >= 0));
        if (todo) {
            const float *t = p.t + row_in * p.rank_pad;
            int te = 0;
            if constexpr (sizeof(T) == 2) {  // the row of t in two parts, as x
                float mx = 0.0f;
                for (int k = 0; k < p.rank; k += 16) {
                    float tv[8];
                    read_t(t, k + h * 8, p.rank, mine >= 0, tv);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float f = __builtin_fabsf(tv[i]);
                        mx = f < __builtin_huge_valf() ? __builtin_fmaxf(mx, f) : mx;
                    }
                }
                mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
                te = top_exp(mx);
            }
            while (todo) {
                const int s = __builtin_amdgcn_readfirstlane(__shfl(mine, __builtin_ctz(todo)));
                const bool own = mine == s;
                todo &= ~uint32_t(__ballot(own));
                floatx16 low[SM];
#pragma unroll
                for (int m = 0; m < SM; ++m)
#pragma unroll
                    for (int i = 0; i < 16; ++i) low[m][i] = 0.0f;
                const T *b[SM];
#pragma unroll
                for (int m = 0; m < SM; ++m)
                    b[m] = static_cast<const T *>(p.b) +
                           (int64_t(s) * p.co + min(c0 + (wm * SM + m) * 32 + l32, p.co - 1)) * p.rank;
                for (int k = 0; k < p.rank; k += 16) {
                    float tv[8];
                    read_t(t, k + h * 8, p.rank, own, tv);
                    if constexpr (sizeof(T) == 2) {
                        halfx8 th, tl;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            _Float16 hi, lo;
                            split2(tv[i], kSplitExp - te, hi, lo);
                            th[i] = hi, tl[i] = lo;
                        }
#pragma unroll
                        for (int m = 0; m < SM; ++m) {
                            const halfx8 bv = vb ? load8<true>(b[m], k + h * 8, p.rank) : load8<false>(b[m], k + h * 8, p.rank);
                            low[m] = mfma16(bv, tl, low[m]);
                            low[m] = mfma16(bv, th, low[m]);
                        }
                    } else {
#pragma unroll
                        for (int m = 0; m < SM; ++m)
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float bv = k + h * 8 + i < p.rank ? float(b[m][k + h * 8 + i]) : 0.0f;
                                low[m] = __builtin_amdgcn_mfma_f32_32x32x2f32(bv, tv[i], low[m], 0, 0, 0);
                            }
                    }
                }
                if constexpr (sizeof(T) == 2)
#pragma unroll
                    for (int m = 0; m < SM; ++m)
                        redo_nan(low[m], own, [&](floatx16 &sum) {
#pragma nounroll
                            for (int k = 0; k < p.rank; k += 16) {
                                float tv[8];
                                read_t(t, k + h * 8, p.rank, own, tv);
                                halfx8 th;
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    _Float16 hi, lo;
                                    split2(tv[i], kSplitExp - te, hi, lo);
                                    th[i] = hi;
                                }
                                sum = mfma16(load8<false>(b[m], k + h * 8, p.rank), th, sum);
                            }
                        });
                const float scale = p.scale[s];
#pragma unroll
                for (int m = 0; m < SM; ++m)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float v = sizeof(T) == 2 ? ldexpf(low[m][i], te - kSplitExp) : low[m][i];
                        acc[m][n][i] = own ? __builtin_fmaf(scale, v, acc[m][n][i]) : acc[m][n][i];
                    }
            }
        }
        if (row >= p.rows) continue;
#pragma unroll
        for (int m = 0; m < SM; ++m)
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const int c = c0 + (wm * SM + m) * 32 + 8 * f + 4 * h;
                float *out = p.out + row * p.co + c;
                const float *res = g.residual ? g.residual + row * p.co + c : nullptr;
                if (c + 4 <= p.co) {
                    floatx4 y = {acc[m][n][4 * f], acc[m][n][4 * f + 1], acc[m][n][4 * f + 2], acc[m][n][4 * f + 3]};
                    if (g.bias)
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] += g.bias[c + e];
                    if (res) y += floatx4(*reinterpret_cast<const float4u *>(res));
                    *reinterpret_cast<float4u *>(out) = y;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < p.co)
                            out[e] = acc[m][n][4 * f + e] + (g.bias ? g.bias[c + e] : 0.0f) + (res ? res[e] : 0.0f);
                }
            }
    }
}

template <int BM, int BN, int KG, int P, bool WPARTS, bool VW>
void launch(Context &ctx, GemmArgs g, WeightType at) {
    g.tiles_m = int(ceil_div(g.l.co, BM));
    const int64_t tn = ceil_div(g.l.rows, BN);
    MH_REQUIRE(tn * g.tiles_m < (int64_t(1) << 30), "lora: too many tiles");
    g.tiles_n = int(tn);
    const dim3 grid{uint32_t(ceil_div(tn * g.tiles_m, 8) * 8)}, tb{256 * KG};
    if (at == kF16) lora_gemm_kernel<BM, BN, KG, P, WPARTS, VW, _Float16><<<grid, tb, 0, ctx.stream>>>(g);
    else lora_gemm_kernel<BM, BN, KG, P, WPARTS, VW, float><<<grid, tb, 0, ctx.stream>>>(g);
    MH_LAUNCH_CHECK();
}

bool wide_weight(const GemmArgs &g) { return g.l.ci % 8 == 0 && aligned16(g.w); }

template <int KG, int P>
void launch_small(Context &ctx, const GemmArgs &g, WeightType wt, WeightType at) {
    if (wt == kF32) launch<64, 64, KG, P, true, true>(ctx, g, at);
    else if (wide_weight(g)) launch<64, 64, KG, P, false, true>(ctx, g, at);
    else launch<64, 64, KG, P, false, false>(ctx, g, at);
}

template <int P>
void launch_tiles(Context &ctx, const GemmArgs &g, WeightType wt, WeightType at) {
    // 8192 rows of 1280 x 1280, the product alone: tiles of 128 x 128 92 us, 192 x 128 88;
    // the whole call for 4096 rows, where the latter leave CUs idle, 65.5, with tiles of 64
    // 59. 2048 rows: 41 with one group of waves, 44 with two; 1024 rows 33 and 30.5; 128 rows
    // 29, 25 and with four groups 23, but 15.8 and 16.4 where the long axis is 320.
    const int wide = wt == kF32 ? 128 : 192;  // columns of the large tile that registers hold
    const int64_t tiles = ceil_div(g.l.rows, 64) * ceil_div(g.l.co, 64);
    if (ceil_div(g.l.rows, 128) * ceil_div(g.l.co, wide) >= ctx.cu_count) {
        if (wt == kF32) launch<128, 128, 1, P, true, true>(ctx, g, at);
        else if (wide_weight(g)) launch<192, 128, 1, P, false, true>(ctx, g, at);
        else launch<192, 128, 1, P, false, false>(ctx, g, at);
    } else if (tiles >= 2 * ctx.cu_count) {
        launch_small<1, P>(ctx, g, wt, at);
    } else if (tiles >= ctx.cu_count || g.l.ci < 1024) {
        launch_small<2, P>(ctx, g, wt, at);
    } else {
        launch_small<4, P>(ctx, g, wt, at);
    }
}

template <int P>
void launch_split_rows(Context &ctx, const SplitRows &a, const SplitRows &b, int ci, int cip) {
    const dim3 grid{uint32_t(ceil_div(a.rows + b.rows, 4))}, tb{256};
    if (ci % 4 == 0 && aligned16(a.x) && aligned16(b.x)) split_rows_kernel<true, P><<<grid, tb, 0, ctx.stream>>>(a, b, ci, cip);
    else split_rows_kernel<false, P><<<grid, tb, 0, ctx.stream>>>(a, b, ci, cip);
    MH_LAUNCH_CHECK();
}

template <int P>
void launch_split_shrink(Context &ctx, const LoraArgs &p, int cip, _Float16 *parts, int *exps) {
    const dim3 grid{uint32_t(ceil_div(p.rows, 16))}, tb{64 * kPassWaves};
    if (p.ci % 8 == 0 && aligned16(p.x) && aligned16(p.a))
        split_shrink_kernel<true, P><<<grid, tb, 0, ctx.stream>>>(p, cip, parts, exps);
    else split_shrink_kernel<false, P><<<grid, tb, 0, ctx.stream>>>(p, cip, parts, exps);
    MH_LAUNCH_CHECK();
}

}  // namespace

void split_rows(Context &ctx, const SplitRows &a, const SplitRows &b, int ci, int cip, int nparts) {
    if (nparts == 1) launch_split_rows<1>(ctx, a, b, ci, cip);
    else launch_split_rows<2>(ctx, a, b, ci, cip);
}

void split_shrink(Context &ctx, const LoraArgs &p, int cip, int nparts, _Float16 *parts, int *exps) {
    if (nparts == 1) launch_split_shrink<1>(ctx, p, cip, parts, exps);
    else launch_split_shrink<2>(ctx, p, cip, parts, exps);
}

void gemm(Context &ctx, const GemmArgs &g, int nparts, WeightType wt, WeightType at) {
    if (nparts == 1) launch_tiles<1>(ctx, g, wt, at);
    else launch_tiles<2>(ctx, g, wt, at);
}

}  // namespace lora
}  // namespace mh
