// Attention over selected blocks of keys: one pass with a running maximum and sum.
//
// For the rows r of a block of queries (query r / G, head hk G + r % G, G query heads
// per key head: all of them share the list) and the keys j of the listed blocks:
//   s_j = c q . k_j (c = scale log2 e),  m = max s_j,  p_j = 2^(s_j - m),  o = sum p_j v_j / sum p_j
// in tiles of KT keys: where the tile's maximum passes m, o and the sum are scaled by 2^(m - m').
//
// A wave takes 32 rows. It forms S^T = K . Q^T, so that a lane holds one row's scores
// (32x32 instructions: column = lane % 32), the maximum and the sum of a row stay in the
// lane but for one exchange with lane +- 32, and the scores are already the B operand of
// O^T = V^T . P^T: its lane half h wants eight keys of sixteen, and holds eight, keys
// 4h .. 4h + 3 and 8 + 4h .. 8 + 4h + 3, so V^T is read with its keys in that order. WR
// waves share a tile of keys, WK groups of waves take every WK-th tile and join in LDS.
//
// kHalf: f16 products (v_mfma_f32_32x32x16_f16), f32 storage rounded and saturated (infinities
// too) as the f16 GEMMs round operands; P rounded to f16 while its sum keeps f32, off by at most
// 2^-11 each, which a sum over keys averages (outputs of f16 tensors then lie 2.6e-4 to 2.9e-4 of
// the largest from 64 bits, where their own rounding alone gives 2.1e-4; P in two parts would
// double the second product). kF32: f32 products (v_mfma_f32_32x32x2_f32, an eighth of the
// rate). kSplit: each f32 operand as two f16 parts, x = hi + lo to 2^-24, and the three
// products above 2^-24 of theirs; queries scaled by a power of two per row, keys and values
// per sixteen tokens, or per token where those are far apart (KeyScale), probabilities by 2^11
// and their key's power against the largest that the row has seen, so that the parts keep all
// bits of queries down to 2^-18, of keys to 2^-12 and of p v to 2^-13 of the largest, and no
// token that a row does not see takes bits from it. Scores, maxima, sums and outputs are f32 in all.
//
// Bound: the matrix instructions and the vector instructions beside them (7 to 8 for each;
// from registers alone 7 leave the card 1278 TFLOP/s of f16 on random values); latency where
// rows are few. Measured: 16384 tokens, 16 heads of 128, f16, 2048 keys per row 346 us (795
// TFLOP/s); 2 x 4096, 8 heads of 80, f32, 1024 keys 131 us, on the f32 instructions 298; 8
// single tokens, 32 / 8 heads of 128, 2048 of up to 16384 keys 24.7 us. For the first: values
// read from LDS transposed by ds_read_b64_tr_b16 instead of gathered 1140 -> 473 us; loads
// without branches and 32-bit offsets 473 -> 375; the maximum's reference moved only when it
// is passed by 2^8 355 -> 350; two buffers, tiles of 32 keys with three waves per SIMD and
// products interleaved with exponentials by scheduling groups changed nothing.
#pragma once

#include <type_traits>

#include "attention.hpp"

namespace mh {
namespace battn {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));

// Products of f16 operands; of f32 ones on the f32 instructions; of f32 ones as three
// products of operands split in two f16 parts.
enum Mode { kHalf, kF32, kSplit };

// The exponents by which the key and the values of a token are scaled where they are split,
// the values' twice and 1 more where some that are not finite were left out. Sixteen tokens
// share theirs, the largest, where all are within 2^kSplitSpread of it; else each has its
// own, which leaves the others their bits whatever lies at tokens that a row does not see.
constexpr int kSplitSpread = 6;
struct KeyScale {
    int k, v;
};

struct Args {
    const void *q, *k, *v;  // kSplit: k, v as written by split_kv, rows of two parts of dk values
    void *out;
    int64_t ldq, ldo;
    uint32_t ldk, ldv;  // bytes
    const int32_t *blocks, *q_len, *kv_len;
    float *part;  // split partials, NULL: none
    float c;      // scale . log2 e
    int n, q_tokens, kv_tokens, hk, g, d, qb, kb_log, nq, top, row_tiles, splits, work;
    bool causal;
    int dk;       // values of a staged row's part: d, or d rounded up to 8 (kSplit)
    int kv_rows;  // rows per item of k and v
    const void *v0;        // kSplit: the values themselves, rows ldv0 bytes apart, heads of d
    uint32_t ldv0;
    const KeyScale *meta;  // [n][hk][kv_rows]
};

constexpr int kNoExp = -1000;  // exponent of values that are all zero or not finite: below all others
constexpr int kSplitExp = 14;  // split operands are scaled to a largest value of 2^14 .. 2^15
// Powers of two by which a row's maximum may pass its reference: probabilities up to 2^8 fit
// f16, split ones (scaled by 2^11) up to 2^3.
constexpr int kLazyHalf = 8, kLazySplit = 3;
constexpr int kSplitP = 11;    // split probabilities are scaled to at most 2^(11 + 3 + kLazyV)
constexpr int kLazyV = 1;      // powers of two by which a key's values may pass their reference

// x 2^e in two f16 parts, x = hi + lo to 2^-24 of it (and 2^-40 of the largest value that e
// was taken from); a value that is not finite is all in hi.
__device__ __forceinline__ void split2(float x, int e, _Float16 &hi, _Float16 &lo) {
    const float y = ldexpf(x, e);
    hi = static_cast<_Float16>(y);
    const float r = y - float(hi);
    lo = static_cast<_Float16>(__builtin_fabsf(y) < __builtin_huge_valf() ? r : 0.0f);
}

constexpr float kNegInf = -__builtin_huge_valf();

// Floats of one wave's partial: the sums of DT x 16 registers and the row's maximum and sum.
constexpr int part_floats(int dt) { return (dt * 16 + 2) * 64; }

template <int MODE, int DT, int WR>
struct Tiling {
    static constexpr int kDP = DT * 32, kCols = MODE == kSplit ? 2 * kDP : kDP;
    static constexpr int kKT = MODE == kHalf && (DT <= 2 ? WR >= 2 : DT <= 4 && WR == 4) ? 64 : 32;  // keys per tile
    static constexpr int kES = MODE == kF32 ? 4 : 2;  // bytes of a staged value
    // staged rows (values), padded so that the rows of a read lie on distinct banks
    static constexpr int kKS = kCols + (MODE == kF32 ? 4 : 8);
    static constexpr int kVS = MODE == kF32 ? kDP + 8 : kCols + (kCols % 64 ? 0 : 32);
    static constexpr int kKBytes = kKT * kKS * kES, kVBytes = kKT * kVS * kES;
    static constexpr int kStage = kKBytes + kVBytes + (MODE == kSplit ? 8 * kKT : 0);  // one key group's tile, its scales
    // key groups: four waves together, fewer where their tiles exceed the LDS of a CU (160 KiB)
    static constexpr int kWK = 4 / WR * kStage <= 144 * 1024 ? 4 / WR : 2 / WR;
    static_assert(kWK >= 1 && kWK * kStage <= 144 * 1024, "tiles exceed the LDS");
    static constexpr int kThreads = 64 * WR * kWK;
    static constexpr int kJoin = WR * part_floats(DT) * 4;
    static constexpr int kLds = kStage * kWK > kJoin || kWK == 1 ? kStage * kWK : kJoin;
};

// Eight consecutive values of a row.
template <typename T>
struct Run8 {
    typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
    static constexpr int kN = int(sizeof(T)) / 2;  // 16-byte loads
    V v[kN];
    template <bool VEC>
    __device__ __forceinline__ void load(const T *p, int valid) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < kN; ++i) v[i] = reinterpret_cast<const V *>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i / (8 / kN)][i % (8 / kN)] = i < valid ? p[i] : T(0);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = V(T(0));
    }
    __device__ __forceinline__ T at(int i) const { return v[i / (8 / kN)][i % (8 / kN)]; }
    __device__ __forceinline__ halfx8 half() const {
        halfx8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 2) {
                h[i] = at(i);
            } else {
                const float x = at(i);
                h[i] = static_cast<_Float16>(__builtin_fabsf(x) > 65504.0f ? __builtin_copysignf(65504.0f, x) : x);
            }
        }
        return h;
    }
    // Zeros in the place of values that are not finite (SATURATED: NaN alone); whether there were any.
    template <bool SATURATED = false>
    __device__ __forceinline__ bool clean() {
        bool any = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = float(at(i));
            const bool ok = SATURATED ? x == x : __builtin_fabsf(x) < __builtin_huge_valf();
            any = any || !ok;
            v[i / (8 / kN)][i % (8 / kN)] = ok ? at(i) : T(0);
        }
        return any;
    }
};

// V^T operand of 32 channels and sixteen keys from staged rows of stride VS: a transposed
// read hands lane i of sixteen the i-th of sixteen channels at four keys, the lanes' own
// addresses being four channels of key lane / 4 each. Keys 4 h .. 4 h + 3, then 8 more on.
template <int VS>
__device__ __forceinline__ halfx8 read_vt(const char *v, int lane) {
    typedef short shortx4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) shortx4 lds4;
    const char *p = v + ((4 * (lane >> 5) + ((lane >> 2) & 3)) * VS + ((lane >> 4) & 1) * 16 + (lane & 3) * 4) * 2;
    const shortx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p));
    const shortx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + 8 * VS * 2));
    return __builtin_bit_cast(halfx8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The value of lane +- 32.
__device__ __forceinline__ float other_half(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

// Key of accumulator register i in lane half h (32 x 32 results: row of the tile).
__device__ __forceinline__ int acc_row(int i, int h) { return 8 * (i / 4) + 4 * h + (i % 4); }

// Waves per SIMD that the registers allow (kSplit with four tiles and two row waves does without
// the second: 49 registers spilled, 245 us against 213 with 8 heads of 128, 2 x 4096 rows).
constexpr int occupancy(int mode, int dt, int wr) {
    if (mode == kSplit && dt == 4 && wr == 2) return 1;
    return mode == kF32 ? 1 : dt <= 4 || (mode == kHalf && dt == 5 && wr >= 2) ? 2 : 1;
}

template <typename T, int MODE, bool VEC, int DT, int WR>
__global__ __launch_bounds__(256, (occupancy(MODE, DT, WR))) void block_attention_kernel(Args a) {
    using L = Tiling<MODE, DT, WR>;
    typedef std::conditional_t<MODE == kSplit, _Float16, T> S;  // k and v
    constexpr bool SPLIT = MODE == kSplit, HALF = MODE != kF32, KVEC = VEC || SPLIT;
    constexpr bool SATURATED = MODE == kHalf && sizeof(T) == 4;  // infinite values are finite operands
    constexpr int kLazy = SPLIT ? kLazySplit : kLazyHalf;
    constexpr int KT = L::kKT, WK = L::kWK, SUB = KT / 32, DP = L::kDP, RUNS = L::kCols / 8;
    constexpr int NT = 64 * WR;                      // threads that stage one tile
    constexpr int KU = (KT * RUNS + NT - 1) / NT;    // runs of 8 channels of K, and of V, per thread
    extern __shared__ __align__(16) char smem[];
    __shared__ int32_t list[kMaxTop];  // first token of every block to visit
    __shared__ int list_n, bad;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % WR, wk = wave / WR, ttid = tid % NT;
    const int col = lane & 31, h = lane >> 5;

    // Work items (item, key head, block of queries, rows, split) in this order: workgroup i
    // runs on XCD i % 8, and each XCD takes one contiguous eighth, few heads' keys.
    const int per_xcd = (a.work + 7) / 8;
    int w = int(blockIdx.x % 8) * per_xcd + int(blockIdx.x / 8);
    if (int(blockIdx.x / 8) >= per_xcd || w >= a.work) return;
    const int work = w;
    const int split = w % a.splits;
    w /= a.splits;
    const int rt = w % a.row_tiles;
    w /= a.row_tiles;
    const int qb = w % a.nq;
    w /= a.nq;
    const int hk = w % a.hk, item = w / a.hk;
    const int q_len = a.q_len ? min(max(a.q_len[item], 0), a.q_tokens) : a.q_tokens;
    const int kv_len = a.kv_len ? min(max(a.kv_len[item], 0), a.kv_tokens) : a.kv_tokens;
    const int i0 = qb * a.qb, i1 = min(i0 + a.qb, q_len);
    const int rows = (i1 - i0) * a.g, r0 = rt * WR * 32;
    if (r0 >= rows) return;
    const int kb = 1 << a.kb_log;
    const int off = kv_len - q_len;
    // the last token that the rows of this workgroup may see
    const int last = a.causal ? min(kv_len, off + i0 + (min(rows, r0 + WR * 32) - 1) / a.g + 1) - 1 : kv_len - 1;

    // The list without what is outside, behind `last` or listed before, by the first wave.
    if (wave == 0) {
        const int32_t *src = a.blocks + ((int64_t(item) * a.nq + qb) * a.hk + hk) * a.top;
        bool ascending = true;
        for (int i = lane; i < a.top; i += 64) {
            const int e = src[i], before = i ? src[i - 1] : -1;
            ascending = ascending && (e < 0 || i == 0 || (before >= 0 && e > before));
        }
        ascending = __all(ascending);
        int n = 0;
        for (int i = lane; i < (a.top + 63) / 64 * 64; i += 64) {
            const int e = i < a.top ? src[i] : -1;
            bool ok = e >= 0 && e <= (last >> a.kb_log) && last >= 0;
            if (ok && !ascending)
#pragma unroll 8
                for (int j = 0; j < i; ++j) ok = ok && src[j] != e;
            const uint64_t all = __ballot(ok);
            if (ok) list[n + __popcll(all & ((uint64_t(1) << lane) - 1))] = e << a.kb_log;
            n += __popcll(all);
        }
        if (lane == 0) list_n = n, bad = 0;
    }

    // Q^T: this lane's row, channels 16 c + 8 h .. + 7 of chunk c (f32: 8 c + 4 h .. + 3).
    const int row = r0 + wr * 32 + col;
    const bool row_ok = row < rows, rows_here = r0 + wr * 32 < rows;  // this lane's, any of the wave's
    const int qi = i0 + (row_ok ? row : 0) / a.g, qe = hk * a.g + (row_ok ? row : 0) % a.g;
    const T *qp = static_cast<const T *>(a.q) + (int64_t(item) * a.q_tokens + qi) * a.ldq + int64_t(qe) * a.d;
    halfx8 qh[HALF ? DT * 2 : 1], ql[SPLIT ? DT * 2 : 1];
    float qf[HALF ? 1 : DT * 16];
    int eq = 0;  // SPLIT: the power of two that the row's products lack, but for the key's
    if constexpr (SPLIT) {
        Run8<T> r[DT * 2];
        float mx = 0.0f;
#pragma unroll
        for (int c = 0; c < DT * 2; ++c) {
            const int ch = c * 16 + h * 8;
            r[c].zero();
            if (ch < a.d) r[c].template load<VEC>(qp + ch, a.d - ch);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = __builtin_fabsf(float(r[c].at(i)));
                mx = v < __builtin_huge_valf() ? __builtin_fmaxf(mx, v) : mx;
            }
        }
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
        const int e = mx == 0.0f ? 0 : __builtin_amdgcn_frexp_expf(mx) - 1;
        eq = e - 2 * kSplitExp;
#pragma unroll
        for (int c = 0; c < DT * 2; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                _Float16 hi, lo;
                split2(float(r[c].at(i)), kSplitExp - e, hi, lo);
                qh[c][i] = hi, ql[c][i] = lo;
            }
    } else if constexpr (HALF) {
#pragma unroll
        for (int c = 0; c < DT * 2; ++c) {
            const int ch = c * 16 + h * 8;
            Run8<T> r;
            r.zero();
            if (ch < a.d) r.template load<VEC>(qp + ch, a.d - ch);
            qh[c] = r.half();
        }
    } else {
#pragma unroll
        for (int c = 0; c < DT * 4; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int ch = c * 8 + h * 4 + j;
                qf[c * 4 + j] = ch < a.d ? float(qp[ch]) : 0.0f;
            }
    }
    const int lim = a.causal ? min(kv_len, off + qi + 1) : kv_len;  // this lane's row sees tokens below it
    // the tokens below which every row of the workgroup, and of the wave, sees all
    const int lim_first = a.causal ? min(kv_len, off + i0 + r0 / a.g + 1) : kv_len;
    const int lim_all = a.causal ? min(kv_len, off + i0 + (r0 + wr * 32) / a.g + 1) : kv_len;

    char *const kst = smem + wk * L::kStage, *const vst = kst + L::kKBytes;
    // Channels behind d of the staged keys: zeros, which the loads never overwrite.
    if (a.dk < DP)
        for (int i = ttid; i < KT * RUNS; i += NT) {
            const int ch = i % (DP / 8) * 8;
            if (ch + 8 > a.dk) {
                char *p = kst + (i / RUNS * L::kKS + i % RUNS * 8) * L::kES;
                reinterpret_cast<floatx4 *>(p)[0] = floatx4{0, 0, 0, 0};
                if constexpr (L::kES == 4) reinterpret_cast<floatx4 *>(p)[1] = floatx4{0, 0, 0, 0};
            }
        }
    __syncthreads();

    // This split's share of the list, whole tiles of keys.
    const int n_all = list_n;
    const int unit = max(1, KT >> a.kb_log);
    const int share = ((n_all + a.splits - 1) / a.splits + unit - 1) / unit * unit;
    const int l0 = min(split * share, n_all), l1 = min(l0 + share, n_all);
    const int keys = (l1 - l0) << a.kb_log;
    const int tiles = (keys + KT - 1) / KT;
    const int64_t head = int64_t(hk) * (SPLIT ? 2 * a.dk : a.dk) * int64_t(sizeof(S));
    const char *kp = static_cast<const char *>(a.k) + uint64_t(item) * a.kv_rows * a.ldk + head;
    const char *vp = static_cast<const char *>(a.v) + uint64_t(item) * a.kv_rows * a.ldv + head;

    // Token of key j of this split; past its end none. Loads of tokens there are not
    // (behind the list or kv_len) read the last one instead and are not used.
    auto token = [&](int j) {
        const int t = list[l0 + (min(j, keys - 1) >> a.kb_log)] + (j & (kb - 1));
        return j < keys ? t : 0x7fffffff;
    };
    // The next tile's runs, their tokens, and whether a row of the wave does not see some of
    // its keys. Runs behind d are loaded from the last channels and not staged.
    Run8<S> kr[KU], vr[KU];
    int tok[KU];
    KeyScale ks{};  // of key ttid % KT
    const KeyScale *meta = SPLIT ? a.meta + (int64_t(item) * a.hk + hk) * a.kv_rows : nullptr;
    int *const kx = reinterpret_cast<int *>(vst + L::kVBytes), *const vx = kx + KT;
    bool masked_next = false;
    constexpr bool kWhole = KT * RUNS % NT == 0;
    auto fetch = [&](int tile) {
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int j = (ttid + u * NT) / RUNS;
            tok[u] = kWhole || j < KT ? token(tile * KT + j) : 0x7fffffff;
        }
        masked_next = !__all(token(tile * KT + lane % KT) < lim_all);
        if constexpr (SPLIT) ks = meta[min(token(tile * KT + ttid % KT), kv_len - 1)];
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int run = (ttid + u * NT) % RUNS, ch = run % (DP / 8) * 8;
            const uint32_t t = min(tok[u], kv_len - 1);
            const int c = (KVEC ? min(ch, a.dk - 8) : ch) + run / (DP / 8) * a.dk;
            kr[u].template load<KVEC>(reinterpret_cast<const S *>(kp + c * int(sizeof(S)) + uint64_t(t) * a.ldk), a.dk - c);
            vr[u].template load<KVEC>(reinterpret_cast<const S *>(vp + c * int(sizeof(S)) + uint64_t(t) * a.ldv), a.dk - c);
        }
    };
    auto put = [&](char *p, const Run8<S> &r) {
        if constexpr (HALF) {
            *reinterpret_cast<halfx8 *>(p) = r.half();
        } else {
#pragma unroll
            for (int e = 0; e < 2; ++e)
                reinterpret_cast<floatx4 *>(p)[e] = floatx4{float(r.at(4 * e)), float(r.at(4 * e + 1)),
                                                            float(r.at(4 * e + 2)), float(r.at(4 * e + 3))};
        }
    };
    auto stage = [&]() {
        if constexpr (SPLIT)
            if (ttid < KT) {
                kx[ttid] = ks.k, vx[ttid] = ks.v >> 1;
                if (ks.v & 1) bad = 1;
            }
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int i = ttid + u * NT, j = i / RUNS, run = i % RUNS, ch = run % (DP / 8) * 8;
            if constexpr (!SPLIT) {
                if (__any(tok[u] >= lim_first)) {
                    // Values of tokens that there are not: zeros, whatever lies there. Values that
                    // are not finite, of tokens that some row does not see (0 times them is NaN in
                    // the products): zeros too, they are added at the end.
                    if (tok[u] >= kv_len) vr[u].zero();
                    else if (tok[u] >= lim_first && vr[u].template clean<SATURATED>()) bad = 1;
                }
            }
            if ((kWhole || j < KT) && ch < a.dk) {
                put(kst + (j * L::kKS + run * 8) * L::kES, kr[u]);
                put(vst + (j * L::kVS + run * 8) * L::kES, vr[u]);
            }
        }
    };

    floatx16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    float m = kNegInf, l = 0.0f;
    int top = kNoExp;  // SPLIT: the exponent that the row's o is scaled by

    const int steps = (tiles + WK - 1) / WK;
    if (wk < tiles) fetch(wk);
    for (int s = 0; s < steps; ++s) {
        const int tile = s * WK + wk;
        const bool live = tile < tiles;
        if (s) __syncthreads();  // the tile before has been read
        if (live) stage();
        const bool masked = masked_next;
        // SPLIT: the exponents of each sixteen keys and values, unless each has its own or they
        // count by what a row sees.
        int ke[2] = {}, ve[2] = {};
        bool each = false;
        if constexpr (SPLIT) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
                ke[x] = __builtin_amdgcn_readlane(ks.k, 16 * x), ve[x] = __builtin_amdgcn_readlane(ks.v, 16 * x) >> 1;
            each = masked || !__all(ks.k == (col < 16 ? ke[0] : ke[1]) && ks.v >> 1 == (col < 16 ? ve[0] : ve[1]));
        }
        __syncthreads();
        if (tile + WK < tiles) fetch(tile + WK);
        if (!live || !rows_here) continue;

        floatx16 sc[SUB];
#pragma unroll
        for (int b = 0; b < SUB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[b][i] = 0.0f;
        if constexpr (HALF) {
            const char *p = kst + (col * L::kKS + h * 8) * 2;
#pragma unroll
            for (int c = 0; c < DT * 2; ++c)
#pragma unroll
                for (int b = 0; b < SUB; ++b) {
                    const halfx8 kh = *reinterpret_cast<const halfx8 *>(p + (b * 32 * L::kKS + c * 16) * 2);
                    if constexpr (SPLIT) {  // the small products first
                        const halfx8 kl = *reinterpret_cast<const halfx8 *>(p + (b * 32 * L::kKS + DP + c * 16) * 2);
                        sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[c], sc[b], 0, 0, 0);
                        sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[c], sc[b], 0, 0, 0);
                    }
                    sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[c], sc[b], 0, 0, 0);
                }
        } else {
            const float *p = reinterpret_cast<const float *>(kst) + col * L::kKS + h * 4;
#pragma unroll
            for (int c = 0; c < DT * 4; ++c)
#pragma unroll
                for (int b = 0; b < SUB; ++b) {
                    const floatx4 kv = *reinterpret_cast<const floatx4 *>(p + b * 32 * L::kKS + c * 8);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        sc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(kv[j], qf[c * 4 + j], sc[b], 0, 0, 0);
                }
        }
        const float c = a.c;
        if (SPLIT && each) {
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const intx4 e = reinterpret_cast<const intx4 *>(kx)[2 * f + h];
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[0][4 * f + i] = ldexpf(sc[0][4 * f + i], e[i] + eq);
            }
        }
        if (masked) {
#pragma unroll
            for (int b = 0; b < SUB; ++b)
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                    const int t0 = token(tile * KT + b * 32 + 8 * f + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (t0 >= lim || t0 + e >= lim) sc[b][4 * f + e] = kNegInf;
                }
        }
        int tv = max(ve[0], ve[1]);  // the largest exponent of the values that the row sees
        if (SPLIT && each) {
            tv = kNoExp;
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const intx4 e = reinterpret_cast<const intx4 *>(vx)[2 * f + h];
#pragma unroll
                for (int i = 0; i < 4; ++i) tv = max(tv, sc[0][4 * f + i] == kNegInf ? kNoExp : e[i]);
            }
            tv = max(tv, __builtin_bit_cast(int, other_half(__builtin_bit_cast(float, tv))));
        } else if (SPLIT) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[0][i] = ldexpf(sc[0][i], ke[i / 8] + eq);
        }
        float mx = sc[0][0];
#pragma unroll
        for (int b = 0; b < SUB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = __builtin_fmaxf(mx, sc[b][i]);
        mx = __builtin_fmaxf(mx, other_half(mx)) * c;
        // The reference m follows the maximum only when that has grown by 2^kLazy: probabilities
        // stay below 2^kLazy and most tiles leave the sums as they are. top follows tv alike.
        if (__any(mx > m + float(kLazy) || (SPLIT && tv > top + kLazyV))) {
            const float mn = __builtin_fmaxf(m, mx);
            const float f = __builtin_amdgcn_exp2f(m - (mn == kNegInf ? 0.0f : mn));  // 0 before the first key
            const int tn = max(top, tv);
            const float fo = SPLIT ? ldexpf(f, top - tn) : f;
            l *= f;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= fo;
            m = mn, top = tn;
        }
        const float mu = m == kNegInf ? 0.0f : m;
        // The fused exponent is off by half a step of m, which is nothing until scores are so large
        // that the largest key's power would leave the range: their products are rounded first.
        const bool far = __any(__builtin_fabsf(mu) > 1048576.0f);
        if (far)
#pragma unroll
            for (int b = 0; b < SUB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[b][i] *= c;
        const float ce = far ? 1.0f : c;
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < SUB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sc[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][i], ce, -mu));
                sum += sc[b][i];
            }
        // An infinite value is all in its first part; its products with second parts are NaN or of
        // either sign. Scores that are NaN are -inf, and their keys without weight, where they are by
        // the first parts alone.
        if constexpr (SPLIT)
            if (__any(sum != sum)) {
                floatx16 s;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = 0.0f;
                const char *p = kst + (col * L::kKS + h * 8) * 2;
#pragma unroll
                for (int c = 0; c < DT * 2; ++c)
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const halfx8 *>(p + c * 32), qh[c], s, 0, 0, 0);
                sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sc[0][i] = sc[0][i] != sc[0][i] && s[i] == kNegInf ? 0.0f : sc[0][i];
                    sum += sc[0][i];
                }
            }
        l += sum;
        if (SPLIT && each) {
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const intx4 e = reinterpret_cast<const intx4 *>(vx)[2 * f + h];
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[0][4 * f + i] = ldexpf(sc[0][4 * f + i], e[i] - top + kSplitP);
            }
        } else if (SPLIT) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[0][i] = ldexpf(sc[0][i], ve[i / 8] - top + kSplitP);
        }
        if constexpr (HALF) {
#pragma unroll
            for (int b = 0; b < SUB; ++b)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    halfx8 p, pl;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float y = sc[b][x * 8 + i];
                        p[i] = static_cast<_Float16>(y);
                        if constexpr (SPLIT) pl[i] = static_cast<_Float16>(y - float(p[i]));
                    }
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        const char *vb = vst + ((b * 32 + x * 16) * L::kVS + t * 32) * 2;
                        const halfx8 v = read_vt<L::kVS>(vb, lane);
                        if constexpr (SPLIT) {
                            const halfx8 vl = read_vt<L::kVS>(vb + DP * 2, lane);
                            o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, p, o[t], 0, 0, 0);
                            o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl, o[t], 0, 0, 0);
                        }
                        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p, o[t], 0, 0, 0);
                    }
                }
        } else {
#pragma unroll
            for (int b = 0; b < SUB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float *p = reinterpret_cast<const float *>(vst) + (b * 32 + acc_row(i, h)) * L::kVS + col;
#pragma unroll
                    for (int t = 0; t < DT; ++t)
                        o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(p[t * 32], sc[b][i], o[t], 0, 0, 0);
                }
        }
    }
    l += __shfl_xor(l, 32);

    if constexpr (SPLIT) {  // the scales taken back
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = ldexpf(o[t][i], top - kSplitExp - kSplitP);
    }

    // Groups of waves join: group 0 takes the others' sums one after another.
    if constexpr (WK > 1) {
        float *slot = reinterpret_cast<float *>(smem) + wr * part_floats(DT);
        for (int src = 1; src < WK; ++src) {
            __syncthreads();
            if (wk == src) {
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) slot[(t * 16 + i) * 64 + lane] = o[t][i];
                slot[DT * 16 * 64 + lane] = m;
                slot[(DT * 16 + 1) * 64 + lane] = l;
            }
            __syncthreads();
            if (wk == 0) {
                const float m2 = slot[DT * 16 * 64 + lane], l2 = slot[(DT * 16 + 1) * 64 + lane];
                const float mn = __builtin_fmaxf(m, m2), mu = mn == kNegInf ? 0.0f : mn;
                const float f = __builtin_amdgcn_exp2f(m - mu), f2 = __builtin_amdgcn_exp2f(m2 - mu);
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        o[t][i] = __builtin_fmaf(o[t][i], f, slot[(t * 16 + i) * 64 + lane] * f2);
                l = __builtin_fmaf(l, f, l2 * f2);
                m = mn;
            }
        }
        if (wk) return;
    }
    // The values that were staged as zeros because they are not finite, for the rows that see them.
    if (bad) {
        const char *v0 = SPLIT ? static_cast<const char *>(a.v0) + uint64_t(item) * a.kv_tokens * a.ldv0 +
                                     int64_t(hk) * a.d * int64_t(sizeof(T))
                               : vp;
        for (int j = 0; j < keys; ++j) {
            const int t = token(j);
            if ((!SPLIT && t < lim_first) || t >= lim) continue;
            const T *v = reinterpret_cast<const T *>(v0 + uint64_t(uint32_t(t)) * (SPLIT ? a.ldv0 : a.ldv));
#pragma unroll
            for (int x = 0; x < DT; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int ch = x * 32 + acc_row(i, h);
                    const float f = ch < a.d ? float(v[ch]) : 0.0f;
                    if (SATURATED ? f != f : !(__builtin_fabsf(f) < __builtin_huge_valf())) o[x][i] += f;
                }
        }
    }
    if (a.part) {
        if (!row_ok) return;
        float *p = a.part + (int64_t(work) * WR + wr) * part_floats(DT);
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) p[(t * 16 + i) * 64 + lane] = o[t][i];
        p[DT * 16 * 64 + lane] = m;
        p[(DT * 16 + 1) * 64 + lane] = l;
        return;
    }
    if (!row_ok) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *op = static_cast<T *>(a.out) + (int64_t(item) * a.q_tokens + qi) * a.ldo + int64_t(qe) * a.d;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int ch = t * 32 + 8 * f + 4 * h;
            if constexpr (VEC) {
                typedef T V4 __attribute__((ext_vector_type(4)));
                if (ch < a.d) {
                    V4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(o[t][4 * f + e] * inv);
                    *reinterpret_cast<V4 *>(op + ch) = v;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (ch + e < a.d) op[ch + e] = static_cast<T>(o[t][4 * f + e] * inv);
            }
        }
}

// Joins the splits of a row tile: a wave per 32 rows and 32 channels, with the lanes'
// places of the partial sums.
template <typename T, int DT, int WR>
__global__ __launch_bounds__(64) void block_attention_join_kernel(Args a) {
    const int lane = threadIdx.x, col = lane & 31, h = lane >> 5;
    const int wr = blockIdx.x % WR, t = blockIdx.y;
    const int base = blockIdx.x / WR;  // (item, key head, block of queries, rows)
    int w = base;
    const int rt = w % a.row_tiles;
    w /= a.row_tiles;
    const int qb = w % a.nq;
    w /= a.nq;
    const int hk = w % a.hk, item = w / a.hk;
    const int q_len = a.q_len ? min(max(a.q_len[item], 0), a.q_tokens) : a.q_tokens;
    const int i0 = qb * a.qb, rows = (min(i0 + a.qb, q_len) - i0) * a.g;
    const int row = (rt * WR + wr) * 32 + col;
    if (rt * WR * 32 >= rows || row >= rows) return;  // its splits wrote nothing
    constexpr int PF = part_floats(DT);
    const float *p = a.part + (int64_t(base) * a.splits * WR + wr) * PF;
    float m = kNegInf;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) m = __builtin_fmaxf(m, p[int64_t(s) * WR * PF + DT * 16 * 64 + lane]);
    const float mu = m == kNegInf ? 0.0f : m;
    float l = 0.0f, o[16] = {};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const float *ps = p + int64_t(s) * WR * PF;
        const float f = __builtin_amdgcn_exp2f(ps[DT * 16 * 64 + lane] - mu);
        l = __builtin_fmaf(ps[(DT * 16 + 1) * 64 + lane], f, l);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __builtin_fmaf(ps[(t * 16 + i) * 64 + lane], f, o[i]);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *op = static_cast<T *>(a.out) + (int64_t(item) * a.q_tokens + i0 + row / a.g) * a.ldo +
            int64_t(hk * a.g + row % a.g) * a.d;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int ch = t * 32 + acc_row(i, h);
        if (ch < a.d) op[ch] = static_cast<T>(o[i] * inv);
    }
}

template <typename T, int MODE, bool VEC, int DT, int WR>
void launch(Context &ctx, const Args &a) {
    using L = Tiling<MODE, DT, WR>;
    const void *fn = reinterpret_cast<const void *>(&block_attention_kernel<T, MODE, VEC, DT, WR>);
    if (L::kLds > 48 * 1024) HIP_CHECK(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, L::kLds));
    const uint32_t grid = uint32_t((a.work + 7) / 8 * 8);
    block_attention_kernel<T, MODE, VEC, DT, WR><<<dim3{grid}, dim3{L::kThreads}, L::kLds, ctx.stream>>>(a);
    MH_LAUNCH_CHECK();
    if (a.splits > 1) {
        const dim3 jg{uint32_t(a.work / a.splits * WR), uint32_t((a.d + 31) / 32)};
        block_attention_join_kernel<T, DT, WR><<<jg, dim3{64}, 0, ctx.stream>>>(a);
        MH_LAUNCH_CHECK();
    }
}

template <typename T, int MODE, bool VEC, int DT>
void launch_rows(Context &ctx, const Args &a, int wr) {
    if constexpr (MODE != kSplit && DT <= 4)  // (as the plan takes them)
        if (wr == 1) return launch<T, MODE, VEC, DT, 1>(ctx, a);
    if (wr == 2) launch<T, MODE, VEC, DT, 2>(ctx, a);
    else launch<T, MODE, VEC, DT, 4>(ctx, a);
}

// dt: 32-channel tiles of the head as chosen by head_tiles.
template <typename T, int MODE>
void launch_mode(Context &ctx, const Args &a, int wr, int dt, bool vec) {
    if (vec) {
        if (dt == 1) launch_rows<T, MODE, true, 1>(ctx, a, wr);
        else if (dt == 2) launch_rows<T, MODE, true, 2>(ctx, a, wr);
        else if (dt == 3) launch_rows<T, MODE, true, 3>(ctx, a, wr);
        else if (dt == 4) launch_rows<T, MODE, true, 4>(ctx, a, wr);
        else if (dt == 5) launch_rows<T, MODE, true, 5>(ctx, a, wr);
        else if constexpr (MODE != kSplit) launch_rows<T, MODE, true, 8>(ctx, a, wr);
    } else {
        if (dt == 4) launch_rows<T, MODE, false, 4>(ctx, a, wr);
        else if (dt == 5) launch_rows<T, MODE, false, 5>(ctx, a, wr);
        else if constexpr (MODE != kSplit) launch_rows<T, MODE, false, 8>(ctx, a, wr);
    }
}

void launch_f16(Context &ctx, const Args &a, int wr, int dt, bool vec);
void launch_f32_half(Context &ctx, const Args &a, int wr, int dt, bool vec);
void launch_f32(Context &ctx, const Args &a, int wr, int dt, bool vec);
// Head tiles that launch_split takes (with two row waves or more).
inline bool split_fits(int dt) { return dt <= 5; }
void launch_split(Context &ctx, const Args &a, int wr, int dt, bool vec);
// k and v [n][kv_tokens] rows (ldk, ldv elements apart) of hk heads of d f32 -> kp, vp
// [n][kv_rows][hk][2][dk] f16 parts of every token below kv_len, scaled by its own power of
// two, zeros behind d; meta [n][hk][kv_rows].
void split_kv(Context &ctx, const float *k, const float *v, int64_t ldk, int64_t ldv, int n, int kv_tokens, int kv_rows,
              int hk, int d, int dk, const int32_t *kv_len, void *kp, void *vp, KeyScale *meta);

}  // namespace battn
}  // namespace mh
