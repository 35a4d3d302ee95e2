// The blocks of keys that each block of queries attends to.
//
// block_means_kernel: m_b = mean of a block's key rows, the state a cache keeps per block.
// Bound: memory, each key read once.
//
// block_select_kernel: score s_b = <q, m_b> with q the mean over the valid queries of a
// block and over the heads that share a key head; the `top` largest, ties to the lower
// index; causal: the blocks of the queries' own tokens before all others. The scores
// decide, so they are f64 sums of f32 products' factors: another order of the sum moves
// them by 1e-16 of their terms, and the selection does not depend on it. Bound: memory,
// the queries read once (the products are a 1 / q_block of the attention's).
//
// Scores as ordered 64-bit keys in LDS; a wave finds the top-th largest bit by bit from
// above, counting the keys at or above a candidate with ballots, and stops once exactly
// `top` are, which takes the exponent's bits and as many as tell the blocks apart.
//
// Measured, means and selection together: 2 x 4096 tokens, 8 heads of 80, f32, 16 of 64
// blocks 18.9 us (5.6 and 14.6 by themselves); 16384 tokens, 16 / 8 heads of 128, f16, 32 of
// 256 blocks 40 us (7.8 and 28.7). Eight waves per workgroup against four: 63 -> 45 and
// 27 -> 18.5 us; products on v_mfma_f64_4x4x4 against 16x16x4, most of whose rows are no
// queries, 45 -> 40 us; on the vector units 154 us.
#include <algorithm>

#include "attention.hpp"

namespace mh {
namespace {

template <typename T, int W>
__device__ __forceinline__ void load_run(const T *p, float (&v)[W]) {
    if constexpr (W == 1) {
        v[0] = float(*p);
    } else {
        typedef T V __attribute__((ext_vector_type(W)));
        const V r = *reinterpret_cast<const V *>(p);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = float(r[i]);
    }
}

__device__ __forceinline__ int clamp_len(const int32_t *len, int item, int most) {
    return len ? min(max(len[item], 0), most) : most;
}

// One workgroup per (item, block, run of 32 column vectors), these innermost; eight row groups of 32
// threads, each summing every eighth row, joined in LDS.
constexpr int kMeanCols = 32, kMeanRows = 8;

template <typename T, int W>
__global__ __launch_bounds__(256) void block_means_kernel(const T *x, int64_t ld, int tokens, int cols, int block,
                                                          const int32_t *first, const int32_t *len, float *means) {
    __shared__ double part[kMeanRows][kMeanCols * W];
    const uint32_t cg = (uint32_t(cols) + kMeanCols * W - 1) / (kMeanCols * W), at = blockIdx.x / cg;
    const int nb = (tokens + block - 1) / block, item = int(at / uint32_t(nb)), b = int(at % uint32_t(nb));
    const int n = clamp_len(len, item, tokens);
    const int r0 = b * block, r1 = min(r0 + block, n);
    if (r0 >= r1 || (first && r0 + block <= first[item])) return;
    const int c = threadIdx.x % kMeanCols, rg = threadIdx.x / kMeanCols;
    const int col0 = int(blockIdx.x % cg) * kMeanCols * W, col = col0 + c * W;
    double sum[W] = {};
    if (col < cols) {
        const T *p = x + int64_t(item) * tokens * ld + col;
#pragma unroll 8
        for (int r = r0 + rg; r < r1; r += kMeanRows) {
            float v[W];
            load_run<T, W>(p + int64_t(r) * ld, v);
#pragma unroll
            for (int i = 0; i < W; ++i) sum[i] += double(v[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) part[rg][c * W + i] = sum[i];
    __syncthreads();
    for (int j = threadIdx.x; j < kMeanCols * W; j += 256) {
        const int cj = col0 + j;
        if (cj >= cols) break;
        double s = 0;
#pragma unroll
        for (int g = 0; g < kMeanRows; ++g) s += part[g][j];
        means[(int64_t(item) * nb + b) * cols + cj] = float(s / double(r1 - r0));
    }
}

struct SelectArgs {
    const void *q;
    int64_t ld;
    const float *means;
    const int32_t *q_len, *kv_len;
    int32_t *blocks;
    int q_tokens, kv_tokens, hk, g, d, qb, kb, nq, nk, top, tiles;
    bool causal;
};

constexpr uint64_t kForced = ~uint64_t(0);

// Order-preserving: NaN lowest, then -inf .. +inf (zeros equal), forced blocks above.
__device__ __forceinline__ uint64_t order_key(double s) {
    if (s != s) return 0;
    s += 0.0;
    const uint64_t b = __builtin_bit_cast(uint64_t, s);
    return (b >> 63) ? ~b : b | (uint64_t(1) << 63);
}

// One workgroup per (item, key head, TQ blocks of queries); W, MW: the runs in which the
// queries and the means are read.
constexpr int kSelWaves = 8;
constexpr int kRegKeys = 8;  // keys per lane that the search holds in registers

template <typename T, int W, int MW, int TQ>
__global__ __launch_bounds__(64 * kSelWaves) void block_select_kernel(SelectArgs a) {
    extern __shared__ uint64_t keys[];  // [TQ][nk]
    constexpr int kQS = kMaxHeadDim + 20;  // rows of a read on distinct banks, sixteen zeros behind d
    __shared__ __align__(16) float qm[TQ][kQS];
    const int tile = blockIdx.x % a.tiles;
    const int hk = (blockIdx.x / a.tiles) % a.hk, item = blockIdx.x / a.tiles / a.hk;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int q_len = clamp_len(a.q_len, item, a.q_tokens), kv_len = clamp_len(a.kv_len, item, a.kv_tokens);
    const int b0 = tile * TQ;
    const int seen_all = (kv_len + a.kb - 1) / a.kb;
    const int l16 = lane & 15, kg = lane >> 4;
    // The first means that the scores take are loaded before the queries.
    const int t_first = __builtin_amdgcn_readfirstlane(wave) * 16;
    float mv[4][4];
    auto load_means = [&](int t0, int c0) {
        const int b = min(t0 + l16, seen_all - 1);
        const float *m = a.means + ((int64_t(item) * a.nk + b) * a.hk + hk) * a.d;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c = c0 + u * 16 + kg * 4;
            if constexpr (MW == 4) {
                load_run<float, 4>(m + min(c, a.d - 4), mv[u]);
#pragma unroll
                for (int e = 0; e < 4; ++e) mv[u][e] = c < a.d ? mv[u][e] : 0.0f;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) mv[u][e] = c + e < a.d ? m[c + e] : 0.0f;
            }
        }
    };
    if (TQ > 1 && t_first < seen_all) load_means(t_first, 0);

    // Mean query of each block: kParts waves per block, lanes over (row group, run of channels).
    constexpr int kParts = kSelWaves / TQ;
    __shared__ double part[kSelWaves][kMaxHeadDim];
    const int runs = a.d / W;
    int span = 1;  // lanes per row: the next power of two
    while (span < runs && span < 64) span *= 2;
    const int groups = 64 / span, cl = lane % span, rg = lane / span;
    // Zeros behind d, which the products' last run of sixteen reads.
    for (int i = tid; i < TQ * 16; i += 64 * kSelWaves) qm[i / 16][a.d + i % 16] = 0.0f;
    {
        const int t = wave / kParts, i0 = (b0 + t) * a.qb, i1 = min(i0 + a.qb, q_len);
        const int rows = max(i1 - i0, 0) * a.g, step = groups * kParts;
        const T *base = static_cast<const T *>(a.q) + (int64_t(item) * a.q_tokens + i0) * a.ld + int64_t(hk) * a.g * a.d;
        for (int c0 = cl; c0 < ((runs + span - 1) / span) * span; c0 += span) {
            double sum[W] = {};
            if (c0 < runs) {
#pragma unroll 8
                for (int r = rg * kParts + wave % kParts; r < rows; r += step) {
                    const int i = r / a.g, e = r - i * a.g;
                    float v[W];
                    load_run<T, W>(base + int64_t(i) * a.ld + e * a.d + c0 * W, v);
#pragma unroll
                    for (int k = 0; k < W; ++k) sum[k] += double(v[k]);
                }
            }
            for (int m = span; m < 64; m *= 2)
#pragma unroll
                for (int k = 0; k < W; ++k) sum[k] += __shfl_xor(sum[k], m);
            if (rg == 0 && c0 < runs)
#pragma unroll
                for (int k = 0; k < W; ++k) part[wave][c0 * W + k] = sum[k];
        }
    }
    __syncthreads();
    for (int i = tid; i < TQ * a.d; i += 64 * kSelWaves) {
        const int t = i / a.d, c = i - t * a.d;
        const int rows = max(min((b0 + t + 1) * a.qb, q_len) - (b0 + t) * a.qb, 0) * a.g;
        double sum = 0;
#pragma unroll
        for (int p = 0; p < kParts; ++p) sum += part[t * kParts + p][c];
        qm[t][c] = rows ? float(sum / double(rows)) : 0.0f;
    }
    __syncthreads();

    // Scores. One block of queries: sixteen lanes per key block. More: 16 key blocks x 4 query
    // blocks on the f64 matrix instruction of four 4 x 4 products (lane: key block lane % 16,
    // query block lane % 4, four channels at 4 (lane / 16); its result is of key block
    // 4 (lane / 4 % 4) + lane / 16), the next means loaded meanwhile.
    if constexpr (TQ == 1) {
        for (int t0 = 0; t0 < seen_all; t0 += 4 * kSelWaves) {
            const int b = t0 + wave * 4 + kg;
            double s = 0;
            if (b < seen_all) {
                const float *m = a.means + ((int64_t(item) * a.nk + b) * a.hk + hk) * a.d;
                for (int c = l16 * MW; c < a.d; c += 16 * MW) {
                    float v[MW];
                    load_run<float, MW>(m + c, v);
#pragma unroll
                    for (int e = 0; e < MW; ++e) s = __builtin_fma(double(qm[0][c + e]), double(v[e]), s);
                }
            }
#pragma unroll
            for (int x = 8; x; x >>= 1) s += __shfl_xor(s, x);
            if (b < seen_all && l16 == 0) keys[b] = order_key(s);
        }
    } else {
        constexpr int QG = TQ / 4 ? TQ / 4 : 1;
        double acc[QG] = {};
        int t0 = t_first, c0 = 0;
        while (t0 < seen_all) {
            float cur[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) cur[u][e] = mv[u][e];
            const bool last = c0 + 64 >= a.d;
            const int t_next = last ? t0 + 16 * kSelWaves : t0, c_next = last ? 0 : c0 + 64;
            if (t_next < seen_all) load_means(t_next, c_next);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (c0 + u * 16 >= a.d) break;
#pragma unroll
                for (int x = 0; x < QG; ++x) {
                    float qv[4];
                    load_run<float, 4>(qm[min(x * 4 + (lane & 3), TQ - 1)] + c0 + u * 16 + kg * 4, qv);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[x] = __builtin_amdgcn_mfma_f64_4x4x4f64(double(cur[u][e]), double(qv[e]), acc[x], 0, 0, 0);
                }
            }
            if (last) {
                const int r = t0 + (lane >> 2 & 3) * 4 + kg;
#pragma unroll
                for (int x = 0; x < QG; ++x) {
                    const int t = x * 4 + (lane & 3);
                    if (t < TQ && r < seen_all) keys[t * a.nk + r] = order_key(acc[x]);
                    acc[x] = 0;
                }
            }
            t0 = t_next, c0 = c_next;
        }
    }
    __syncthreads();

    if (wave < TQ && b0 + wave < a.nq) {
        const int t = wave, qb = b0 + t;
        int32_t *out = a.blocks + ((int64_t(item) * a.nq + qb) * a.hk + hk) * a.top;
        const int i0 = qb * a.qb, i1 = min(i0 + a.qb, q_len);
        int seen = i1 > i0 ? seen_all : 0, f0 = 0, f1 = 0;  // blocks f0 .. f1 - 1 come first
        if (a.causal && seen) {
            const int lo = kv_len - q_len + i0, hi = kv_len - q_len + i1 - 1;
            seen = hi < 0 ? 0 : hi / a.kb + 1;
            f0 = max(lo, 0) / a.kb, f1 = seen;
        }
        uint64_t *k = keys + t * a.nk;
        int count = 0;
        if (seen > a.top) {
            for (int b = f0 + lane; b < f1; b += 64) k[b] = kForced;
            __threadfence_block();
            uint64_t at = 0;  // the largest key with at least `top` keys at or above it
            int above = seen;
            if (seen <= 64 * kRegKeys) {  // keys in registers
                uint64_t r[kRegKeys];
#pragma unroll
                for (int j = 0; j < kRegKeys; ++j) r[j] = lane + j * 64 < seen ? k[lane + j * 64] : 0;
                for (int bit = 63; bit >= 0 && above != a.top; --bit) {
                    const uint64_t cand = at | (uint64_t(1) << bit);
                    int n = 0;
#pragma unroll
                    for (int j = 0; j < kRegKeys; ++j)
                        if (j * 64 < seen) n += __popcll(__ballot(r[j] >= cand));
                    if (n >= a.top) at = cand, above = n;
                }
            } else {
                for (int bit = 63; bit >= 0 && above != a.top; --bit) {
                    const uint64_t cand = at | (uint64_t(1) << bit);
                    int n = 0;
                    for (int b = lane; b < (seen + 63) / 64 * 64; b += 64)
                        n += __popcll(__ballot(b < seen && k[b] >= cand));
                    if (n >= a.top) at = cand, above = n;
                }
            }
            // above == top: every key at or above; else the lower indices of those equal to it
            int greater = 0;
            const bool ties = above != a.top;
            if (ties)
                for (int b = lane; b < (seen + 63) / 64 * 64; b += 64)
                    greater += __popcll(__ballot(b < seen && k[b] > at));
            int quota = ties ? a.top - greater : seen;
            for (int b = lane; b < (seen + 63) / 64 * 64; b += 64) {
                const uint64_t v = b < seen ? k[b] : 0;
                const uint64_t below = (uint64_t(1) << lane) - 1;
                const bool gt = b < seen && (ties ? v > at : v >= at);
                const bool eq = b < seen && ties && v == at;
                const uint64_t eqs = __ballot(eq);
                const bool take = gt || (eq && __popcll(eqs & below) < quota);
                const uint64_t takes = __ballot(take);
                if (take) out[count + __popcll(takes & below)] = b;
                count += __popcll(takes);
                quota -= min(quota, int(__popcll(eqs)));
            }
        } else {
            for (int b = lane; b < seen; b += 64) out[b] = b;
            count = seen;
        }
        for (int i = count + lane; i < a.top; i += 64) out[i] = -1;
    }
}

template <typename T, int W, int MW>
void select_w(Context &ctx, SelectArgs &a, int n) {
    // Blocks of queries per workgroup: up to eight share the reads of the means, as many
    // as leave the card two workgroups per CU and their keys in 32 KiB of LDS. 128 blocks of
    // 24 heads: 8 24.9 us, 4 22.8, 2 31.7, 1 39.1; 64 blocks of 8 heads: 14.5, 11.0, 10.0, 9.3;
    // single tokens of 64 requests, 8 heads: 14.6, 13.0, 13.2, 12.6.
    int tq = 8;
    while (tq > 1 && (tq > a.nq || int64_t(tq) * a.nk * 8 > 32 * 1024 ||
                      int64_t(n) * a.hk * ceil_div(a.nq, tq) < 2 * ctx.cu_count))
        tq /= 2;
    a.tiles = int(ceil_div(a.nq, tq));
    const int64_t blocks = int64_t(n) * a.hk * a.tiles;
    MH_REQUIRE(blocks < (int64_t(1) << 31), "block_select: too many blocks of queries");
    const uint32_t lds = uint32_t(tq) * a.nk * 8;
    const dim3 grid{uint32_t(blocks)}, block{64 * kSelWaves};
    if (tq == 8) {
        block_select_kernel<T, W, MW, 8><<<grid, block, lds, ctx.stream>>>(a);
    } else if (tq == 4) {
        block_select_kernel<T, W, MW, 4><<<grid, block, lds, ctx.stream>>>(a);
    } else if (tq == 2) {
        block_select_kernel<T, W, MW, 2><<<grid, block, lds, ctx.stream>>>(a);
    } else {
        const void *fn = reinterpret_cast<const void *>(&block_select_kernel<T, W, MW, 1>);
        if (lds > 48 * 1024) HIP_CHECK(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
        block_select_kernel<T, W, MW, 1><<<grid, block, lds, ctx.stream>>>(a);
    }
    MH_LAUNCH_CHECK();
}

template <typename T, int W>
void select_q(Context &ctx, SelectArgs &a, int n) {
    if (a.d % 4 == 0 && aligned16(a.means)) select_w<T, W, 4>(ctx, a, n);
    else select_w<T, W, 1>(ctx, a, n);
}

template <typename T>
bool runs_of(int w, const void *p, int64_t ld, int64_t cols) {
    return cols % w == 0 && ld % w == 0 && reinterpret_cast<uintptr_t>(p) % (w * sizeof(T)) == 0;
}

template <typename T>
void means_t(Context &ctx, HeadRows x, int n, int tokens, int d, const int32_t *first, const int32_t *len, int block,
             float *means) {
    constexpr int V = 16 / int(sizeof(T));
    const int cols = x.heads * d;
    const bool vec = runs_of<T>(V, x.p, x.ld, cols);
    const int64_t nb = ceil_div(tokens, block), cg = ceil_div(cols, kMeanCols * (vec ? V : 1));
    MH_REQUIRE(cg * nb < (int64_t(1) << 31) / n, "block_means: too many blocks");
    const dim3 grid{uint32_t(cg * nb * n)}, tb{256};
    const T *p = static_cast<const T *>(x.p);
    if (vec) block_means_kernel<T, V><<<grid, tb, 0, ctx.stream>>>(p, x.ld, tokens, cols, block, first, len, means);
    else block_means_kernel<T, 1><<<grid, tb, 0, ctx.stream>>>(p, x.ld, tokens, cols, block, first, len, means);
    MH_LAUNCH_CHECK();
}

}  // namespace

void block_means(Context &ctx, HeadRows x, WeightType type, int n, int tokens, int d, const int32_t *first,
                 const int32_t *len, int block, float *means) {
    if (!n || !tokens) return;
    if (type == kF16) means_t<_Float16>(ctx, x, n, tokens, d, first, len, block, means);
    else means_t<float>(ctx, x, n, tokens, d, first, len, block, means);
}

void block_select(Context &ctx, HeadRows q, WeightType type, const BlockShape &s, const float *k_means,
                  int32_t *blocks) {
    if (!s.n || !s.q_tokens) return;
    SelectArgs a{};
    a.q = q.p, a.ld = q.ld, a.means = k_means, a.q_len = s.q_len, a.kv_len = s.kv_len, a.blocks = blocks;
    a.q_tokens = s.q_tokens, a.kv_tokens = s.kv_tokens, a.hk = s.heads_kv, a.g = s.heads_q / s.heads_kv, a.d = s.d;
    a.qb = s.q_block, a.kb = s.kv_block, a.nq = s.q_blocks(), a.nk = s.kv_blocks(), a.top = s.top, a.causal = s.causal;
    if (type == kF16) {
        if (runs_of<_Float16>(8, q.p, q.ld, s.d)) select_q<_Float16, 8>(ctx, a, s.n);
        else select_q<_Float16, 1>(ctx, a, s.n);
    } else {
        if (runs_of<float>(4, q.p, q.ld, s.d)) select_q<float, 4>(ctx, a, s.n);
        else select_q<float, 1>(ctx, a, s.n);
    }
}

}  // namespace mh
