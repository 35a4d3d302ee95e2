// Attention over a cache in 8 bits (cache8.hpp): one pass with a running maximum and sum.
//
// For a row of queries r and the keys j that it sees, with codes kc, vc and their blocks' scales:
//   s_j = c ks_j (q . kc_j)  (c = scale log2 e),  m = max s_j,  p_j = 2^(s_j - m),
//   o = sum p_j vs_j vc_j / sum p_j.
// Codes are integers of 8 bits and exact in f16, so both products run on the f16 matrix
// instructions and the scales join outside of them: ks in the scores, vs in the probabilities.
#pragma once

#include "cache8.hpp"

namespace mh {
namespace c8a {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));

constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kChunk = 64;  // tokens that a wave takes at once

struct Args {
    const void *q;
    void *out;
    int64_t ldq, ldo;
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int32_t *table, *q_len, *kv_len;
    float *part;  // split partials, NULL: none
    float c;      // scale . log2 e
    int n, q_tokens, hk, g, d, dp, blocks, pages, block_log, row_tiles, splits, work;
    int causal, window, sinks;
};

// Eight codes as f16: a byte b in the low bits of 1024 is 1024 + b.
__device__ __forceinline__ halfx8 halves(uint32_t lo, uint32_t hi) {
    halfx8 r;
    const halfx2 bias{_Float16(-1152.0f), _Float16(-1152.0f)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = __builtin_amdgcn_perm(0x64646464u, i < 2 ? lo : hi, i % 2 ? 0x04030402u : 0x04010400u);
        const halfx2 h = __builtin_bit_cast(halfx2, w) + bias;
        r[2 * i] = h[0], r[2 * i + 1] = h[1];
    }
    return r;
}

// The positions that a tile of rows looks at, and the chunks of kChunk tokens that hold them.
struct Range {
    int q_len, kv_len, off;  // position of row t: t + off
    int rows;                // of the tile's item and key head: q_len * g
    int head_chunks, first_chunk, chunks;  // chunks 0 .. head_chunks - 1, then first_chunk ..
    __device__ __forceinline__ int chunk(int i) const { return i < head_chunks ? i : first_chunk + i - head_chunks; }
};

__device__ __forceinline__ Range range_of(const Args &a, int item, int r0, int tile) {
    Range r;
    const int cap = a.blocks << a.block_log;
    r.q_len = a.q_len ? min(max(a.q_len[item], 0), a.q_tokens) : a.q_tokens;
    r.kv_len = a.kv_len ? min(max(a.kv_len[item], 0), cap) : cap;
    r.off = r.kv_len - r.q_len;
    r.rows = r.q_len * a.g;
    const int t0 = r0 / a.g, t1 = (min(r.rows, r0 + tile) - 1) / a.g;  // the tile's tokens
    const int end = a.causal ? min(r.kv_len, r.off + t1 + 1) : r.kv_len;
    const int begin = a.window ? min(max(r.off + t0 - a.window + 1, 0), max(end, 0)) : 0;
    const int sinks = min(a.sinks, begin);
    r.first_chunk = begin / kChunk;
    r.head_chunks = min((sinks + kChunk - 1) / kChunk, r.first_chunk);
    r.chunks = end > 0 && r0 < r.rows ? r.head_chunks + (end + kChunk - 1) / kChunk - r.first_chunk : 0;
    return r;
}

// Exponents of two by which a row's maximum may pass its reference: probabilities of up to
// 2^kLazy times a scale below 1 fit f16, split ones with 2^kSplitP more.
constexpr int kLazyHalf = 8, kLazySplit = 3, kSplitP = 11;
constexpr int kNoExp = -1000;
// How far a block's exponent of values may lie below the one that the sums are scaled by before
// that follows it down, and how far below the largest seen.
constexpr int kBelow = 10, kDeepest = 80;
constexpr int kSplitQ = 14;  // split queries are scaled to a largest value of 2^14 .. 2^15

// Few rows per key head: a wave takes 16 * NQ rows and every fourth chunk of 64 tokens of its
// workgroup's share, straight from memory into registers.
//
// S^T = K . Q^T on 16x16x32 instructions: a lane holds row lane % 16 of the queries and, with key
// row r of tile t standing for token 16 (r / 4) + 4 t + r % 4 of the chunk, the sixteen tokens
// 16 g .. 16 g + 15 of its group g = lane / 16. These are the B operand of O^T = V^T . P^T as they
// stand, and their values one load of 16 bytes from a channel's row; keys are 16 bytes of a
// token's row as two steps of the instruction. A block holds whole groups of 16 tokens, so page,
// scales and whether the page is there are the lane's own.
template <typename T, int PARTS, int DT, int NQ>
__global__ __launch_bounds__(256) void cache8_rows_kernel(Args a) {
    constexpr int DC = (DT + 3) / 4;  // chunks of 64 channels
    constexpr int kLazy = PARTS == 2 ? kLazySplit : kLazyHalf;
    constexpr int kOut = NQ * DT * 4 + NQ * 2;  // floats of a lane's partial: sums, then m and l
    extern __shared__ float joined[];           // [4][kOut][64]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;

    const int per_xcd = (a.work + 7) / 8;
    int w = int(blockIdx.x % 8) * per_xcd + int(blockIdx.x / 8);
    if (int(blockIdx.x / 8) >= per_xcd || w >= a.work) return;
    const int work = w;
    const int split = w % a.splits;
    w /= a.splits;
    const int r0 = w % a.row_tiles * 16 * NQ;
    w /= a.row_tiles;
    const int hk = w % a.hk, item = w / a.hk;
    const Range rg = range_of(a, item, r0, 16 * NQ);
    if (r0 >= rg.rows) return;
    const int share = (rg.chunks + a.splits - 1) / a.splits;
    const int c0 = min(split * share, rg.chunks), c1 = min(c0 + share, rg.chunks);

    // Q^T: this lane's rows, channels 64 c + 16 g + 8 s .. + 7 of step 2 c + s.
    halfx8 q[NQ][PARTS][DC * 2];
    float cq[NQ];           // what a row's products lack: c and its power of two
    int lo[NQ], hi[NQ];     // the row sees tokens lo .. hi - 1 and those below min(lo, sinks)
    const T *qp[NQ];
    bool row_ok[NQ];
    int64_t row_at[NQ], row_ch[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int row = r0 + n * 16 + col;
        row_ok[n] = row < rg.rows;
        const int t = (row_ok[n] ? row : r0) / a.g, h = hk * a.g + (row_ok[n] ? row : r0) % a.g;
        row_at[n] = int64_t(item) * a.q_tokens + t, row_ch[n] = int64_t(h) * a.d;
        qp[n] = static_cast<const T *>(a.q) + row_at[n] * a.ldq + row_ch[n];
        const int at = t + rg.off;
        hi[n] = a.causal ? min(rg.kv_len, at + 1) : rg.kv_len;
        lo[n] = a.window ? max(at - a.window + 1, 0) : 0;
        float x[DC * 2][8];
        float mx = 0.0f;
        bool odd = false;
#pragma unroll
        for (int s = 0; s < DC * 2; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int ch = (s / 2) * 64 + g * 16 + (s % 2) * 8 + i;
                const float v = ch < a.d ? float(qp[n][ch]) : 0.0f;
                x[s][i] = v;
                const bool fine = __builtin_fabsf(v) < __builtin_huge_valf();
                odd = odd || !fine;
                mx = fine ? __builtin_fmaxf(mx, __builtin_fabsf(v)) : mx;
            }
        int e = 0;
        if constexpr (sizeof(T) == 4) {  // scaled by a power of two per row, so that no value leaves f16
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
            e = mx == 0.0f ? 0 : __builtin_amdgcn_frexp_expf(mx) - 1 - kSplitQ;
        }
#pragma unroll
        for (int s = 0; s < DC * 2; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = sizeof(T) == 4 ? ldexpf(x[s][i], -e) : x[s][i];
                q[n][0][s][i] = static_cast<_Float16>(y);
                if constexpr (PARTS == 2) q[n][1][s][i] = static_cast<_Float16>(odd ? 0.0f : y - float(q[n][0][s][i]));
            }
        cq[n] = ldexpf(a.c, e);
    }

    const int64_t tile = int64_t(a.dp) << a.block_log;  // codes of a page and head
    const int block = 1 << a.block_log;
    // The chunk's codes: keys of four tiles, values of DT tiles; the lane's scales.
    uintx4 kc[4][DC], vc[DT];
    float ks, vs;
    bool there;
    int kch[DC];
#pragma unroll
    for (int c = 0; c < DC; ++c) kch[c] = c * 64 + g * 16 < a.dp ? c * 64 + g * 16 : 0;
    auto page_of = [&](int token, bool &ok) {
        const int b = token >> a.block_log;
        const int page = b < a.blocks ? a.table[int64_t(item) * a.blocks + b] : -1;
        ok = page >= 0 && page < a.pages;
        return (ok ? int64_t(page) : 0) * a.hk + hk;
    };
    auto load_k = [&](int chunk) {
        const int t0 = chunk * kChunk + 16 * (col >> 2);
        bool ok;
        const uint8_t *p = a.k + page_of(t0, ok) * tile + ((t0 & (block - 1)) + (col & 3)) * a.dp;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < DC; ++c) kc[t][c] = *reinterpret_cast<const uintx4 *>(p + 4 * t * a.dp + kch[c]);
    };
    auto load_v = [&](int chunk) {
        const int t0 = chunk * kChunk + 16 * g;
        const int64_t at = page_of(t0, there);
        there = there && t0 < rg.kv_len;  // (blocks behind it may never have been written)
        ks = a.ks[at], vs = a.vs[at];
        const uint8_t *p = a.v + at * tile + (t0 & (block - 1)) + (col << a.block_log);
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (t * 16 < a.dp) vc[t] = *reinterpret_cast<const uintx4 *>(p + (t * 16 << a.block_log));
    };

    floatx4 o[NQ][DT];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        m[n] = kNegInf, l[n] = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[n][t] = floatx4{0, 0, 0, 0};
    }
    int ve = kNoExp, ve_max = kNoExp;  // the exponent that the sums are scaled by, and the largest seen

    int i = c0 + wave;
    if (i < c1) load_k(rg.chunk(i)), load_v(rg.chunk(i));
    for (; i < c1; i += 4) {
        const int base = rg.chunk(i) * kChunk;
        floatx4 sc[NQ][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) sc[n][t] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < DC * 2; ++s) {
                const uintx4 w = kc[t][s / 2];
                const halfx8 h = s % 2 ? halves(w[2], w[3]) : halves(w[0], w[1]);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    if constexpr (PARTS == 2)
                        sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, q[n][1][s], sc[n][t], 0, 0, 0);
                    sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, q[n][0][s], sc[n][t], 0, 0, 0);
                }
            }
        }
        const bool more = i + 4 < c1;
        const float ks_now = ks, vs_now = vs;
        const bool there_now = there;
        if (more) load_k(rg.chunk(i + 4));

        // The sums' exponent follows the blocks' scales of values.
        int tv = there_now && vs_now > 0.0f ? __builtin_amdgcn_frexp_expf(vs_now) : kNoExp;
        tv = max(tv, __shfl_xor(tv, 16));
        tv = __builtin_amdgcn_readfirstlane(max(tv, __shfl_xor(tv, 32)));
        if (tv > ve || (tv > kNoExp && tv < ve - kBelow)) {
            ve_max = max(ve_max, tv);
            const int to = max(tv, ve_max - kDeepest);
            if (to != ve) {
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int t = 0; t < DT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][t][e] = ldexpf(o[n][t][e], ve - to);
                ve = to;
            }
        }
        const float vrel = there_now && vs_now > 0.0f ? ldexpf(vs_now, (PARTS == 2 ? kSplitP : 0) - ve) : 0.0f;

        halfx8 p[NQ][PARTS][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float c = __builtin_fminf(ks_now * cq[n], 0x1.fffffep127f);  // (0 times it is 0)
            const int t0 = base + 16 * g;
            const bool whole = there_now && t0 + 16 <= hi[n] && (t0 >= lo[n] || t0 + 16 <= a.sinks);
            float mx = kNegInf;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[n][t][e] *= c;
            if (!__all(whole)) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = t0 + 4 * t + e;
                        if (!(there_now && j < hi[n] && (j >= lo[n] || j < a.sinks))) sc[n][t][e] = kNegInf;
                    }
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = __builtin_fmaxf(mx, sc[n][t][e]);
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
            if (__any(mx > m[n] + float(kLazy))) {
                const float mn = __builtin_fmaxf(m[n], mx);
                const float f = __builtin_amdgcn_exp2f(m[n] - (mn == kNegInf ? 0.0f : mn));
                l[n] *= f;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][t][e] *= f;
                m[n] = mn;
            }
            const float mu = m[n] == kNegInf ? 0.0f : m[n];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = __builtin_amdgcn_exp2f(sc[n][t][e] - mu);
                    l[n] += y;
                    float z = y * vrel;
                    // (both parts are of z rounded to f32; a product fused with its conversion is not)
                    if constexpr (PARTS == 2) asm("" : "+v"(z));
                    const _Float16 h = static_cast<_Float16>(z);
                    p[n][0][t / 2][(t % 2) * 4 + e] = h;
                    if constexpr (PARTS == 2) p[n][1][t / 2][(t % 2) * 4 + e] = static_cast<_Float16>(z - float(h));
                }
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            if (t * 16 >= a.dp) continue;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const halfx8 h = halves(vc[t][2 * s], vc[t][2 * s + 1]);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    if constexpr (PARTS == 2)
                        o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, p[n][1][s], o[n][t], 0, 0, 0);
                    o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, p[n][0][s], o[n][t], 0, 0, 0);
                }
            }
        }
        if (more) load_v(rg.chunk(i + 4));
    }

    // Scales taken back; the waves' sums joined in LDS, each wave then finishing some of them.
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                joined[(wave * kOut + (n * DT + t) * 4 + e) * 64 + lane] =
                    ldexpf(o[n][t][e], ve == kNoExp ? 0 : ve - (PARTS == 2 ? kSplitP : 0));
        joined[(wave * kOut + NQ * DT * 4 + 2 * n) * 64 + lane] = m[n];
        joined[(wave * kOut + NQ * DT * 4 + 2 * n + 1) * 64 + lane] = l[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        float mw[4], top = kNegInf, sum = 0.0f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            mw[x] = joined[(x * kOut + NQ * DT * 4 + 2 * n) * 64 + lane];
            top = __builtin_fmaxf(top, mw[x]);
        }
        const float mu = top == kNegInf ? 0.0f : top;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            mw[x] = __builtin_amdgcn_exp2f(mw[x] - mu);
            sum = __builtin_fmaf(joined[(x * kOut + NQ * DT * 4 + 2 * n + 1) * 64 + lane], mw[x], sum);
        }
        const float inv = a.part ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
        float *part = a.part ? a.part + ((int64_t(work) * NQ + n) * 16 + col) * (DT * 16 + 2) : nullptr;
        if (part && wave == 0 && g == 0) part[DT * 16] = top, part[DT * 16 + 1] = sum;
        T *op = static_cast<T *>(a.out) + row_at[n] * a.ldo + row_ch[n];
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            if (t % 4 != wave || t * 16 >= a.d) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float y = 0.0f;
#pragma unroll
                for (int x = 0; x < 4; ++x) y = __builtin_fmaf(joined[(x * kOut + (n * DT + t) * 4 + e) * 64 + lane], mw[x], y);
                const int ch = t * 16 + 4 * g + e;
                if (part) part[ch] = y;
                else if (row_ok[n] && ch < a.d) op[ch] = static_cast<T>(y * inv);
            }
        }
    }
}

// Joins the splits of a row: a wave per row.
template <typename T, int DT, int NQ>
__global__ __launch_bounds__(64) void cache8_join_kernel(Args a) {
    const int lane = threadIdx.x, col = blockIdx.x % (16 * NQ);
    const int base = blockIdx.x / (16 * NQ);
    int w = base;
    const int r0 = w % a.row_tiles * 16 * NQ;
    w /= a.row_tiles;
    const int hk = w % a.hk, item = w / a.hk;
    const int q_len = a.q_len ? min(max(a.q_len[item], 0), a.q_tokens) : a.q_tokens;
    const int row = r0 + col;
    if (row >= q_len * a.g) return;
    constexpr int PF = DT * 16 + 2;
    const float *p = a.part + (int64_t(base) * a.splits * NQ * 16 + col) * PF;
    const int64_t step = int64_t(NQ) * 16 * PF;
    float m = kNegInf;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) m = __builtin_fmaxf(m, p[s * step + DT * 16]);
    const float mu = m == kNegInf ? 0.0f : m;
    float l = 0.0f, o[(DT * 16 + 63) / 64] = {};
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
        const float f = __builtin_amdgcn_exp2f(p[s * step + DT * 16] - mu);
        l = __builtin_fmaf(p[s * step + DT * 16 + 1], f, l);
#pragma unroll
        for (int i = 0; i < (DT * 16 + 63) / 64; ++i)
            if (i * 64 + lane < a.d) o[i] = __builtin_fmaf(p[s * step + i * 64 + lane], f, o[i]);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *op = static_cast<T *>(a.out) + (int64_t(item) * a.q_tokens + row / a.g) * a.ldo + int64_t(hk * a.g + row % a.g) * a.d;
#pragma unroll
    for (int i = 0; i < (DT * 16 + 63) / 64; ++i)
        if (i * 64 + lane < a.d) op[i * 64 + lane] = static_cast<T>(o[i] * inv);
}

template <typename T, int PARTS, int DT, int NQ>
void launch_rows(Context &ctx, const Args &a) {
    const size_t lds = size_t(4) * (NQ * DT * 4 + NQ * 2) * 64 * 4;
    const void *fn = reinterpret_cast<const void *>(&cache8_rows_kernel<T, PARTS, DT, NQ>);
    if (lds > 48 * 1024) HIP_CHECK(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
    cache8_rows_kernel<T, PARTS, DT, NQ><<<dim3{uint32_t((a.work + 7) / 8 * 8)}, dim3{256}, lds, ctx.stream>>>(a);
    MH_LAUNCH_CHECK();
    if (a.part) {
        cache8_join_kernel<T, DT, NQ><<<dim3{uint32_t(a.work / a.splits * 16 * NQ)}, dim3{64}, 0, ctx.stream>>>(a);
        MH_LAUNCH_CHECK();
    }
}

template <typename T, int PARTS>
void launch_rows_dt(Context &ctx, const Args &a, int nq, int dt) {
    auto by_nq = [&](auto n) {
        constexpr int DT = decltype(n)::value;
        if (nq == 1) launch_rows<T, PARTS, DT, 1>(ctx, a);
        else if constexpr (DT <= 8) launch_rows<T, PARTS, DT, 2>(ctx, a);
    };
    if (dt == 4) by_nq(std::integral_constant<int, 4>{});
    else if (dt == 5) by_nq(std::integral_constant<int, 5>{});
    else if (dt == 6) by_nq(std::integral_constant<int, 6>{});
    else if (dt == 8) by_nq(std::integral_constant<int, 8>{});
    else if (dt == 10) by_nq(std::integral_constant<int, 10>{});
    else by_nq(std::integral_constant<int, 16>{});
}

void launch_f16(Context &ctx, const Args &a, int nq, int dt);
void launch_f32(Context &ctx, const Args &a, int nq, int dt);
void launch_f32_half(Context &ctx, const Args &a, int nq, int dt);

}  // namespace c8a
}  // namespace mh
