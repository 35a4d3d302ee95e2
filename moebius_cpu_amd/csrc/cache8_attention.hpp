// Attention over a cache in 8 bits (cache8.hpp): one pass with a running maximum and sum.
//
// For a row of queries r and the keys j that it sees, with codes kc, vc and their blocks' scales:
//   s_j = c ks_j (q . kc_j)  (c = scale log2 e),  m = max s_j,  p_j = 2^(s_j - m),
//   o = sum p_j vs_j vc_j / sum p_j.
// Codes are integers of 8 bits and exact in f16, so both products run on the f16 matrix
// instructions and the scales join outside of them: ks in the scores, vs in the probabilities.
//
// The probabilities meet vs in f16, whose range is short, so the sums are held against a power of two
// near the scales of the values that are being read. It moves when those do, and where the blocks of
// one chunk differ by more than 2^kBelow their groups are taken one after another.
//
// f32 queries and all probabilities are two f16 parts, at the cost of a product more: one part alone is off by
// as much as an f16 output's own rounding. FAST contexts take one of each.
#pragma once

#include <type_traits>

#include "cache8.hpp"

namespace mh {
namespace c8a {

typedef float floatx2 __attribute__((ext_vector_type(2)));
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
    int q_tokens, hk, g, d, dp, blocks, pages, block_log, row_tiles, splits, work;
    int causal, window, sinks;
    int wide;  // rows of q in vectors of eight, of out in vectors of four
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

// Which of the sixteen tokens from t0 on a row sees that sees lo .. hi - 1 and those below sinks and hi:
// bits, as branches of every token's own cost more than a chunk's products.
__device__ __forceinline__ uint32_t seen_bits(int t0, int lo, int hi, int sinks) {
    auto below = [&](int limit) { return (1u << min(max(limit - t0, 0), 16)) - 1u; };
    return below(hi) & (~below(lo) | below(sinks));
}

// Exponents of two by which a row's maximum may pass its reference (in one f16 part, in two), and what the scales
// of values beside the probabilities are lifted by: 2^kLazy times a scale below 2^kUp fits f16, and the more of its
// range lies below, the smaller the probabilities that keep their bits. Rescales are rarer where kLazy is larger,
// which pays where a probability costs least.
constexpr int kLazyHalf = 8, kUpHalf = 7, kLazySplit = 3, kUpSplit = 12;
constexpr int kNoExp = -1000;
// How far an exponent of a chunk's values may lie below the one that the sums are scaled by before that follows the
// chunk down: a scale beside a probability is 2^(kUp - 1 - kBelow) or more, so that a probability is held to 2^-25 of
// that, 2^-28 and 2^-33 of its row's largest, where its own 2^-11 or 2^-22 is less. Rows may see only the small values
// of a chunk, thousands of them with small probabilities, which then must not round to nothing.
// kDeepest: how far below the largest seen it goes; 2^72 times the sums of 2^30 keys, 127 2^(kLazy + kUp) each,
// are below the end of f32.
constexpr int kBelow = 3, kDeepest = 72;
constexpr int kReadsAhead = 6;  // fragments of 16 bytes per lane on their way from LDS
constexpr int kSplitQ = 14;  // split queries are scaled to a largest value of 2^14 .. 2^15

// Eight channels of a row of queries from ch on, zeros behind d.
template <typename T>
__device__ __forceinline__ void load8(const T *p, int ch, int d, int wide, float (&x)[8]) {
    typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int kE = 16 / int(sizeof(T));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    if (wide) {
        if (ch < d)
#pragma unroll
            for (int j = 0; j < 8 / kE; ++j) {
                const V v = reinterpret_cast<const V *>(p + ch)[j];
#pragma unroll
                for (int i = 0; i < kE; ++i) x[j * kE + i] = float(v[i]);
            }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (ch + i < d) x[i] = float(p[ch + i]);
    }
}

// Few rows per key head: a wave takes 16 * NQ rows and every WV-th chunk of 64 tokens of its
// workgroup's share, straight from memory into registers.
//
// S^T = K . Q^T on 16x16x32 instructions: a lane holds row lane % 16 of the queries and, with key
// row r of tile t standing for token 16 (r / 4) + 4 t + r % 4 of the chunk, the sixteen tokens
// 16 g .. 16 g + 15 of its group g = lane / 16. These are the B operand of O^T = V^T . P^T as they
// stand, and their values one load of 16 bytes from a channel's row; keys are 16 bytes of a
// token's row as two steps of the instruction. A block holds whole groups of 16 tokens, so page,
// scales and whether the page is there are the lane's own.
//
// Bound: memory, and the latency of its loads where the tokens are few. Codes are read once and never
// shared between rows that are not in one wave, which is why nothing is staged. Single tokens of 8 items with up
// to 16384 tokens, 32 heads over 8 of 128 (210 MB of codes): 42 us of the call's 51, 5 TB/s, the join 5. One token
// over 300, 8 heads of 80, f32: 9.1 us, one workgroup's chain of lengths, page, codes and products.
template <typename T, int PARTS, int DT, int NQ, int WV>
__global__ __launch_bounds__(64 * WV, (WV / 4)) void cache8_rows_kernel(Args a) {
    constexpr int DC = (DT + 3) / 4;  // chunks of 64 channels
    // Probabilities of f16 in two parts on FAST contexts too: the kernel waits for memory, and takes 0.3 us more of 50.
    constexpr int PP = sizeof(T) == 2 ? 2 : PARTS;
    constexpr int kLazy = PP == 2 ? kLazySplit : kLazyHalf, kUp = PP == 2 ? kUpSplit : kUpHalf;
    constexpr int kOut = NQ * DT * 4 + NQ * 2;  // floats of a lane's partial: sums, then m and l
    extern __shared__ float joined[];           // [WV][kOut][64]
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
        for (int s = 0; s < DC * 2; ++s) {
            load8(qp[n], (s / 2) * 64 + g * 16 + (s % 2) * 8, a.d, a.wide, x[s]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = __builtin_fabsf(x[s][i]);
                odd = odd || !(v < __builtin_huge_valf());
                mx = v < __builtin_huge_valf() ? __builtin_fmaxf(mx, v) : mx;
            }
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
    // Pages of the chunk that is loaded next, a chunk ahead of its codes: of the lane's key rows, of its
    // group (looked at when they are used, not waited for where they are read).
    int kpage = -1, vpage = -1;
    auto page_at = [&](int token) { return a.table[int64_t(item) * a.blocks + min(token >> a.block_log, a.blocks - 1)]; };
    auto next_pages = [&](int chunk) {
        kpage = page_at(chunk * kChunk + 16 * (col >> 2));
        vpage = page_at(chunk * kChunk + 16 * g);
    };
    auto at_page = [&](int page) {
        return int64_t(uint32_t(page) < uint32_t(a.pages) ? page : 0) * a.hk + hk;
    };
    auto load_k = [&](int chunk) {
        const int t0 = chunk * kChunk + 16 * (col >> 2);
        const uint8_t *p = a.k + at_page(kpage) * tile + ((t0 & (block - 1)) + (col & 3)) * a.dp;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < DC; ++c) kc[t][c] = *reinterpret_cast<const uintx4 *>(p + 4 * t * a.dp + kch[c]);
    };
    auto load_v = [&](int chunk) {
        const int t0 = chunk * kChunk + 16 * g;
        const int64_t at = at_page(vpage);
        there = uint32_t(vpage) < uint32_t(a.pages) && t0 < rg.kv_len;  // (blocks behind it may never have been written)
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
    if (i < c1) {
        next_pages(rg.chunk(i));
        load_k(rg.chunk(i)), load_v(rg.chunk(i));
        next_pages(rg.chunk(i + WV));
    }
    for (int visit = 0; i < c1;) {
        const int base = rg.chunk(i) * kChunk;
        const float ks_now = ks, vs_now = vs;
        const int ev = there && vs > 0.0f ? __builtin_amdgcn_frexp_expf(vs) : kNoExp;
        int tv = max(ev, __shfl_xor(ev, 16));
        tv = __builtin_amdgcn_readfirstlane(max(tv, __shfl_xor(tv, 32)));
        int tl = tv;
        bool there_now = there, last = true;
        if (a.block_log < 6) {
            // Groups of tokens whose scales of values are far apart are taken in visits of their own to the
            // chunk, as a row may see the small ones alone: next to the largest their probabilities would
            // leave f16.
            tl = ev == kNoExp ? -kNoExp : ev;
            tl = min(tl, __shfl_xor(tl, 16));
            tl = __builtin_amdgcn_readfirstlane(min(tl, __shfl_xor(tl, 32)));
            if (tv > kNoExp && tv - tl > kBelow) {
                there_now = there && g == visit;
                tv = tl = __builtin_amdgcn_readlane(ev, 16 * visit);
                last = visit == 3;
            }
        }
        visit = last ? 0 : visit + 1;
        const int next = last ? i + WV : i;
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
        const bool more = next < c1;
        if (more) {
            if (!last) next_pages(rg.chunk(i));
            load_k(rg.chunk(next));
        }

        // The sums' exponent follows the blocks' scales of values.
        if (tv > ve || (tv > kNoExp && tl < ve - kBelow)) {
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
        const float vrel = there_now && vs_now > 0.0f ? ldexpf(vs_now, kUp - ve) : 0.0f;

        halfx8 p[NQ][PP][2];
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
                const uint32_t bits = there_now ? seen_bits(t0, lo[n], hi[n], a.sinks) : 0u;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[n][t][e] = bits & (1u << (4 * t + e)) ? sc[n][t][e] : kNegInf;
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = __builtin_fmaxf(mx, sc[n][t][e]);
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
            if (__any(mx - m[n] > float(kLazy))) {  // (a sum of both would round past it where scores are large)
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
                    if constexpr (PP == 2) asm("" : "+v"(z));
                    const _Float16 h = static_cast<_Float16>(z);
                    p[n][0][t / 2][(t % 2) * 4 + e] = h;
                    if constexpr (PP == 2) p[n][1][t / 2][(t % 2) * 4 + e] = static_cast<_Float16>(z - float(h));
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
                    if constexpr (PP == 2)
                        o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, p[n][1][s], o[n][t], 0, 0, 0);
                    o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, p[n][0][s], o[n][t], 0, 0, 0);
                }
            }
        }
        if (more) {
            load_v(rg.chunk(next));
            next_pages(rg.chunk(next + WV));
        }
        i = next;
    }

    // The waves' means joined in LDS, each wave then finishing some of them. A sum is divided before its power of two
    // is put back: of values near the end of f32 the mean is finite, the sum is not.
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
        const float by = l[n] == 0.0f ? 0.0f : 1.0f / l[n];
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                joined[(wave * kOut + (n * DT + t) * 4 + e) * 64 + lane] =
                    ldexpf(o[n][t][e] * by, ve == kNoExp ? 0 : ve - kUp);
        joined[(wave * kOut + NQ * DT * 4 + 2 * n) * 64 + lane] = m[n];
        joined[(wave * kOut + NQ * DT * 4 + 2 * n + 1) * 64 + lane] = l[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        float mw[WV], top = kNegInf, sum = 0.0f;
#pragma unroll
        for (int x = 0; x < WV; ++x) {
            mw[x] = joined[(x * kOut + NQ * DT * 4 + 2 * n) * 64 + lane];
            top = __builtin_fmaxf(top, mw[x]);
        }
        const float mu = top == kNegInf ? 0.0f : top;
#pragma unroll
        for (int x = 0; x < WV; ++x) {
            mw[x] = joined[(x * kOut + NQ * DT * 4 + 2 * n + 1) * 64 + lane] * __builtin_amdgcn_exp2f(mw[x] - mu);
            sum += mw[x];
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int x = 0; x < WV; ++x) mw[x] *= inv;  // a wave's share of the row's probabilities
        float *part = a.part ? a.part + ((int64_t(work) * NQ + n) * 16 + col) * (DT * 16 + 2) : nullptr;
        if (part && row_ok[n] && wave == 0 && g == 0) part[DT * 16] = top, part[DT * 16 + 1] = sum;
        T *op = static_cast<T *>(a.out) + row_at[n] * a.ldo + row_ch[n];
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            if (t % WV != wave || t * 16 >= a.d) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float y = 0.0f;
#pragma unroll
                for (int x = 0; x < WV; ++x) y = __builtin_fmaf(joined[(x * kOut + (n * DT + t) * 4 + e) * 64 + lane], mw[x], y);
                const int ch = t * 16 + 4 * g + e;
                if (!row_ok[n]) continue;
                if (part) part[ch] = y;
                else if (ch < a.d) op[ch] = static_cast<T>(y);
            }
        }
    }
}

typedef float floatx16 __attribute__((ext_vector_type(16)));

// The value of lane +- 32.
__device__ __forceinline__ float other_half(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

// LDS of the staged chunks: keys [64][KS * 16] and values [KS * 16 rounded up to 32][64] as f16, rows
// padded by 16 bytes (the rows of a read then lie on distinct banks); NB of each.
template <int KS, int NB>
struct Stage {
    static constexpr int kDT = (KS + 1) / 2;                   // tiles of 32 channels
    static constexpr int kKS = KS * 16 + 8, kVS = kChunk + 8;  // halves of a row
    static constexpr int kK = kChunk * kKS * 2, kV = kDT * 32 * kVS * 2;
    static constexpr int kV0 = NB * kK, kBytes = kV0 + NB * kV;
};

// Orders the MFMAs of a block and the reads from LDS that feed them, N1 reads for P1 MFMAs each and then N2
// for P2: some reads ahead of the first product, then one beside each (the compiler's own order waits for
// every second read).
template <int N1, int P1, int N2 = 0, int P2 = 1>
__device__ __forceinline__ void feed() {
    constexpr int kReads = N1 + N2, kFirst = kReads < kReadsAhead ? kReads : kReadsAhead;
    __builtin_amdgcn_sched_group_barrier(0x100, kFirst, 0);
#pragma unroll
    for (int i = 0; i < N1; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, P1, 0);
        if (i + kFirst < kReads) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
#pragma unroll
    for (int i = N1; i < kReads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, P2, 0);
        if (i + kFirst < kReads) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
}

// Loads that are the same for all lanes, of memory that nothing writes while the kernel runs: through
// the scalar unit.
template <typename X>
__device__ __forceinline__ X scalar_load(const X *p) {
    return *reinterpret_cast<const __attribute__((address_space(4))) X *>(reinterpret_cast<uintptr_t>(p));
}

// Many rows per key head: W waves of 32 rows share chunks of 64 tokens, which are turned into f16
// once, on their way into LDS.
//
// S^T = K . Q^T and O^T = V^T . P^T on 32x32x16 instructions: a lane holds one row's scores (column
// lane % 32), and with LDS row r of a half chunk holding token 16 (r / 4 % 2) + 4 (r / 8) + r % 4 they
// are those of the 16 tokens of its half h = lane / 32: one block, one pair of scales, and the B
// operand of the second product as they stand.
//
// A chunk takes two phases with a barrier behind each: the products (O^T of the chunk before, S^T of
// this one), then the exponentials and the staging of chunks to come. Where W is 8, waves 4 .. 7 are
// a phase behind, so that of the two waves of a SIMD one feeds the matrix unit while the other takes
// the vector unit; keys are then staged two chunks ahead and values one, in three buffers, as the
// waves behind still read one that the others are done with. Else one buffer is enough, and the
// workgroups of a CU drift apart.
//
// Bound: issue, of matrix and vector instructions that take turns (0.61 and 0.58 of a SIMD's cycles at heads of 128,
// LDS 0.28), and the clock, which gives way under them. 4096 rows of a prompt of 16384, 32 heads over 8 of 128, f16:
// 1252 to 1305 us with the card's clock, three products where a plain one has two (up to 1150 TFLOP/s of them);
// probabilities in one part, as on FAST contexts, 965 to 1007 (every wave for itself from memory 2738, shared without
// turns 1115). 4096 x 13312 of 16 heads, not causal: 715 to 727, in one part 545 to 564. f32, queries in two parts too,
// 2 x 4096 x 4096 of 8 heads of 80: 174 to 179, FAST 120.
//
// WIDE: blocks of 64 or 128 tokens, so that a chunk lies in one page and has one scale of keys and one of
// values, read through the scalar unit. Else its four groups of 16 tokens have their own: lane l
// reads the page of group l % 4 and, of keys or (l & 4) of values, its scale.
//
// PARTS: f16 parts of a query, PP: of a probability.
template <typename T, int PARTS, int PP, int KS, int W, bool WIDE>
__global__ __launch_bounds__(64 * W, (W == 4 && KS <= 4 ? 3 : KS <= (PARTS == 2 ? 8 : 10) ? 2 : 1)) void cache8_tiles_kernel(Args a) {
    constexpr bool TURNS = W == 8;
    constexpr int NP = WIDE ? 1 : 4;  // groups of tokens with a page of their own
    constexpr int NB = TURNS ? 3 : 1, AHEAD = TURNS ? 1 : 0;  // keys are staged AHEAD + 1 chunks ahead, values AHEAD
    using L = Stage<KS, NB>;
    constexpr int DT = L::kDT, NT = 64 * W;
    constexpr int kLazy = PP == 2 ? kLazySplit : kLazyHalf, kUp = PP == 2 ? kUpSplit : kUpHalf;
    // Whether scales of values join the exponents: a multiplication less for each probability, at an error of
    // 2^-20 of it, which is nothing beside f16's but more than f32 calls have.
    constexpr bool LOGS = sizeof(T) == 2 || PP == 1;
    constexpr int U = (kChunk * KS + NT - 1) / NT;  // 16-byte runs of codes per thread, of keys and of values
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;

    const int per_xcd = (a.work + 7) / 8;
    int w = int(blockIdx.x % 8) * per_xcd + int(blockIdx.x / 8);
    if (int(blockIdx.x / 8) >= per_xcd || w >= a.work) return;
    const int work = w;
    const int split = w % a.splits;
    w /= a.splits;
    const int r0 = w % a.row_tiles * 32 * W;
    w /= a.row_tiles;
    const int hk = w % a.hk, item = w / a.hk;
    const Range rg = range_of(a, item, r0, 32 * W);
    if (r0 >= rg.rows) return;
    const int share = (rg.chunks + a.splits - 1) / a.splits;
    const int c0 = min(split * share, rg.chunks), n = min(c0 + share, rg.chunks) - c0;

    // Q^T: this lane's row, channels 16 c + 8 h .. + 7 of step c.
    const int wrow = r0 + wave * 32, row = wrow + col;
    const bool row_ok = row < rg.rows;
    const int t = (row_ok ? row : r0) / a.g, qh = hk * a.g + (row_ok ? row : r0) % a.g;
    const int64_t row_at = int64_t(item) * a.q_tokens + t;
    const T *qp = static_cast<const T *>(a.q) + row_at * a.ldq + int64_t(qh) * a.d;
    halfx8 q[PARTS][KS];
    float cq = a.c;
    {
        float x[KS][8];
        float mx = 0.0f;
        bool odd = false;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            load8(qp, s * 16 + h * 8, a.d, a.wide, x[s]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = __builtin_fabsf(x[s][i]);
                odd = odd || !(v < __builtin_huge_valf());
                mx = v < __builtin_huge_valf() ? __builtin_fmaxf(mx, v) : mx;
            }
        }
        int e = 0;
        if constexpr (sizeof(T) == 4) {  // scaled by a power of two per row, so that no value leaves f16
            mx = __builtin_fmaxf(mx, other_half(mx));
            e = mx == 0.0f ? 0 : __builtin_amdgcn_frexp_expf(mx) - 1 - kSplitQ;
            cq = ldexpf(a.c, e);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = sizeof(T) == 4 ? ldexpf(x[s][i], -e) : x[s][i];
                q[0][s][i] = static_cast<_Float16>(y);
                if constexpr (PARTS == 2) q[1][s][i] = static_cast<_Float16>(odd ? 0.0f : y - float(q[0][s][i]));
            }
    }
    // The row sees tokens lo .. hi - 1 and those below min(hi, sinks), all rows of the wave those of
    // lo_all .. hi_all - 1 and below min(hi_all, sinks).
    const int at = t + rg.off, hi = a.causal ? min(rg.kv_len, at + 1) : rg.kv_len;
    const int lo = a.window ? max(at - a.window + 1, 0) : 0;
    const int t_first = wrow / a.g, t_last = max(min(rg.rows, wrow + 32) - 1, 0) / a.g;
    const int hi_all = a.causal ? min(rg.kv_len, t_first + rg.off + 1) : rg.kv_len;
    const int lo_all = a.window ? max(t_last + rg.off - a.window + 1, 0) : 0;

    // Channels behind dp of the staged keys: zeros, which the chunks never overwrite.
    if (a.dp < KS * 16)
        for (int i = tid; i < NB * kChunk * 2; i += NT)
            for (int ch = a.dp; ch < KS * 16; ch += 16)
                *reinterpret_cast<uintx4 *>(smem + ((i / 2) * L::kKS + ch + i % 2 * 8) * 2) = uintx4{0, 0, 0, 0};

    const int runs = a.dp / 16;  // 16-byte runs of a token's keys
    const uint32_t tile = uint32_t(a.dp) << a.block_log;
    const int block = 1 << a.block_log;
    // This thread's runs: token and channel of keys, channel and group of values, and their places in LDS
    // (threads behind the last run repeat it).
    int ktk[U], koff[U], kput[U], voff[U], vgrp[U], vput[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = min(tid + u * NT, kChunk * runs - 1);
        const int tk = i / runs, run = i - tk * runs, j = tk & 31;
        ktk[u] = tk, koff[u] = WIDE ? tk * a.dp + run * 16 : run * 16;
        kput[u] = (((tk & 32) + 4 * (j >> 4) + 8 * ((j & 15) >> 2) + (j & 3)) * L::kKS + run * 16) * 2;
        vgrp[u] = i & 3, voff[u] = ((i >> 2) << a.block_log) + (WIDE ? (i & 3) * 16 : 0);
        vput[u] = ((i >> 2) * L::kVS + (i & 3) * 16) * 2;
    }
    // Pages of the chunks i + 1 .. i + AHEAD + 2 behind chunk i: read a chunk or more ahead of the codes,
    // and looked at when they are used, so that nothing waits for them.
    int page[AHEAD + 2];
    auto read_page = [&](int i) {
        const int base = rg.chunk(c0 + i) * kChunk + (WIDE ? 0 : (lane & 3) * 16);
        const int32_t *p = a.table + int64_t(item) * a.blocks + min(base >> a.block_log, a.blocks - 1);
        if constexpr (WIDE) return scalar_load(p);
        else return *p;
    };
    auto there = [&](int pg) { return uint32_t(pg) < uint32_t(a.pages); };
    auto at_page = [&](int pg) { return (there(pg) ? uint32_t(pg) : 0u) * uint32_t(a.hk) + uint32_t(hk); };
    // at_page of a thread's group
    auto at_group = [&](int pg, int group) {
        const uint32_t own = at_page(pg);
        if constexpr (WIDE) return own;
        uint32_t at = __builtin_amdgcn_readlane(own, 0);
#pragma unroll
        for (int x = 1; x < 4; ++x) at = group == x ? uint32_t(__builtin_amdgcn_readlane(own, x)) : at;
        return at;
    };
    uintx4 kr[U], vr[U];
    auto fetch_k = [&](int i, int pg) {
        const int base = rg.chunk(c0 + i) * kChunk;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int off = WIDE ? (base & (block - 1)) * a.dp + koff[u] : ((base + ktk[u]) & (block - 1)) * a.dp + koff[u];
            kr[u] = *reinterpret_cast<const uintx4 *>(a.k + uint64_t(at_group(pg, ktk[u] >> 4)) * tile + uint32_t(off));
        }
    };
    auto fetch_v = [&](int i, int pg) {
        const int base = rg.chunk(c0 + i) * kChunk;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int off = WIDE ? (base & (block - 1)) + voff[u] : ((base + vgrp[u] * 16) & (block - 1)) + voff[u];
            vr[u] = *reinterpret_cast<const uintx4 *>(a.v + uint64_t(at_group(pg, vgrp[u])) * tile + uint32_t(off));
        }
    };
    auto stage_k = [&](int i) {
        char *const buf = smem + i % NB * L::kK;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            halfx8 *p = reinterpret_cast<halfx8 *>(buf + kput[u]);
            p[0] = halves(kr[u][0], kr[u][1]), p[1] = halves(kr[u][2], kr[u][3]);
        }
    };
    auto stage_v = [&](int i) {
        char *const buf = smem + L::kV0 + i % NB * L::kV;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            halfx8 *p = reinterpret_cast<halfx8 *>(buf + vput[u]);
            p[0] = halves(vr[u][0], vr[u][1]), p[1] = halves(vr[u][2], vr[u][3]);
        }
    };

    floatx16 o[DT], sc[2];
    halfx8 p[PP][4];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = kNegInf, l = 0.0f;
    int ve = kNoExp, ve_max = kNoExp;

    auto scores = [&](int i) {
        const char *const kp = smem + i % NB * L::kK + (col * L::kKS + h * 8) * 2;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[b][e] = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const halfx8 k = *reinterpret_cast<const halfx8 *>(kp + b * 32 * L::kKS * 2 + s * 32);
                if constexpr (PARTS == 2) sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[1][s], sc[b], 0, 0, 0);
                sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[0][s], sc[b], 0, 0, 0);
            }
    };
    auto values = [&](int i) {
        const char *const vp = smem + L::kV0 + i % NB * L::kV + (col * L::kVS + h * 16) * 2;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const halfx8 v = *reinterpret_cast<const halfx8 *>(vp + ((s / 2) * 32 + (s % 2) * 8 + d * 32 * L::kVS) * 2);
                if constexpr (PP == 2) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[1][s], o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[0][s], o[d], 0, 0, 0);
            }
    };
    // What the chunk's scales make of its scores and probabilities, formed beside the products: the
    // factor of the scores, the scales of values against the power of two of the sums (LOGS: the
    // logarithm, and the inverse, which takes it out of the sum).
    float ks[2], vrel[2], inv[2];
    int shift = 0;       // how far that power of two moves
    bool whole = false;  // every row of the wave sees all of the chunk
    // The scales of chunk i + 1, and which of its groups have a page; then those of the chunk at hand.
    float ks_next = 0.0f, vs_next = 0.0f;  // (WIDE alone)
    float scale_next = 0.0f;               // (else: the lane's)
    bool ok_next = false, ok[NP];
    // Groups whose scales of values are far apart are taken in visits of their own to the chunk, as a row
    // may see the small ones alone: next to the largest their probabilities would leave f16.
    float k_here[NP], v_here[NP];
    int visit = 0, visits = 1;
    auto follow = [&](int tv, int tl) {  // largest and smallest exponent of the chunk's values
        const bool go = tv > ve || (tv > kNoExp && tl < ve - kBelow);
        ve_max = go ? max(ve_max, tv) : ve_max;
        const int to = go ? max(tv, ve_max - kDeepest) : ve;
        shift = ve - to;
        ve = to;
    };
    auto factors = [&](int b, float k, float v) {
        // (codes at a scale of 0 are 0: any factor will do)
        const float x = v > 0.0f ? ldexpf(v, kUp - ve) : 1.0f;
        if constexpr (!LOGS) {
            vrel[b] = x;
        } else {
            const float y = __builtin_fmaxf(x, 0x1p-90f);  // (values far below the largest count as nothing)
            vrel[b] = __builtin_amdgcn_logf(y), inv[b] = __builtin_amdgcn_rcpf(y);
        }
        // (0 times the smallest is 0, and a masked score stays -inf)
        ks[b] = __builtin_fminf(__builtin_fmaxf(k * cq, 0x1p-126f), 0x1.fffffep127f);
    };
    auto prepare = [&](int i) {
        const int base = rg.chunk(c0 + i) * kChunk;
        whole = base + kChunk <= hi_all && (base >= lo_all || base + kChunk <= a.sinks);
        int ev[NP];
        if constexpr (WIDE) {
            ok[0] = ok_next;
            k_here[0] = ok[0] ? ks_next : 0.0f, v_here[0] = ok[0] ? vs_next : 0.0f;
        } else if (visit == 0) {
            // (blocks behind the last token may never have been written)
            const float x = ok_next && base + 16 * (lane & 3) < rg.kv_len ? scale_next : -1.0f;
#pragma unroll
            for (int g = 0; g < NP; ++g) {
                k_here[g] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), g));
                v_here[g] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 4 + g));
            }
        }
        int tv = kNoExp, tl = -kNoExp;
        float k[NP], v[NP];
#pragma unroll
        for (int x = 0; x < NP; ++x) {
            k[x] = k_here[x], v[x] = v_here[x];
            // the exponent as frexp gives it; below the normal range as at its end
            const int bits = __builtin_bit_cast(int, v[x]);
            ev[x] = bits > 0 ? max(bits >> 23, 1) - 126 : kNoExp;
            tv = max(tv, ev[x]);
            tl = bits > 0 ? min(tl, ev[x]) : tl;
            if (!WIDE) ok[x] = bits >= 0;
        }
        if constexpr (!WIDE) {
            visits = tv > kNoExp && tv - tl > kBelow ? NP : 1;
            if (visits > 1) {
                tv = kNoExp;
#pragma unroll
                for (int x = 0; x < NP; ++x) {
                    ok[x] = ok[x] && x == visit;
                    v[x] = x == visit ? v[x] : 0.0f;
                    tv = x == visit ? ev[x] : tv;
                }
                tl = tv;
            }
        }
#pragma unroll
        for (int x = 0; x < NP; ++x) whole = whole && ok[x];
        follow(tv, tl);
        factors(0, h ? k[1 % NP] : k[0], h ? v[1 % NP] : v[0]);
        if constexpr (WIDE) ks[1] = ks[0], vrel[1] = vrel[0], inv[1] = inv[0];
        else factors(1, h ? k[3 % NP] : k[2 % NP], h ? v[3 % NP] : v[2 % NP]);
    };
    bool far = false;
    auto softmax = [&](int i) {
        if (shift) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] = ldexpf(o[d][e], shift);
        }
        if (!whole) {
            const int base = rg.chunk(c0 + i) * kChunk;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const bool page = h ? ok[(2 * b + 1) % NP] : ok[2 * b % NP];
                const uint32_t bits = page ? seen_bits(base + b * 32 + h * 16, lo, hi, a.sinks) : 0u;
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[b][e] = bits & (1u << e) ? sc[b][e] : kNegInf;
            }
        }
        float mx[4];  // (several chains: a dependent instruction waits for twice its issue)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            mx[x] = sc[x / 2][x % 2 * 8];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx[x] = __builtin_fmaxf(mx[x], sc[x / 2][x % 2 * 8 + e]);
        }
        float top = __builtin_fmaxf(__builtin_fmaxf(mx[0], mx[1]) * ks[0], __builtin_fmaxf(mx[2], mx[3]) * ks[1]);
        top = __builtin_fmaxf(top, other_half(top));
        if (__any(top - m > float(kLazy))) {  // (as above)
            const float mn = __builtin_fmaxf(m, top);
            const float f = __builtin_amdgcn_exp2f(m - (mn == kNegInf ? 0.0f : mn));
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= f;
            m = mn;
            far = __any(__builtin_fabsf(m) > 1048576.0f && m != kNegInf);
        }
        const float mu = m == kNegInf ? 0.0f : m;
        // The fused exponent is off by half a step of m, which is nothing until scores are so large
        // that the largest key's power would leave the range: their products are rounded first.
        if (far) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[b][e] = sc[b][e] * ks[b] - mu + (LOGS ? vrel[b] : 0.0f);
        } else {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float off = LOGS ? vrel[b] - mu : -mu;
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[b][e] = __builtin_fmaf(sc[b][e], ks[b], off);
            }
        }
        float sum[4] = {};
        float minus = -1.0f;  // (not known to the compiler, which would make a conversion and a subtraction of the fused form)
        asm("" : "+s"(minus));
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                // Two at once: the conversion of a pair, and second parts fused with taking the first ones back,
                // half of the instructions of one after another: windows over heads of 64 80 -> 73 us, prompts of 128
                // 1328 -> 1300, f32 images 186 -> 178.
                floatx2 z;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float y = __builtin_amdgcn_exp2f(sc[b][e + x]);
                    sum[2 * b + x] += y;
                    float w = LOGS ? y : y * vrel[b];
                    // (both parts are of a value rounded to f32; a product fused with its conversion is not)
                    if constexpr (!LOGS) asm("" : "+v"(w));
                    z[x] = w;
                }
                const halfx2 first = __builtin_convertvector(z, halfx2);
#pragma unroll
                for (int x = 0; x < 2; ++x) p[0][2 * b + e / 8][e % 8 + x] = first[x];
                if constexpr (PP == 2) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) z[x] = __builtin_fmaf(float(first[x]), minus, z[x]);
                    const halfx2 second = __builtin_convertvector(z, halfx2);
#pragma unroll
                    for (int x = 0; x < 2; ++x) p[1][2 * b + e / 8][e % 8 + x] = second[x];
                }
            }
        if constexpr (!LOGS) l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        else l = __builtin_fmaf(sum[0] + sum[1], inv[0], __builtin_fmaf(sum[2] + sum[3], inv[1], l));
    };

    auto scales = [&]() {  // of the chunk whose page is the first in line
        const uint32_t at = at_page(page[0]);
        if constexpr (WIDE) ks_next = scalar_load(a.ks + at), vs_next = scalar_load(a.vs + at);
        else scale_next = (lane & 4 ? a.vs : a.ks)[at];
        ok_next = there(page[0]);
    };
    auto move_up = [&](int pg) {
#pragma unroll
        for (int j = 0; j < AHEAD + 1; ++j) page[j] = page[j + 1];
        page[AHEAD + 1] = pg;
    };
    if (a.blocks > 0) {  // (without blocks there is no table either)
#pragma unroll
        for (int x = 0; x < AHEAD + 2; ++x) page[x] = read_page(x);  // (chunks 0 ..)
        scales();
        fetch_k(0, page[0]);
        fetch_v(0, page[0]);
        stage_k(0);
        fetch_k(1, page[1]);
        if constexpr (TURNS) {
            stage_v(0);
            fetch_v(1, page[1]);
            stage_k(1);
            fetch_k(2, page[AHEAD + 1]);
        }
        move_up(read_page(AHEAD + 2));
        __syncthreads();
        if (TURNS && wave >= 4) __syncthreads();
        if (n > 0) {
            scores(0);
            feed<2 * KS, PARTS>();
            prepare(0);
        }
        __syncthreads();
        for (int i = 0; i < n;) {
            const bool first = WIDE || visit == 0, last = WIDE || visit + 1 == visits;
            scales();
            const int page_new = read_page(i + AHEAD + 3);
            softmax(i);
            if (last && i + AHEAD + 1 < n) stage_k(i + AHEAD + 1);
            if (first && i + AHEAD < n) stage_v(i + AHEAD);
            fetch_v(i + AHEAD + 1, page[AHEAD]);
            if (last) {
                fetch_k(i + AHEAD + 2, page[AHEAD + 1]);
                move_up(page_new);
            }
            __syncthreads();
            __builtin_amdgcn_s_setprio(1);
            const int next = last ? i + 1 : i;
            values(i);
            scores(next);  // (behind the last chunk: of what the buffer holds, and not used)
            feed<4 * DT, PP, 2 * KS, PARTS>();
            __builtin_amdgcn_s_setprio(0);
            visit = last ? 0 : visit + 1;
            i = next;
            if (i < n) prepare(i);
            __syncthreads();
        }
        if (TURNS && wave < 4) __syncthreads();
    }
    if (!row_ok) return;
    l += other_half(l);
    const int back = ve == kNoExp ? 0 : ve - kUp;
    const float by = l == 0.0f ? 0.0f : 1.0f / l;  // (before the power of two is put back, as above)
    if (a.part) {
        float *part = a.part + (int64_t(work) * 32 * W + wave * 32 + col) * (DT * 32 + 2);
        if (h == 0) part[DT * 32] = m, part[DT * 32 + 1] = l;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) part[d * 32 + 8 * (e / 4) + 4 * h + e % 4] = ldexpf(o[d][e] * by, back);
        return;
    }
    T *op = static_cast<T *>(a.out) + row_at * a.ldo + int64_t(qh) * a.d;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int ch = d * 32 + 8 * f + 4 * h;
            typedef T V4 __attribute__((ext_vector_type(4)));
            V4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(ldexpf(o[d][4 * f + e] * by, back));
            if (a.wide) {
                if (ch < a.d) *reinterpret_cast<V4 *>(op + ch) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (ch + e < a.d) op[ch + e] = v[e];
            }
        }
}

// Joins the splits of a row, TILE rows per workgroup of the split, PF floats of means each (then the
// maximum and the sum of the probabilities): a workgroup per row, every fourth split to a wave.
template <typename T, int TILE, int PF>
__global__ __launch_bounds__(256) void cache8_join_kernel(Args a) {
    constexpr int C = (PF + 63) / 64;
    __shared__ float joined[3][C][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = blockIdx.x % TILE, base = blockIdx.x / TILE;
    int w = base;
    const int r0 = w % a.row_tiles * TILE;
    w /= a.row_tiles;
    const int hk = w % a.hk, item = w / a.hk;
    const int q_len = a.q_len ? min(max(a.q_len[item], 0), a.q_tokens) : a.q_tokens;
    const int row = r0 + col;
    if (row >= q_len * a.g) return;
    const float *p = a.part + (int64_t(base) * a.splits * TILE + col) * (PF + 2);
    const int64_t step = int64_t(TILE) * (PF + 2);
    float m = kNegInf;
    for (int s = lane; s < a.splits; s += 64) m = __builtin_fmaxf(m, p[s * step + PF]);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) m = __builtin_fmaxf(m, __shfl_xor(m, x));
    const float mu = m == kNegInf ? 0.0f : m;
    float l = 0.0f, o[C] = {};
    for (int s = lane; s < a.splits; s += 64)
        l = __builtin_fmaf(p[s * step + PF + 1], __builtin_amdgcn_exp2f(p[s * step + PF] - mu), l);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 4
    for (int s = wave; s < a.splits; s += 4) {
        const float f = p[s * step + PF + 1] * __builtin_amdgcn_exp2f(p[s * step + PF] - mu) * inv;
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (i * 64 + lane < a.d) o[i] = __builtin_fmaf(p[s * step + i * 64 + lane], f, o[i]);
    }
#pragma unroll
    for (int i = 0; i < C; ++i)
        if (wave) joined[wave - 1][i][lane] = o[i];
    __syncthreads();
    if (wave) return;
    T *op = static_cast<T *>(a.out) + (int64_t(item) * a.q_tokens + row / a.g) * a.ldo + int64_t(hk * a.g + row % a.g) * a.d;
#pragma unroll
    for (int i = 0; i < C; ++i)
        if (i * 64 + lane < a.d)
            op[i * 64 + lane] = static_cast<T>(o[i] + joined[0][i][lane] + joined[1][i][lane] + joined[2][i][lane]);
}

template <typename T, int TILE, int PF>
void launch_join(Context &ctx, const Args &a) {
    if (!a.part) return;
    cache8_join_kernel<T, TILE, PF><<<dim3{uint32_t(a.work / a.splits * TILE)}, dim3{256}, 0, ctx.stream>>>(a);
    MH_LAUNCH_CHECK();
}

template <typename T, int PARTS, int DT, int NQ>
void launch_rows(Context &ctx, const Args &a) {
    // Two waves per SIMD where 256 registers hold one. Single tokens, 8 items of 16384 tokens, 32 heads over 8 of 128, us
    // with eight and with four: f16 49, 57, f32 49, 57; of 256: 185, 107 and 242, 106; five f32 queries of 128: 140, 76.
    constexpr int WV = DT == 16 || (PARTS == 2 && NQ == 2 && DT == 8) ? 4 : 8;
    const size_t lds = size_t(WV) * (NQ * DT * 4 + NQ * 2) * 64 * 4;
    const void *fn = reinterpret_cast<const void *>(&cache8_rows_kernel<T, PARTS, DT, NQ, WV>);
    if (lds > 48 * 1024) HIP_CHECK(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
    cache8_rows_kernel<T, PARTS, DT, NQ, WV><<<dim3{uint32_t((a.work + 7) / 8 * 8)}, dim3{64 * WV}, lds, ctx.stream>>>(a);
    MH_LAUNCH_CHECK();
    launch_join<T, 16 * NQ, DT * 16>(ctx, a);
}

template <typename T, int PARTS, int PP, int KS, int W, bool WIDE>
void launch_tiles(Context &ctx, const Args &a) {
    using L = Stage<KS, W == 8 ? 3 : 1>;
    const size_t lds = L::kBytes;
    static_assert(lds <= 160 * 1024, "chunks exceed the LDS");
    const void *fn = reinterpret_cast<const void *>(&cache8_tiles_kernel<T, PARTS, PP, KS, W, WIDE>);
    HIP_CHECK(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
    cache8_tiles_kernel<T, PARTS, PP, KS, W, WIDE><<<dim3{uint32_t((a.work + 7) / 8 * 8)}, dim3{64 * W}, lds, ctx.stream>>>(a);
    MH_LAUNCH_CHECK();
    launch_join<T, 32 * W, L::kDT * 32>(ctx, a);
}

// by(the constant dt), tiles of 16 channels as chosen by head_tiles.
template <typename F>
void by_tiles(int dt, F &&by) {
    if (dt == 4) by(std::integral_constant<int, 4>{});
    else if (dt == 5) by(std::integral_constant<int, 5>{});
    else if (dt == 6) by(std::integral_constant<int, 6>{});
    else if (dt == 8) by(std::integral_constant<int, 8>{});
    else if (dt == 10) by(std::integral_constant<int, 10>{});
    else by(std::integral_constant<int, 16>{});
}

// nq tiles of 16 rows for each workgroup.
template <typename T, int PARTS>
void rows_alone(Context &ctx, const Args &a, int nq, int dt) {
    by_tiles(dt, [&](auto n) {
        constexpr int DT = decltype(n)::value;
        if (nq == 1) launch_rows<T, PARTS, DT, 1>(ctx, a);
        else if constexpr (DT <= 8) launch_rows<T, PARTS, DT, 2>(ctx, a);
    });
}

// Waves of 32 rows that share a chunk, four or eight.
template <typename T, int PARTS, int PP>
void rows_shared(Context &ctx, const Args &a, int waves, int dt) {
    const bool wide = a.block_log >= 6;
    by_tiles(dt, [&](auto n) {
        constexpr int DT = decltype(n)::value;
        if constexpr (DT <= 8)
            if (waves == 8) return wide ? launch_tiles<T, PARTS, PP, DT, 8, true>(ctx, a) : launch_tiles<T, PARTS, PP, DT, 8, false>(ctx, a);
        wide ? launch_tiles<T, PARTS, PP, DT, 4, true>(ctx, a) : launch_tiles<T, PARTS, PP, DT, 4, false>(ctx, a);
    });
}

// Rows alone where waves is 0. Halves: probabilities (and f32 queries) rounded to f16 once, as FAST contexts ask for;
// f16 rows alone have no such form, as theirs costs nothing.
void launch_f16(Context &ctx, const Args &a, int nq, int waves, int dt);
void launch_f16_half(Context &ctx, const Args &a, int waves, int dt);
void launch_f32(Context &ctx, const Args &a, int nq, int waves, int dt);
void launch_f32_half(Context &ctx, const Args &a, int nq, int waves, int dt);

}  // namespace c8a
}  // namespace mh
