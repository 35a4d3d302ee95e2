// Keys and values quantised to 8 bits as they are written into the pages of a cache, and
// read back.
//
// A block of tokens and a head of it share a scale: with a = max |x| over the block's finite
// values, s = a (1 / 127) in f32 and the code is x / s rounded to the nearest integer (ties to
// even), so a value is off by at most s / 2. Where a block holds tokens already, s is the
// larger of its scale and the new tokens', and the codes it holds are rounded to the new one.
// The quotient is rounded as if exact: c = rint(x * (1 / s)) is the nearest integer or one
// beside it, x - c s is exact in f32 (fused; within s of zero, and a multiple of the smaller of
// both operands' last places), and its distance to s / 2 decides.
//
// Bound: memory, 1 byte written for the 2 or 4 read. A workgroup takes a block of one head,
// keys or values, in patches of 4 tokens x 8 channels that stay in registers between the
// maximum and the codes, so that x is read once. Values are turned through LDS.
#include <algorithm>
#include <type_traits>

#include "cache8.hpp"

namespace mh {
namespace {

typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

struct RowArgs {
    const void *in[2];   // write: k, v
    void *out[2];        // read: k, v
    int64_t ld[2];
    uint8_t *code[2];
    float *scale[2];
    const int32_t *table, *first, *len;
    int tokens, blocks, pages, heads, d, dp, runs, block_log, touched;  // runs of 8 channels: 8 runs <= dp
    uint32_t by_runs;  // 2^16 / runs rounded up: p / runs = p by_runs >> 16 for p < 1024 and runs of at most 32
};

// What a workgroup works on: tokens lo .. hi - 1 of one page and head.
struct Spot {
    int item, head, which, base, first, lo, hi;
    int page;
    __device__ __forceinline__ bool there(const RowArgs &a) const { return page >= 0 && page < a.pages; }
    __device__ __forceinline__ int64_t at(const RowArgs &a) const { return int64_t(page) * a.heads + head; }
};

// Whether there are such tokens; the page is read but not waited for.
__device__ __forceinline__ bool find(const RowArgs &a, Spot &s) {
    // Heads first: the workgroups that run together then cover whole rows of tokens. 16384 tokens of 16
    // heads of 128: written in 47.5 us, 55.6 with the blocks first; read back in 35.7 and 34.4.
    int w = blockIdx.x;
    s.head = w % a.heads;
    w /= a.heads;
    const int b = w % a.touched;
    w /= a.touched;
    s.which = w % 2;
    s.item = w / 2;
    const int block = 1 << a.block_log, cap = a.blocks << a.block_log;
    s.first = a.first ? min(max(a.first[s.item], 0), cap) : 0;
    const int len = min(a.len ? min(max(a.len[s.item], 0), a.tokens) : a.tokens, cap - s.first);
    const int blk = (s.first >> a.block_log) + b;
    s.base = blk << a.block_log;
    s.lo = max(s.first - s.base, 0);
    s.hi = min(s.first + len - s.base, block);
    if (s.lo >= s.hi) return false;
    s.page = a.table[int64_t(s.item) * a.blocks + blk];
    return true;
}

// Eight values of a row, `valid` of them there.
template <typename T, bool VEC>
struct Eight {
    typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
    static constexpr int kN = int(sizeof(T)) / 2, kE = 16 / int(sizeof(T));
    V v[kN];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = V(T(0));
    }
    __device__ __forceinline__ void load(const T *p, int valid) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < kN; ++i) v[i] = reinterpret_cast<const V *>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i / kE][i % kE] = i < valid ? p[i] : T(0);
        }
    }
    __device__ __forceinline__ void store(T *p, int valid) const {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < kN; ++i) reinterpret_cast<V *>(p)[i] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < valid) p[i] = v[i / kE][i % kE];
        }
    }
    // The largest magnitude, as the bits of its f32.
    __device__ __forceinline__ uint32_t largest() const {
        if constexpr (sizeof(T) == 2) {
            typedef uint16_t U2 __attribute__((ext_vector_type(2)));
            typedef uint32_t U4 __attribute__((ext_vector_type(4)));
            const U4 b = __builtin_bit_cast(U4, v[0]);
            U2 m{0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(U2, uint32_t(b[i] & 0x7FFF7FFFu)));
            const uint16_t x = m[0] > m[1] ? m[0] : m[1];
            return __builtin_bit_cast(uint32_t, float(__builtin_bit_cast(_Float16, x))) & 0x7FFFFFFFu;
        } else {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = v[i / kE][i % kE];
                m = max(m, __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu);
            }
            return m;
        }
    }
    __device__ __forceinline__ float at(int i) const { return float(v[i / kE][i % kE]); }
    __device__ __forceinline__ void set(int i, float x) { v[i / kE][i % kE] = static_cast<T>(x); }
};

// The scale s and what dividing by it takes; scales near the end of the range are lifted so
// that their quotients keep their bits.
struct Divider {
    float s, inv, half, up;
    __device__ __forceinline__ explicit Divider(float scale) {
        up = scale < 0x1p-64f ? 0x1p64f : 1.0f;
        s = scale * up;
        inv = s > 0.0f ? 1.0f / s : 0.0f;
        half = 0.5f * s;
    }
    // x / s rounded to the nearest integer within +-127, plus 128; NaN is zero.
    __device__ __forceinline__ uint32_t code(float x) const {
        x *= up;
        float c = __builtin_rintf(x * inv);
        const float e = __builtin_fmaf(-c, s, x), far = __builtin_fabsf(e);
        const bool odd = (int(c) & 1) != 0;
        if (far > half || (far == half && odd)) c += __builtin_copysignf(1.0f, e);
        c = __builtin_fminf(__builtin_fmaxf(c, -127.0f), 127.0f);
        return c == c && s > 0.0f && x == x ? uint32_t(int(c) + 128) : 128u;
    }
};

// The last bytes of four words, the first lowest.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
}

// Four codes rounded from scale s0 to s: their product and its quotient decide exactly in f64.
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float s0, float s) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = int((w >> (8 * i)) & 255) - 128;
        const double q = __builtin_rint(double(c) * double(s0) / double(s));
        r |= uint32_t(int(__builtin_fmin(__builtin_fmax(q, -127.0), 127.0)) + 128) << (8 * i);
    }
    return r;
}

template <typename T, int PU, bool VEC>
__global__ __launch_bounds__(256) void cache8_write_kernel(RowArgs a) {
    extern __shared__ uint32_t turned[];  // values: [dp][block / 4 + 1]
    __shared__ float wave_max[4];
    Spot s;
    if (!find(a, s)) return;
    const int tid = threadIdx.x, nt = blockDim.x;
    const int block = 1 << a.block_log, held = s.lo;
    const int q0 = s.lo / 4, q1 = (s.hi + 3) / 4, patches = (q1 - q0) * a.runs;
    const bool values = s.which == 1;
    const int64_t ld = a.ld[s.which];
    const T *x = static_cast<const T *>(a.in[s.which]) + (int64_t(s.item) * a.tokens + (s.base - s.first)) * ld +
                 int64_t(s.head) * a.d;
    Eight<T, VEC> r[PU][4];
    const bool full = s.lo == 0 && s.hi == block;
#pragma unroll
    for (int u = 0; u < PU; ++u) {
        const int p = tid + u * nt, row = int(uint32_t(p) * a.by_runs >> 16), run = p - row * a.runs, t = (q0 + row) * 4;
        const T *const at = x + int64_t(t) * ld + run * 8;
        if (full && p < patches) {
#pragma unroll
            for (int e = 0; e < 4; ++e) r[u][e].load(at + e * ld, a.d - run * 8);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                r[u][e].zero();
                if (p < patches && t + e >= s.lo && t + e < s.hi) r[u][e].load(at + e * ld, a.d - run * 8);
            }
        }
    }
    if (!s.there(a)) return;
    float *const scale = a.scale[s.which] + s.at(a);
    const float s0 = held ? *scale : 0.0f;
    // The largest magnitude by its bits, in which infinities and NaN are above all others.
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < PU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, r[u][e].largest());
    float mx = __builtin_bit_cast(float, top);
    if (__any(!(mx < __builtin_huge_valf()))) {
        mx = 0.0f;
#pragma unroll
        for (int u = 0; u < PU; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = __builtin_fabsf(r[u][e].at(i));
                    mx = v < __builtin_huge_valf() ? __builtin_fmaxf(mx, v) : mx;
                }
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) mx = __builtin_fmaxf(mx, __shfl_xor(mx, o));
    if (nt > 64) {
        if ((tid & 63) == 0) wave_max[tid >> 6] = mx;
        __syncthreads();
        for (int w = 0; w < nt / 64; ++w) mx = __builtin_fmaxf(mx, wave_max[w]);
    }
    const float sc = __builtin_fmaxf(s0, mx * (1.0f / 127.0f));
    const bool grown = held && sc > s0;
    // (the barrier above, or the wave's own order, lies between the reads of s0 and this store)
    if (tid == 0) *scale = sc;
    const Divider by(sc);

    // The codes of every patch: of keys by channel (word 2 e + i / 4 of channels i of token e), of values
    // by token (word i of channel i).
    uint32_t w[PU][8];
    auto quantise = [&](auto by_token, auto by_value) {
#pragma unroll
        for (int u = 0; u < PU; ++u) {
            uint32_t c[4][8];
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 8; ++i) c[e][i] = by_value(r[u][e].at(i));
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const int e = x / 2, i = x % 2 * 4;
                if (decltype(by_token)::value) w[u][x] = low_bytes(c[0][x], c[1][x], c[2][x], c[3][x]);
                else w[u][x] = low_bytes(c[e][i], c[e][i + 1], c[e][i + 2], c[e][i + 3]);
            }
        }
    };
    // 1.5 2^23 + 128 more, a quotient rounds to an integer as f32 adds, and its last byte is the code. It
    // is the right one where x (1 / s), which is off by at most 2^-17, is not that near to a tie.
    float tie = 0.0f;
    auto codes = [&](auto by_token) {
        if (sc >= 0x1p-64f)
            quantise(by_token, [&](float x) {
                constexpr float kUp = 12582912.0f + 128.0f;
                const float t = __builtin_fmaf(x, by.inv, kUp);
                tie = __builtin_fmaxf(tie, __builtin_fabsf(__builtin_fmaf(x, by.inv, kUp - t)));
                return __builtin_bit_cast(uint32_t, t);
            });
        if (__any(!(sc >= 0x1p-64f && tie < 0.5f - 0x1p-16f && top < 0x7F800000u)))
            quantise(by_token, [&](float x) { return by.code(x); });
    };
    if (values) codes(std::true_type{});
    else codes(std::false_type{});

    if (!values) {
        uint8_t *const k = a.code[0] + s.at(a) * block * a.dp;
#pragma unroll
        for (int u = 0; u < PU; ++u) {
            const int p = tid + u * nt, row = int(uint32_t(p) * a.by_runs >> 16), run = p - row * a.runs, q = q0 + row;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = q * 4 + e;
                if (p >= patches || t < s.lo || t >= s.hi) continue;
                *reinterpret_cast<uintx2 *>(k + t * a.dp + run * 8) = uintx2{w[u][2 * e], w[u][2 * e + 1]};
            }
        }
        if (grown)
            for (int i = tid; i < held * a.dp / 4; i += nt) {
                uint32_t *p = reinterpret_cast<uint32_t *>(k) + i;
                *p = rescaled(*p, s0, sc);
            }
        return;
    }
    const int ldt = block / 4 + 1;
#pragma unroll
    for (int u = 0; u < PU; ++u) {
        const int p = tid + u * nt, row = int(uint32_t(p) * a.by_runs >> 16), run = p - row * a.runs, q = q0 + row;
        if (p >= patches) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) turned[(run * 8 + i) * ldt + q] = w[u][i];
    }
    __syncthreads();
    uint32_t *const v = reinterpret_cast<uint32_t *>(a.code[1] + s.at(a) * block * a.dp);
    if (s.lo == 0 && s.hi == block) {  // all of the block: 16 tokens of a channel at once
        const int log = a.block_log - 4;
        for (int i = tid; i < a.runs * 8 << log; i += nt) {
            const int ch = i >> log, at = (i & ((1 << log) - 1)) * 4;
            const uint32_t *const t = turned + ch * ldt + at;
            typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<uintx4 *>(v + ch * (block / 4) + at) = uintx4{t[0], t[1], t[2], t[3]};
        }
        return;
    }
    const int c0 = grown ? 0 : q0, nq = q1 - c0;
    for (int i = tid; i < a.runs * 8 * nq; i += nt) {
        const int ch = i / nq, q = c0 + i % nq;
        uint32_t *const p = v + ch * (block / 4) + q;
        const int lo = max(s.lo - 4 * q, 0), hi = min(s.hi - 4 * q, 4);  // the new tokens of these four
        const uint32_t word = lo < hi ? turned[ch * ldt + q] : 0u;
        if (!grown && hi - lo < 4) {  // the tokens beside the new ones stay as they are
            for (int e = lo; e < hi; ++e) reinterpret_cast<uint8_t *>(p)[e] = uint8_t(word >> (8 * e));
            continue;
        }
        uint32_t mask = 0xFFFFFFFFu, kept = 0;
        if (hi - lo < 4) {  // tokens before the new ones at the new scale, those behind them as they were
            mask = lo < hi ? (hi == 4 ? 0xFFFFFFFFu : (1u << (8 * hi)) - 1u) & ~((1u << (8 * lo)) - 1u) : 0u;
            const uint32_t old = *p;
            const uint32_t before = 4 * q + 3 < s.lo ? 0xFFFFFFFFu : (1u << (8 * min(max(s.lo - 4 * q, 0), 3))) - 1u;
            kept = (rescaled(old, s0, sc) & before) | (old & ~before);
        }
        *p = (word & mask) | (kept & ~mask);
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void cache8_read_kernel(RowArgs a) {
    Spot s;
    if (!find(a, s) || !s.there(a)) return;
    const int tid = threadIdx.x, nt = blockDim.x;
    const int block = 1 << a.block_log;
    const int q0 = s.lo / 4, q1 = (s.hi + 3) / 4, patches = (q1 - q0) * a.runs;
    const int64_t ld = a.ld[s.which];
    T *y = static_cast<T *>(a.out[s.which]) + (int64_t(s.item) * a.tokens + (s.base - s.first)) * ld +
           int64_t(s.head) * a.d;
    const float sc = a.scale[s.which][s.at(a)];
    const uint8_t *const code = a.code[s.which] + s.at(a) * block * a.dp;
    for (int p = tid; p < patches; p += nt) {
        const int row = int(uint32_t(p) * a.by_runs >> 16), run = p - row * a.runs, q = q0 + row;
        Eight<T, VEC> r[4];
        if (s.which == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uintx2 w = *reinterpret_cast<const uintx2 *>(code + (q * 4 + e) * a.dp + run * 8);
#pragma unroll
                for (int i = 0; i < 8; ++i) r[e].set(i, float(int((w[i / 4] >> (8 * (i % 4))) & 255) - 128) * sc);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(code + (run * 8 + i) * block + q * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e].set(i, float(int((w >> (8 * e)) & 255) - 128) * sc);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int t = q * 4 + e;
            if (t >= s.lo && t < s.hi) r[e].store(y + int64_t(t) * ld + run * 8, a.d - run * 8);
        }
    }
}

RowArgs row_args(const Cache8 &c, const PageTable &t, HeadRows k, HeadRows v, int tokens, const int32_t *first,
                 const int32_t *len) {
    RowArgs a{};
    a.in[0] = k.p, a.in[1] = v.p;
    a.out[0] = const_cast<void *>(k.p), a.out[1] = const_cast<void *>(v.p);
    a.ld[0] = k.ld, a.ld[1] = v.ld;
    a.code[0] = c.k, a.code[1] = c.v, a.scale[0] = c.k_scale, a.scale[1] = c.v_scale;
    a.table = t.table, a.first = first, a.len = len;
    a.tokens = tokens, a.blocks = t.blocks, a.pages = c.pages, a.heads = c.heads;
    a.d = c.d, a.dp = c.dp(), a.runs = int(ceil_div(c.d, 8)), a.by_runs = uint32_t((65536 + a.runs - 1) / a.runs), a.block_log = c.block_log;
    // blocks that a run of tokens from anywhere (first NULL: from 0) lies in
    a.touched = int(std::min<int64_t>(t.blocks, (int64_t(tokens) + (first ? c.block() - 1 : 0) + c.block() - 1) >> c.block_log));
    return a;
}

bool wide(HeadRows x, int d, int size) {
    return d % 8 == 0 && x.ld % (16 / size) == 0 && aligned16(x.p);
}

uint32_t grid_of(const RowArgs &a, int n) {
    const int64_t g = int64_t(n) * a.heads * 2 * a.touched;
    MH_REQUIRE(g < (int64_t(1) << 31), "cache8: too many blocks of tokens");
    return uint32_t(g);
}

// Patches that the new tokens of a block make at most.
int most_patches(const RowArgs &a, bool anywhere) {
    const int quads = 1 << (a.block_log - 2);
    return std::min(quads, int(ceil_div(std::min(a.tokens, 1 << a.block_log) + (anywhere ? 3 : 0), 4))) * a.runs;
}

}  // namespace

void cache8_write(Context &ctx, const Cache8 &c, const PageTable &t, HeadRows k, HeadRows v, WeightType type, int tokens,
                  const int32_t *first, const int32_t *len) {
    if (!t.n || !tokens || !t.blocks) return;
    const RowArgs a = row_args(c, t, k, v, tokens, first, len);
    const int size = type == kF16 ? 2 : 4;
    const bool vec = wide(k, c.d, size) && wide(v, c.d, size);
    const int patches = most_patches(a, first != nullptr && tokens > 1);
    const int pu = int(ceil_div(patches, 256)), nt = int(ceil_div(patches, pu * 64) * 64);
    const size_t lds = size_t(a.dp) * (c.block() / 4 + 1) * 4;
    const dim3 grid{grid_of(a, t.n)}, threads{uint32_t(nt)};
    auto go = [&](auto kernel) { kernel<<<grid, threads, lds, ctx.stream>>>(a); };
    auto by_size = [&](auto zero, auto vecs) {
        using T = decltype(zero);
        constexpr bool V = decltype(vecs)::value;
        if (pu == 1) go(cache8_write_kernel<T, 1, V>);
        else if (pu == 2) go(cache8_write_kernel<T, 2, V>);
        else go(cache8_write_kernel<T, 4, V>);
    };
    if (type == kF16) {
        if (vec) by_size(_Float16(0), std::true_type{});
        else by_size(_Float16(0), std::false_type{});
    } else {
        if (vec) by_size(0.0f, std::true_type{});
        else by_size(0.0f, std::false_type{});
    }
    MH_LAUNCH_CHECK();
}

void cache8_read(Context &ctx, const Cache8 &c, const PageTable &t, HeadRows k, HeadRows v, WeightType type, int tokens,
                 const int32_t *first, const int32_t *len) {
    if (!t.n || !tokens || !t.blocks) return;
    const RowArgs a = row_args(c, t, k, v, tokens, first, len);
    const int size = type == kF16 ? 2 : 4;
    const bool vec = wide(k, c.d, size) && wide(v, c.d, size);
    const int patches = most_patches(a, first != nullptr && tokens > 1);
    const dim3 grid{grid_of(a, t.n)}, threads{uint32_t(patches <= 64 ? 64 : patches <= 128 ? 128 : 256)};
    if (type == kF16) {
        if (vec) cache8_read_kernel<_Float16, true><<<grid, threads, 0, ctx.stream>>>(a);
        else cache8_read_kernel<_Float16, false><<<grid, threads, 0, ctx.stream>>>(a);
    } else {
        if (vec) cache8_read_kernel<float, true><<<grid, threads, 0, ctx.stream>>>(a);
        else cache8_read_kernel<float, false><<<grid, threads, 0, ctx.stream>>>(a);
    }
    MH_LAUNCH_CHECK();
}

}  // namespace mh
