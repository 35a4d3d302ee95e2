// Instantiations of block_attention.hpp for f32 storage as two f16 parts, and the kernel
// that splits keys and values once for all blocks of queries that read them.
#include <algorithm>

#include "block_attention.hpp"

namespace mh {
namespace battn {
namespace {

// One workgroup per (item, 16 tokens, 32 where GL is 8, key head) and side (keys, values), a
// group of GL lanes per token and eight channels a lane: the exponents that each sixteen
// share or have by themselves (KeyScale), then the parts. Tokens at or behind kv_len are not
// written. Bound: memory, 8 bytes per value.
template <bool VEC, int GL>
__global__ __launch_bounds__(GL == 32 ? 512 : 256) void split_kv_kernel(const float *k, const float *v, int64_t ldk,
                                                                        int64_t ldv, int kv_tokens, int kv_rows, int hk,
                                                                        int d, int dk, const int32_t *kv_len,
                                                                        _Float16 *kp, _Float16 *vp, KeyScale *meta) {
    constexpr int kRows = (GL == 32 ? 512 : 256) / GL, kNone = 0x7fffffff;
    __shared__ __align__(16) int exps[kRows];  // of the tokens, kNone: not there
    const bool is_v = blockIdx.y;
    const int tiles = (kv_tokens + kRows - 1) / kRows;
    const int head = blockIdx.x % hk, tile = blockIdx.x / hk % tiles, item = blockIdx.x / hk / tiles;
    const int len = kv_len ? min(max(kv_len[item], 0), kv_tokens) : kv_tokens;
    const int lane = threadIdx.x & 63, r = threadIdx.x / GL, t = tile * kRows + r, ch = threadIdx.x % GL * 8;
    const int64_t ld = is_v ? ldv : ldk;
    const float *src = (is_v ? v : k) + (int64_t(item) * kv_tokens + t) * ld + int64_t(head) * d;
    Run8<float> x;
    x.zero();
    if (t < len && ch < dk) x.template load<VEC>(src + ch, d - ch);
    float mx = 0.0f;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float a = __builtin_fabsf(x.at(e));
        const bool ok = a < __builtin_huge_valf();
        mx = ok ? __builtin_fmaxf(mx, a) : mx;
        bad = bad || !ok;
    }
#pragma unroll
    for (int m = GL / 2; m; m >>= 1) mx = __builtin_fmaxf(mx, __shfl_xor(mx, m));
    bad = __ballot(bad) >> (lane / GL * GL) & ((uint64_t(1) << GL) - 1);
    int e = mx == 0.0f ? kNoExp : __builtin_amdgcn_frexp_expf(mx) - 1;
    if (ch == 0) exps[r] = t < len ? e : kNone;
    __syncthreads();
    int hi = kNoExp, lo = kNone;
    bool zero = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const intx4 q = reinterpret_cast<const intx4 *>(exps)[r / 16 * 4 + i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            hi = max(hi, q[j] == kNone ? kNoExp : q[j]);
            lo = min(lo, q[j] == kNoExp ? kNone : q[j]);
            zero = zero || q[j] == kNoExp;
        }
    }
    // (zeros take any exponent as keys, as values none: they would count among what a row sees)
    if (hi != kNoExp && hi - lo <= kSplitSpread && !(is_v && zero)) e = hi;
    if (!is_v && e == kNoExp) e = 0;
    if (t >= len) return;
    const int64_t at = (int64_t(item) * kv_rows + t) * hk + head;
    if (ch < dk) {
        if (is_v && bad) x.clean();
        halfx8 p, q;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            _Float16 big, small;
            split2(x.at(c), kSplitExp - e, big, small);
            p[c] = big, q[c] = small;
        }
        _Float16 *o = (is_v ? vp : kp) + at * 2 * dk + ch;
        *reinterpret_cast<halfx8 *>(o) = p;
        *reinterpret_cast<halfx8 *>(o + dk) = q;
    }
    if (ch == 0) {
        KeyScale &s = meta[(int64_t(item) * hk + head) * kv_rows + t];
        if (is_v) s.v = 2 * e + bad;
        else s.k = e;
    }
}

template <bool VEC>
void launch_split_kv(Context &ctx, const float *k, const float *v, int64_t ldk, int64_t ldv, int n, int kv_tokens,
                     int kv_rows, int hk, int d, int dk, const int32_t *kv_len, _Float16 *kp, _Float16 *vp,
                     KeyScale *meta) {
    const int gl = dk <= 64 ? 8 : dk <= 128 ? 16 : 32, threads = gl == 32 ? 512 : 256;
    const int64_t groups = int64_t(n) * ceil_div(kv_tokens, threads / gl) * hk;
    MH_REQUIRE(groups < (int64_t(1) << 31), "block_attention: too many keys");
    const dim3 grid{uint32_t(groups), 2}, tb{uint32_t(threads)};
    auto run = [&](auto kernel) {
        kernel<<<grid, tb, 0, ctx.stream>>>(k, v, ldk, ldv, kv_tokens, kv_rows, hk, d, dk, kv_len, kp, vp, meta);
    };
    if (gl == 8) run(split_kv_kernel<VEC, 8>);
    else if (gl == 16) run(split_kv_kernel<VEC, 16>);
    else run(split_kv_kernel<VEC, 32>);
    MH_LAUNCH_CHECK();
}

}  // namespace

void split_kv(Context &ctx, const float *k, const float *v, int64_t ldk, int64_t ldv, int n, int kv_tokens, int kv_rows,
              int hk, int d, int dk, const int32_t *kv_len, void *kp, void *vp, KeyScale *meta) {
    const bool vec = d % 8 == 0 && ldk % 4 == 0 && ldv % 4 == 0 && aligned16(k) && aligned16(v);
    auto *kh = static_cast<_Float16 *>(kp), *vh = static_cast<_Float16 *>(vp);
    if (vec) launch_split_kv<true>(ctx, k, v, ldk, ldv, n, kv_tokens, kv_rows, hk, d, dk, kv_len, kh, vh, meta);
    else launch_split_kv<false>(ctx, k, v, ldk, ldv, n, kv_tokens, kv_rows, hk, d, dk, kv_len, kh, vh, meta);
}

void launch_split(Context &ctx, const Args &a, int wr, int dt, bool vec) { launch_mode<float, kSplit>(ctx, a, wr, dt, vec); }

}  // namespace battn
}  // namespace mh
