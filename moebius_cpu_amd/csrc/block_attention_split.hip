// Instantiations of block_attention.hpp for f32 storage as two f16 parts, and the kernel
// that splits keys and values once for all blocks of queries that read them.
#include <algorithm>

#include "block_attention.hpp"

namespace mh {
namespace battn {
namespace {

// One workgroup per (item, block, key head) and side (keys, values): the largest exponent
// of the block's finite values, then the parts. Bound: memory, 8 bytes per value.
template <bool VEC>
__global__ __launch_bounds__(256) void split_kv_kernel(const float *k, const float *v, int64_t ldk, int64_t ldv,
                                                       int kv_tokens, int blocks, int hk, int d, int dk, int kb,
                                                       const int32_t *kv_len, _Float16 *kp, _Float16 *vp,
                                                       SplitMeta *meta) {
    __shared__ float wave_max[4];
    __shared__ int wave_bad[4];
    const bool is_v = blockIdx.y;
    const int head = blockIdx.x % hk, b = blockIdx.x / hk % blocks, item = blockIdx.x / hk / blocks;
    const int len = kv_len ? min(max(kv_len[item], 0), kv_tokens) : kv_tokens;
    const int rows = min(kb, len - b * kb), runs = dk / 8;  // rows may be negative
    const int64_t ld = is_v ? ldv : ldk;
    const float *src = (is_v ? v : k) + (int64_t(item) * kv_tokens + b * kb) * ld + int64_t(head) * d;
    float mx = 0.0f;
    bool bad = false;
    auto get = [&](int i) {
        const int r = i / runs, ch = i % runs * 8;
        Run8<float> x;
        x.zero();
        if (r < rows) x.template load<VEC>(src + int64_t(r) * ld + ch, d - ch);
        return x;
    };
    for (int i = threadIdx.x; i < kb * runs; i += 256) {
        const Run8<float> x = get(i);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = __builtin_fabsf(x.at(e));
            const bool ok = a < __builtin_huge_valf();
            mx = ok ? __builtin_fmaxf(mx, a) : mx;
            bad = bad || !ok;
        }
    }
    for (int m = 32; m; m >>= 1) mx = __builtin_fmaxf(mx, __shfl_xor(mx, m));
    bad = __any(bad);
    if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = mx, wave_bad[threadIdx.x >> 6] = bad;
    __syncthreads();
    mx = __builtin_fmaxf(__builtin_fmaxf(wave_max[0], wave_max[1]), __builtin_fmaxf(wave_max[2], wave_max[3]));
    bad = wave_bad[0] | wave_bad[1] | wave_bad[2] | wave_bad[3];
    const int e = mx == 0.0f ? 0 : __builtin_amdgcn_frexp_expf(mx) - 1;
    _Float16 *dst = (is_v ? vp : kp) + ((int64_t(item) * blocks + b) * kb * hk + head) * 2 * dk;
    for (int i = threadIdx.x; i < kb * runs; i += 256) {
        Run8<float> x = get(i);
        if (is_v && bad) x.clean();
        halfx8 hi, lo;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            _Float16 p, q;
            split2(x.at(c), kSplitExp - e, p, q);
            hi[c] = p, lo[c] = q;
        }
        _Float16 *o = dst + int64_t(i / runs) * hk * 2 * dk + i % runs * 8;
        *reinterpret_cast<halfx8 *>(o) = hi;
        *reinterpret_cast<halfx8 *>(o + dk) = lo;
    }
    if (threadIdx.x == 0) {
        SplitMeta *m = meta + (int64_t(item) * blocks + b) * hk + head;
        if (is_v) m->v_exp = mx == 0.0f ? kNoExp : e, m->v_bad = bad;
        else m->k_exp = e;
    }
}

}  // namespace

void split_kv(Context &ctx, const float *k, const float *v, int64_t ldk, int64_t ldv, int n, int kv_tokens, int hk,
              int d, int dk, int kb, const int32_t *kv_len, void *kp, void *vp, SplitMeta *meta) {
    const int blocks = int(ceil_div(kv_tokens, kb));
    const int64_t groups = int64_t(n) * blocks * hk;
    MH_REQUIRE(groups < (int64_t(1) << 31), "block_attention: too many blocks of keys");
    const bool vec = d % 8 == 0 && ldk % 4 == 0 && ldv % 4 == 0 && aligned16(k) && aligned16(v);
    const dim3 grid{uint32_t(groups), 2}, tb{256};
    auto *kh = static_cast<_Float16 *>(kp), *vh = static_cast<_Float16 *>(vp);
    if (vec)
        split_kv_kernel<true><<<grid, tb, 0, ctx.stream>>>(k, v, ldk, ldv, kv_tokens, blocks, hk, d, dk, kb, kv_len, kh,
                                                           vh, meta);
    else
        split_kv_kernel<false><<<grid, tb, 0, ctx.stream>>>(k, v, ldk, ldv, kv_tokens, blocks, hk, d, dk, kb, kv_len, kh,
                                                            vh, meta);
    MH_LAUNCH_CHECK();
}

void launch_split(Context &ctx, const Args &a, int wr, int dt, bool vec) { launch_mode<float, kSplit>(ctx, a, wr, dt, vec); }

}  // namespace battn
}  // namespace mh
