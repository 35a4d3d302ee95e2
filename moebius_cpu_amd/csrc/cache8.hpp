// A cache of keys and values in 8 bits, and attention over it: the C++ functions
// behind the entry points of include/moebius_hip.h. All are asynchronous on
// ctx.stream. None has a counterpart in the reference.
#pragma once

#include <cstdint>

#include "attention.hpp"

namespace mh {

// Pages of `block` tokens (16 << 0 .. 3): codes of keys [pages][heads][block][dp], of values
// [pages][heads][dp][block] (dp: d rounded up to 16), a code b standing for (b - 128) scale, and
// f32 scales [pages][heads]. Values lie channel by channel because the attention multiplies V^T
// by the probabilities, whose operand holds consecutive tokens of one channel in a lane.
struct Cache8 {
    uint8_t *k = nullptr, *v = nullptr;
    float *k_scale = nullptr, *v_scale = nullptr;
    int pages = 0, heads = 0, d = 0, block_log = 0;
    int dp() const { return (d + 15) / 16 * 16; }
    int block() const { return 1 << block_log; }
};

// Token p of item i lies in page table[i][p >> block_log]; entries outside 0 .. pages - 1: not there.
struct PageTable {
    const int32_t *table = nullptr;  // [n][blocks]
    int n = 0, blocks = 0;
};

// Tokens t < len[item] (NULL: tokens) of k and v [n][tokens] rows go to first[item] + t (NULL: t).
void cache8_write(Context &ctx, const Cache8 &c, const PageTable &t, HeadRows k, HeadRows v, WeightType type, int tokens,
                  const int32_t *first, const int32_t *len);
// What the cache holds at first[item] + t, t < len[item], to rows t of k and v.
void cache8_read(Context &ctx, const Cache8 &c, const PageTable &t, HeadRows k, HeadRows v, WeightType type, int tokens,
                 const int32_t *first, const int32_t *len);

// Row t of an item stands at position t + kv_len - q_len and sees the tokens j < kv_len, where
// causal j <= its position, and where window > 0 those less than window before it or j < sinks.
struct Cache8Attention {
    Cache8 c;
    PageTable t;
    HeadRows q;
    WeightType type = kF32;
    int q_tokens = 0;
    void *out = nullptr;
    int64_t ld_out = 0;
    const int32_t *q_len = nullptr, *kv_len = nullptr;
    float scale = 0;
    bool causal = false;
    int window = 0, sinks = 0;
};
size_t cache8_attention_scratch(const Context &ctx, const Cache8Attention &a);
void cache8_attention(Context &ctx, const Cache8Attention &a, void *scratch);

}  // namespace mh
