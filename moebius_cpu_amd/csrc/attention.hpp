// Operators of transformers over image and video tokens, and low-rank adapters
// beside a shared projection: the C++ functions behind the entry points of
// include/moebius_hip.h. All are asynchronous on ctx.stream. None has a
// counterpart in the reference, whose UNet mixes tokens with lambda layers.
#pragma once

#include <cstdint>

#include "common.hpp"
#include "kernels.hpp"

namespace mh {

// Heads of tokens: element (row, head, channel) of a tensor at row * ld + head * d +
// channel, f32 or f16 (WeightType, the storage types of the library).
struct HeadRows {
    const void *p = nullptr;
    int64_t ld = 0;
    int heads = 0;
};

// ---- rotary positions (rope.hip)
enum class RopePairing : uint32_t { Interleaved = 0, Halves = 1 };

constexpr int kRopeMaxAxes = 4;

// Rotary positions over up to four axes: the head's first 2 * pair_end[axes - 1]
// channels in pairs, pairs pair_end[a - 1] .. pair_end[a] - 1 turned by
// pos[row % pos_rows][a] * freq[pair] radians.
struct RopeTable {
    const int32_t *pos = nullptr;   // [pos_rows][axes]
    const double *freq = nullptr;   // [pairs], radians per position
    int64_t pos_rows = 0;
    int axes = 0;
    int pair_end[kRopeMaxAxes] = {0, 0, 0, 0};
    RopePairing pairing = RopePairing::Interleaved;
    bool inverse = false;
};

void rope_frequencies(double theta, int axes, const uint32_t *axis_dims, double *freq);
// x and out (which may be x) of `rows` rows; channels behind the pairs are copied.
void rope_axes(Context &ctx, HeadRows x, WeightType type, int64_t rows, int d, const RopeTable &t, void *out,
               int64_t ld_out);
// RMS norm of each head of q and k (gamma f32 [d] or NULL), then the rotation.
void qk_norm_rope(Context &ctx, HeadRows q, HeadRows k, WeightType type, int64_t rows, int d, const float *gamma_q,
                  const float *gamma_k, float eps, const RopeTable &t, void *q_out, int64_t ld_qo, void *k_out,
                  int64_t ld_ko);

// ---- attention over selected blocks of keys (block_select.hip, block_attention*)
constexpr int kMaxHeadDim = 256;    // channels of a head that the selection and the attention take
constexpr int kMaxKeyBlocks = 8192; // key blocks of an item that the selection orders
constexpr int kMaxTop = 1024;       // selected blocks per block of queries

// means [n][ceil(tokens / block)][heads][d] f32: each block's mean over its tokens below
// len[item] (NULL: tokens), f64 sums rounded once. Blocks without such a token, and
// those wholly below first[item] (NULL: 0), are left as they were.
void block_means(Context &ctx, HeadRows x, WeightType type, int n, int tokens, int d, const int32_t *first,
                 const int32_t *len, int block, float *means);

// The geometry that the selection and the attention share: n items of q_tokens rows of
// q.heads heads and kv_tokens rows of heads_kv heads, in blocks of q_block and kv_block.
struct BlockShape {
    int n = 0, q_tokens = 0, kv_tokens = 0, heads_q = 0, heads_kv = 0, d = 0, q_block = 0, kv_block = 0, top = 0;
    bool causal = false;
    const int32_t *q_len = nullptr, *kv_len = nullptr;  // [n], NULL: full
    int q_blocks() const { return int(ceil_div(q_tokens, q_block)); }
    int kv_blocks() const { return int(ceil_div(kv_tokens, kv_block)); }
};
void block_select(Context &ctx, HeadRows q, WeightType type, const BlockShape &s, const float *k_means,
                  int32_t *blocks);

// out [n][q_tokens][heads_q][d] (rows ld_out apart) = softmax(scale q . k) v over the tokens
// of each block of queries' list blocks [n][q blocks][heads_kv][top] below kv_len and, where
// causal, at most i + kv_len - q_len for query i. Indices outside 0 .. blocks - 1 are skipped,
// one listed twice counts once; a row that sees no key is zero, rows at or above q_len are
// left as they were. scratch: block_attention_scratch bytes (0: none needed), 16-byte aligned.
struct BlockAttention {
    BlockShape s;
    HeadRows q, k, v;
    void *out = nullptr;
    int64_t ld_out = 0;
    const int32_t *blocks = nullptr;
    float scale = 0;
};
size_t block_attention_scratch(const Context &ctx, const BlockShape &s, WeightType type);
void block_attention(Context &ctx, const BlockAttention &a, WeightType type, void *scratch);

// ---- low-rank adapters beside a shared projection (lora.hip)
constexpr int kMaxRank = 256;

// out [rows][c_out] = x . W^T + bias + residual + scale[s] (x . a[s]^T) . b[s]^T, written once, for
// every row whose s = slot[row / rows_per_slot] is one of 0 .. slots - 1; a [slots][rank][c_in],
// b [slots][c_out][rank]. Other rows are the projection alone. scratch: lora_scratch bytes, 16-byte aligned.
struct Lora {
    const void *a = nullptr, *b = nullptr;
    WeightType type = kF32;
    int slots = 0, rank = 0;
    const float *scale = nullptr;   // [slots]
    const int32_t *slot = nullptr;  // [ceil(rows / rows_per_slot)]
    int64_t rows_per_slot = 1;
};
size_t lora_scratch(const Context &ctx, int64_t rows, int c_in, int c_out, WeightType wt, int rank);
void conv1x1_lora(Context &ctx, const float *x, int64_t rows, int c_in, const void *weight, WeightType wt, int c_out,
                  const float *bias, const float *residual, const Lora &l, float *out, void *scratch);

}  // namespace mh
