// The entry points of include/moebius_hip.h for transformers over image and video
// tokens and for adapters: argument checks, which need no device, then the context
// and the functions of attention.hpp.
#include <algorithm>
#include <cmath>
#include <string>

#include "attention.hpp"
#include "capi_context.hpp"
#include "capi_rows.hpp"

namespace {

using mh::capi::aligned4;
using mh::capi::C;
using mh::capi::check_scratch;
using mh::capi::dim;
using mh::capi::guard;
using mh::capi::need;
using mh::capi::no_overlap;
using mh::capi::Rows;
using mh::capi::rows_of;
using mh::capi::same_or_apart;
using mh::capi::size_of;
using mh::capi::wtype;

mh::RopeTable rope_table(const MhRope *r, uint32_t d) {
    need(r, "rope");
    need(r->positions, "positions");
    need(r->freq, "freq");
    if (reinterpret_cast<uintptr_t>(r->positions) % 4 || reinterpret_cast<uintptr_t>(r->freq) % 8)
        mh::fail(mh::kInvalidArgument, "rope: positions or freq are not aligned to their type");
    if (r->axes < 1 || r->axes > uint32_t(mh::kRopeMaxAxes)) mh::fail(mh::kInvalidArgument, "rope: 1 to 4 axes");
    if (r->pairing > MH_ROPE_HALVES) mh::fail(mh::kInvalidArgument, "rope: unknown pairing");
    if (r->pos_rows == 0) mh::fail(mh::kInvalidArgument, "rope: no positions");
    if (r->reserved) mh::fail(mh::kInvalidArgument, "rope: reserved is not 0");
    mh::RopeTable t;
    t.pos = r->positions;
    t.freq = r->freq;
    t.pos_rows = int64_t(std::min<uint64_t>(r->pos_rows, 0xFFFFFFFFull));
    t.axes = int(r->axes);
    uint64_t sum = 0;
    for (uint32_t a = 0; a < r->axes; ++a) {
        if (r->axis_dims[a] == 0 || r->axis_dims[a] % 2) mh::fail(mh::kInvalidArgument, "rope: axis dims are even and not 0");
        sum += r->axis_dims[a];
        if (sum > d) mh::fail(mh::kInvalidArgument, "rope: axis dims exceed the head");
        t.pair_end[a] = int(sum / 2);
    }
    t.pairing = mh::RopePairing(r->pairing);
    t.inverse = r->inverse != 0;
    return t;
}

void few_rows(uint64_t rows) {
    if (rows >= (uint64_t(1) << 31)) mh::fail(mh::kInvalidArgument, "2^31 rows or more");
}

// (offsets within a tile of a projection are 32 bits)
void few_channels(uint32_t c_in, uint32_t c_out) {
    if (std::max(c_in, c_out) > (1u << 22)) mh::fail(mh::kInvalidArgument, "Conv1x1: more than 2^22 channels");
}

mh::BlockShape block_shape(const MhBlockShape *s) {
    need(s, "shape");
    mh::BlockShape b;
    b.n = dim(s->n, "n");
    b.q_tokens = dim(s->q_tokens, "q_tokens");
    b.kv_tokens = dim(s->kv_tokens, "kv_tokens");
    if (s->heads_q == 0 || s->heads_kv == 0 || s->d == 0) mh::fail(mh::kInvalidArgument, "shape: no heads or channels");
    b.heads_q = dim(s->heads_q, "heads_q");
    b.heads_kv = dim(s->heads_kv, "heads_kv");
    if (b.heads_q % b.heads_kv) mh::fail(mh::kInvalidArgument, "heads_q is not a multiple of heads_kv");
    if (b.heads_q / b.heads_kv > 65536) mh::fail(mh::kInvalidArgument, "more than 65536 query heads per key head");
    if (s->d > uint32_t(mh::kMaxHeadDim)) mh::fail(mh::kInvalidArgument, "heads of more than 256 channels");
    b.d = int(s->d);
    if (s->q_block < 1 || s->q_block > 1024) mh::fail(mh::kInvalidArgument, "q_block is 1 .. 1024");
    b.q_block = int(s->q_block);
    if (s->kv_block != 16 && s->kv_block != 32 && s->kv_block != 64 && s->kv_block != 128)
        mh::fail(mh::kInvalidArgument, "kv_block is 16, 32, 64 or 128");
    b.kv_block = int(s->kv_block);
    if (s->top < 1 || s->top > uint32_t(mh::kMaxTop)) mh::fail(mh::kInvalidArgument, "top is 1 .. 1024");
    b.top = int(s->top);
    b.causal = s->causal != 0;
    if (reinterpret_cast<uintptr_t>(s->q_len) % 4 || reinterpret_cast<uintptr_t>(s->kv_len) % 4)
        mh::fail(mh::kInvalidArgument, "lengths are not aligned to their type");
    b.q_len = s->q_len;
    b.kv_len = s->kv_len;
    return b;
}

}  // namespace

extern "C" {

int32_t mh_rope_frequencies(double theta, uint32_t axes, const uint32_t *axis_dims, double *freq) {
    return guard([&] {
        need(axis_dims, "axis_dims");
        need(freq, "freq");
        if (!(theta > 0) || !std::isfinite(theta)) mh::fail(mh::kInvalidArgument, "rope: theta is positive and finite");
        if (axes < 1 || axes > uint32_t(mh::kRopeMaxAxes)) mh::fail(mh::kInvalidArgument, "rope: 1 to 4 axes");
        for (uint32_t a = 0; a < axes; ++a)
            if (axis_dims[a] == 0 || axis_dims[a] % 2 || axis_dims[a] > (1u << 20))
                mh::fail(mh::kInvalidArgument, "rope: axis dims are even and not 0");
        mh::rope_frequencies(theta, int(axes), axis_dims, freq);
    });
}

int32_t mh_rope_axes(MhContext *ctx, const void *x, uint32_t dtype, uint64_t rows, uint32_t heads, uint32_t d,
                     uint64_t ld_x, const MhRope *rope, void *out, uint64_t ld_out) {
    return guard([&] {
        few_rows(rows);
        const mh::WeightType t = wtype(dtype);
        const Rows in = rows_of(x, rows, heads, d, ld_x, t, "x"), to = rows_of(out, rows, heads, d, ld_out, t, "out");
        const mh::RopeTable table = rope_table(rope, d);
        same_or_apart(in, to, "x and out");
        mh::Context &c = C(ctx);
        mh::rope_axes(c, {x, in.ld, int(heads)}, t, in.rows, int(d), table, out, to.ld);
    });
}

int32_t mh_qk_norm_rope(MhContext *ctx, const void *q, uint64_t ld_q, uint32_t heads_q, const void *k, uint64_t ld_k,
                        uint32_t heads_k, uint32_t dtype, uint64_t rows, uint32_t d, const float *gamma_q,
                        const float *gamma_k, float eps, const MhRope *rope, void *q_out, uint64_t ld_qo, void *k_out,
                        uint64_t ld_ko) {
    return guard([&] {
        few_rows(rows);
        const mh::WeightType t = wtype(dtype);
        const Rows qi = rows_of(q, rows, heads_q, d, ld_q, t, "q"), ki = rows_of(k, rows, heads_k, d, ld_k, t, "k");
        const Rows qo = rows_of(q_out, rows, heads_q, d, ld_qo, t, "q_out");
        const Rows ko = rows_of(k_out, rows, heads_k, d, ld_ko, t, "k_out");
        if (!(eps >= 0) || !std::isfinite(eps)) mh::fail(mh::kInvalidArgument, "eps is finite and not negative");
        aligned4(gamma_q, "gamma_q");
        aligned4(gamma_k, "gamma_k");
        const mh::RopeTable table = rope_table(rope, d);
        same_or_apart(qi, qo, "q and q_out");
        same_or_apart(ki, ko, "k and k_out");
        no_overlap(qi, ko, "q and k_out");
        no_overlap(ki, qo, "k and q_out");
        no_overlap(qo, ko, "q_out and k_out");
        mh::Context &c = C(ctx);
        mh::qk_norm_rope(c, {q, qi.ld, int(heads_q)}, {k, ki.ld, int(heads_k)}, t, qi.rows, int(d), gamma_q, gamma_k,
                         eps, table, q_out, qo.ld, k_out, ko.ld);
    });
}

int32_t mh_block_means(MhContext *ctx, const void *x, uint32_t dtype, uint32_t n, uint32_t tokens, uint32_t heads,
                       uint32_t d, uint64_t ld, const int32_t *first, const int32_t *len, uint32_t block,
                       float *means) {
    return guard([&] {
        const mh::WeightType t = wtype(dtype);
        const uint64_t rows = uint64_t(dim(n, "n")) * uint64_t(dim(tokens, "tokens"));
        const Rows in = rows_of(x, rows, heads, d, ld, t, "x");
        if (block < 1 || block > 1024) mh::fail(mh::kInvalidArgument, "block is 1 .. 1024");
        if (rows) need(means, "means");
        aligned4(first, "first");
        aligned4(len, "len");
        aligned4(means, "means");
        mh::Context &c = C(ctx);
        mh::block_means(c, {x, in.ld, int(heads)}, t, int(n), int(tokens), int(d), first, len, int(block), means);
    });
}

int32_t mh_block_select(MhContext *ctx, const void *q, uint32_t dtype, uint64_t ld_q, const MhBlockShape *shape,
                        const float *k_means, int32_t *blocks) {
    return guard([&] {
        const mh::WeightType t = wtype(dtype);
        const mh::BlockShape s = block_shape(shape);
        const Rows in = rows_of(q, uint64_t(s.n) * s.q_tokens, s.heads_q, s.d, ld_q, t, "q");
        if (in.rows) need(blocks, "blocks");
        if (in.rows && s.kv_tokens) need(k_means, "k_means");
        aligned4(blocks, "blocks");
        aligned4(k_means, "k_means");
        if (s.kv_blocks() > mh::kMaxKeyBlocks) mh::fail(mh::kInvalidArgument, "more than 8192 blocks of keys");
        if (s.causal && s.top < std::min(s.kv_blocks(), (s.q_block + s.kv_block - 2) / s.kv_block + 1))
            mh::fail(mh::kInvalidArgument, "top does not hold the blocks of the queries' own tokens");
        mh::Context &c = C(ctx);
        mh::block_select(c, {q, in.ld, s.heads_q}, t, s, k_means, blocks);
    });
}

int32_t mh_block_attention_scratch(MhContext *ctx, uint32_t dtype, const MhBlockShape *shape, uint64_t *bytes) {
    return guard([&] {
        need(bytes, "bytes");
        const mh::WeightType t = wtype(dtype);
        const mh::BlockShape s = block_shape(shape);
        mh::Context &c = C(ctx);
        *bytes = mh::block_attention_scratch(c, s, t);
    });
}

int32_t mh_block_attention(MhContext *ctx, const void *q, uint64_t ld_q, const void *k, uint64_t ld_k, const void *v,
                           uint64_t ld_v, uint32_t dtype, const MhBlockShape *shape, const int32_t *blocks, float scale,
                           void *out, uint64_t ld_out, void *scratch, uint64_t scratch_bytes) {
    return guard([&] {
        const mh::WeightType t = wtype(dtype);
        mh::BlockAttention a;
        a.s = block_shape(shape);
        const uint64_t q_rows = uint64_t(a.s.n) * a.s.q_tokens, kv_rows = uint64_t(a.s.n) * a.s.kv_tokens;
        const Rows qi = rows_of(q, q_rows, a.s.heads_q, a.s.d, ld_q, t, "q");
        const Rows ki = rows_of(k, kv_rows, a.s.heads_kv, a.s.d, ld_k, t, "k");
        const Rows vi = rows_of(v, kv_rows, a.s.heads_kv, a.s.d, ld_v, t, "v");
        const Rows to = rows_of(out, q_rows, a.s.heads_q, a.s.d, ld_out, t, "out");
        if (q_rows) need(blocks, "blocks");
        aligned4(blocks, "blocks");
        if (ki.ld * int64_t(ki.size) >= (1 << 25) || vi.ld * int64_t(vi.size) >= (1 << 25))
            mh::fail(mh::kInvalidArgument, "rows of k or v 32 MiB apart or more");
        if (!(scale > 0) || !std::isfinite(scale)) mh::fail(mh::kInvalidArgument, "scale is positive and finite");
        no_overlap(qi, to, "q and out");
        no_overlap(ki, to, "k and out");
        no_overlap(vi, to, "v and out");
        mh::Context &c = C(ctx);
        const size_t needed = mh::block_attention_scratch(c, a.s, t);
        scratch = check_scratch(c, scratch, scratch_bytes, needed);
        if (needed && !scratch) scratch = c.ws.get(needed, c.stream);
        a.q = {q, qi.ld, a.s.heads_q};
        a.k = {k, ki.ld, a.s.heads_kv};
        a.v = {v, vi.ld, a.s.heads_kv};
        a.out = out;
        a.ld_out = to.ld;
        a.blocks = blocks;
        a.scale = scale;
        mh::block_attention(c, a, t, scratch);
    });
}

int32_t mh_conv1x1_lora_scratch(MhContext *ctx, uint64_t rows, uint32_t c_in, uint32_t c_out, uint32_t weight_dtype,
                                uint32_t rank, uint64_t *bytes) {
    return guard([&] {
        need(bytes, "bytes");
        few_rows(rows);
        if (rank < 1 || rank > uint32_t(mh::kMaxRank)) mh::fail(mh::kInvalidArgument, "rank is 1 .. 256");
        const mh::WeightType t = wtype(weight_dtype);
        few_channels(c_in, c_out);
        mh::Context &c = C(ctx);
        *bytes = mh::lora_scratch(c, int64_t(rows), dim(c_in, "c_in"), dim(c_out, "c_out"), t, int(rank));
    });
}

int32_t mh_conv1x1_lora(MhContext *ctx, const float *x, uint64_t rows, uint32_t c_in, const void *weight,
                        uint32_t weight_dtype, uint32_t c_out, const float *bias, const float *residual,
                        const MhAdapters *adapters, const int32_t *slot, uint64_t rows_per_slot, float *out,
                        void *scratch, uint64_t scratch_bytes) {
    return guard([&] {
        few_rows(rows);
        need(weight, "weight");
        need(adapters, "adapters");
        if (rows) {
            need(x, "x");
            need(out, "out");
            need(slot, "slot");
        }
        if (c_in == 0 || c_out == 0) mh::fail(mh::kInvalidArgument, "Conv1x1: empty channel axis");
        if (rows_per_slot == 0 || rows_per_slot >= (uint64_t(1) << 31))
            mh::fail(mh::kInvalidArgument, "rows_per_slot is 1 .. 2^31 - 1");
        few_channels(c_in, c_out);
        mh::Lora l;
        l.type = wtype(adapters->dtype);
        if (adapters->rank < 1 || adapters->rank > uint32_t(mh::kMaxRank))
            mh::fail(mh::kInvalidArgument, "rank is 1 .. 256");
        if (adapters->reserved) mh::fail(mh::kInvalidArgument, "adapters: reserved is not 0");
        l.rank = int(adapters->rank);
        l.slots = dim(adapters->slots, "slots");
        if (l.slots) {
            need(adapters->a, "adapters a");
            need(adapters->b, "adapters b");
            need(adapters->scale, "adapters scale");
        }
        if (reinterpret_cast<uintptr_t>(adapters->a) % size_of(l.type) ||
            reinterpret_cast<uintptr_t>(adapters->b) % size_of(l.type))
            mh::fail(mh::kInvalidArgument, "adapters are not aligned to their type");
        for (const void *q : {static_cast<const void *>(x), static_cast<const void *>(out), static_cast<const void *>(bias),
                              static_cast<const void *>(residual), static_cast<const void *>(slot),
                              static_cast<const void *>(adapters->scale)})
            aligned4(q, "x, out, bias, residual, slot or scale");
        if (reinterpret_cast<uintptr_t>(weight) % size_of(wtype(weight_dtype)))
            mh::fail(mh::kInvalidArgument, "weight is not aligned to its type");
        l.a = adapters->a, l.b = adapters->b, l.scale = adapters->scale;
        l.slot = slot;
        l.rows_per_slot = int64_t(rows_per_slot);
        const Rows to{reinterpret_cast<const char *>(out), int64_t(rows), int64_t(c_out), int64_t(c_out), 4};
        const Rows in{reinterpret_cast<const char *>(x), int64_t(rows), int64_t(c_in), int64_t(c_in), 4};
        no_overlap(in, to, "x and out");
        Rows res = to;
        res.p = reinterpret_cast<const char *>(residual);
        if (residual) same_or_apart(res, to, "residual and out");
        mh::Context &c = C(ctx);
        const size_t needed = mh::lora_scratch(c, int64_t(rows), dim(c_in, "c_in"), dim(c_out, "c_out"),
                                               wtype(weight_dtype), l.rank);
        scratch = check_scratch(c, scratch, scratch_bytes, needed);
        mh::conv1x1_lora(c, x, int64_t(rows), int(c_in), weight, wtype(weight_dtype), dim(c_out, "c_out"), bias,
                         residual, l, out, scratch);
    });
}

}  // extern "C"
