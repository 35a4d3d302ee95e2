// The entry points of include/moebius_hip.h for a cache in 8 bits, the attention over it
// and gated norms: argument checks, which need no device, then the context and the
// functions of cache8.hpp and gated_norm.hpp.
#include <cmath>
#include <string>

#include "cache8.hpp"
#include "capi_context.hpp"
#include "capi_rows.hpp"
#include "gated_norm.hpp"

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
using mh::capi::size_of;
using mh::capi::wtype;

struct Held {
    mh::Cache8 c;
    uint64_t codes, scales;  // bytes of each array
};

Held sizes(uint32_t pages, uint32_t heads, uint32_t d, uint32_t block) {
    Held h;
    if (pages == 0) mh::fail(mh::kInvalidArgument, "cache: no pages");
    if (heads == 0 || d == 0) mh::fail(mh::kInvalidArgument, "cache: no heads or channels");
    if (d > uint32_t(mh::kMaxHeadDim)) mh::fail(mh::kInvalidArgument, "cache: heads of more than 256 channels");
    if (block != 16 && block != 32 && block != 64 && block != 128)
        mh::fail(mh::kInvalidArgument, "cache: block is 16, 32, 64 or 128");
    h.c.pages = dim(pages, "pages");
    h.c.heads = dim(heads, "heads");
    if (uint64_t(pages) * heads >= (uint64_t(1) << 31)) mh::fail(mh::kInvalidArgument, "cache too large");
    h.c.d = int(d);
    h.c.block_log = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7;
    h.codes = uint64_t(pages) * heads * block * h.c.dp();
    h.scales = uint64_t(pages) * heads * 4;
    return h;
}

Held cache_of(const MhCache8 *c) {
    need(c, "cache");
    Held h = sizes(c->pages, c->heads, c->d, c->block);
    need(c->k, "cache k");
    need(c->v, "cache v");
    need(c->k_scale, "cache k_scale");
    need(c->v_scale, "cache v_scale");
    if (!mh::aligned16(c->k) || !mh::aligned16(c->v))
        mh::fail(mh::kInvalidArgument, "cache: codes are not 16-byte aligned");
    aligned4(c->k_scale, "cache k_scale");
    aligned4(c->v_scale, "cache v_scale");
    h.c.k = c->k, h.c.v = c->v, h.c.k_scale = c->k_scale, h.c.v_scale = c->v_scale;
    return h;
}

mh::PageTable table_of(const MhPageTable *t, int block) {
    need(t, "table");
    mh::PageTable p;
    p.n = dim(t->n, "n");
    p.blocks = dim(t->blocks, "blocks");
    if (int64_t(p.blocks) * block > (1 << 30)) mh::fail(mh::kInvalidArgument, "table: more than 2^30 tokens per item");
    if (p.n && p.blocks) need(t->pages, "table pages");
    aligned4(t->pages, "table pages");
    p.table = t->pages;
    return p;
}

// A run of bytes as the overlap check takes it.
Rows bytes_of(const void *p, uint64_t bytes) {
    return Rows{static_cast<const char *>(p), bytes ? 1 : 0, int64_t(bytes), int64_t(bytes), 1};
}

void apart_from_cache(const Rows &r, const Held &h, const char *what) {
    for (const void *p : {h.c.k, h.c.v}) no_overlap(r, bytes_of(p, h.codes), what);
    for (const void *p : {h.c.k_scale, h.c.v_scale}) no_overlap(r, bytes_of(p, h.scales), what);
}

void own_arrays(const Held &h) {
    const Rows r[4] = {bytes_of(h.c.k, h.codes), bytes_of(h.c.v, h.codes), bytes_of(h.c.k_scale, h.scales),
                       bytes_of(h.c.v_scale, h.scales)};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < i; ++j) no_overlap(r[i], r[j], "the arrays of the cache");
}

Rows small(const int32_t *p, uint64_t count) { return bytes_of(p, p ? count * 4 : 0); }

mh::NormSpec norm_of(const MhNorm &n, const char *what) {
    const std::string name = what;
    mh::NormSpec s;
    if (n.kind > MH_NORM_LAYER) mh::fail(mh::kInvalidArgument, name + ": unknown norm");
    s.kind = mh::NormKind(n.kind);
    if (s.kind == mh::NormKind::None) {
        if (n.gamma || n.beta) mh::fail(mh::kInvalidArgument, name + ": gamma or beta without a norm");
        return s;
    }
    if (!(n.eps >= 0) || !std::isfinite(n.eps)) mh::fail(mh::kInvalidArgument, name + ": eps is finite and not negative");
    s.eps = n.eps;
    aligned4(n.gamma, "gamma");
    aligned4(n.beta, "beta");
    s.gamma = n.gamma, s.beta = n.beta;
    return s;
}

}  // namespace

extern "C" {

int32_t mh_cache8_sizes(uint32_t pages, uint32_t heads, uint32_t d, uint32_t block, uint64_t *code_bytes,
                        uint64_t *scale_bytes) {
    return guard([&] {
        need(code_bytes, "code_bytes");
        need(scale_bytes, "scale_bytes");
        const Held h = sizes(pages, heads, d, block);
        *code_bytes = h.codes, *scale_bytes = h.scales;
    });
}

int32_t mh_cache8_write(MhContext *ctx, const MhCache8 *cache, const MhPageTable *table, const void *k, uint64_t ld_k,
                        const void *v, uint64_t ld_v, uint32_t dtype, uint32_t tokens, const int32_t *first,
                        const int32_t *len) {
    return guard([&] {
        const mh::WeightType t = wtype(dtype);
        const Held h = cache_of(cache);
        const mh::PageTable p = table_of(table, h.c.block());
        const uint64_t rows = uint64_t(p.n) * uint64_t(dim(tokens, "tokens"));
        const Rows kr = rows_of(k, rows, h.c.heads, h.c.d, ld_k, t, "k"), vr = rows_of(v, rows, h.c.heads, h.c.d, ld_v, t, "v");
        aligned4(first, "first");
        aligned4(len, "len");
        own_arrays(h);
        apart_from_cache(kr, h, "k and the cache");
        apart_from_cache(vr, h, "v and the cache");
        apart_from_cache(small(p.table, uint64_t(p.n) * p.blocks), h, "the table and the cache");
        apart_from_cache(small(first, p.n), h, "first and the cache");
        apart_from_cache(small(len, p.n), h, "len and the cache");
        mh::Context &c = C(ctx);
        mh::cache8_write(c, h.c, p, {k, kr.ld, h.c.heads}, {v, vr.ld, h.c.heads}, t, int(tokens), first, len);
    });
}

int32_t mh_cache8_read(MhContext *ctx, const MhCache8 *cache, const MhPageTable *table, void *k, uint64_t ld_k, void *v,
                       uint64_t ld_v, uint32_t dtype, uint32_t tokens, const int32_t *first, const int32_t *len) {
    return guard([&] {
        const mh::WeightType t = wtype(dtype);
        const Held h = cache_of(cache);
        const mh::PageTable p = table_of(table, h.c.block());
        const uint64_t rows = uint64_t(p.n) * uint64_t(dim(tokens, "tokens"));
        const Rows kr = rows_of(k, rows, h.c.heads, h.c.d, ld_k, t, "k"), vr = rows_of(v, rows, h.c.heads, h.c.d, ld_v, t, "v");
        aligned4(first, "first");
        aligned4(len, "len");
        no_overlap(kr, vr, "k and v");
        for (const Rows *r : {&kr, &vr}) {
            apart_from_cache(*r, h, "k or v and the cache");
            no_overlap(*r, small(p.table, uint64_t(p.n) * p.blocks), "k or v and the table");
            no_overlap(*r, small(first, p.n), "k or v and first");
            no_overlap(*r, small(len, p.n), "k or v and len");
        }
        mh::Context &c = C(ctx);
        mh::cache8_read(c, h.c, p, {k, kr.ld, h.c.heads}, {v, vr.ld, h.c.heads}, t, int(tokens), first, len);
    });
}

}  // extern "C"

namespace {

mh::Cache8Attention attention_of(const MhCacheAttention *s, uint32_t dtype, const MhCache8 *cache,
                                 const MhPageTable *table) {
    need(s, "shape");
    mh::Cache8Attention a;
    a.c = cache_of(cache).c;
    a.t = table_of(table, a.c.block());
    a.type = wtype(dtype);
    a.q_tokens = dim(s->q_tokens, "q_tokens");
    if (s->heads_q == 0) mh::fail(mh::kInvalidArgument, "shape: no heads");
    a.q.heads = dim(s->heads_q, "heads_q");
    if (a.q.heads % a.c.heads) mh::fail(mh::kInvalidArgument, "heads_q is not a multiple of the cache's heads");
    if (a.q.heads / a.c.heads > 65536) mh::fail(mh::kInvalidArgument, "more than 65536 query heads per key head");
    if (int64_t(a.q_tokens) * (a.q.heads / a.c.heads) >= (int64_t(1) << 30))
        mh::fail(mh::kInvalidArgument, "2^30 rows of a key head or more");
    if (s->window > (1u << 30) || s->sinks > (1u << 30)) mh::fail(mh::kInvalidArgument, "window or sinks too large");
    if (s->reserved) mh::fail(mh::kInvalidArgument, "shape: reserved is not 0");
    if (s->sinks && !s->window) mh::fail(mh::kInvalidArgument, "sinks without a window");
    a.causal = s->causal != 0;
    a.window = int(s->window), a.sinks = int(s->sinks);
    aligned4(s->q_len, "q_len");
    aligned4(s->kv_len, "kv_len");
    a.q_len = s->q_len, a.kv_len = s->kv_len;
    return a;
}

}  // namespace

extern "C" {

int32_t mh_cache8_attention_scratch(MhContext *ctx, uint32_t dtype, const MhCacheAttention *shape, const MhCache8 *cache,
                                    const MhPageTable *table, uint64_t *bytes) {
    return guard([&] {
        need(bytes, "bytes");
        const mh::Cache8Attention a = attention_of(shape, dtype, cache, table);
        mh::Context &c = C(ctx);
        *bytes = mh::cache8_attention_scratch(c, a);
    });
}

int32_t mh_cache8_attention(MhContext *ctx, const void *q, uint64_t ld_q, uint32_t dtype, const MhCacheAttention *shape,
                            const MhCache8 *cache, const MhPageTable *table, float scale, void *out, uint64_t ld_out,
                            void *scratch, uint64_t scratch_bytes) {
    return guard([&] {
        mh::Cache8Attention a = attention_of(shape, dtype, cache, table);
        const uint64_t rows = uint64_t(a.t.n) * a.q_tokens;
        const Rows qi = rows_of(q, rows, a.q.heads, a.c.d, ld_q, a.type, "q");
        const Rows to = rows_of(out, rows, a.q.heads, a.c.d, ld_out, a.type, "out");
        if (!(scale > 0) || !std::isfinite(scale)) mh::fail(mh::kInvalidArgument, "scale is positive and finite");
        no_overlap(qi, to, "q and out");
        const Held h = cache_of(cache);
        apart_from_cache(to, h, "out and the cache");
        no_overlap(to, small(a.t.table, uint64_t(a.t.n) * a.t.blocks), "out and the table");
        no_overlap(to, small(a.q_len, a.t.n), "out and q_len");
        no_overlap(to, small(a.kv_len, a.t.n), "out and kv_len");
        mh::Context &c = C(ctx);
        const size_t needed = mh::cache8_attention_scratch(c, a);
        scratch = check_scratch(c, scratch, scratch_bytes, needed);
        if (needed && !scratch) scratch = c.ws.get(needed, c.stream);
        a.q.p = q, a.q.ld = qi.ld;
        a.out = out, a.ld_out = to.ld;
        a.scale = scale;
        mh::cache8_attention(c, a, scratch);
    });
}

int32_t mh_gated_norm(MhContext *ctx, const MhGatedNorm *n) {
    return guard([&] {
        need(n, "gated norm");
        mh::GatedNorm g;
        if (n->rows >= (uint64_t(1) << 31)) mh::fail(mh::kInvalidArgument, "2^31 rows or more");
        if (n->rows_per_item == 0 || n->rows_per_item >= (uint64_t(1) << 31))
            mh::fail(mh::kInvalidArgument, "rows_per_item is 1 .. 2^31 - 1");
        if (n->c == 0 || n->c > uint32_t(mh::kGatedNormMaxC)) mh::fail(mh::kInvalidArgument, "c is 1 .. 32768");
        if (!std::isfinite(n->keep)) mh::fail(mh::kInvalidArgument, "keep is finite");
        g.rows = int64_t(n->rows), g.rows_per_item = int64_t(n->rows_per_item), g.c = int(n->c), g.keep = n->keep;
        g.x_type = wtype(n->x_dtype), g.branch_type = wtype(n->branch_dtype);
        g.post = norm_of(n->post, "post"), g.pre = norm_of(n->pre, "pre");
        const Rows x = rows_of(n->x, n->rows, 1, n->c, n->ld_x, g.x_type, "x");
        g.x = n->x, g.ld_x = x.ld;
        Rows in[2] = {x, Rows{}}, out[2] = {};
        if (n->branch) {
            in[1] = rows_of(n->branch, n->rows, 1, n->c, n->ld_branch, g.branch_type, "branch");
            g.branch = n->branch, g.ld_branch = in[1].ld;
        } else if (n->gate || g.post.kind != mh::NormKind::None) {
            mh::fail(mh::kInvalidArgument, "gate or post without a branch");
        }
        if (n->x_out) {
            out[0] = rows_of(n->x_out, n->rows, 1, n->c, n->ld_x_out, g.x_type, "x_out");
            g.x_out = n->x_out, g.ld_x_out = out[0].ld;
        }
        if (n->y) {
            out[1] = rows_of(n->y, n->rows, 1, n->c, n->ld_y, g.branch_type, "y");
            g.y = n->y, g.ld_y = out[1].ld;
        } else if (n->scale || n->shift || g.pre.kind != mh::NormKind::None) {
            mh::fail(mh::kInvalidArgument, "pre, scale or shift without y");
        }
        if (!n->x_out && !n->y) mh::fail(mh::kInvalidArgument, "neither x_out nor y");
        if (out[0].rows && out[1].rows) no_overlap(out[0], out[1], "x_out and y");
        const uint64_t items = (n->rows + n->rows_per_item - 1) / n->rows_per_item;
        // vectors of the items, and of the norms
        auto vectors = [&](const float *p, uint64_t count, uint64_t ld, const char *what) {
            if (!p) return;
            const Rows r = rows_of(p, count, 1, n->c, ld, mh::kF32, what);
            for (const Rows &o : out)
                if (o.rows) no_overlap(r, o, "a vector and x_out or y");
        };
        vectors(n->gate, items, n->ld_gate, "gate");
        vectors(n->scale, items, n->ld_scale, "scale");
        vectors(n->shift, items, n->ld_shift, "shift");
        vectors(g.post.gamma, 1, n->c, "gamma"), vectors(g.post.beta, 1, n->c, "beta");
        vectors(g.pre.gamma, 1, n->c, "gamma"), vectors(g.pre.beta, 1, n->c, "beta");
        for (const Rows &i : in)
            for (const Rows &o : out) {
                // in place: every value is read by the thread that writes it, and before
                if (!i.rows || !o.rows || (i.p == o.p && i.ld == o.ld && i.size == o.size)) continue;
                no_overlap(i, o, "x or branch and x_out or y");
            }
        g.gate = {n->gate, int64_t(n->ld_gate)}, g.scale = {n->scale, int64_t(n->ld_scale)};
        g.shift = {n->shift, int64_t(n->ld_shift)};
        mh::Context &c = C(ctx);
        mh::gated_norm(c, g);
    });
}

}  // extern "C"
