// Which variant of the attention over a cache in 8 bits runs, and the scratch its splits
// join through.
#include <algorithm>

#include "cache8_attention.hpp"

namespace mh {
namespace {

// Tiles of 16 channels of the instantiated kernels that hold a head of d channels.
int head_tiles(int d) {
    const int t = int(ceil_div(d, 16));
    return t <= 4 ? 4 : t <= 6 ? t : t <= 8 ? 8 : t <= 10 ? 10 : 16;
}

struct Plan {
    int nq, waves, dt, row_tiles, splits;  // waves > 0: of 32 rows that share chunks in LDS, else nq tiles of 16 rows
    int64_t items;
    size_t bytes;
};

Plan plan(const Context &ctx, const Cache8Attention &a) {
    Plan p;
    const int64_t rows = int64_t(a.q_tokens) * (a.q.heads / a.c.heads);
    p.dt = head_tiles(a.c.d);
    p.nq = rows > 16 && p.dt <= 8 ? 2 : 1;
    int64_t tokens = int64_t(a.t.blocks) << a.c.block_log;
    if (a.window) tokens = std::min(tokens, int64_t(a.window) + a.sinks + a.q_tokens);
    // Waves that share chunks: eight, or four where there are few rows, heads of 64 (of which a CU then
    // holds three workgroups) or heads that three buffers of LDS do not hold. They pay where they fill
    // the card or the tokens are many. us shared (the better of four and eight waves), alone:
    //                                   32 heads over 8 of 128   16 over 4 of 64   8 of 80   f32: of 128   of 64
    //   1 item, 256 queries, 2000 tokens        45, 29                24, 20        22, 18     52, 38    26, 23
    //   1, 1000, 1000                           75, 59                40, 22        33, 15     85, 74    44, 25
    //   8, 24, 16384                            126, 150              48, 59        87, 44     159, 237  55, 64
    //   8, 64, 4000                             84, 90                42, 29        38, 31     102, 128  45, 32
    //   4, 200, 4000                            133, 167              62, 56        45, 35     157, 243  68, 62
    // A few hundred rows of large heads over a few thousand tokens are where the rule leaves most behind.
    const int waves = rows > 128 && p.dt > 4 && p.dt <= 8 ? 8 : 4;
    const int64_t fill = int64_t(a.t.n) * a.c.heads * ceil_div(rows, 32 * waves);
    p.waves = rows > 64 && (4 * fill >= 3 * ctx.cu_count || tokens > 4096) ? waves : 0;
    const int tile = p.waves ? 32 * p.waves : 16 * p.nq;
    p.row_tiles = int(ceil_div(rows, tile));
    p.items = int64_t(a.t.n) * a.c.heads * p.row_tiles;
    // The tokens are split over workgroups where the rows alone leave CUs idle, up to one workgroup per
    // CU (two of four waves that share), into shares of 256 tokens or more, where there are more than
    // 512. Single tokens, 32 heads over 8 of 128, f16, us with this rule and with up to two workgroups
    // per CU: 8 items of 16384 tokens 49, 55, of 4096 21, 27 (16 over 4 of 64, 16384: 19, 21; 8 of 80:
    // 34, 39); 1 of 300 9.4 whole, 11.7 in two. 8 items of 24 queries over 16384 in workgroups of four
    // waves: 127 with two, 146 with one, 143 with three (heads of 64: 48, 65, 49).
    // Tokens are the table's, as lengths are on the device: one query over 300 tokens takes 15.8 under a
    // table for 16384 and 9.5 under one of its own.
    const int64_t room = (p.waves == 4 && p.dt <= 8 ? 2 : 1) * int64_t(ctx.cu_count) / std::max<int64_t>(p.items, 1);
    p.splits = tokens > 512 ? int(std::max<int64_t>(1, std::min(ceil_div(tokens, 256), room))) : 1;
    const int floats = (p.waves ? (p.dt + 1) / 2 * 32 : p.dt * 16) + 2;
    p.bytes = p.splits > 1 ? size_t(p.items) * p.splits * tile * floats * sizeof(float) : 0;
    return p;
}

}  // namespace

size_t cache8_attention_scratch(const Context &ctx, const Cache8Attention &a) {
    if (!a.t.n || !a.q_tokens) return 0;
    return plan(ctx, a).bytes;
}

void cache8_attention(Context &ctx, const Cache8Attention &c, void *scratch) {
    if (!c.t.n || !c.q_tokens) return;
    const Plan p = plan(ctx, c);
    MH_REQUIRE(p.items * p.splits < (int64_t(1) << 26), "cache8_attention: too many rows");
    c8a::Args a{};
    a.q = c.q.p, a.out = c.out, a.ldq = c.q.ld, a.ldo = c.ld_out;
    a.k = c.c.k, a.v = c.c.v, a.ks = c.c.k_scale, a.vs = c.c.v_scale;
    a.table = c.t.table, a.q_len = c.q_len, a.kv_len = c.kv_len;
    a.part = p.splits > 1 ? static_cast<float *>(scratch) : nullptr;
    a.c = c.scale * 1.44269504088896340736f;
    a.q_tokens = c.q_tokens, a.hk = c.c.heads, a.g = c.q.heads / c.c.heads, a.d = c.c.d, a.dp = c.c.dp();
    a.blocks = c.t.blocks, a.pages = c.c.pages, a.block_log = c.c.block_log;
    a.row_tiles = p.row_tiles, a.splits = p.splits, a.work = int(p.items * p.splits);
    a.causal = c.causal, a.window = c.window, a.sinks = c.sinks;
    const int size = c.type == kF16 ? 2 : 4;
    a.wide = c.c.d % 8 == 0 && c.q.ld % (16 / size) == 0 && aligned16(c.q.p) && c.ld_out % 4 == 0 &&
             reinterpret_cast<uintptr_t>(c.out) % (4 * size) == 0;
    const bool fast = ctx.precision == Precision::Fast;
    if (c.type == kF16 && fast && p.waves) c8a::launch_f16_half(ctx, a, p.waves, p.dt);
    else if (c.type == kF16) c8a::launch_f16(ctx, a, p.nq, p.waves, p.dt);
    else if (fast) c8a::launch_f32_half(ctx, a, p.nq, p.waves, p.dt);
    else c8a::launch_f32(ctx, a, p.nq, p.waves, p.dt);
}

}  // namespace mh
