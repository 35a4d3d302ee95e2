// Which variant of the block attention runs, and the scratch its splits join through.
#include <algorithm>

#include "block_attention.hpp"

namespace mh {
namespace {

bool vec_rows(const void *p, int64_t ld, int d, int size) {
    return d % 8 == 0 && ld % (16 / size) == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

// 32-channel tiles of the instantiated kernels that hold a head of d channels.
int head_tiles(int d, bool vec) {
    const int t = int(ceil_div(d, 32));
    if (!vec) return t <= 4 ? 4 : 8;
    return t <= 5 ? t : 8;
}

// Waves of 32 rows that share a tile of keys: as many as the rows of a block of queries
// fill, up to four.
int row_waves(const BlockShape &s) {
    const int64_t rows = int64_t(std::min(s.q_block, s.q_tokens)) * (s.heads_q / s.heads_kv);
    return rows > 64 ? 4 : rows > 32 ? 2 : 1;
}

struct Plan {
    int wr, row_tiles, splits;
    int64_t items;  // workgroups without the splits
};

// The list is split over workgroups where the rows alone leave CUs idle, into shares of
// at least 128 keys.
Plan plan(const Context &ctx, const BlockShape &s) {
    Plan p;
    p.wr = row_waves(s);
    const int64_t rows = int64_t(std::min(s.q_block, s.q_tokens)) * (s.heads_q / s.heads_kv);
    p.row_tiles = int(ceil_div(rows, p.wr * 32));
    p.items = int64_t(s.n) * s.heads_kv * s.q_blocks() * p.row_tiles;
    const int64_t keys = std::min<int64_t>(int64_t(s.top) * s.kv_block, s.kv_tokens);
    int64_t splits = p.items >= ctx.cu_count ? 1 : std::min<int64_t>(2 * ctx.cu_count / std::max<int64_t>(p.items, 1), keys / 128);
    p.splits = int(std::max<int64_t>(1, std::min<int64_t>(splits, 64)));
    return p;
}

}  // namespace

size_t block_attention_scratch(const Context &ctx, const BlockShape &s) {
    if (!s.n || !s.q_tokens) return 0;
    const Plan p = plan(ctx, s);
    if (p.splits == 1) return 0;
    // the most that any storage and alignment of these sizes needs
    return size_t(p.items) * p.splits * p.wr * battn::part_floats(head_tiles(s.d, false)) * sizeof(float);
}

void block_attention(Context &ctx, const BlockAttention &b, WeightType type, void *scratch) {
    const BlockShape &s = b.s;
    if (!s.n || !s.q_tokens) return;
    const Plan p = plan(ctx, s);
    MH_REQUIRE(p.items * p.splits < (int64_t(1) << 30), "block_attention: too many blocks of queries");
    const int size = type == kF16 ? 2 : 4;
    const bool vec = vec_rows(b.q.p, b.q.ld, s.d, size) && vec_rows(b.k.p, b.k.ld, s.d, size) &&
                     vec_rows(b.v.p, b.v.ld, s.d, size) && vec_rows(b.out, b.ld_out, s.d, size);
    battn::Args a{};
    a.q = b.q.p, a.k = b.k.p, a.v = b.v.p, a.out = b.out;
    a.ldq = b.q.ld, a.ldo = b.ld_out;
    MH_REQUIRE(b.k.ld * size < (int64_t(1) << 32) && b.v.ld * size < (int64_t(1) << 32),
               "block_attention: rows of keys or values 4 GiB apart or more");
    a.ldk = uint32_t(b.k.ld * size), a.ldv = uint32_t(b.v.ld * size);
    a.blocks = b.blocks, a.q_len = s.q_len, a.kv_len = s.kv_len;
    a.part = p.splits > 1 ? static_cast<float *>(scratch) : nullptr;
    a.c = b.scale * 1.44269504088896340736f;
    a.n = s.n, a.q_tokens = s.q_tokens, a.kv_tokens = s.kv_tokens, a.hk = s.heads_kv, a.g = s.heads_q / s.heads_kv;
    a.d = s.d, a.qb = s.q_block, a.nq = s.q_blocks(), a.top = s.top;
    while ((1 << a.kb_log) < s.kv_block) ++a.kb_log;
    a.row_tiles = p.row_tiles, a.splits = p.splits, a.work = int(p.items * p.splits), a.causal = s.causal;
    const int dt = head_tiles(s.d, vec);
    if (type == kF16) battn::launch_f16(ctx, a, p.wr, dt, vec);
    else if (b.half) battn::launch_f32_half(ctx, a, p.wr, dt, vec);
    else battn::launch_f32(ctx, a, p.wr, dt, vec);
}

}  // namespace mh
