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
    if (!vec) return t <= 4 ? 4 : t == 5 ? 5 : 8;
    return t <= 5 ? t : 8;
}

// Waves of 32 rows that share a tile of keys: as many as the rows of a block of queries
// fill, up to four. 24 heads of 64, 8192 rows in blocks of 128, 2048 keys each: four 142 us,
// two 165; 8 heads, 4096 rows in blocks of 64, 1024 keys: two 20.6, one 31.7, four 27.8; in
// blocks of 32: one 30.7, two 34.0. Heads of more than 128 channels take two even where one
// has no rows, as the registers that stage a tile are then shared by both: 8 heads of 160,
// 2 x 4096 rows in blocks of 32, 1024 keys 130 us, 230 with one; single tokens of 8 requests,
// 32 / 8 heads, 2048 keys 28.7 and 39.2; f32 148 and 177 (16 requests).
int row_waves(const BlockShape &s) {
    const int64_t rows = int64_t(std::min(s.q_block, s.q_tokens)) * (s.heads_q / s.heads_kv);
    return rows > 64 ? 4 : rows > 32 || s.d > 128 ? 2 : 1;
}

struct Plan {
    int wr, row_tiles, splits;
    int64_t items;  // workgroups without the splits
    bool split;     // f32 operands as two f16 parts
};

// The list is split over workgroups where the rows alone leave CUs idle: into a power of
// two of shares (equal ones of most lists), of 256 keys (f32 128), or down to 128 (f32, and
// where two or four waves of rows share the keys, 64) where that leaves CUs idle, up to two
// workgroups per CU (f32 one).
// Single tokens, 8 heads of 128, f16, caches that are not in the L2, us without splits, with
// this rule, with half and with twice as many: 1 item of 4096 keys 95, 17.6, 22, 18.3; 4 of
// 2048 46, 19.1, 21.9, 20.7; 8 of 2048 47, 24.6, 24.9, 31; 16 of 2048 52.8, 35.9, 37.4, 40.1;
// 1 of 512 15.1, 12.1, 13.7, 12.1; 4 of 256 10.9 without, 12.6 with two; 40 of 2048 76.3
// without, 88.7 with two. f32: 2 of 2048 118, 26.8, 30; 8 of 1024 65, 34, 44, 44; 1 of 256
// 23.6, 19.9, 20.3. Blocks of 128 rows, 1 head of 160, 296 keys: 19.7, 15, 17.4 (f32 41.5,
// 29.8, 33.8).
//
// f32 products are split where the keys and values, which that reads and writes once, are
// then read at least kSplitReuse times by waves full of rows: 4096 keys, 8 heads of 80, read
// once 30.4 us (25.0 on the f32 instructions), twice 34.6 (33.5), four times 43.5 (49.5),
// sixteen times 69 (149). Where one wave's rows are all, kSplitReuseFew times, as half of the
// row waves then stand idle: 2 heads of 80 of 2 items, 8 times 36.5 (31.6), 16 times 39.7 (60.2)
// and 57.7 (56.0), 32 times 88 (90), 128 times 170 (345).
constexpr int64_t kSplitReuse = 2, kSplitReuseFew = 16;
Plan plan(const Context &ctx, const BlockShape &s, WeightType type, bool half) {
    Plan p;
    p.wr = row_waves(s);
    const int64_t rows = int64_t(std::min(s.q_block, s.q_tokens)) * (s.heads_q / s.heads_kv);
    p.row_tiles = int(ceil_div(rows, p.wr * 32));
    p.items = int64_t(s.n) * s.heads_kv * s.q_blocks() * p.row_tiles;
    const int64_t keys = std::min<int64_t>(int64_t(s.top) * s.kv_block, s.kv_tokens);
    p.splits = 1;
    const bool f32 = type == kF32 && !half;
    const int64_t items = std::max<int64_t>(p.items, 1), cus = ctx.cu_count, least = f32 || p.wr > 1 ? 64 : 128;
    if (items < cus && keys >= 4 * least) {
        const int64_t most = std::min<int64_t>((f32 ? 1 : 2) * cus / items,
                                               std::max<int64_t>(keys / (f32 ? 128 : 256), std::min<int64_t>(4, cus / items)));
        while (2 * p.splits <= most) p.splits *= 2;
    }
    p.split = f32 && s.kv_tokens > 0 && battn::split_fits(head_tiles(s.d, false)) &&
              battn::split_fits(head_tiles(s.d, true)) &&
              int64_t(s.q_blocks()) * p.row_tiles * keys >= (p.wr == 1 ? kSplitReuseFew : kSplitReuse) * s.kv_tokens;
    if (p.split) p.wr = std::max(p.wr, 2);
    return p;
}

// Scratch: the splits' partial sums, then the parts of keys and of values and their scales.
struct Layout {
    size_t part = 0, parts = 0, meta = 0;  // bytes of each (parts: of keys, and of values)
    size_t total() const { return part + 2 * parts + meta; }
};

Layout layout(const BlockShape &s, const Plan &p) {
    auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
    Layout l;
    if (p.splits > 1)  // the most that any alignment of these sizes needs
        l.part = up(size_t(p.items) * p.splits * p.wr * battn::part_floats(head_tiles(s.d, false)) * sizeof(float));
    if (p.split) {
        const size_t rows = size_t(s.n) * s.kv_blocks() * s.kv_block * s.heads_kv;
        l.parts = up(rows * 2 * size_t(ceil_div(s.d, 8) * 8) * 2);
        l.meta = up(rows * sizeof(battn::KeyScale));
    }
    return l;
}

}  // namespace

size_t block_attention_scratch(const Context &ctx, const BlockShape &s, WeightType type) {
    if (!s.n || !s.q_tokens) return 0;
    return layout(s, plan(ctx, s, type, ctx.precision == Precision::Fast)).total();
}

void block_attention(Context &ctx, const BlockAttention &b, WeightType type, void *scratch) {
    const BlockShape &s = b.s;
    if (!s.n || !s.q_tokens) return;
    const bool half = type == kF16 || ctx.precision == Precision::Fast;
    const Plan p = plan(ctx, s, type, half);
    const Layout l = layout(s, p);
    MH_REQUIRE(p.items * p.splits < (int64_t(1) << 30), "block_attention: too many blocks of queries");
    const int size = type == kF16 ? 2 : 4;
    const bool vec_q = vec_rows(b.q.p, b.q.ld, s.d, size) && vec_rows(b.out, b.ld_out, s.d, size);
    const bool vec = vec_q && (p.split || (vec_rows(b.k.p, b.k.ld, s.d, size) && vec_rows(b.v.p, b.v.ld, s.d, size)));
    char *mem = static_cast<char *>(scratch);
    battn::Args a{};
    a.q = b.q.p, a.k = b.k.p, a.v = b.v.p, a.out = b.out;
    a.ldq = b.q.ld, a.ldo = b.ld_out;
    a.ldk = uint32_t(b.k.ld * size), a.ldv = uint32_t(b.v.ld * size);
    a.blocks = b.blocks, a.q_len = s.q_len, a.kv_len = s.kv_len;
    a.part = p.splits > 1 ? reinterpret_cast<float *>(mem) : nullptr;
    a.c = b.scale * 1.44269504088896340736f;
    a.n = s.n, a.q_tokens = s.q_tokens, a.kv_tokens = s.kv_tokens, a.hk = s.heads_kv, a.g = s.heads_q / s.heads_kv;
    a.d = s.d, a.qb = s.q_block, a.nq = s.q_blocks(), a.top = s.top;
    while ((1 << a.kb_log) < s.kv_block) ++a.kb_log;
    a.row_tiles = p.row_tiles, a.splits = p.splits, a.work = int(p.items * p.splits), a.causal = s.causal;
    a.dk = s.d, a.kv_rows = s.kv_tokens;
    const int dt = head_tiles(s.d, vec);
    if (p.split) {
        a.dk = int(ceil_div(s.d, 8) * 8);
        a.kv_rows = s.kv_blocks() * s.kv_block;
        a.v0 = b.v.p, a.ldv0 = a.ldv;
        char *kp = mem + l.part, *vp = kp + l.parts;
        auto *meta = reinterpret_cast<battn::KeyScale *>(vp + l.parts);
        battn::split_kv(ctx, static_cast<const float *>(b.k.p), static_cast<const float *>(b.v.p), b.k.ld, b.v.ld, s.n,
                        s.kv_tokens, a.kv_rows, s.heads_kv, s.d, a.dk, s.kv_len, kp, vp, meta);
        a.k = kp, a.v = vp, a.meta = meta;
        const uint64_t row = uint64_t(s.heads_kv) * 2 * a.dk * 2;
        MH_REQUIRE(row < (uint64_t(1) << 25), "block_attention: rows of keys or values of 32 MiB or more");
        a.ldk = a.ldv = uint32_t(row);
        battn::launch_split(ctx, a, p.wr, dt, vec);
    } else if (type == kF16) {
        battn::launch_f16(ctx, a, p.wr, dt, vec);
    } else if (half) {
        battn::launch_f32_half(ctx, a, p.wr, dt, vec);
    } else {
        battn::launch_f32(ctx, a, p.wr, dt, vec);
    }
}

}  // namespace mh
