// Which kernels take a masked attention call, how long walks are cut into parts, and
// the scratch that this needs: by the sizes alone. Host only and free of HIP.
#pragma once

#include "cross_attention_plan.hpp"

namespace nrs {

// A unit is an unbroken set of an item's rows (or keys, in the backward) that a
// workgroup holds; its walk is the tiles of the other side that any of them sees.
// How many these are, only the device knows. A walk is cut into parts of `part` tiles,
// from its own first tile on, each a workgroup's; the grid has `parts` of them for
// every unit, and those that a unit does not need end at once.
struct MaskedWalk {
    int64_t units = 0;
    int part = 1, parts = 1;
};

// Parts no longer than `share` tiles (at least `least`) of walks of up to `tiles`.
inline void cut_walk(MaskedWalk& w, int64_t tiles, int64_t share, int64_t least) {
    const int64_t part = std::max<int64_t>(1, std::min(tiles, std::max(share, least)));
    w.part = (int)part;
    w.parts = (int)std::max<int64_t>(1, (tiles + part - 1) / part);
}

struct MaskedForwardPlan {
    bool tiles;  // the kernel of many rows
    int unit_rows;
    MaskedWalk walk;             // of many rows
    CrossForwardPlan line;       // of few, whose tiles are shared as cross attention's are
    size_t part, stats, counts;  // scratch, in 4-byte words (counts, or the line's shares)
    size_t bytes() const { return 4 * (part + stats + counts); }
    int64_t blocks() const { return tiles ? walk.units * walk.parts : line.blocks; }
};

inline MaskedForwardPlan plan_masked_forward(int64_t batch, int64_t heads, int64_t kv_heads,
                                             int64_t seq_q, int64_t seq_k, int64_t d_head,
                                             int64_t cus) {
    const int64_t R = seq_q * (heads / kv_heads), items = batch * kv_heads;
    // (kFewRows is where cross attention's kernels are level, whose few rows' walk this is;
    // masked attention's own two were not timed against each other)
    MaskedForwardPlan p{R > kFewRows, 16, {}, {}, 0, 0, 0};
    if (items == 0 || R == 0) return p;
    if (!p.tiles) {
        p.line = plan_cross_forward(batch, heads, kv_heads, seq_q, seq_k, d_head, cus);
        // Up to 384 keys (six tiles to a wave) the join costs more than the shares save: 8
        // requests of 300 keys, 8 heads of 32, 15.7 us shared and 9.4 like this, one of 256
        // keys, 8 of 64, 14.5 and 11.0; 512 keys 14.7 and 16.6.
        if (seq_k <= 384 && p.line.groups > 0) {
            p.line.groups = 0;
            p.line.blocks = items * ((R + 15) / 16);
            p.line.part = p.line.stats = p.line.shares = 0;
        }
        p.unit_rows = p.line.unit_rows;
        p.part = p.line.part;
        p.stats = p.line.stats;
        p.counts = p.line.shares;
        return p;
    }
    // 256 rows to a workgroup when an unmasked call has 64 steps of such a one for every
    // compute unit, else 128
    const int64_t steps =
        items * ((R + 255) / 256) * ((seq_k * cross_tile_width((int)d_head) + 4095) / 4096);
    p.unit_rows = R > 128 && steps >= 64 * cus ? 256 : 128;
    const int64_t keys = cross_tile_keys((int)d_head, p.unit_rows / 32);
    const int64_t tiles = (seq_k + keys - 1) / keys;
    const int64_t at_once = p.unit_rows == 128 && d_head <= 96 ? 2 * cus : cus;
    p.walk.units = items * ((R + p.unit_rows - 1) / p.unit_rows);
    // The longest part is half a workgroup's even share of the tiles of an unmasked call (a
    // causal one has half as many), so that it ends no later than the others' sum; the
    // whole of it where units are more than the workgroups at once, as the longest begin
    // first (4 x 3000 rows, 8 heads of 64, 384 on 256: 227 us, by halves 245; but 2 x 2000, 8 of
    // 128, 256 on 256: 222 and 181); 1024 keys at least, which a join costs (4 x 1021, 16 of
    // 64, 512 units on 512: whole walks 80 us, by halves of 512 keys 86; where units are few,
    // nothing shorter was timed). At once are two workgroups to a compute unit, also up to
    // 32 columns, where three have room: by three 8000 rows, 8 heads of 32, take 222 us in place
    // of 261, but 4 x 3000 134 in place of 127.
    cut_walk(p.walk, tiles, p.walk.units * tiles / (p.walk.units > at_once ? at_once : 2 * at_once),
             1024 / keys);
    if (p.walk.parts > 1) {
        const int64_t rows = p.walk.parts * p.walk.units * p.unit_rows;
        p.part = (size_t)((rows * d_head + 3) / 4 * 4);
        p.stats = (size_t)(2 * rows);
        p.counts = (size_t)p.walk.units;
    }
    return p;
}

// Waves of a workgroup of the backward, 16 rows or keys each.
constexpr int masked_backward_waves(int D) { return D > 96 ? 8 : 4; }

struct MaskedBackwardPlan {
    MaskedWalk q, kv;
    int64_t row_tiles;  // tiles of rows that a walk of dk and dv meets, of an item
    // scratch, in 4-byte words: rows' log sums and deltas, queries' ranges, tiles' ends,
    // the gradients' parts and their counts
    size_t rows, ranges, ends, q_part, kv_part, counts;
    size_t bytes() const { return 4 * (rows + ranges + ends + q_part + 2 * kv_part + counts); }
};

inline MaskedBackwardPlan plan_masked_backward(int64_t batch, int64_t heads, int64_t kv_heads,
                                               int64_t seq_q, int64_t seq_k, int64_t d_head,
                                               int64_t cus) {
    const int64_t R = seq_q * (heads / kv_heads), items = batch * kv_heads;
    MaskedBackwardPlan p{};
    const int waves = masked_backward_waves((int)d_head);
    const int64_t tile = cross_tile_keys((int)d_head, waves), own = 16 * waves;
    // (two workgroups of four waves to a compute unit, also up to 64 columns, where three have
    // room: by three 2 x 3000 rows, 8 heads of 32, take 288 us in place of 276, 16384 rows of a
    // head of 64 1051 in place of 1086, 4 x 1021 of 16 the same 251)
    const int64_t at_once = waves == 8 ? cus : 2 * cus;
    p.row_tiles = (R + tile - 1) / tile;
    const int64_t key_tiles = (seq_k + tile - 1) / tile;
    p.rows = (size_t)((2 * items * R + 3) / 4 * 4);
    p.ranges = (size_t)(4 * batch * seq_q);
    p.ends = (size_t)(4 * batch * p.row_tiles);
    p.q.units = items * ((R + own - 1) / own);
    p.kv.units = items * ((seq_k + own - 1) / own);
    // A step of dq is three products a tile, one of dk and dv four. Asked for both
    // gradients or not, the plan is that of both: each has the same bits by itself.
    const int64_t even = (3 * p.q.units * key_tiles + 4 * p.kv.units * p.row_tiles) / at_once;
    cut_walk(p.q, key_tiles, even / 6, 8);
    cut_walk(p.kv, p.row_tiles, even / 8, 8);
    if (p.q.parts > 1) p.q_part = (size_t)((p.q.parts * items * R * d_head + 3) / 4 * 4);
    if (p.kv.parts > 1) p.kv_part = (size_t)((p.kv.parts * items * seq_k * d_head + 3) / 4 * 4);
    p.counts = (size_t)((p.q.units + p.kv.units + 3) / 4 * 4);
    return p;
}

}  // namespace nrs
