// Which kernels take a cross attention call, how its work is shared among
// workgroups, and the scratch that this needs. Host only and free of HIP, so that a
// CPU test can ask.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace nrs {

constexpr int kRowWaves = 4;  // waves of a workgroup of the kernels of few rows and of a short side
constexpr int kMaxSharedBatch = 1024;  // batch items of a shared launch

// A workgroup of the many rows' forward owns 256 rows (8 waves) or 128 (4), one of
// the backward 128 rows or keys: 32 to a wave up to d_head 32, else 16.
constexpr int kCrossBackwardRows = 128;
// Columns of a tile: a multiple of 32, and 96 for those in between (2 x 1037 rows,
// 2506 keys, 2 heads of 96: backward 153 us, in tiles of 128 columns 229).
constexpr int cross_tile_width(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }
// A quarter as many threads share a row in the kernels that go by rows.
constexpr int cross_row_width(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
// Keys (or rows) that a workgroup of that many waves takes at a time.
constexpr int cross_tile_keys(int D, int waves) {
    return (waves == 8 || D > 64 ? 4096 : 2048) / cross_tile_width(D) / 32 * 32;
}

struct CrossForwardPlan {
    bool tiles;      // the kernel of many rows
    bool few_keys;   // the kernel of many rows over up to 16 keys
    int unit_rows;   // of a unit (the scratch of a call with fewer holds no more)
    int groups;      // workgroups that share all units, 0: one each
    bool few_units;  // fewer than those workgroups
    int64_t blocks;  // workgroups of the launch
    size_t part, stats, shares;  // scratch, in 4-byte words
    size_t bytes() const { return 4 * (part + stats + shares); }
};

// Rows of an item up to which the kernel of few rows takes the call. Against the
// kernel of many rows: 32 rows, 16384 keys (16 items of 128) 83 us and 100, 33 rows
// 122 and 104; but 1500 keys (256 items of 64) are level at 16 rows (45 and 51; 24
// rows 74 and 51), and 200 keys (256 items of 32) before 8 (16 and 10).
constexpr int64_t kFewRows = 32;

// The scratch does not depend on key_len being there; the kernels read it.
inline CrossForwardPlan plan_cross_forward(int64_t batch, int64_t heads, int64_t kv_heads,
                                           int64_t seq_q, int64_t seq_k, int64_t d_head,
                                           int64_t cus) {
    const int64_t R = seq_q * (heads / kv_heads), items = batch * kv_heads;
    CrossForwardPlan p{R > kFewRows && seq_k > 16, R > kFewRows && seq_k <= 16, 16, 0, false, 0, 0, 0, 0};
    if (items == 0 || R == 0) return p;
    if (p.few_keys) {
        // four workgroups to a compute unit, a tile of 16 rows to a wave at least
        p.blocks = items * std::max<int64_t>(
            1, std::min<int64_t>(4 * cus / items, (R + 15) / 16 / kRowWaves));
        return p;
    }
    int64_t units, groups, tiles;
    bool share;
    if (!p.tiles) {
        units = items * ((R + 15) / 16);
        tiles = (seq_k + 15) / 16;
        // Shared unless there are enough units by themselves; at least two
        // tiles of 16 keys to a wave. Workgroups to a compute unit
        // by the bytes that each has on the way (a tile of K and V to a wave):
        // 1, 2 and 4 of them take 47, 48 and 51 us at d_head 128 (2 x 16384
        // keys, 8 key heads) and 38, 30 and 26 us, 3 26 us, at d_head 64 (32
        // items of up to 1500 keys, 8 key heads).
        groups = std::min<int64_t>((d_head > 64 ? 1 : d_head > 32 ? 3 : 6) * cus,
                                   units * tiles / (2 * kRowWaves));
        share = groups > units;
        p.unit_rows = (int)std::min<int64_t>(R, 16);
    } else {
        // 256 rows to a workgroup when the call has eight steps of such a one
        // for every compute unit, else 128: 7 x 266 x 425, 8 heads of 128
        // (6 steps), 65 us with 256 and 53 with 128; 4 x 512 x 1500, 16 heads of
        // 64 (12), 86 and 101
        const int width = cross_tile_width((int)d_head);
        const int64_t steps = items * ((R + 255) / 256) * ((seq_k * width + 4095) / 4096);
        p.unit_rows = R > 128 && steps >= 8 * cus ? 256 : 128;
        units = items * ((R + p.unit_rows - 1) / p.unit_rows);
        const int64_t keys = cross_tile_keys((int)d_head, p.unit_rows / 32);
        tiles = (seq_k + keys - 1) / keys;
        // Workgroups at once, and the time of the fullest one in key tiles: a
        // piece's beginning and end cost two tiles, a join four.
        const int64_t at_once = p.unit_rows == 128 && d_head <= 96 ? 2 * cus : cus;
        groups = std::min<int64_t>(at_once, units * tiles / 2);
        share = groups > 1 && (units + at_once - 1) / at_once * (tiles + 2) >
                                  (units * (tiles + 2) + groups - 1) / groups + 8;
    }
    p.blocks = units;
    // (places on the line are 32-bit numbers)
    if (share && batch <= kMaxSharedBatch && units * tiles <= INT32_MAX) {
        p.groups = (int)groups;
        p.few_units = units < groups;
        p.blocks = groups;
        const int64_t slots = (groups + std::min(groups, units)) * p.unit_rows;
        p.part = (size_t)((slots * d_head + 3) / 4 * 4);
        p.stats = (size_t)((2 * slots + 3) / 4 * 4);
        p.shares = (size_t)(2 * units);
    }
    return p;
}

// Rows or keys of an item up to which the backward's kernel of a short side takes
// the call, against the kernel of many: 35 rows, 5256 keys (256 items of 128)
// 1140 us and 2255; 33 keys, 4067 rows (32 items of 98) 177 and 283; but 64 keys,
// 1000 rows (64 items of 64) 81 and 55, 64 rows, 1500 keys 88 and 62.
constexpr int64_t kShort = 48;

struct CrossBackwardPlan {
    int q_splits, kv_splits;
    int64_t rows, keys;  // of all items
    bool short_rows, short_keys;  // the kernel of a short side
    size_t prepared, q_part, kv_part;  // floats of each kind of scratch
    size_t bytes() const { return sizeof(float) * (prepared + q_part + 2 * kv_part); }
};

// A workgroup to a compute unit: a walk that is longer than half a compute
// unit's even part of all the work is shared out, one of dq, which begin last,
// than a quarter, so that the last walks to end leave less idle (2 x 777 rows of
// 16 heads, 4096 keys and fewer, 4 key heads of 128: 1042 us with both by halves,
// 1000 like this; whole walks took 8% longer than halves). A step of dq is three
// products a tile, one of dk and dv four. Asked for both gradients or not, the plan
// is that of both: each has the same bits by itself.
inline CrossBackwardPlan plan_cross_backward(int64_t batch, int64_t heads, int64_t kv_heads,
                                             int64_t seq_q, int64_t seq_k, int64_t d_head,
                                             int64_t cus) {
    const int64_t R = seq_q * (heads / kv_heads), items = batch * kv_heads;
    CrossBackwardPlan p{1, 1, items * R, items * seq_k, false, false, 0, 0, 0};
    p.prepared = (size_t)((2 * p.rows + 3) / 4 * 4);  // needed without keys, too
    if (p.rows == 0 || p.keys == 0) return p;
    const int64_t tile = cross_tile_keys((int)d_head, d_head > 32 ? 8 : 4), own = kCrossBackwardRows;
    const int64_t q_len = (seq_k + tile - 1) / tile, kv_len = (R + tile - 1) / tile;
    const int64_t q_groups = items * ((R + own - 1) / own),
                  kv_groups = items * ((seq_k + own - 1) / own);
    const int64_t even = std::max<int64_t>(16, (3 * q_groups * q_len + 4 * kv_groups * kv_len) / (2 * cus));
    auto shares = [](int64_t cost, int64_t len, int64_t part) {
        return (int)std::max<int64_t>(1, std::min<int64_t>({(cost + part - 1) / part, len, 64}));
    };
    p.q_splits = shares(3 * q_len, q_len, std::max<int64_t>(16, even / 2));
    p.kv_splits = shares(4 * kv_len, kv_len, even);
    p.short_rows = R <= kShort;
    p.short_keys = !p.short_rows && seq_k <= kShort;
    if (p.short_rows || p.short_keys) {
        // three workgroups to a compute unit, two tiles of 16 to a wave at least
        const int64_t tiles = ((p.short_rows ? seq_k : R) + 15) / 16;
        const int splits = (int)std::max<int64_t>(
            1, std::min<int64_t>({3 * cus / items, tiles / (2 * kRowWaves), 64}));
        p.q_splits = p.short_rows ? splits : 1;
        p.kv_splits = p.short_keys ? splits : 1;
    }
    if (p.q_splits > 1) p.q_part = (size_t)((p.q_splits * p.rows * d_head + 3) / 4 * 4);
    if (p.kv_splits > 1) p.kv_part = (size_t)((p.kv_splits * p.keys * d_head + 3) / 4 * 4);
    return p;
}

}  // namespace nrs
