// Arguments and device helpers shared by the cross attention kernels
// (cross_attention.hip: few rows, joins and sums, entry points;
// cross_attention_tile.hip: many rows, the backward).
//
// The query heads of one key head are further rows of the same product: with
// group = heads / kv_heads, row r of an item (batch item, key head) is query
// r / group of head kv_head * group + r % group, R = seq_q * group rows in
// all. Keys past the item's length are never read.
#pragma once

#include "buffer_ops.hpp"
#include "fastdiv.hpp"

namespace nrs {

struct CrossArgs {
    const float *q, *k, *v, *dout, *o;
    float *out, *stats;  // stats: [batch][heads][seq_q][2], base-2 reference and sum
    float *dq, *dk, *dv;
    const int32_t* key_len;  // per batch item, null: all keys
    int B, H, KV, G, Sq, Sk, D, ld_q, ld_kv, ld_out;
    FastDiv by_group;     // division by G
    float scale, scale2;  // scale2 = scale * log2(e)
    float beta_q, beta_kv;
    // forward of many rows: workgroups that share an item's keys. Past 1,
    // `part` has [splits][items][R][D] sums, not yet divided, and part_stats
    // their reference and sum, [items][R][splits][2]
    int rows, splits;  // rows: of a workgroup
    // forward of few rows: workgroups that share the launch's key tiles, or 0.
    // Then `part` has [slots][min(R, 16)][D], part_stats [slots][min(R, 16)][2]
    // and `shares` the first and the last workgroup of each unit
    int groups;
    float* part;
    float* part_stats;
    int32_t* shares;
    // backward
    float *neg_lse, *neg_delta;  // [items][R]: -log2 sum 2^u and -dout . out
    int q_splits, kv_splits;     // workgroups that share a dq (dk and dv) tile's walk
    float *dq_part, *dk_part, *dv_part;  // [splits][items][rows][D] when shared
    int q_blocks;                // workgroups of the dq part of the launch
};

struct __attribute__((packed, aligned(4))) Quad {  // 128 bits at any float
    f32x4 v;
};

__device__ __forceinline__ int live_keys(const CrossArgs& a, int b) {
    return a.key_len ? max(0, min(a.key_len[b], a.Sk)) : a.Sk;
}

// Element offset of row r of (b, kv) in a tensor of queries.
__device__ __forceinline__ int64_t query_offset(const CrossArgs& a, int b, int kv, int r, int ld) {
    const int s = (int)fast_div((uint32_t)r, a.by_group);
    return ((int64_t)b * a.Sq + s) * ld + (int64_t)(kv * a.G + (r - s * a.G)) * a.D;
}

__device__ __forceinline__ int64_t key_offset(const CrossArgs& a, int b, int kv, int r) {
    return ((int64_t)b * a.Sk + r) * a.ld_kv + (int64_t)kv * a.D;
}

__device__ __forceinline__ float* row_stats(const CrossArgs& a, int b, int kv, int r) {
    const int s = (int)fast_div((uint32_t)r, a.by_group);
    return a.stats + (((int64_t)b * a.H + kv * a.G + (r - s * a.G)) * a.Sq + s) * 2;
}

// The kernels of cross_attention_tile.hip, and the sizes by which calls are
// planned. A workgroup of the forward owns 256 rows (8 waves) or 128 (4), one of
// the backward 128 rows or keys, two workgroups to a compute unit up to d_head
// 64: the time of one of 8 waves at 4 x 1000 x 1500 (16 heads of 64: 534 us,
// 553), and fewer idle waves where an item has few rows or keys.
constexpr int kCrossBackwardRows = 128;
constexpr int cross_tile_width(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
// Keys (or rows) that a workgroup of that many waves takes at a time.
constexpr int cross_tile_keys(int D, int waves) {
    return (waves == 8 || D > 64 ? 4096 : 2048) / cross_tile_width(D);
}
void cross_tile_forward(const CrossArgs& a);
void cross_tile_backward(const CrossArgs& a);

}  // namespace nrs
