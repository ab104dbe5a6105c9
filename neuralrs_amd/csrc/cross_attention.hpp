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
#include "cross_attention_plan.hpp"
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
    // The forward. A unit is `unit_rows` rows of an item (16, or a workgroup's of
    // the kernel of many rows), the last one of an item maybe fewer. With
    // `groups` 0 a workgroup takes a unit; else the key tiles of all units lie
    // one after the other, and `groups` workgroups take equal parts of that
    // line, whatever the items' lengths. A unit that a part begins or ends in
    // leaves sums, not yet divided, in a slot of `part` [slots][unit_rows][D],
    // with their reference and sum in part_stats [slots][unit_rows][2]; `shares`
    // has the first and the last workgroup of each unit. A workgroup goes on with
    // an earlier one's unit once at most, in slot `workgroup`, and leaves a unit
    // that it began to a later one once at most, in slot groups + workgroup, or
    // groups + unit where there are fewer units.
    int unit_rows, groups;
    bool few_units;  // fewer than workgroups
    float* part;
    float* part_stats;
    int32_t* shares;
    // backward
    float *neg_lse, *neg_delta;  // [items][R]: -log2 sum 2^u and -dout . out
    int q_splits, kv_splits;     // workgroups that share a dq (dk and dv) tile's walk
    float *dq_part, *dk_part, *dv_part;  // [splits][items][rows][D] when shared
    int q_blocks;                // workgroups of the dq part of the launch
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

// The slot of the sums of a unit that workgroup `first` began and left.
__device__ __forceinline__ int begun_slot(const CrossArgs& a, int unit, int first) {
    return a.groups + (a.few_units ? unit : first);
}

// A workgroup's part of the line of key tiles: an unbroken run of (unit, tiles)
// pieces. `per_item` units to a batch item, tiles of `keys` keys.
template <int NT>
struct LinePart {
    int b, base, p, end, per_item, keys;
    // of the piece at hand:
    int sub, L, t0, t1, tiles;

    // False if the part is empty. All NT threads call it; `scan` and `found` are
    // shared memory. A scan of the items' lengths finds where each begins on
    // the line, and the item of the part's first tile.
    __device__ __forceinline__ bool begin(const CrossArgs& a, int per_item_, int keys_,
                                          int (&scan)[NT / 64], int (&found)[2]) {
        per_item = per_item_;
        keys = keys_;
        const int t = threadIdx.x, lane = t & 63, w = t >> 6, each = (a.B + NT - 1) / NT;
        int own = 0;
        for (int i = 0; i < each; ++i)
            if (t * each + i < a.B) own += (live_keys(a, t * each + i) + keys - 1) / keys * per_item;
        int upto = own;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int v = __shfl_up(upto, d, 64);
            if (lane >= d) upto += v;
        }
        if (lane == 63) scan[w] = upto;
        __syncthreads();
        int at = upto - own, total = 0;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) {
            at += i < w ? scan[i] : 0;
            total += scan[i];
        }
        // a tile to a workgroup at least: those that share a unit, which the join
        // takes from the first to the last, have none without a part between them
        const int parts = min(a.groups, total);
        if ((int)blockIdx.x >= parts) return false;
        p = (int)((int64_t)total * blockIdx.x / parts);
        end = (int)((int64_t)total * (blockIdx.x + 1) / parts);
        for (int i = 0; i < each && t * each + i < a.B; ++i) {
            const int n = (live_keys(a, t * each + i) + keys - 1) / keys * per_item;
            if (at <= p && p < at + n) {
                found[0] = t * each + i;
                found[1] = at;
            }
            at += n;
        }
        __syncthreads();
        b = found[0];
        base = found[1];
        return true;
    }
    // The next piece, if any: tiles t0 .. t1 - 1 of unit b * per_item + sub.
    __device__ __forceinline__ bool next(const CrossArgs& a) {
        if (p >= end) return false;
        for (;;) {  // (items without keys have no tiles)
            L = live_keys(a, b);
            tiles = (L + keys - 1) / keys;
            if (p < base + tiles * per_item) break;
            base += tiles * per_item;
            ++b;
        }
        sub = (p - base) / tiles;
        t0 = p - base - sub * tiles;
        t1 = min(tiles, t0 + end - p);
        p += t1 - t0;
        const int unit = b * per_item + sub;
        if (threadIdx.x == 0) {
            if (t0 == 0) a.shares[2 * unit] = blockIdx.x;
            if (t1 == tiles) a.shares[2 * unit + 1] = blockIdx.x;
        }
        return true;
    }
    // Where the piece's sums go: -1 if it is all of its unit.
    __device__ __forceinline__ int64_t slot(const CrossArgs& a) const {
        if (t0 > 0) return blockIdx.x;
        return t1 == tiles ? -1 : begun_slot(a, b * per_item + sub, blockIdx.x);
    }
};

// The kernels of cross_attention_tile.hip.
void cross_tile_forward(const CrossArgs& a, unsigned blocks);
// The rows' statistics, then (unless only they are wanted) what is asked for of
// dq and dk, dv.
void cross_tile_backward(const CrossArgs& a, bool only_rows);

}  // namespace nrs
