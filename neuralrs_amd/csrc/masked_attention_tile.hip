// Masked attention of many rows, forward and backward, on the bf16 matrix cores: the
// tiles, products and softmax of cross_attention_tile.hip, over each row's own range of
// keys.
//
// A workgroup walks the tiles that any of its rows (or keys) sees, a wave leaves out
// those that none of its own does, and only tiles that some see in part pay for
// the comparison. Values that are not finite would reach rows that do not see them as
// 0 * NaN in the matrix products, so a row of a tile that holds one is staged as zeros
// and marked, and whoever sees it gets a NaN in place of the score.
//
// What bounds it is that a wave's steps (operands from LDS, matrix instructions,
// exponentials and splits) follow one another, and two waves to a SIMD hide a part of it: in
// the last three launches below matrix instructions run 55%, 47% and 63% of the time that a
// compute unit has work, vector instructions issue 43%, 40% and 38%, LDS is busy 25%, 38% and
// 28%. Splitting the met side costs 5 to 10% (measured by leaving it out), so tiles split
// beforehand would not pay for the pass that makes them.
//   32 x 128 rows, 8 heads of 32, causal       forward 10.5 us, backward 17.4 to 18.1
//   4 x 1021, 16 of 64, documents, bias        48 and 87: walks of 7 tiles, their beginnings
//   2 x 4000, 16 of 128 on 4, prefix, cap      769 (181 TFLOP/s of what is seen), backward 2682
//                                              (130; 181 with the two products it repeats)
//   8192, 32 of 128 on 8, causal, forward      2526 (217)
#include <algorithm>

#include "attention_tile.hpp"
#include "masked_attention.hpp"

namespace nrs {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A wave's issue priority while it feeds the matrix cores, over that of the other wave on
// its SIMD, which then takes the cycles between for its exponentials and splits (2 x 4000
// rows of 16 heads of 128, training: 4198 us -> 3931; a prompt of 8192 rows of 32 heads:
// 2818 -> 2730). ON: where that pays, not for heads up to 64 columns in the backward
// (4 x 1021 of 16: 273 us -> 282) or a wave alone (a prompt of 2000: 152 -> 160).
template <bool ON>
__device__ __forceinline__ void priority(int level) {
    if constexpr (ON) {
        if (level)
            __builtin_amdgcn_s_setprio(1);
        else
            __builtin_amdgcn_s_setprio(0);
    }
}

// The same in the backward. Up to 64 columns three waves share a SIMD, if the parts of a
// step keep their order: an operand that is asked for before its part has its turn would take
// the registers of the third (4 x 1021 rows of 16 heads of 64, both directions: two waves 267 us,
// three in any order 264 and, with documents and a bias, of which 50 registers spill, 160 for
// 146, three like this 254 and 138; with a cap 14 registers spill like this, 280 us, and two
// waves take 292, 16384 rows of one head 1218 and 1300).
template <int D>
__device__ __forceinline__ void phase(int level) {
    if constexpr (D > 64)
        priority<true>(level);
    else
        __builtin_amdgcn_sched_barrier(0);
}

// The least and the largest of 32 or 16 neighbouring lanes.
template <int LANES>
__device__ __forceinline__ int lanes_min(int x) {
#pragma unroll
    for (int i = 1; i < LANES; i *= 2) x = min(x, __shfl_xor(x, i, 64));
    return x;
}
template <int LANES>
__device__ __forceinline__ int lanes_max(int x) {
#pragma unroll
    for (int i = 1; i < LANES; i *= 2) x = max(x, __shfl_xor(x, i, 64));
    return x;
}

// The same in scalar registers: for all lanes alike.
__device__ __forceinline__ TileEnds uniform(TileEnds x) {
    return TileEnds{__builtin_amdgcn_readfirstlane(x.least), __builtin_amdgcn_readfirstlane(x.most),
                    __builtin_amdgcn_readfirstlane(x.from), __builtin_amdgcn_readfirstlane(x.to)};
}

// TileEnds of the ranges of a wave's rows, which every LANES of its lanes hold, LIVE of them rows.
template <int LANES>
__device__ __forceinline__ TileEnds ends_of(int lo, int hi, bool live) {
    const bool any = hi > lo;
    return uniform(TileEnds{lanes_min<LANES>(live && any ? lo : INT32_MAX),
                            lanes_max<LANES>(live && any ? hi : 0),
                            lanes_max<LANES>(!live ? 0 : any ? lo : INT32_MAX),
                            lanes_min<LANES>(!live ? INT32_MAX : any ? hi : 0)});
}

// A tile's way into LDS, with the rows of it that hold a NaN, an infinity or a magnitude
// of 2^127 and more as zeros and marked: mark[row] and mark[KT] are `stamp`.
template <class C, bool FULL>
__device__ __forceinline__ void store_marked(Stage<C, FULL>& x, const CrossArgs& a, u32x4* lds,
                                             int* mark, int stamp) {
#pragma unroll
    for (int u = 0; u < C::U; ++u) {
        const int i = threadIdx.x + C::NT * u, row = i / C::Q, q = i % C::Q;
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // (what follows the head in its row is not part of it)
            if (FULL || 4 * q + e % 4 + (e / 4) * (C::D / 2) < a.D)
                most = __builtin_elementwise_maximum(most, __builtin_fabsf(x.x[u][e / 4][e % 4]));
        }
        if (!(most < 0x1p127f)) {
            x.x[u][0] = x.x[u][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            mark[row] = mark[C::KT] = stamp;
        }
    }
    x.store(a, lds);
}

// Turns products into scores in base 2: those of the rows' 32 (or 2 x 4) places o(i)
// past `far`, the distance of place 0.
template <int MODE, int N, class V, class O>
__device__ __forceinline__ void add_bias(V& s, float far, float slope2, O o) {
    if (MODE == kPlain) return;
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = fmaf(-slope2, fabsf(far - (float)o(i)), s[i]);
}

__device__ __forceinline__ constexpr int place32(int i) { return 8 * (i / 4) + i % 4; }

// (narrow heads leave room for three: 2 x 1500 rows, 16 heads of 32, 51 us, with two 59; with
// 64 columns few calls have that many workgroups, and a wave has fewer registers: 8000
// rows of 2 heads 129 us, with two 143, but 4 x 1021 of 16 heads 81 and 78)
constexpr int forward_waves_per_simd(int D, int waves) {
    return D <= 32 && waves == 4 ? 3 : waves_per_simd(D, waves);
}

template <int D, int WAVES, bool FULL, int MODE>
__global__ __launch_bounds__(64 * WAVES, forward_waves_per_simd(D, WAVES)) void masked_tile_fwd_kernel(
    MaskedArgs a) {
    using C = TileCfg<D, WAVES>;
    __shared__ u32x4 lds[2][2 * C::SET];
    __shared__ int marks[2][C::KT + 1], ends[2][WAVES];
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the last rows of all items first, as causal walks of theirs are the longest
    const int R = a.Sq * a.G, items = a.B * a.KV, tiles = (R + 32 * WAVES - 1) / (32 * WAVES);
    const int no = a.parts - 1 - (int)(blockIdx.x / a.units), place = blockIdx.x % a.units;
    const int item = place % items, tile = tiles - 1 - place / items;
    const int b = item / a.KV, kv = item - b * a.KV, unit = item * tiles + tile;
    const int row = (tile * WAVES + w) * 32 + c;
    const bool live = row < R;
    const int s_row = live ? (int)fast_div((uint32_t)row, a.by_group) : 0;
    RowRange range = row_range(a, b, s_row);
    if (!live) range.lo = range.hi = range.at = 0;
    const TileEnds seen = ends_of<32>(range.lo, range.hi, live);
    if (lane == 0) {
        ends[0][w] = seen.least;
        ends[1][w] = seen.most;
    }
    for (int i = threadIdx.x; i < 2 * (C::KT + 1); i += C::NT) marks[0][i] = 0;
    __syncthreads();
    int least = INT32_MAX, most = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        least = min(least, ends[0][i]);
        most = max(most, ends[1][i]);
    }
    least = __builtin_amdgcn_readfirstlane(least);
    most = __builtin_amdgcn_readfirstlane(most);
    const int first = most > 0 ? least / C::KT : 0, last = (most + C::KT - 1) / C::KT;
    const int used = max(1, (last - first + a.part_tiles - 1) / a.part_tiles);
    if (no >= used) return;
    if (a.parts > 1 && no == 0 && threadIdx.x == 0) a.counts[unit] = used;
    const int t0 = first + no * a.part_tiles, t1 = min(last, t0 + a.part_tiles);

    Stage<C, FULL> k, v;
    auto load = [&](int t) {
        const int n = min(C::KT, most - t * C::KT);
        k.template load<false>(a, a.k, a.ld_kv, b, kv, t * C::KT, n);
        v.template load<false>(a, a.v, a.ld_kv, b, kv, t * C::KT, n);
    };
    // From the last tile down: in a causal call a row's nearest keys come first, whose
    // scores a bias by distance makes the largest, and the reference stays
    // near the maximum; from the first tile up, it lagged by up to 2^8, and the rounding
    // of scores that far above it cost 0.9e-6 of the result in place of 0.2e-6.
    auto store = [&](int t) {
        const int buf = (t1 - 1 - t) & 1;
        store_marked(k, a, lds[buf], marks[buf], t + 1);
        store_marked(v, a, lds[buf] + C::SET, marks[buf], t + 1);
    };
    if (t0 < t1) load(t1 - 1);
    const int s = live ? row - s_row * a.G : 0;
    const float slope2 = MODE != kPlain && a.slopes ? a.slopes[kv * a.G + s] * kLog2e : 0.0f;
    u32x4 qf[C::NS][3];
    own_pieces<C, FULL>(qf, a, a.q + (live ? query_offset(a, b, kv, row, a.ld_q) : 0), live, h,
                        a.scale_own);
    f32x16 acc[C::NJ];
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc[j] = all16(0.0f);
    float m = 0.0f, l = 0.0f;
    bool fresh = true;  // no key seen yet
    if (t0 < t1) {
        store(t1 - 1);
        if (t0 + 1 < t1) load(t1 - 2);
        __syncthreads();
    }
    for (int t = t1 - 1; t >= t0; --t) {
        const u32x4* const kl = lds[(t1 - 1 - t) & 1];
        const u32x4* const vl = kl + C::SET;
        const int* const mark = marks[(t1 - 1 - t) & 1];
        const int k0 = t * C::KT;
        if (k0 < seen.most && k0 + C::KT > seen.least) {
            f32x16 p[C::NB];
            priority<WAVES == 8>(1);
#pragma unroll
            for (int kb = 0; kb < C::NB; ++kb) {
                // (from zero, not from -m: 16 registers less, which wide heads spilled)
                p[kb] = products<C>(kl, qf, kb, all16(0.0f), c, h);
                if (MODE == kCap)
                    cap_scores<16>(p[kb], a.cap2, a.by_cap, m);
                else
                    p[kb] = p[kb] - m;
                if (MODE != kCap || a.slopes)
                    add_bias<MODE, 16>(p[kb], (float)(range.at - (k0 + kb * 32 + 4 * h)), slope2,
                                       place32);
            }
            priority<WAVES == 8>(0);
            if (__builtin_amdgcn_readfirstlane(mark[C::KT]) == t + 1) {
#pragma unroll
                for (int kb = 0; kb < C::NB; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (mark[kb * 32 + 4 * h + place32(i)] == t + 1) p[kb][i] = NAN;
            }
            if (k0 < seen.from || k0 + C::KT > seen.to) {
                const uint32_t span = range.hi - range.lo;
#pragma unroll
                for (int kb = 0; kb < C::NB; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t at = k0 + kb * 32 + 4 * h - range.lo + place32(i);
                        p[kb][i] = at < span ? p[kb][i] : -INFINITY;
                    }
            }
            float top = p[0][0];
#pragma unroll
            for (int kb = 0; kb < C::NB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, p[kb][i]);
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const bool begins = fresh && top > -INFINITY, moves = begins || top > 8.0f;
            if (__any(moves)) {
                const float shift = moves ? top : 0.0f;
                const float alpha = begins ? 0.0f : __builtin_amdgcn_exp2f(-shift);
                m += shift;
                l *= alpha;
                fresh = fresh && !begins;
#pragma unroll
                for (int kb = 0; kb < C::NB; ++kb) p[kb] = p[kb] - shift;
#pragma unroll
                for (int j = 0; j < C::NJ; ++j) acc[j] = acc[j] * alpha;
            }
#pragma unroll
            for (int kb = 0; kb < C::NB; ++kb)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] = __builtin_amdgcn_exp2f(p[kb][8 * u + i]);
                        l += x[i];
                    }
                    u32x4 pieces[3];
                    split8(x, pieces);
                    priority<WAVES == 8>(1);
                    add_transposed<C>(acc, vl, kb, u, pieces, lane);
                    priority<WAVES == 8>(0);
                }
        }
        if (t > t0) {
            // the other buffer was last read in step t + 1, which every wave
            // had left before the barrier that ended it
            store(t - 1);
            if (t - 1 > t0) load(t - 2);
            __syncthreads();
        }
    }
    l += __shfl_xor(l, 32, 64);
    if (!live) return;
    const bool whole = used == 1, none = l == 0.0f;
    const int64_t at = ((int64_t)no * a.units + unit) * (32 * WAVES) + w * 32 + c;
    store_own<C, FULL>(whole ? a.out + query_offset(a, b, kv, row, a.ld_out) : a.part + at * a.D,
                       acc, !whole ? 1.0f : none ? 0.0f : 1.0f / l, 0.0f, a.D, h);
    if (h == 0 && (!whole || a.stats)) {
        float* st = whole ? row_stats(a, b, kv, row) : a.part_stats + 2 * at;
        st[0] = !whole && none ? -INFINITY : m;  // (the join takes those for no part)
        st[1] = l;
    }
}

// What the backward starts from: per row -log2 of its sum of exponentials (-infinity
// where no key is seen) and -dout . out, D / 4 lanes to a row; by the workgroups
// behind those, the ranges of all queries and what the rows of each tile have in common,
// 32 lanes to a tile of TILE rows.
template <int D, int TILE>
__global__ __launch_bounds__(256) void masked_prepare_kernel(MaskedArgs a, int row_blocks) {
    constexpr int LANES = D / 4;
    const int R = a.Sq * a.G;
    if ((int)blockIdx.x < row_blocks) {
        const int x = threadIdx.x % LANES;
        const int64_t at = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
        if (at >= (int64_t)a.B * a.KV * R) return;
        const int item = (int)(at / R), r = (int)(at - (int64_t)item * R);
        const int b = item / a.KV, kv = item - b * a.KV;
        const int64_t off = query_offset(a, b, kv, r, a.ld_out) + 4 * x;
        float dot = 0.0f;
        if (4 * x + 4 <= a.D) {
            const f32x4 g = reinterpret_cast<const Quad*>(a.dout + off)->v,
                        o = reinterpret_cast<const Quad*>(a.o + off)->v;
#pragma unroll
            for (int e = 0; e < 4; ++e) dot = fmaf(g[e], o[e], dot);
        } else {
            for (int e = 0; 4 * x + e < a.D; ++e) dot = fmaf(a.dout[off + e], a.o[off + e], dot);
        }
#pragma unroll
        for (int i = 1; i < LANES; i *= 2) dot += __shfl_xor(dot, i, 64);
        if (x == 0) {
            const float* st = row_stats(a, b, kv, r);
            a.neg_lse[at] = st[1] == 0.0f ? -INFINITY : -(st[0] + __builtin_amdgcn_logf(st[1]));
            a.neg_delta[at] = -dot;
        }
        return;
    }
    const int64_t no = (int64_t)(blockIdx.x - row_blocks) * 8 + threadIdx.x / 32;
    if (no >= (int64_t)a.B * a.row_tiles) return;
    const int b = (int)(no / a.row_tiles), r0 = (int)(no - (int64_t)b * a.row_tiles) * TILE;
    const int s0 = (int)fast_div((uint32_t)r0, a.by_group),
              s1 = (int)fast_div((uint32_t)min(r0 + TILE, R) - 1, a.by_group);
    TileEnds all{INT32_MAX, 0, 0, INT32_MAX};
    for (int s = s0 + (threadIdx.x & 31); s <= s1; s += 32) {
        const RowRange range = row_range(a, b, s);
        const bool any = range.hi > range.lo;
        all.least = min(all.least, any ? range.lo : INT32_MAX);
        all.most = max(all.most, range.hi);
        all.from = max(all.from, any ? range.lo : INT32_MAX);
        all.to = min(all.to, range.hi);
        // (a query on the edge of two tiles is written by both, the same)
        a.ranges[(int64_t)b * a.Sq + s] = RowKeys{range.lo, range.hi, range.at, 0};
    }
    all = TileEnds{lanes_min<32>(all.least), lanes_max<32>(all.most), lanes_max<32>(all.from),
                   lanes_min<32>(all.to)};
    if ((threadIdx.x & 31) == 0) a.ends[no] = all;
}

// out = met . own^T of block kb of a tile, the small products of the pieces in a sum of
// their own: rounded as products16's closer form, which reads the large ones' operand a
// second time.
template <class C>
__device__ __forceinline__ void close16(f32x4 (&out)[2], const u32x4* set,
                                        const u32x4 (&own)[C::D / 32][3], int kb, int c, int g) {
    f32x4 small[2];
#pragma unroll
    for (int half = 0; half < 2; ++half)
        out[half] = small[half] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < C::D / 32; ++s) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            u32x4 met[3];
#pragma unroll
            for (int p = 0; p < 3; ++p) met[p] = piece16<C>(set, kb * 32 + 16 * half, s, p, c, g);
            f32x4& o = small[half];
            o = mfma16(met[2], own[s][0], o);
            o = mfma16(met[1], own[s][1], o);
            o = mfma16(met[0], own[s][2], o);
            o = mfma16(met[1], own[s][0], o);
            o = mfma16(met[0], own[s][1], o);
            out[half] = mfma16(met[0], own[s][0], out[half]);
        }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) out[half] = out[half] + small[half];
}

__device__ __forceinline__ constexpr int place16(int i) { return 16 * (i / 4) + i % 4; }

// dq of a workgroup's rows, 16 to a wave: P = 2^(score - lse), dS = P (v . dout - delta) and, with a
// cap, times 1 - tanh^2; dQ = scale * K^T dS.
template <int D, int WAVES, bool FULL, int MODE>
__device__ __forceinline__ void masked_dq_walk(const MaskedArgs& a, u32x4* lds, int (*marks)[TileCfg<D, WAVES>::KT + 1],
                                               int (*shared_ends)[WAVES], int block) {
    using C = TileCfg<D, WAVES>;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Sq * a.G, tiles = (R + 16 * WAVES - 1) / (16 * WAVES), items = a.B * a.KV;
    const int no = a.q_parts - 1 - block / a.q_units, place = block % a.q_units;
    const int item = place % items, tile = tiles - 1 - place / items;
    const int b = item / a.KV, kv = item - b * a.KV, unit = item * tiles + tile;
    const int row = (tile * WAVES + w) * 16 + c;
    const bool live = row < R;
    const int s_row = live ? (int)fast_div((uint32_t)row, a.by_group) : 0;
    RowKeys range = a.ranges[(int64_t)b * a.Sq + s_row];
    if (!live) range = RowKeys{0, 0, 0, 0};
    const TileEnds seen = ends_of<16>(range.lo, range.hi, live);
    if (lane == 0) {
        shared_ends[0][w] = seen.least;
        shared_ends[1][w] = seen.most;
    }
    __syncthreads();
    int least = INT32_MAX, most = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        least = min(least, shared_ends[0][i]);
        most = max(most, shared_ends[1][i]);
    }
    least = __builtin_amdgcn_readfirstlane(least);
    most = __builtin_amdgcn_readfirstlane(most);
    const int first = most > 0 ? least / C::KT : 0, last = (most + C::KT - 1) / C::KT;
    const int used = max(1, (last - first + a.q_part_tiles - 1) / a.q_part_tiles);
    if (no >= used) return;
    if (a.q_parts > 1 && no == 0 && threadIdx.x == 0) a.q_counts[unit] = used;
    const int t0 = first + no * a.q_part_tiles, t1 = min(last, t0 + a.q_part_tiles);
    Stage<C, FULL> k, v;
    auto load = [&](int t) {
        const int n = min(C::KT, most - t * C::KT);
        k.template load<false>(a, a.k, a.ld_kv, b, kv, t * C::KT, n);
        v.template load<false>(a, a.v, a.ld_kv, b, kv, t * C::KT, n);
    };
    auto store = [&](int t) {
        const int buf = (t - t0) & 1;
        store_marked(k, a, lds + buf * 2 * C::SET, marks[buf], t + 1);
        store_marked(v, a, lds + buf * 2 * C::SET + C::SET, marks[buf], t + 1);
    };
    if (t0 < t1) load(t0);
    const float slope2 =
        MODE != kPlain && a.slopes && live ? a.slopes[kv * a.G + row - s_row * a.G] * kLog2e : 0.0f;
    u32x4 qf[D / 32][3], gf[D / 32][3];
    own16<C, FULL>(qf, a, a.q + (live ? query_offset(a, b, kv, row, a.ld_q) : 0), live, g,
                   a.scale_own);
    own16<C, FULL>(gf, a, a.dout + (live ? query_offset(a, b, kv, row, a.ld_out) : 0), live, g, 1.0f);
    const float nl = live ? a.neg_lse[(int64_t)item * R + row] : -INFINITY;
    const float nd = live ? a.neg_delta[(int64_t)item * R + row] : 0.0f;
    f32x4 acc[D / 16];
#pragma unroll
    for (int j = 0; j < D / 16; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (t0 < t1) {
        store(t0);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        const u32x4* const kl = lds + ((t - t0) & 1) * 2 * C::SET;
        const int* const mark = marks[(t - t0) & 1];
        const bool marked = __builtin_amdgcn_readfirstlane(mark[C::KT]) == t + 1;
#pragma unroll
        for (int kb = 0; kb < C::NB; ++kb) {
            const int k0 = t * C::KT + kb * 32;
            if (k0 >= seen.most || k0 + 32 <= seen.least) continue;
            f32x4 s[2], dp[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) dp[half] = f32x4{nd, nd, nd, nd};
            phase<D>(1);
            close16<C>(s, kl, qf, kb, c, g);
            products16<C, false>(dp, kl + C::SET, gf, kb, c, g);
            phase<D>(0);
            float x[8], y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = s[i / 4][i % 4];
                y[i] = dp[i / 4][i % 4];
            }
            if (MODE == kCap) cap_scores_and_slopes(x, y, a.cap2, a.by_cap);
            if (MODE != kCap || a.slopes)
                add_bias<MODE, 8>(x, (float)(range.at - (k0 + 4 * g)), slope2, place16);
            if (marked) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (mark[kb * 32 + 4 * g + place16(i)] == t + 1) x[i] = NAN;
            }
            if (k0 < seen.from || k0 + 32 > seen.to) {
                // (both: a hidden value may be as large as to make its product infinite)
                const uint32_t span = range.hi - range.lo;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool sees = k0 + 4 * g - range.lo + place16(i) < span;
                    x[i] = sees ? x[i] : -INFINITY;
                    y[i] = sees ? y[i] : 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(x[i] + nl) * y[i];
            u32x4 p[3];
            split8(x, p);
            phase<D>(1);
            add16<C>(acc, kl, kb, p, lane);
            phase<D>(0);
        }
        if (t + 1 < t1) {
            store(t + 1);
            if (t + 2 < t1) load(t + 2);
            __syncthreads();
        }
    }
    if (!live) return;
    if (used > 1)
        store16<C, FULL>(a.dq_part + (((int64_t)no * items + item) * R + row) * a.D, acc, 1.0f, 0.0f,
                         a.D, g);
    else
        store16<C, FULL>(a.dq + query_offset(a, b, kv, row, a.ld_q), acc, a.scale, a.beta_q, a.D, g);
}

// dk and dv of a workgroup's keys, 16 to a wave: the same P and dS with the rows met, dV = dO^T P,
// dK = scale * Q^T dS.
template <int D, int WAVES, bool FULL, int MODE>
__device__ __forceinline__ void masked_dkv_walk(const MaskedArgs& a, u32x4* lds, int (*marks)[TileCfg<D, WAVES>::KT + 1],
                                                f32x4* starts, int (*shared_ends)[WAVES], int block) {
    using C = TileCfg<D, WAVES>;
    constexpr int ROWS = MODE == kPlain ? 4 : 6;  // -lse, -delta, lo, keys; place, slope
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Sq * a.G, tiles = (a.Sk + 16 * WAVES - 1) / (16 * WAVES), items = a.B * a.KV;
    const int no = a.parts - 1 - block / a.units, place = block % a.units;
    const int item = place % items, tile = place / items;
    const int b = item / a.KV, kv = item - b * a.KV, unit = item * tiles + tile;
    const int key0 = (tile * WAVES + w) * 16, key = key0 + c;
    // the tiles of rows of which any sees a key of the workgroup
    const TileEnds* const ends = a.ends + (int64_t)b * a.row_tiles;
    int first = INT32_MAX, last = 0;
    for (int t = threadIdx.x; t < a.row_tiles; t += C::NT)
        if (ends[t].least < (tile + 1) * 16 * WAVES && ends[t].most > tile * 16 * WAVES) {
            first = min(first, t);
            last = t + 1;
        }
    first = lanes_min<64>(first);
    last = lanes_max<64>(last);
    if (lane == 0) {
        shared_ends[0][w] = first;
        shared_ends[1][w] = last;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        first = min(first, shared_ends[0][i]);
        last = max(last, shared_ends[1][i]);
    }
    first = __builtin_amdgcn_readfirstlane(min(first, last));
    last = __builtin_amdgcn_readfirstlane(last);
    const int used = max(1, (last - first + a.part_tiles - 1) / a.part_tiles);
    if (no >= used) return;
    if (a.parts > 1 && no == 0 && threadIdx.x == 0) a.counts[unit] = used;
    const int t0 = first + no * a.part_tiles, t1 = min(last, t0 + a.part_tiles);
    // (keys past the item's length are never read)
    const bool live = key < live_keys(a, b) && t0 < t1;
    Stage<C, FULL> q, go;
    float start[2], slope = 0.0f;  // of threads below KT: of a row of the tile
    RowKeys range;
    TileEnds next;
    auto load = [&](int t) {
        const int r0 = t * C::KT, n = min(C::KT, R - r0);
        q.template load<true>(a, a.q, a.ld_q, b, kv, r0, n);
        go.template load<true>(a, a.dout, a.ld_out, b, kv, r0, n);
        start[0] = -INFINITY;
        start[1] = 0.0f;
        range = RowKeys{0, 0, 0, 0};
        if ((int)threadIdx.x < n) {
            const int r = r0 + threadIdx.x, s = (int)fast_div((uint32_t)r, a.by_group);
            start[0] = a.neg_lse[(int64_t)item * R + r];
            start[1] = a.neg_delta[(int64_t)item * R + r];
            range = a.ranges[(int64_t)b * a.Sq + s];
            if (MODE != kPlain && a.slopes) slope = a.slopes[kv * a.G + r - s * a.G];
        }
        next = ends[t];
    };
    auto store = [&](int t) {
        const int buf = (t - t0) & 1;
        store_marked(q, a, lds + buf * 2 * C::SET, marks[buf], t + 1);
        store_marked(go, a, lds + buf * 2 * C::SET + C::SET, marks[buf], t + 1);
        if ((int)threadIdx.x < C::KT) {
            float* const to = reinterpret_cast<float*>(starts) + buf * ROWS * C::KT + threadIdx.x;
            to[0] = start[0];
            to[C::KT] = start[1];
            to[2 * C::KT] = __builtin_bit_cast(float, range.lo);
            to[3 * C::KT] = __builtin_bit_cast(float, range.hi - range.lo);
            if (MODE != kPlain) {
                to[4 * C::KT] = (float)(range.at - tile * 16 * WAVES);
                to[5 * C::KT] = slope * kLog2e;
            }
        }
    };
    if (t0 < t1) load(t0);
    u32x4 kf[D / 32][3], vf[D / 32][3];
    own16<C, FULL>(kf, a, a.k + (live ? key_offset(a, b, kv, key) : 0), live, g, a.scale_own);
    own16<C, FULL>(vf, a, a.v + (live ? key_offset(a, b, kv, key) : 0), live, g, 1.0f);
    f32x4 acc_k[D / 16], acc_v[D / 16];
#pragma unroll
    for (int j = 0; j < D / 16; ++j) acc_k[j] = acc_v[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    TileEnds seen{};
    if (t0 < t1) {
        seen = uniform(next);
        store(t0);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        const u32x4* const ql = lds + buf * 2 * C::SET;
        const int* const mark = marks[buf];
        if (seen.least < key0 + 16 && seen.most > key0) {
            const bool marked = __builtin_amdgcn_readfirstlane(mark[C::KT]) == t + 1;
            const bool part = key0 < seen.from || key0 + 16 > seen.to;
#pragma unroll
            for (int rb = 0; rb < C::NB; ++rb) {
                const f32x4* const st = starts + (buf * ROWS * C::KT + rb * 32) / 4 + g;
                f32x4 s[2], dp[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) dp[half] = st[C::KT / 4 + 4 * half];
                phase<D>(1);
                close16<C>(s, ql, kf, rb, c, g);
                products16<C, false>(dp, ql + C::SET, vf, rb, c, g);
                phase<D>(0);
                float x[8], y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = s[i / 4][i % 4];
                    y[i] = dp[i / 4][i % 4];
                }
                if (MODE == kCap) cap_scores_and_slopes(x, y, a.cap2, a.by_cap);
                if (MODE == kBias || (MODE == kCap && a.slopes)) {
                    const float place_key = (float)(key - tile * 16 * WAVES);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const f32x4 at = st[4 * C::KT / 4 + 4 * half], by = st[5 * C::KT / 4 + 4 * half];
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            x[4 * half + r] = fmaf(-by[r], fabsf(at[r] - place_key), x[4 * half + r]);
                    }
                }
                if (marked) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (mark[rb * 32 + 4 * g + place16(i)] == t + 1) x[i] = NAN;
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const f32x4 nl = st[4 * half];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = 4 * half + r;
                        x[i] = __builtin_amdgcn_exp2f(x[i] + nl[r]);
                        y[i] *= x[i];
                    }
                }
                if (part) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const i32x4 lo = __builtin_bit_cast(i32x4, st[2 * C::KT / 4 + 4 * half]);
                        const u32x4 span = __builtin_bit_cast(u32x4, st[3 * C::KT / 4 + 4 * half]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int i = 4 * half + r;
                            const bool sees = (uint32_t)(key - lo[r]) < span[r];
                            x[i] = sees ? x[i] : 0.0f;
                            y[i] = sees ? y[i] : 0.0f;
                        }
                    }
                }
                u32x4 p[3];
                split8(x, p);
                phase<D>(1);
                add16<C>(acc_v, ql + C::SET, rb, p, lane);
                phase<D>(0);
                split8(y, p);
                phase<D>(1);
                add16<C>(acc_k, ql, rb, p, lane);
                phase<D>(0);
            }
        }
        if (t + 1 < t1) {
            seen = uniform(next);
            store(t + 1);
            if (t + 2 < t1) load(t + 2);
            __syncthreads();
        }
    }
    if (key >= a.Sk) return;
    if (used > 1) {
        const int64_t at = (((int64_t)no * items + item) * a.Sk + key) * a.D;
        store16<C, FULL>(a.dk_part + at, acc_k, 1.0f, 0.0f, a.D, g);
        store16<C, FULL>(a.dv_part + at, acc_v, 1.0f, 0.0f, a.D, g);
        return;
    }
    if (t0 >= t1 && a.beta_kv == 1.0f) return;
    const int64_t at = key_offset(a, b, kv, key);
    store16<C, FULL>(a.dk + at, acc_k, a.scale, a.beta_kv, a.D, g);
    store16<C, FULL>(a.dv + at, acc_v, 1.0f, a.beta_kv, a.D, g);
}

// One launch for both: they need nothing of each other, and the workgroups of one fill
// the compute units that the other leaves idle (the longer walks begin first).
template <int D, int WAVES, bool FULL, int MODE>
__global__ __launch_bounds__(64 * WAVES, D <= 64 ? 3 : 2) void masked_tile_bwd_kernel(MaskedArgs a) {
    using C = TileCfg<D, WAVES>;
    __shared__ u32x4 lds[4 * C::SET];
    __shared__ f32x4 starts[2 * (MODE == kPlain ? 4 : 6) * C::KT / 4];
    __shared__ int marks[2][C::KT + 1], ends[2][WAVES];
    for (int i = threadIdx.x; i < 2 * (C::KT + 1); i += C::NT) marks[0][i] = 0;
    const int kv_blocks = gridDim.x - a.q_blocks;
    if ((int)blockIdx.x >= kv_blocks)
        masked_dq_walk<D, WAVES, FULL, MODE>(a, lds, marks, ends, blockIdx.x - kv_blocks);
    else
        masked_dkv_walk<D, WAVES, FULL, MODE>(a, lds, marks, starts, ends, blockIdx.x);
}

int mode_of(const MaskedArgs& a) { return a.cap2 > 0.0f ? kCap : a.slopes ? kBias : kPlain; }

template <int D, int WAVES, int MODE>
void launch_forward(const MaskedArgs& a, unsigned blocks) {
    auto kernel = a.D == D ? masked_tile_fwd_kernel<D, WAVES, true, MODE>
                           : masked_tile_fwd_kernel<D, WAVES, false, MODE>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * WAVES), 0, stream(), a);
}

template <int D, int MODE>
void launch_backward(const MaskedArgs& a, unsigned blocks) {
    constexpr int WAVES = masked_backward_waves(D);
    auto kernel = a.D == D ? masked_tile_bwd_kernel<D, WAVES, true, MODE>
                           : masked_tile_bwd_kernel<D, WAVES, false, MODE>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * WAVES), 0, stream(), a);
}

template <int D>
void forward(const MaskedArgs& a, unsigned blocks) {
    const int mode = mode_of(a);
    if (a.unit_rows == 256)
        (mode == kCap    ? launch_forward<D, 8, kCap>
         : mode == kBias ? launch_forward<D, 8, kBias>
                         : launch_forward<D, 8, kPlain>)(a, blocks);
    else
        (mode == kCap    ? launch_forward<D, 4, kCap>
         : mode == kBias ? launch_forward<D, 4, kBias>
                         : launch_forward<D, 4, kPlain>)(a, blocks);
}

template <int D>
void backward(MaskedArgs a) {
    const int64_t rows = (int64_t)a.B * a.KV * a.Sq * a.G;
    if (rows > 0) {
        constexpr int WIDE = cross_row_width(D), PER = 1024 / WIDE;
        const int64_t row_blocks = (rows + PER - 1) / PER,
                      end_blocks = ((int64_t)a.B * a.row_tiles + 7) / 8;
        hipLaunchKernelGGL((masked_prepare_kernel<WIDE, TileCfg<D, masked_backward_waves(D)>::KT>),
                           dim3((unsigned)(row_blocks + end_blocks)), dim3(256), 0, stream(), a,
                           (int)row_blocks);
    }
    const int64_t q_blocks = a.dq ? (int64_t)a.q_units * a.q_parts : 0;
    const int64_t kv_blocks = a.dk ? (int64_t)a.units * a.parts : 0;
    const int mode = mode_of(a);
    auto launch = [&](int64_t q, int64_t kv) {
        a.q_blocks = (int)q;
        if (q + kv > 0)
            (mode == kCap    ? launch_backward<D, kCap>
             : mode == kBias ? launch_backward<D, kBias>
                             : launch_backward<D, kPlain>)(a, (unsigned)(q + kv));
    };
    if (q_blocks + kv_blocks < (1 << 23)) {
        launch(q_blocks, kv_blocks);
    } else {  // a launch has fewer than 2^32 threads
        launch(0, kv_blocks);
        launch(q_blocks, 0);
    }
}

}  // namespace

void masked_tile_forward(const MaskedArgs& a, unsigned blocks) {
    (a.D <= 32   ? forward<32>
     : a.D <= 64 ? forward<64>
     : a.D <= 96 ? forward<96>
                 : forward<128>)(a, blocks);
}

void masked_tile_backward(const MaskedArgs& a) {
    (a.D <= 32   ? backward<32>
     : a.D <= 64 ? backward<64>
     : a.D <= 96 ? backward<96>
                 : backward<128>)(a);
}

}  // namespace nrs
