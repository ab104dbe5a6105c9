// Arguments and device helpers shared by the masked attention kernels
// (masked_attention.hip: few rows, joins and sums, entry points;
// masked_attention_tile.hip: many rows, the backward).
//
// Rows are those of cross_attention.hpp: row r of an item (batch item, key head) is
// query r / group of head kv_head * group + r % group. Every row sees an unbroken
// range of its item's keys: causal, prefix, document and length masks are one each,
// and so is what they have in common.
#pragma once

#include "cross_attention.hpp"
#include "masked_attention_plan.hpp"

namespace nrs {

constexpr float kLog2e = 1.4426950408889634f;

// A row's keys and place, as the backward keeps them.
struct __attribute__((aligned(16))) RowKeys {
    int lo, hi, at, unused;
};
// Of the rows of a tile: all that any of them sees lies in least .. most - 1, and what
// lies in from .. to - 1 is seen by each.
struct __attribute__((aligned(16))) TileEnds {
    int least, most, from, to;
};

struct MaskedArgs : CrossArgs {
    bool causal;
    const int32_t *q_start, *prefix_len;    // per batch item, or null
    const int32_t *key_begin, *key_end;     // per batch item and query, or null
    const float* slopes;                    // per head, or null
    float scale_own;                        // of the rows' (or keys') operands: scale * log2(e)
    float cap2, by_cap;                     // cap * log2(e), 1 / that
    // the forward's walk, or the backward's two
    int units, part_tiles, parts, q_units, q_part_tiles, q_parts;
    int row_tiles;
    int32_t *counts, *q_counts;             // parts of each unit
    RowKeys* ranges;                        // [batch][seq_q]
    TileEnds* ends;                         // [batch][row_tiles]
};

// The keys that a row sees, lo .. hi - 1 (lo = hi: none), and where it stands among
// them for the bias: at its own position, or the nearest key if that is not among them.
// The distance from there differs from the row's own by the same amount for all
// of its keys, which changes no weight, and keeps the last bits of a far row's scores.
struct RowRange {
    int lo, hi, at;
};

__device__ __forceinline__ RowRange row_range(const MaskedArgs& a, int b, int s) {
    const int64_t at = (int64_t)(a.q_start ? a.q_start[b] : a.Sk - a.Sq) + s;
    const int64_t i = (int64_t)b * a.Sq + s;
    int hi = live_keys(a, b);
    if (a.causal) {
        int64_t seen = at + 1;
        if (a.prefix_len) seen = max(seen, (int64_t)a.prefix_len[b]);
        hi = (int)min((int64_t)hi, seen);
    }
    if (a.key_end) hi = min(hi, a.key_end[i]);
    RowRange r;
    r.lo = a.key_begin ? max(0, a.key_begin[i]) : 0;
    r.hi = hi;
    if (r.lo >= r.hi) r.lo = r.hi = 0;
    r.at = (int)max((int64_t)r.lo, min((int64_t)r.hi - 1, at));
    return r;
}

// cap2 tanh(x / cap2) is x times this, for y = x / cap2 up to 0.6: tanh y = y (1 + z P(z)), z =
// y^2, P of degree 4 (the least largest relative error of that form: 0.05 * 2^-24).
__device__ __forceinline__ float tanh_by_y(float y) {
    const float z = y * y;
    float p = fmaf(z, -0.00589516f, 0.02079597f);
    p = fmaf(z, p, -0.05378383f);
    p = fmaf(z, p, 0.13331924f);
    p = fmaf(z, p, -0.33333298f);
    return fmaf(z, p, 1.0f);
}

// s[i] = cap2 tanh(s[i] / cap2) - from, of scores in base 2, by_cap = 1 / cap2. The operands
// of the products know nothing of the cap, which may be as large or small as a float can
// be. Past 0.6 tanh |y| = 1 - 2 / (1 + e^(2 |y|)), where a wave has such. (Two loops: with a
// branch for each score 2 x 1500 rows of 16 heads of 32 take 77 us in place of 60.)
template <int N, class V>
__device__ __forceinline__ void cap_scores(V& s, float cap2, float by_cap, float from) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(s[i]));
    if (!__any(most > 0.6f * cap2)) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = fmaf(s[i], tanh_by_y(s[i] * by_cap), -from);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float y = s[i] * by_cap;
        const float e = __builtin_amdgcn_exp2f(fabsf(y) * (2.0f * kLog2e));
        const float big = fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
        s[i] = fabsf(y) > 0.6f ? fmaf(copysignf(cap2, y), big, -from)
                               : fmaf(s[i], tanh_by_y(y), -from);
    }
}

// The same from 0, and d[i] *= 1 - tanh^2: past 0.6 that is 4 e / (1 + e)^2, e = e^(-2 |y|),
// which has all its bits where 1 - tanh^2 cancels (near 8 caps 3 bits are left of that). (A
// branch for each score: the backward's kernels spill the registers that two loops take,
// 16384 rows of a head of 64 1499 us in place of 1222.)
template <int N>
__device__ __forceinline__ void cap_scores_and_slopes(float (&s)[N], float (&d)[N], float cap2,
                                                      float by_cap) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(s[i]));
    const bool far = __any(most > 0.6f * cap2);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float x = s[i], y = x * by_cap, p = tanh_by_y(y);
        const float t = y * p;
        float slope = fmaf(-t, t, 1.0f);
        s[i] = x * p;
        if (far) {
            const float e = __builtin_amdgcn_exp2f(fabsf(y) * (-2.0f * kLog2e));
            const float r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
            const bool past = fabsf(y) > 0.6f;
            s[i] = past ? copysignf(cap2, x) * fmaf(-2.0f, er, 1.0f) : s[i];
            slope = past ? 4.0f * er * r : slope;
        }
        d[i] *= slope;
    }
}

// What is added to a product to get a score, by what a call asks for.
enum { kPlain = 0, kBias = 1, kCap = 2 };  // kCap: with a bias, too (of slope 0 if none)

// The kernels of masked_attention_tile.hip.
void masked_tile_forward(const MaskedArgs& a, unsigned blocks);
// The rows' statistics and ranges, then what is asked for of dq and dk, dv.
void masked_tile_backward(const MaskedArgs& a);

}  // namespace nrs
