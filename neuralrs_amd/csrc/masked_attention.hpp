// Arguments and device helpers shared by the masked attention kernels.
//
// Rows are those of cross_attention.hpp: row r of an item (batch item, key head) is
// query r / group of head kv_head * group + r % group. Every row sees an unbroken
// range of its item's keys: causal, prefix, document and length masks are one each,
// and so is what they have in common.
#pragma once

#include "cross_attention.hpp"

namespace nrs {

struct MaskedArgs : CrossArgs {
    bool causal;
    const int32_t *q_start, *prefix_len;    // per batch item, or null
    const int32_t *key_begin, *key_end;     // per batch item and query, or null
    const float* slopes;                    // per head, or null
    float cap;                              // 0: none
};

// The keys that a row sees, lo .. hi - 1 (lo = hi: none), and where it stands among
// them.
struct RowRange {
    int lo, hi;
    int64_t at;
};

__device__ __forceinline__ RowRange row_range(const MaskedArgs& a, int b, int s) {
    RowRange r;
    r.at = (int64_t)(a.q_start ? a.q_start[b] : a.Sk - a.Sq) + s;
    const int64_t i = (int64_t)b * a.Sq + s;
    int64_t hi = live_keys(a, b);
    if (a.causal) {
        int64_t seen = r.at + 1;
        if (a.prefix_len) seen = max(seen, (int64_t)a.prefix_len[b]);
        hi = min(hi, seen);
    }
    if (a.key_end) hi = min(hi, (int64_t)a.key_end[i]);
    const int64_t lo = a.key_begin ? max(0, a.key_begin[i]) : 0;
    r.lo = (int)lo;
    r.hi = (int)max(lo, hi);
    return r;
}

// The distance to the nearest key of a row's range: biases are taken relative to
// that key's, which changes every score of the row by the same amount, so that far
// rows do not lose their scores' last bits in the size of the bias.
__device__ __forceinline__ int64_t nearest(const RowRange& r) {
    return r.at < r.lo ? r.lo - r.at : r.at >= r.hi ? r.at - (r.hi - 1) : 0;
}

}  // namespace nrs
