// Attention whose rows see ranges of keys, with capped scores and a bias by
// distance, forward and backward, all f32.
//
// Here: the forward of few rows (tokens being decoded), the joins and sums of walks in
// parts, and the entry points. Which kernels take a call, and the parts, are planned in
// masked_attention_plan.hpp.
#include "attention_rows.hpp"
#include "masked_attention.hpp"

#include <cmath>

namespace nrs {
namespace {

// All that any query of an item sees, least .. most - 1 (0 .. -1: nothing).
struct Span {
    int least, most;
    __device__ __forceinline__ int first() const { return least / 16; }
    __device__ __forceinline__ int tiles() const {
        return most > 0 ? (most + 15) / 16 - least / 16 : 0;
    }
};

__device__ __forceinline__ Span item_span(const MaskedArgs& a, int b) {
    Span all{INT32_MAX, 0};
    for (int s = 0; s < a.Sq; ++s) {
        const RowRange r = row_range(a, b, s);
        if (r.hi > 0) all.least = min(all.least, r.lo);
        all.most = max(all.most, r.hi);
    }
    return all;
}

// A workgroup's part of the line of all items' tiles of 16 keys, as LinePart
// (cross_attention.hpp): there an item's tiles are those of its length, here those that
// any of its queries sees.
template <int NT>
struct SpanLine {
    Span* spans;  // of all items, in shared memory
    int b, base, p, end, per_item;
    int sub, t0, t1, tiles;  // of the piece at hand: tiles t0 .. t1 - 1, from the span's first

    // False if the part is empty. All NT threads call it; `scan` and `found` are shared.
    __device__ __forceinline__ bool begin(const MaskedArgs& a, int per_item_, int (&scan)[NT / 64],
                                          int (&found)[2]) {
        per_item = per_item_;
        const int t = threadIdx.x, lane = t & 63, w = t >> 6, each = (a.B + NT - 1) / NT;
        int own = 0;
        for (int i = t * each; i < min((t + 1) * each, a.B); ++i) {
            spans[i] = item_span(a, i);
            own += spans[i].tiles() * per_item;
        }
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
        // a tile to a workgroup at least, so that those that share a unit follow each other
        const int parts = min(a.groups, total);
        if ((int)blockIdx.x >= parts) return false;
        p = (int)((int64_t)total * blockIdx.x / parts);
        end = (int)((int64_t)total * (blockIdx.x + 1) / parts);
        for (int i = t * each; i < min((t + 1) * each, a.B); ++i) {
            const int n = spans[i].tiles() * per_item;
            if (at <= p && p < at + n) {
                found[0] = i;
                found[1] = at;
            }
            at += n;
        }
        __syncthreads();
        b = found[0];
        base = found[1];
        return true;
    }
    __device__ __forceinline__ bool next(const MaskedArgs& a) {
        if (p >= end) return false;
        for (;;) {  // (items that see nothing have no tiles)
            tiles = __builtin_amdgcn_readfirstlane(spans[b].tiles());
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
    __device__ __forceinline__ int64_t slot(const MaskedArgs& a) const {
        if (t0 > 0) return blockIdx.x;
        return t1 == tiles ? -1 : begun_slot(a, b * per_item + sub, blockIdx.x);
    }
};

// Few rows (tokens being decoded): K and V stream from memory once, straight into
// registers, as operands of v_mfma_f32_16x16x4_f32. A unit is 16 rows of an item; a
// workgroup's waves take turns at tiles of 16 keys, each with its next tile on the way,
// and are joined at the end. 4 x 16384 keys and fewer, 8 key heads of 128, 4 rows each, capped:
// 76 us, 4.7 TB/s; 32 items of up to 1500 keys, 8 heads of 64, a row each: 29 us, 3.9 TB/s,
// where a wave sees five tiles behind the lengths' and the rows' own round trips.
template <int NJ, int MODE>
struct MaskedRows {
    const MaskedArgs& a;
    float (&sums)[kRowWaves][4 * NJ][64];
    float (&tops)[kRowWaves][16];
    float (&totals)[kRowWaves][16];

    // Tiles t0 .. t1 - 1 of the rows from r0 on of (b, kv), whose item sees `span`: all of
    // them (slot < 0) or a part.
    __device__ __forceinline__ void run(int b, int kv, int r0, Span span, int t0, int t1,
                                        int64_t slot) const {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
        const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int R = a.Sq * a.G, most = __builtin_amdgcn_readfirstlane(span.most);
        f32x4 qf[NJ], acc[NJ], kf[NJ];
        float vf[4][NJ];
        auto load_keys = [&](int t) {
            Rows<false>(a, a.k, b, kv, a.ld_kv, 16 * t, min(16, most - 16 * t))
                .template along<NJ>(kf, c, g);
        };
        auto load_values = [&](int t) {
            const Rows<false> vs(a, a.v, b, kv, a.ld_kv, 16 * t, min(16, most - 16 * t));
#pragma unroll
            for (int r = 0; r < 4; ++r) vs.template across<NJ>(vf[r], 4 * g + r, c);
        };
        if (t0 + w < t1) {
            load_keys(t0 + w);
            load_values(t0 + w);
        }
        const bool live = r0 + c < R;
        const int s_row = live ? (r0 + c) / a.G : 0;
        RowRange range = row_range(a, b, s_row);
        if (!live) range.lo = range.hi = range.at = 0;
        // what all rows see
        int from = !live ? 0 : range.hi > 0 ? range.lo : INT32_MAX, to = live ? range.hi : INT32_MAX;
#pragma unroll
        for (int i = 1; i < 16; i *= 2) {
            from = max(from, __shfl_xor(from, i, 64));
            to = min(to, __shfl_xor(to, i, 64));
        }
        const float slope2 = MODE != kPlain && a.slopes && live
                                 ? a.slopes[kv * a.G + r0 + c - s_row * a.G] * kLog2e
                                 : 0.0f;
        Rows<true>(a, a.q, b, kv, a.ld_q, r0, min(16, R - r0)).template along<NJ>(qf, c, g);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            qf[j] = qf[j] * a.scale_own;
            acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        float m = -INFINITY, l = 0.0f;
        for (int t = t0 + w; t < t1; t += kRowWaves) {
            f32x4 p = dot_rows<NJ>(kf, qf);
            if (t + kRowWaves < t1) load_keys(t + kRowWaves);
            if (MODE == kCap) cap_scores<4>(p, a.cap2, a.by_cap, 0.0f);
            if (MODE != kPlain) {
                const float far = (float)(range.at - (16 * t + 4 * g));
#pragma unroll
                for (int r = 0; r < 4; ++r) p[r] = fmaf(-slope2, fabsf(far - (float)r), p[r]);
            }
            if (16 * t < from || 16 * t + 16 > to) {
                // a value that is not finite must not meet the weight 0 of a row that does
                // not see it: the key gets zeros, and a NaN for a score
                int bad = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float most_v = 0.0f;
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
                        if (c * NJ + j < a.D)
                            most_v = __builtin_elementwise_maximum(most_v, __builtin_fabsf(vf[r][j]));
                    bad |= most_v < INFINITY ? 0 : 1 << r;
                }
#pragma unroll
                for (int i = 1; i < 16; i *= 2) bad |= __shfl_xor(bad, i, 64);
                const uint32_t keys = range.hi - range.lo;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (bad >> r & 1) {
                        p[r] = NAN;
#pragma unroll
                        for (int j = 0; j < NJ; ++j) vf[r][j] = 0.0f;
                    }
                    p[r] = (uint32_t)(16 * t + 4 * g + r - range.lo) < keys ? p[r] : -INFINITY;
                }
            }
            float top = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(fmaxf(top, __shfl_xor(top, 32, 64)), m);
            const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= alpha;
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[j] = acc[j] * alpha;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[r] = p[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(p[r] - m);
                l += p[r];
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[j] = mfma16(vf[r][j], p[r], acc[j]);
            }
            if (t + kRowWaves < t1) load_values(t + kRowWaves);
        }
        l = across_groups(l);
        if (g == 0) {
            tops[w][c] = m;
            totals[w][c] = l;
        }
        __syncthreads();
        float top = tops[0][c];
#pragma unroll
        for (int i = 1; i < kRowWaves; ++i) top = fmaxf(top, tops[i][c]);
        const float f = Joined<32>::weight(m, l, top);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NJ; ++j) sums[w][r * NJ + j][lane] = acc[j][r] * f;
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < kRowWaves; ++i) {
            const float of = Joined<32>::weight(tops[i][c], totals[i][c], top);
            total += totals[i][c] * of;
        }
        __syncthreads();
        if (live) {
            // wave w adds the waves' register w: NJ neighbouring columns of row c
            static_assert(kRowWaves == 4, "a register of an accumulator to each wave");
            const bool whole = slot < 0, none = total == 0.0f;
            const float scale = !whole ? 1.0f : none ? 0.0f : 1.0f / total;
            const int64_t at = slot * a.unit_rows + c;
            float* dst = whole ? a.out + query_offset(a, b, kv, r0 + c, a.ld_out) : a.part + at * a.D;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                float v = 0.0f;
#pragma unroll
                for (int i = 0; i < kRowWaves; ++i) v += sums[i][w * NJ + j][lane];
                const int d = (4 * g + w) * NJ + j;
                if (d < a.D) dst[d] = v * scale;
            }
            if (w == 0 && g == 0 && (!whole || a.stats)) {
                float* st = whole ? row_stats(a, b, kv, r0 + c) : a.part_stats + 2 * at;
                st[0] = whole && none ? 0.0f : top;
                st[1] = total;
            }
        }
        __syncthreads();  // before the shared arrays serve the next unit
    }
};

template <int NJ, int MODE>
__global__ __launch_bounds__(64 * kRowWaves) void masked_rows_fwd_kernel(MaskedArgs a) {
    __shared__ float sums[kRowWaves][4 * NJ][64];
    __shared__ float tops[kRowWaves][16], totals[kRowWaves][16];
    __shared__ int scan[kRowWaves], found[2];
    __shared__ Span spans[kMaxSharedBatch];
    const MaskedRows<NJ, MODE> walk{a, sums, tops, totals};
    const int row_tiles = (a.Sq * a.G + 15) / 16, per_item = a.KV * row_tiles;
    if (a.groups == 0) {
        const int unit = blockIdx.x, b = unit / per_item, sub = unit - b * per_item;
        const Span span = item_span(a, b);
        walk.run(b, sub / row_tiles, sub % row_tiles * 16, span, span.most > 0 ? span.first() : 0,
                 span.most > 0 ? span.first() + span.tiles() : 0, -1);
        return;
    }
    SpanLine<64 * kRowWaves> line{spans};
    if (!line.begin(a, per_item, scan, found)) return;
    while (line.next(a)) {
        const Span span = spans[line.b];
        walk.run(line.b, line.sub / row_tiles, line.sub % row_tiles * 16, span,
                 span.first() + line.t0, span.first() + line.t1, line.slot(a));
    }
}

// The parts of a row of the kernel of many rows: their number, and where each is.
struct WalkParts {
    int n, unit, units, unit_rows, in_unit;
    __device__ __forceinline__ WalkParts(const MaskedArgs& a, int item, int r)
        : unit(item * ((a.Sq * a.G + a.unit_rows - 1) / a.unit_rows) + r / a.unit_rows),
          units(a.units), unit_rows(a.unit_rows), in_unit(r % a.unit_rows) {
        n = a.counts[unit];
    }
    __device__ __forceinline__ int64_t at(int s) const {
        return ((int64_t)s * units + unit) * unit_rows + in_unit;
    }
};

template <int LANES>
__device__ __forceinline__ void store_joined(const MaskedArgs& a, const Joined<LANES>& sum, int item,
                                             int r, int live) {
    const int x = threadIdx.x % LANES, b = item / a.KV, kv = item - b * a.KV;
    const bool none = sum.total == 0.0f;
    const float scale = none ? 0.0f : 1.0f / sum.total;
    float* dst = a.out + query_offset(a, b, kv, r, a.ld_out) + 4 * x;
    if (live == 4)
        reinterpret_cast<Quad*>(dst)->v = sum.v * scale;
    else
        for (int e = 0; e < live; ++e) dst[e] = sum.v[e] * scale;
    if (a.stats && x == 0) {
        float* st = row_stats(a, b, kv, r);
        st[0] = none ? 0.0f : sum.top;
        st[1] = sum.total;
    }
}

// Joins the parts of masked_rows_fwd_kernel, which may be many, a workgroup to a row:
// eight groups of 32 threads take an eighth of them each and are added up in LDS.
__global__ __launch_bounds__(256) void masked_rows_join_kernel(MaskedArgs a) {
    __shared__ f32x4 sums[8][32];
    __shared__ float tops[8], totals[8];
    const int x = threadIdx.x % 32, group = threadIdx.x / 32, R = a.Sq * a.G;
    const int item = blockIdx.x / R, r = blockIdx.x - item * R;
    const int live = max(0, min(4, a.D - 4 * x));
    const RowParts parts(a, item, r, item_span(a, item / a.KV).most > 0);
    if (parts.n == 1) return;  // one workgroup took all of the unit
    Joined<32> sum;
    sum.add(parts.n * group / 8, parts.n * (group + 1) / 8, live,
            [&](int s) { return a.part_stats + 2 * parts.at(s); },
            [&](int s) { return a.part + parts.at(s) * a.D; });
    sums[group][x] = sum.v;
    if (x == 0) {
        tops[group] = sum.top;
        totals[group] = sum.total;
    }
    __syncthreads();
    if (group != 0) return;
    for (int i = 1; i < 8; ++i) {
        const float most = fmaxf(sum.top, tops[i]);
        const float f = Joined<32>::weight(sum.top, sum.total, most),
                    of = Joined<32>::weight(tops[i], totals[i], most);
        sum.v = sum.v * f + sums[i][x] * of;
        sum.total = sum.total * f + totals[i] * of;
        sum.top = most;
    }
    store_joined(a, sum, item, r, live);
}

// Joins the parts of masked_tile_fwd_kernel, which are few: D / 4 threads to a row.
template <int D>
__global__ __launch_bounds__(256) void masked_join_kernel(MaskedArgs a) {
    constexpr int LANES = D / 4;
    const int R = a.Sq * a.G, x = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (row >= (int64_t)a.B * a.KV * R) return;
    const int item = (int)(row / R), r = (int)(row - (int64_t)item * R);
    const int live = max(0, min(4, a.D - 4 * x));
    const WalkParts parts(a, item, r);
    if (parts.n == 1) return;
    Joined<LANES> sum;
    sum.add(0, parts.n, live, [&](int s) { return a.part_stats + 2 * parts.at(s); },
            [&](int s) { return a.part + parts.at(s) * a.D; });
    store_joined(a, sum, item, r, live);
}

// Adds the parts of a gradient in order: dst = f * sum + beta * dst, D / 4 threads to a
// row. KEYS: rows are keys, blockIdx.y is 0 for dk and 1 for dv.
template <int D, bool KEYS>
__global__ __launch_bounds__(256) void masked_sum_kernel(MaskedArgs a) {
    constexpr int LANES = D / 4;
    const int n = KEYS ? a.Sk : a.Sq * a.G, x = threadIdx.x % LANES;
    const int64_t at = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const int64_t rows = (int64_t)a.B * a.KV * n;
    if (at >= rows) return;
    const int item = (int)(at / n), r = (int)(at - (int64_t)item * n);
    const int b = item / a.KV, kv = item - b * a.KV;
    const int own = 16 * masked_backward_waves(a.D), unit = item * ((n + own - 1) / own) + r / own;
    const int parts = (KEYS ? a.counts : a.q_counts)[unit];
    if (parts == 1) return;  // one workgroup took all of it
    const bool second = KEYS && blockIdx.y == 1;
    const float beta = KEYS ? a.beta_kv : a.beta_q, f = second ? 1.0f : a.scale;
    const float* part = (KEYS ? (second ? a.dv_part : a.dk_part) : a.dq_part) + at * a.D + 4 * x;
    float* dst = (KEYS ? (second ? a.dv : a.dk) + key_offset(a, b, kv, r)
                       : a.dq + query_offset(a, b, kv, r, a.ld_q)) + 4 * x;
    if (4 * x + 4 <= a.D) {
        f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int s = 0; s < parts; ++s)
            v = v + reinterpret_cast<const Quad*>(part + s * rows * a.D)->v;
        v = v * f;
        Quad* const to = reinterpret_cast<Quad*>(dst);
        if (beta != 0.0f) v = v + beta * to->v;
        to->v = v;
    } else {
        for (int e = 0; 4 * x + e < a.D; ++e) {
            float v = 0.0f;
            for (int s = 0; s < parts; ++s) v += part[s * rows * a.D + e];
            dst[e] = beta != 0.0f ? v * f + beta * dst[e] : v * f;
        }
    }
}

template <int D>
void launch_sums(const MaskedArgs& a, bool dq, bool dkv) {
    constexpr int PER = 1024 / D;
    const int64_t rows = (int64_t)a.B * a.KV * a.Sq * a.G, keys = (int64_t)a.B * a.KV * a.Sk;
    if (dq)
        hipLaunchKernelGGL((masked_sum_kernel<D, false>), dim3((unsigned)((rows + PER - 1) / PER)),
                           dim3(256), 0, stream(), a);
    if (dkv)
        hipLaunchKernelGGL((masked_sum_kernel<D, true>), dim3((unsigned)((keys + PER - 1) / PER), 2),
                           dim3(256), 0, stream(), a);
}

template <int D>
void launch_join(const MaskedArgs& a, int64_t rows) {
    constexpr int PER = 1024 / D;
    hipLaunchKernelGGL(masked_join_kernel<D>, dim3((unsigned)((rows + PER - 1) / PER)),
                       dim3(256), 0, stream(), a);
}

template <int NJ>
void launch_rows(const MaskedArgs& a, unsigned blocks) {
    auto kernel = a.cap2 > 0.0f ? masked_rows_fwd_kernel<NJ, kCap>
                  : a.slopes    ? masked_rows_fwd_kernel<NJ, kBias>
                                : masked_rows_fwd_kernel<NJ, kPlain>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kRowWaves), 0, stream(), a);
}

int check(const char* what, const nrs_attention_mask* mask, int64_t batch, int64_t heads,
          int64_t kv_heads, int64_t seq_q, int64_t seq_k, int64_t d_head, int64_t ld_q,
          int64_t ld_kv, int64_t ld_out, float scale) {
    if (int rc = cross_check_shape(what, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q,
                                   ld_kv, ld_out))
        return rc;
    if (!mask) return NRS_OK;
    // (the reciprocal of a smaller one is past the largest float)
    NRS_ARG_CHECK(mask->cap == 0.0f || (mask->cap >= 0x1p-126f && std::isfinite(mask->cap * kLog2e)),
                  "%s: cap must be 0 (none) or a number from 2^-126 to below 2^127, is %g", what,
                  (double)mask->cap);
    NRS_ARG_CHECK(mask->cap == 0.0f || std::isfinite((float)((double)scale / mask->cap)),
                  "%s: scale / cap is %g / %g", what, (double)scale, (double)mask->cap);
    NRS_ARG_CHECK(mask->causal || !mask->prefix_len, "%s: a prefix without a causal mask", what);
    return NRS_OK;
}

MaskedArgs arguments(const nrs_attention_mask* mask, int64_t batch, int64_t heads,
                     int64_t kv_heads, int64_t seq_q, int64_t seq_k, int64_t d_head, int64_t ld_q,
                     int64_t ld_kv, int64_t ld_out, float scale) {
    MaskedArgs a{};
    if (mask) {
        a.causal = mask->causal != 0;
        a.q_start = mask->q_start;
        a.key_len = mask->key_len;
        a.prefix_len = mask->prefix_len;
        a.key_begin = mask->key_begin;
        a.key_end = mask->key_end;
        a.slopes = mask->slopes;
    }
    // (taken in 64 bits, rounded once)
    const double log2e = 1.4426950408889634, cap2 = (mask ? mask->cap : 0.0f) * log2e;
    a.scale_own = (float)(scale * log2e);
    a.cap2 = (float)cap2;
    a.by_cap = cap2 > 0.0 ? (float)(1.0 / cap2) : 0.0f;
    a.B = (int)batch;
    a.H = (int)heads;
    a.KV = (int)kv_heads;
    a.G = (int)(heads / kv_heads);
    a.Sq = (int)seq_q;
    a.Sk = (int)seq_k;
    a.D = (int)d_head;
    a.ld_q = (int)ld_q;
    a.ld_kv = (int)ld_kv;
    a.ld_out = (int)ld_out;
    a.by_group = make_fastdiv((uint32_t)a.G);
    a.scale = scale;
    return a;
}

}  // namespace
}  // namespace nrs

extern "C" {

int nrs_masked_attention_supported(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q,
                                   int64_t seq_k, int64_t d_head, int64_t ld_q, int64_t ld_kv,
                                   int64_t ld_out) {
    return nrs_cross_attention_supported(batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                                         ld_out);
}

int nrs_masked_attention_workspace(size_t* bytes, int64_t batch, int64_t heads, int64_t kv_heads,
                                   int64_t seq_q, int64_t seq_k, int64_t d_head, int backward) {
    const char* what = "masked attention workspace";
    NRS_ARG_CHECK(bytes, "%s: null pointer", what);
    const int64_t ld = int64_t(1) << 20;
    if (int rc = nrs::cross_check_shape(what, batch, heads, kv_heads, seq_q, seq_k, d_head, ld, ld,
                                        ld))
        return rc;
    const int cus = nrs::num_cus();
    *bytes =
        backward
            ? nrs::plan_masked_backward(batch, heads, kv_heads, seq_q, seq_k, d_head, cus).bytes()
            : nrs::plan_masked_forward(batch, heads, kv_heads, seq_q, seq_k, d_head, cus).bytes();
    return NRS_OK;
}

int nrs_masked_attention_forward(float* out, float* stats, const float* q, const float* k,
                                 const float* v, const nrs_attention_mask* mask, int64_t batch,
                                 int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_k,
                                 int64_t d_head, int64_t ld_q, int64_t ld_kv, int64_t ld_out,
                                 float scale, void* work, size_t work_bytes) {
    const char* what = "masked attention forward";
    if (int rc = nrs::check(what, mask, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                            ld_out, scale))
        return rc;
    if (batch == 0 || seq_q == 0) return NRS_OK;
    NRS_ARG_CHECK(out && q && ((k && v) || seq_k == 0), "%s: null pointer", what);
    NRS_REQUIRE_INIT();
    if (int rc = nrs::check_device(what)) return rc;
    const auto plan = nrs::plan_masked_forward(batch, heads, kv_heads, seq_q, seq_k, d_head,
                                               nrs::num_cus());
    float* scratch = nullptr;
    if (int rc = nrs::call_scratch(&scratch, plan.bytes(), work, work_bytes, what)) return rc;
    auto a = nrs::arguments(mask, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                            ld_out, scale);
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.stats = stats;
    a.unit_rows = plan.unit_rows;
    a.units = (int)plan.walk.units;
    a.part_tiles = plan.walk.part;
    a.parts = plan.walk.parts;
    a.groups = plan.line.groups;
    a.few_units = plan.line.few_units;
    a.part = scratch;
    a.part_stats = scratch + plan.part;
    a.shares = a.counts = reinterpret_cast<int32_t*>(scratch + plan.part + plan.stats);
    const unsigned blocks = (unsigned)plan.blocks();
    const int64_t rows = batch * heads * seq_q;
    if (plan.tiles) {
        nrs::masked_tile_forward(a, blocks);
        NRS_LAUNCH_CHECK(what);
        const int width = nrs::cross_row_width(a.D);
        if (a.parts > 1)
            (width == 32   ? nrs::launch_join<32>
             : width == 64 ? nrs::launch_join<64>
                           : nrs::launch_join<128>)(a, rows);
    } else {
        (a.D <= 16   ? nrs::launch_rows<1>
         : a.D <= 32 ? nrs::launch_rows<2>
         : a.D <= 64 ? nrs::launch_rows<4>
                     : nrs::launch_rows<8>)(a, blocks);
        NRS_LAUNCH_CHECK(what);
        if (a.groups > 0)
            hipLaunchKernelGGL(nrs::masked_rows_join_kernel, dim3((unsigned)rows), dim3(256), 0,
                               nrs::stream(), a);
    }
    NRS_LAUNCH_CHECK(what);
    return NRS_OK;
}

int nrs_masked_attention_backward(float* dq, float* dk, float* dv, const float* dout,
                                  const float* out, const float* q, const float* k, const float* v,
                                  const float* stats, const nrs_attention_mask* mask,
                                  int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q,
                                  int64_t seq_k, int64_t d_head, int64_t ld_q, int64_t ld_kv,
                                  int64_t ld_out, float scale, float beta_q, float beta_kv,
                                  void* work, size_t work_bytes) {
    const char* what = "masked attention backward";
    if (int rc = nrs::check(what, mask, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                            ld_out, scale))
        return rc;
    NRS_ARG_CHECK((dk == nullptr) == (dv == nullptr), "%s: dk and dv go together", what);
    if (batch == 0) return NRS_OK;
    const bool rows = seq_q > 0, keys = seq_k > 0;
    NRS_ARG_CHECK((!rows || (dout && out && q && stats)) && (!keys || (k && v)),
                  "%s: null pointer", what);
    NRS_REQUIRE_INIT();
    if (int rc = nrs::check_device(what)) return rc;
    const auto plan = nrs::plan_masked_backward(batch, heads, kv_heads, seq_q, seq_k, d_head,
                                                nrs::num_cus());
    float* scratch = nullptr;
    if (int rc = nrs::call_scratch(&scratch, plan.bytes(), work, work_bytes, what)) return rc;
    auto a = nrs::arguments(mask, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                            ld_out, scale);
    a.q = q;
    a.k = k;
    a.v = v;
    a.dout = dout;
    a.o = out;
    a.stats = const_cast<float*>(stats);  // only read here
    a.dq = rows ? dq : nullptr;
    a.dk = keys ? dk : nullptr;
    a.dv = keys ? dv : nullptr;
    a.beta_q = beta_q;
    a.beta_kv = beta_kv;
    a.q_units = (int)plan.q.units;
    a.q_part_tiles = plan.q.part;
    a.q_parts = plan.q.parts;
    a.units = (int)plan.kv.units;
    a.part_tiles = plan.kv.part;
    a.parts = plan.kv.parts;
    a.row_tiles = (int)plan.row_tiles;
    float* next = scratch;
    auto take = [&next](size_t words) {
        float* const p = next;
        next += words;
        return p;
    };
    a.neg_lse = take(plan.rows);
    a.neg_delta = a.neg_lse + batch * heads * seq_q;
    a.ranges = reinterpret_cast<nrs::RowKeys*>(take(plan.ranges));
    a.ends = reinterpret_cast<nrs::TileEnds*>(take(plan.ends));
    a.dq_part = take(plan.q_part);
    a.dk_part = take(plan.kv_part);
    a.dv_part = take(plan.kv_part);
    a.q_counts = reinterpret_cast<int32_t*>(take(plan.counts));
    a.counts = a.q_counts + plan.q.units;
    if (!a.dq && !a.dk) return NRS_OK;
    nrs::masked_tile_backward(a);
    NRS_LAUNCH_CHECK(what);
    const int width = nrs::cross_row_width(a.D);
    (width == 32   ? nrs::launch_sums<32>
     : width == 64 ? nrs::launch_sums<64>
                   : nrs::launch_sums<128>)(a, a.dq && a.q_parts > 1, a.dk && a.parts > 1);
    NRS_LAUNCH_CHECK(what);
    return NRS_OK;
}

}  // extern "C"
