// Rows as operands of the f32 matrix instructions, and the join of a row's parts, for
// the attention kernels of few rows.
#pragma once

#include "cross_attention.hpp"

namespace nrs {

__device__ __forceinline__ f32x4 mfma16(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// 16 rows (rows, relative to `row0`, of this item and key head) of a tensor of
// keys (GROUPED false) or queries.
template <bool GROUPED>
struct Rows {
    __amdgpu_buffer_rsrc_t rs;
    int ld, row0, n;  // n: live rows of the tile
    const CrossArgs& a;
    int q0;

    __device__ __forceinline__ Rows(const CrossArgs& a, const float* base, int b, int kv, int ld,
                                    int row0, int rows)
        : ld(ld), row0(row0), n(rows), a(a), q0(GROUPED ? row0 / a.G : 0) {
        int64_t first, span;
        if (GROUPED) {
            first = ((int64_t)b * a.Sq + q0) * ld + (int64_t)kv * a.G * a.D;
            span = (int64_t)((row0 + rows - 1) / a.G - q0) * ld + (int64_t)a.G * a.D;
        } else {
            first = ((int64_t)b * a.Sk + row0) * ld + (int64_t)kv * a.D;
            span = (int64_t)(rows - 1) * ld + a.D;
        }
        rs = buffer_rsrc(base + first, span * 4);
    }
    // Byte offset of the tile's row i, or out of range.
    __device__ __forceinline__ int at(int i, int d) const {
        if (i >= n || d >= a.D) return kOutOfRange;
        if (!GROUPED) return (i * ld + d) * 4;
        const int r = row0 + i;
        return ((r / a.G - q0) * ld + (r % a.G) * a.D + d) * 4;
    }
    // d = 16 i + 4 g + e of row c, zero past d_head: an operand of a product
    // over d, whose order of summation is free.
    template <int NJ>
    __device__ __forceinline__ void along(f32x4 (&f)[NJ], int c, int g) const {
#pragma unroll
        for (int i = 0; i < NJ; ++i) {
            const int d = 16 * i + 4 * g;
            f[i] = buffer_load4(rs, at(c, d));
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e >= a.D) f[i][e] = 0.0f;
        }
    }
    // Columns c * NJ .. c * NJ + NJ - 1 of row i (any value past d_head): the
    // operand of a product over rows, its d spread over the lanes.
    template <int NJ>
    __device__ __forceinline__ void across(float (&f)[NJ], int i, int c) const {
        if constexpr (NJ == 1) {
            f[0] = buffer_load1(rs, at(i, c));
        } else if constexpr (NJ == 2) {
            const f32x2 v = buffer_load2(rs, at(i, c * 2));
            f[0] = v[0];
            f[1] = v[1];
        } else {
#pragma unroll
            for (int j = 0; j < NJ; j += 4) {
                const f32x4 v = buffer_load4(rs, at(i, c * NJ + j));
#pragma unroll
                for (int e = 0; e < 4; ++e) f[j + e] = v[e];
            }
        }
    }
};

// acc[m][n] = sum over d of x[m][d] y[n][d]: lane (c, g) gets rows 4g + r of
// column c.
template <int NJ>
__device__ __forceinline__ f32x4 dot_rows(const f32x4 (&x)[NJ], const f32x4 (&y)[NJ]) {
    f32x4 acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NJ; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = mfma16(x[i][e], y[i][e], acc);
    return acc;
}

__device__ __forceinline__ float across_groups(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

// The sums of a row's parts: the reference and the sum of part s at stats(s),
// its columns at part(s). LANES threads share the columns, four each; lane s of
// them looks up part s, and the parts are asked for eight at a time.
template <int LANES>
struct Joined {
    float top = -INFINITY, total = 0.0f;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};

    // The weight of sums taken against m when the reference is `top`: a part
    // without keys has none (NaN sums are not taken for that).
    __device__ __forceinline__ static float weight(float m, float l, float top) {
        return m == -INFINITY && l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    }

    template <class S, class P>
    __device__ __forceinline__ void add(int s0, int s1, int live, S stats, P part) {
        const int x = threadIdx.x % LANES;
        for (int c0 = s0; c0 < s1; c0 += LANES) {
            float m = -INFINITY, l = 0.0f;
            if (c0 + x < s1) {
                const float* st = stats(c0 + x);
                m = st[0];
                l = st[1];
            }
            float most = m;
#pragma unroll
            for (int i = 1; i < LANES; i *= 2) most = fmaxf(most, __shfl_xor(most, i, LANES));
            most = fmaxf(most, top);
            const float old = weight(top, total, most), f = weight(m, l, most);
            float sum = l * f;
#pragma unroll
            for (int i = 1; i < LANES; i *= 2) sum += __shfl_xor(sum, i, LANES);
            total = total * old + sum;
            top = most;
            v = v * old;
            for (int s = c0; s < min(c0 + LANES, s1); s += 8) {
                f32x4 x8[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x8[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    if (s + i >= s1) continue;
                    const float* src = part(s + i) + 4 * x;
                    if (live == 4)
                        x8[i] = reinterpret_cast<const Quad*>(src)->v;
                    else
                        for (int e = 0; e < live; ++e) x8[i][e] = src[e];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) v = v + x8[i] * __shfl(f, s + i - c0, LANES);
            }
        }
    }

    __device__ __forceinline__ void store(const CrossArgs& a, int b, int kv, int r, int live) const {
        const int x = threadIdx.x % LANES;
        const bool any = live_keys(a, b) > 0;
        const float scale = any ? 1.0f / total : 0.0f;
        float* dst = a.out + query_offset(a, b, kv, r, a.ld_out) + 4 * x;
        if (live == 4)
            reinterpret_cast<Quad*>(dst)->v = v * scale;
        else
            for (int e = 0; e < live; ++e) dst[e] = v[e] * scale;
        if (a.stats && x == 0) {
            float* st = row_stats(a, b, kv, r);
            st[0] = any ? top : 0.0f;
            st[1] = any ? total : 0.0f;
        }
    }
};

// The parts of row r of an item: their number (0: no key is seen by its unit) and where in rows
// of `part` each one is.
struct RowParts {
    int n = 0, unit_rows, begun = 0, line = 0;  // the rows of part 0, and of one before part 1
    __device__ __forceinline__ RowParts(const CrossArgs& a, int item, int r, bool any)
        : unit_rows(a.unit_rows) {
        if (!any) return;
        const int units = (a.Sq * a.G + unit_rows - 1) / unit_rows, in_item = r / unit_rows;
        const int unit = item * units + in_item, first = a.shares[2 * unit];
        n = a.shares[2 * unit + 1] - first + 1;
        const int in_unit = r - in_item * unit_rows;
        begun = begun_slot(a, unit, first) * unit_rows + in_unit;
        line = first * unit_rows + in_unit;
    }
    __device__ __forceinline__ int64_t at(int s) const {
        return s == 0 ? begun : line + s * unit_rows;
    }
};

}  // namespace nrs
