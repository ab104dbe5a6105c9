// Attention of a decoder's rows over an encoder's states: queries and keys of
// different lengths, several query heads to a key head, a length of live keys
// for each batch item. Forward and backward, all f32.
//
// Here: the forward of few rows (a token being decoded), the join of an item's
// keys shared among workgroups, the backward and the entry points. Which kernels
// take a call is planned in cross_attention_plan.hpp.
#include "attention_rows.hpp"

#include <algorithm>

namespace nrs {
namespace {

// Few rows: K and V stream from HBM straight into registers, as operands of
// v_mfma_f32_16x16x4_f32 (16 rows at 157 TFLOP/s keep pace with 8 TB/s of f32
// keys and values). Waves of a workgroup take turns at tiles of 16 keys, each
// with its next tile on the way, and are joined at the end. 2 x 16384 keys, 8 key
// heads of 128, 4 rows each: 45 us, 5.9 TB/s; 32 items of up to 1500 keys, 8 heads
// of 64, a row each: 26 us, 4.4 TB/s, where a wave sees five tiles.
template <int NJ>
struct RowsWalk {
    const CrossArgs& a;
    float (&sums)[kRowWaves][4 * NJ][64];
    float (&tops)[kRowWaves][16];
    float (&totals)[kRowWaves][16];

    // Tiles t0 .. t1 - 1 of unit `unit` (rows r0 .. of (b, kv)), L live keys:
    // the whole of it (slot < 0) or a part.
    __device__ __forceinline__ void run(int b, int kv, int r0, int L, int t0, int t1,
                                        int64_t slot) const {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
        const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int R = a.Sq * a.G;
        f32x4 qf[NJ], acc[NJ], kf[NJ];
        float vf[4][NJ];
        auto load_keys = [&](int t) {
            Rows<false>(a, a.k, b, kv, a.ld_kv, 16 * t, min(16, L - 16 * t))
                .template along<NJ>(kf, c, g);
        };
        auto load_values = [&](int t) {
            const Rows<false> vs(a, a.v, b, kv, a.ld_kv, 16 * t, min(16, L - 16 * t));
#pragma unroll
            for (int r = 0; r < 4; ++r) vs.template across<NJ>(vf[r], 4 * g + r, c);
        };
        if (t0 + w < t1) {
            load_keys(t0 + w);
            load_values(t0 + w);
        }
        Rows<true>(a, a.q, b, kv, a.ld_q, r0, min(16, R - r0)).template along<NJ>(qf, c, g);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            qf[j] = qf[j] * a.scale2;
            acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        float m = -INFINITY, l = 0.0f;
        for (int t = t0 + w; t < t1; t += kRowWaves) {
            f32x4 p = dot_rows<NJ>(kf, qf);
            if (t + kRowWaves < t1) load_keys(t + kRowWaves);
            float mt = -INFINITY;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (16 * t + 4 * g + r >= L) p[r] = -INFINITY;
                mt = fmaxf(mt, p[r]);
            }
            mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
            mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
            const float top = fmaxf(m, mt);
            const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= alpha;
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[j] = acc[j] * alpha;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[r] = 16 * t + 4 * g + r < L ? __builtin_amdgcn_exp2f(p[r] - m) : 0.0f;
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
        // a wave without keys adds nothing; NaN must not be taken for that
        const float f = m == -INFINITY && l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NJ; ++j) sums[w][r * NJ + j][lane] = acc[j][r] * f;
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < kRowWaves; ++i) {
            const float li = totals[i][c];
            total += tops[i][c] == -INFINITY && li == 0.0f
                         ? 0.0f
                         : li * __builtin_amdgcn_exp2f(tops[i][c] - top);
        }
        __syncthreads();
        if (r0 + c < R) {
            // wave w adds the waves' register w: NJ neighbouring columns of row c
            static_assert(kRowWaves == 4, "a register of an accumulator to each wave");
            const bool whole = slot < 0;
            const float scale = !whole ? 1.0f : L > 0 ? 1.0f / total : 0.0f;
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
                st[0] = whole && L == 0 ? 0.0f : top;
                st[1] = total;
            }
        }
        __syncthreads();  // before the shared arrays serve the next unit
    }
};

template <int NJ>
__global__ __launch_bounds__(64 * kRowWaves) void cross_rows_fwd_kernel(CrossArgs a) {
    __shared__ float sums[kRowWaves][4 * NJ][64];
    __shared__ float tops[kRowWaves][16], totals[kRowWaves][16];
    __shared__ int scan[kRowWaves], found[2];
    const RowsWalk<NJ> walk{a, sums, tops, totals};
    const int row_tiles = (a.Sq * a.G + 15) / 16, per_item = a.KV * row_tiles;
    if (a.groups == 0) {
        const int unit = blockIdx.x, b = unit / per_item, sub = unit - b * per_item;
        const int L = live_keys(a, b);
        walk.run(b, sub / row_tiles, sub % row_tiles * 16, L, 0, (L + 15) / 16, -1);
        return;
    }
    LinePart<64 * kRowWaves> part;
    if (!part.begin(a, per_item, 16, scan, found)) return;
    while (part.next(a))
        walk.run(part.b, part.sub / row_tiles, part.sub % row_tiles * 16, part.L, part.t0, part.t1,
                 part.slot(a));
}

// Joins the parts of cross_rows_fwd_kernel, a workgroup to a row: eight groups of
// 32 threads take an eighth of them each and are added up in LDS: 4.8 us for 64
// rows of 17 parts, a launch and its round trips.
__global__ __launch_bounds__(256) void cross_rows_join_kernel(CrossArgs a) {
    __shared__ f32x4 sums[8][32];
    __shared__ float tops[8], totals[8];
    const int x = threadIdx.x % 32, group = threadIdx.x / 32, R = a.Sq * a.G;
    const int item = blockIdx.x / R, r = blockIdx.x - item * R, b = item / a.KV;
    const int live = max(0, min(4, a.D - 4 * x));
    const RowParts parts(a, item, r, live_keys(a, b) > 0);
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
                    g = Joined<32>::weight(tops[i], totals[i], most);
        sum.v = sum.v * f + sums[i][x] * g;
        sum.total = sum.total * f + totals[i] * g;
        sum.top = most;
    }
    sum.store(a, b, item - b * a.KV, r, live);
}

// Joins the parts of cross_tile_fwd_kernel, which are few: D / 4 threads to a row,
// whole vectors (32768 rows of 64, two parts: 7.8 us, 10 behind the kernel that
// leaves them).
template <int D>
__global__ __launch_bounds__(256) void cross_join_kernel(CrossArgs a) {
    constexpr int LANES = D / 4;
    const int R = a.Sq * a.G, x = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (row >= (int64_t)a.B * a.KV * R) return;
    const int item = (int)(row / R), r = (int)(row - (int64_t)item * R), b = item / a.KV;
    const int live = max(0, min(4, a.D - 4 * x));
    const RowParts parts(a, item, r, live_keys(a, b) > 0);
    if (parts.n == 1) return;
    Joined<LANES> sum;
    sum.add(0, parts.n, live, [&](int s) { return a.part_stats + 2 * parts.at(s); },
            [&](int s) { return a.part + parts.at(s) * a.D; });
    sum.store(a, b, item - b * a.KV, r, live);
}

// A short side in LDS: 16 T rows of two tensors, zeros past `n` and past d_head.
// from(which, row) is where a row begins.
template <int NJ, int T, class F>
__device__ __forceinline__ void fill_short(float (&own)[2][16 * T][16 * NJ + 4], int n, int D,
                                           F from) {
    for (int i = threadIdx.x; i < 2 * 16 * T * 4 * NJ; i += 64 * kRowWaves) {
        const int which = i / (16 * T * 4 * NJ), at = i % (16 * T * 4 * NJ), row = at / (4 * NJ),
                  d = at % (4 * NJ) * 4;
        f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (row < n) {
            const float* const src = from(which, row);
            if (d + 4 <= D)
                v = reinterpret_cast<const Quad*>(src + d)->v;
            else
                for (int e = 0; d + e < D; ++e) v[e] = src[d + e];
        }
        *reinterpret_cast<f32x4*>(&own[which][row][d]) = v;
    }
}

// Adds, over the own rows 4g + r at `rows`, weight[r] (own row, tile's row c) times
// the row: lane (c, g) of to[j] gets column c NJ + j of the tile's rows 4g + r.
template <int NJ>
__device__ __forceinline__ void add_short(f32x4 (&to)[NJ], const float (*rows)[16 * NJ + 4],
                                          f32x4 weight, int c, int g) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float* const src = &rows[4 * g + r][c * NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) to[j] = mfma16(weight[r], src[j], to[j]);
    }
}

// Row 4g + r of a tile, as add_short leaves it, NJ neighbouring columns to a lane:
// 16 lanes store a row one after the other.
template <int NJ>
__device__ __forceinline__ void store_short(float* dst, const f32x4 (&x)[NJ], int r, float f,
                                            float beta, int D, int c) {
#pragma unroll
    for (int j = 0; j < NJ; j += 4) {
        const int d = c * NJ + j;
        if (NJ % 4 == 0 && d + 4 <= D) {
            f32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = x[(j + i) % NJ][r] * f;
            Quad* const to = reinterpret_cast<Quad*>(dst + d);
            if (beta != 0.0f) v = v + beta * to->v;
            to->v = v;
        } else {
#pragma unroll
            for (int i = 0; i < (NJ < 4 ? NJ : 4); ++i) {
                const float v = x[(j + i) % NJ][r] * f;
                if (d + i < D) dst[d + i] = beta != 0.0f ? v + beta * dst[d + i] : v;
            }
        }
    }
}

// The forward of many rows over up to 16 keys: K and V stay in LDS, and the rows
// stream in tiles of 16 that the waves take in turns, read once and written once.
// 8 x 1951 rows of 56 heads, 10 keys, 8 key heads of 96: 156 us, 4.3 TB/s (the
// kernel of many keys 253); 50 x 102 rows of 112 heads, 6 keys, 16 key heads of 40:
// 58 us and 105. With more keys, up to 48, it was faster (57 and 73 us) or slower
// (20 and 17) by the sizes.
template <int NJ>
__global__ __launch_bounds__(64 * kRowWaves) void cross_short_fwd_kernel(CrossArgs a) {
    __shared__ f32x4 shared[2 * 16 * (16 * NJ + 4) / 4];
    float(&own)[2][16][16 * NJ + 4] = *reinterpret_cast<float(*)[2][16][16 * NJ + 4]>(shared);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Sq * a.G, items = a.B * a.KV, item = blockIdx.x % items;
    const int no = blockIdx.x / items, shares = gridDim.x / items;
    const int b = item / a.KV, kv = item - b * a.KV, L = live_keys(a, b);
    fill_short<NJ, 1>(own, L, a.D, [&](int which, int row) {
        return (which ? a.v : a.k) + key_offset(a, b, kv, row);
    });
    __syncthreads();
    const int tiles = (R + 15) / 16, t1 = (int)((int64_t)tiles * (no + 1) / shares);
    for (int t = (int)((int64_t)tiles * no / shares) + w; t < t1; t += kRowWaves) {
        const int r0 = 16 * t, n = min(16, R - r0);
        f32x4 q[NJ], p = f32x4{0.0f, 0.0f, 0.0f, 0.0f}, sum[NJ];
        Rows<true>(a, a.q, b, kv, a.ld_q, r0, n).template along<NJ>(q, c, g);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            q[j] = q[j] * a.scale2;
            sum[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            const f32x4 x = *reinterpret_cast<const f32x4*>(&own[0][c][16 * j + 4 * g]);
#pragma unroll
            for (int e = 0; e < 4; ++e) p = mfma16(x[e], q[j][e], p);
        }
        float top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (4 * g + r < L) top = fmaxf(top, p[r]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            p[r] = 4 * g + r < L ? __builtin_amdgcn_exp2f(p[r] - top) : 0.0f;
            total += p[r];
        }
        add_short<NJ>(sum, own[1], p, c, g);
        total = across_groups(total);
        const float f = L > 0 ? 1.0f / total : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float own_f = __shfl(f, 4 * g + r, 64);
            if (4 * g + r < n)
                store_short<NJ>(a.out + query_offset(a, b, kv, r0 + 4 * g + r, a.ld_out), sum, r,
                                own_f, 0.0f, a.D, c);
        }
        if (a.stats && g == 0 && c < n) {
            float* const st = row_stats(a, b, kv, r0 + c);
            st[0] = L > 0 ? top : 0.0f;
            st[1] = total;
        }
    }
}

// The backward where one side is short (up to 16 T rows of an item, or KEYS:
// keys). The short side is the workgroup's own, X and Y (Q and dO, or K and V) in
// LDS; the long side streams from memory once, in tiles of 16 that the waves take
// in turns, as operands of the f32 matrix instructions. Of a tile
//   S = X Xm^T, dP = Y Ym^T, P = 2^(S - lse), dS = P (dP - delta),
// lane (c, g) with rows 4g + r of X and row c of the tile. Products over the short
// side finish the tile's gradients (dK = scale dS^T Q and dV = P^T dO, or
// dQ = scale dS K); those over the tile, with P and dS turned about in LDS, add to
// the short side's own (dQ, or dK and dV), which the waves and the workgroups that
// share an item join at the end.
// 16 x 5 rows of 112 heads, 5256 keys (16 key heads of 128): 1119 us, of which the
// matrix instructions are some 525 and the 2.8 GB some 560, with a wave to a SIMD;
// 5 x 2 rows, 9000 keys, 4 heads of 128: 109 us, 3.4 TB/s. Three workgroups to a
// compute unit: six took 1262 us in the first and 148 in the second. The next tile
// asked for a tile ahead took 1242 and 121, and 284 in place of 230 at 19 x 4 rows,
// 12867 keys, 3 key heads of 40 (178 now that rows are stored by neighbouring lanes).
template <int NJ, int T, bool KEYS>
__global__ __launch_bounds__(64 * kRowWaves) void cross_short_bwd_kernel(CrossArgs a) {
    constexpr int W = 16 * NJ + 4, OWN = 2 * 16 * T * W, SUMS = kRowWaves * 4 * NJ * 64;
    __shared__ f32x4 shared[(OWN > SUMS ? OWN : SUMS) / 4];
    __shared__ f32x4 turned[kRowWaves][KEYS ? 2 : 1][16][5];
    __shared__ f32x4 starts[2][4 * T];  // !KEYS: -lse and -delta of the own rows
    float(&own)[2][16 * T][W] = *reinterpret_cast<float(*)[2][16 * T][W]>(shared);
    float(&sums)[kRowWaves][4 * NJ][64] = *reinterpret_cast<float(*)[kRowWaves][4 * NJ][64]>(shared);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Sq * a.G, items = a.B * a.KV, item = blockIdx.x % items;
    const int no = blockIdx.x / items, shares = KEYS ? a.kv_splits : a.q_splits;
    const int b = item / a.KV, kv = item - b * a.KV, L = live_keys(a, b);
    const bool finish = KEYS ? a.dq != nullptr : a.dk != nullptr;  // the tiles' gradients
    const bool add = KEYS ? a.dk != nullptr : a.dq != nullptr;     // the short side's
    // live rows of the short side and of the long one, and those to be written
    const int own_n = KEYS ? a.Sk : R, n = KEYS ? L : R;
    const int met = KEYS ? (L > 0 ? R : 0) : L, all = KEYS ? R : a.Sk;
    const float* const lse = a.neg_lse + (int64_t)item * R;
    const float* const delta = a.neg_delta + (int64_t)item * R;
    fill_short<NJ, T>(own, n, a.D, [&](int which, int row) {
        if (KEYS) return (which ? a.v : a.k) + key_offset(a, b, kv, row);
        return which ? a.dout + query_offset(a, b, kv, row, a.ld_out)
                     : a.q + query_offset(a, b, kv, row, a.ld_q);
    });
    if (!KEYS && threadIdx.x < 16 * T) {
        const bool live = (int)threadIdx.x < n;
        reinterpret_cast<float*>(starts[0])[threadIdx.x] = live ? lse[threadIdx.x] : -INFINITY;
        reinterpret_cast<float*>(starts[1])[threadIdx.x] = live ? delta[threadIdx.x] : 0.0f;
    }
    __syncthreads();
    f32x4 acc[T][NJ], acc_y[KEYS ? T : 1][NJ];
#pragma unroll
    for (int ot = 0; ot < T; ++ot)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            acc[ot][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (KEYS) acc_y[ot][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    auto add_met = [&](f32x4(&to)[NJ], const float (&x)[4][NJ], f32x4 weight) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NJ; ++j) to[j] = mfma16(x[r][j], weight[r], to[j]);
    };
    // w[4g + r][c] -> w[c][4g + r]
    auto turn = [&](f32x4 x, int which) {
        f32x4(&at)[16][5] = turned[w][which];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        at[c][g] = x;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        f32x4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = reinterpret_cast<const float*>(at[4 * g + r])[c];
        return y;
    };
    const int tiles = (all + 15) / 16, t1 = (int)((int64_t)tiles * (no + 1) / shares);
    for (int t = (int)((int64_t)tiles * no / shares) + w; t < t1; t += kRowWaves) {
        const int m0 = 16 * t, nm = min(16, met - m0);
        f32x4 dx[NJ], dy[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) dx[j] = dy[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (nm > 0) {
            const Rows<KEYS> xs(a, KEYS ? a.q : a.k, b, kv, KEYS ? a.ld_q : a.ld_kv, m0, nm),
                ys(a, KEYS ? a.dout : a.v, b, kv, KEYS ? a.ld_out : a.ld_kv, m0, nm);
            f32x4 mx[NJ], my[NJ];
            float cx[4][NJ], cy[4][NJ];
            xs.template along<NJ>(mx, c, g);
            ys.template along<NJ>(my, c, g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (add) xs.template across<NJ>(cx[r], 4 * g + r, c);
                if (KEYS && add) ys.template across<NJ>(cy[r], 4 * g + r, c);
            }
            const float met_lse = KEYS && c < nm ? lse[m0 + c] : -INFINITY;
            const float met_delta = KEYS && c < nm ? delta[m0 + c] : 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) mx[j] = mx[j] * a.scale2;
#pragma unroll
            for (int ot = 0; ot < T; ++ot) {
                if (16 * ot >= n) break;
                f32x4 p = f32x4{0.0f, 0.0f, 0.0f, 0.0f}, ds = p;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int at = 16 * j + 4 * g;
                    const f32x4 x = *reinterpret_cast<const f32x4*>(&own[0][16 * ot + c][at]),
                                y = *reinterpret_cast<const f32x4*>(&own[1][16 * ot + c][at]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p = mfma16(x[e], mx[j][e], p);
                        ds = mfma16(y[e], my[j][e], ds);
                    }
                }
                const f32x4 nl = starts[0][4 * ot + g], nd = starts[1][4 * ot + g];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool live = c < nm && 16 * ot + 4 * g + r < n;
                    p[r] = live ? __builtin_amdgcn_exp2f(p[r] + (KEYS ? met_lse : nl[r])) : 0.0f;
                    ds[r] = live ? p[r] * (ds[r] + (KEYS ? met_delta : nd[r])) : 0.0f;
                }
                if (finish) {
                    add_short<NJ>(dx, &own[0][16 * ot], ds, c, g);
                    if (!KEYS) add_short<NJ>(dy, &own[1][16 * ot], p, c, g);
                }
                if (add) {
                    add_met(acc[ot], cx, turn(ds, 0));
                    if constexpr (KEYS) add_met(acc_y[ot], cy, turn(p, 1));
                }
            }
        }
        if (finish) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = 4 * g + r;
                if (m0 + m >= all) continue;
                if (KEYS) {
                    store_short<NJ>(a.dq + query_offset(a, b, kv, m0 + m, a.ld_q), dx, r, a.scale,
                                    a.beta_q, a.D, c);
                } else if (m < nm || a.beta_kv != 1.0f) {  // else a dead key's, left as it is
                    const int64_t at = key_offset(a, b, kv, m0 + m);
                    store_short<NJ>(a.dk + at, dx, r, a.scale, a.beta_kv, a.D, c);
                    store_short<NJ>(a.dv + at, dy, r, 1.0f, a.beta_kv, a.D, c);
                }
            }
        }
    }
    if (!add) return;
#pragma unroll
    for (int ot = 0; ot < T; ++ot) {
        if (16 * ot >= own_n) break;
#pragma unroll
        for (int which = 0; which < (KEYS ? 2 : 1); ++which) {
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    sums[w][r * NJ + j][lane] = which ? acc_y[KEYS ? ot : 0][j][r] : acc[ot][j][r];
            __syncthreads();
            const int o = 16 * ot + c;
            // (shares of dead keys are not looked at, and a beta of 1 leaves them)
            const bool left = KEYS && o >= n && (shares > 1 || a.beta_kv == 1.0f);
            if (o < own_n && !left) {
                float* const dst =
                    shares > 1 ? (!KEYS ? a.dq_part : which ? a.dv_part : a.dk_part) +
                                     (((int64_t)no * items + item) * own_n + o) * a.D
                    : !KEYS    ? a.dq + query_offset(a, b, kv, o, a.ld_q)
                               : (which ? a.dv : a.dk) + key_offset(a, b, kv, o);
                const float f = shares > 1 || which ? 1.0f : a.scale;
                const float beta = shares > 1 ? 0.0f : KEYS ? a.beta_kv : a.beta_q;
                // wave w adds the waves' register w: NJ neighbouring columns of o
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    float v = 0.0f;
#pragma unroll
                    for (int i = 0; i < kRowWaves; ++i) v += sums[i][w * NJ + j][lane];
                    const int d = (4 * g + w) * NJ + j;
                    if (d < a.D) dst[d] = beta != 0.0f ? v * f + beta * dst[d] : v * f;
                }
            }
        }
    }
}

template <int NJ, bool KEYS>
void launch_short(const CrossArgs& a) {
    const int n = KEYS ? a.Sk : a.Sq * a.G;
    auto kernel = n <= 16   ? cross_short_bwd_kernel<NJ, 1, KEYS>
                  : n <= 32 ? cross_short_bwd_kernel<NJ, 2, KEYS>
                            : cross_short_bwd_kernel<NJ, 3, KEYS>;
    const unsigned blocks = (unsigned)(a.B * a.KV * (KEYS ? a.kv_splits : a.q_splits));
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kRowWaves), 0, stream(), a);
}

// Adds the shares of a gradient in order: dst = f * sum + beta * dst, D / 4
// threads to a row (8192 keys of 4 heads of 128, two shares: 16 us). KEYS: rows are keys (dead ones have no shares), blockIdx.y
// is 0 for dk and 1 for dv.
template <int D, bool KEYS>
__global__ __launch_bounds__(256) void cross_sum_kernel(CrossArgs a) {
    constexpr int LANES = D / 4;
    const int n = KEYS ? a.Sk : a.Sq * a.G, x = threadIdx.x % LANES;
    const int64_t at = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const int64_t rows = (int64_t)a.B * a.KV * n;
    if (at >= rows) return;
    const int item = (int)(at / n), r = (int)(at - (int64_t)item * n);
    const int b = item / a.KV, kv = item - b * a.KV;
    const bool live = !KEYS || r < live_keys(a, b), second = KEYS && blockIdx.y == 1;
    const float beta = KEYS ? a.beta_kv : a.beta_q, f = second ? 1.0f : a.scale;
    if (!live && beta == 1.0f) return;
    const float* part = (KEYS ? (second ? a.dv_part : a.dk_part) : a.dq_part) + at * a.D + 4 * x;
    float* dst = (KEYS ? (second ? a.dv : a.dk) + key_offset(a, b, kv, r)
                       : a.dq + query_offset(a, b, kv, r, a.ld_q)) + 4 * x;
    const int shares = live ? (KEYS ? a.kv_splits : a.q_splits) : 0;
    if (4 * x + 4 <= a.D) {
        f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int s = 0; s < shares; ++s)
            v = v + reinterpret_cast<const Quad*>(part + s * rows * a.D)->v;
        v = v * f;
        Quad* const to = reinterpret_cast<Quad*>(dst);
        if (beta != 0.0f) v = v + beta * to->v;
        to->v = v;
    } else {
        for (int e = 0; 4 * x + e < a.D; ++e) {
            float v = 0.0f;
            for (int s = 0; s < shares; ++s) v += part[s * rows * a.D + e];
            dst[e] = beta != 0.0f ? v * f + beta * dst[e] : v * f;
        }
    }
}

template <int D>
void launch_sums(const CrossArgs& a, int64_t rows, int64_t keys, bool dq, bool dkv) {
    constexpr int PER = 1024 / D;
    if (dq)
        hipLaunchKernelGGL((cross_sum_kernel<D, false>), dim3((unsigned)((rows + PER - 1) / PER)),
                           dim3(256), 0, stream(), a);
    if (dkv)
        hipLaunchKernelGGL((cross_sum_kernel<D, true>), dim3((unsigned)((keys + PER - 1) / PER), 2),
                           dim3(256), 0, stream(), a);
}

template <class F>
void for_width(int d, F f) {
    if (d <= 16)
        f(std::integral_constant<int, 1>());
    else if (d <= 32)
        f(std::integral_constant<int, 2>());
    else if (d <= 64)
        f(std::integral_constant<int, 4>());
    else
        f(std::integral_constant<int, 8>());
}

constexpr int64_t kMaxLd = 1 << 20, kMaxLen = 1 << 26, kMaxGroups = 1 << 22;

const char* refusal(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_k,
                    int64_t d_head, int64_t ld_q, int64_t ld_kv, int64_t ld_out) {
    if (batch < 0 || seq_q < 0 || seq_k < 0 || heads < 1 || kv_heads < 1)
        return "a size is negative or there are no heads";
    if (heads % kv_heads != 0) return "heads must be a multiple of kv_heads";
    if (d_head < 1 || d_head > 128) return "d_head must be 1 to 128";
    if (heads > kMaxLd / d_head || ld_q < heads * d_head || ld_out < heads * d_head ||
        ld_kv < kv_heads * d_head)
        return "a row stride is shorter than its heads";
    if (ld_q > kMaxLd || ld_kv > kMaxLd || ld_out > kMaxLd) return "a row stride is past 2^20";
    if (seq_q > kMaxLen || seq_k > kMaxLen) return "a length is past 2^26";
    // A launch has fewer than 2^32 threads, 256 for 16 rows or keys at most. Each
    // factor is below 2^47: divided, not multiplied.
    const int64_t rows = (seq_q * (heads / kv_heads) + 15) / 16, keys = (seq_k + 15) / 16;
    if (std::max<int64_t>({rows, keys, 1}) > kMaxGroups / kv_heads ||
        batch > kMaxGroups / kv_heads / std::max<int64_t>({rows, keys, 1}))
        return "more than 2^26 rows or keys (in groups of 16 of an item)";
    return nullptr;
}

}  // namespace

int cross_check_shape(const char* what, int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q,
                      int64_t seq_k, int64_t d_head, int64_t ld_q, int64_t ld_kv, int64_t ld_out) {
    const char* why =
        refusal(batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv, ld_out);
    NRS_ARG_CHECK(!why,
                  "%s: %s (batch %lld, heads %lld, kv_heads %lld, seq_q %lld, seq_k %lld, d_head "
                  "%lld, ld_q %lld, ld_kv %lld, ld_out %lld)",
                  what, why, (long long)batch, (long long)heads, (long long)kv_heads,
                  (long long)seq_q, (long long)seq_k, (long long)d_head, (long long)ld_q,
                  (long long)ld_kv, (long long)ld_out);
    return NRS_OK;
}

}  // namespace nrs

extern "C" {

int nrs_cross_attention_supported(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q,
                                  int64_t seq_k, int64_t d_head, int64_t ld_q, int64_t ld_kv,
                                  int64_t ld_out) {
    return nrs::refusal(batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv, ld_out) ? 0 : 1;
}

int nrs_cross_attention_workspace(size_t* bytes, int64_t batch, int64_t heads, int64_t kv_heads,
                                  int64_t seq_q, int64_t seq_k, int64_t d_head, int backward) {
    NRS_ARG_CHECK(bytes, "cross attention workspace: null pointer");
    if (int rc = nrs::cross_check_shape("cross attention workspace", batch, heads, kv_heads, seq_q,
                                  seq_k, d_head, nrs::kMaxLd, nrs::kMaxLd, nrs::kMaxLd))
        return rc;
    const int cus = nrs::num_cus();
    *bytes =
        backward
            ? nrs::plan_cross_backward(batch, heads, kv_heads, seq_q, seq_k, d_head, cus).bytes()
            : nrs::plan_cross_forward(batch, heads, kv_heads, seq_q, seq_k, d_head, cus).bytes();
    return NRS_OK;
}

int nrs_cross_attention_forward(float* out, float* stats, const float* q, const float* k,
                                const float* v, const int32_t* key_len, int64_t batch,
                                int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_k,
                                int64_t d_head, int64_t ld_q, int64_t ld_kv, int64_t ld_out,
                                float scale, void* work, size_t work_bytes) {
    const char* what = "cross attention forward";
    if (int rc = nrs::cross_check_shape(what, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                                  ld_out))
        return rc;
    if (batch == 0 || seq_q == 0) return NRS_OK;
    NRS_ARG_CHECK(out && q && ((k && v) || seq_k == 0), "%s: null pointer", what);
    NRS_REQUIRE_INIT();
    if (int rc = nrs::check_device(what)) return rc;
    const auto plan = nrs::plan_cross_forward(batch, heads, kv_heads, seq_q, seq_k, d_head,
                                              nrs::num_cus());
    const int64_t rows = batch * heads * seq_q;
    float* scratch = nullptr;
    if (int rc = nrs::call_scratch(&scratch, plan.bytes(), work, work_bytes, what)) return rc;
    nrs::CrossArgs a{};
    a.unit_rows = plan.unit_rows;
    a.groups = plan.groups;
    a.few_units = plan.few_units;
    a.part = scratch;
    a.part_stats = scratch + plan.part;
    a.shares = reinterpret_cast<int32_t*>(scratch + plan.part + plan.stats);
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.stats = stats;
    a.key_len = key_len;
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
    a.by_group = nrs::make_fastdiv((uint32_t)a.G);
    a.scale = scale;
    a.scale2 = scale * 1.4426950408889634f;
    if (plan.few_keys) {
        nrs::for_width(a.D, [&](auto nj) {
            hipLaunchKernelGGL(nrs::cross_short_fwd_kernel<decltype(nj)::value>,
                               dim3((unsigned)plan.blocks), dim3(64 * nrs::kRowWaves), 0,
                               nrs::stream(), a);
        });
    } else if (plan.tiles) {
        nrs::cross_tile_forward(a, (unsigned)plan.blocks);
    } else {
        nrs::for_width(a.D, [&](auto nj) {
            hipLaunchKernelGGL(nrs::cross_rows_fwd_kernel<decltype(nj)::value>,
                               dim3((unsigned)plan.blocks), dim3(64 * nrs::kRowWaves), 0,
                               nrs::stream(), a);
        });
    }
    NRS_LAUNCH_CHECK(what);
    if (a.groups > 0 && !plan.tiles) {
        hipLaunchKernelGGL(nrs::cross_rows_join_kernel, dim3((unsigned)rows), dim3(256), 0,
                           nrs::stream(), a);
    } else if (a.groups > 0) {
        const int width = nrs::cross_row_width(a.D), per = 1024 / width;
        auto join = width == 32   ? nrs::cross_join_kernel<32>
                    : width == 64 ? nrs::cross_join_kernel<64>
                                  : nrs::cross_join_kernel<128>;
        hipLaunchKernelGGL(join, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0,
                           nrs::stream(), a);
    }
    NRS_LAUNCH_CHECK(what);
    return NRS_OK;
}

int nrs_cross_attention_backward(float* dq, float* dk, float* dv, const float* dout,
                                 const float* out, const float* q, const float* k, const float* v,
                                 const float* stats, const int32_t* key_len, int64_t batch,
                                 int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_k,
                                 int64_t d_head, int64_t ld_q, int64_t ld_kv, int64_t ld_out,
                                 float scale, float beta_q, float beta_kv, void* work,
                                 size_t work_bytes) {
    const char* what = "cross attention backward";
    if (int rc = nrs::cross_check_shape(what, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                                  ld_out))
        return rc;
    NRS_ARG_CHECK((dk == nullptr) == (dv == nullptr), "%s: dk and dv go together", what);
    if (batch == 0) return NRS_OK;
    const bool rows = seq_q > 0, keys = seq_k > 0;
    NRS_ARG_CHECK((!rows || (dout && out && q && stats)) && (!keys || (k && v)),
                  "%s: null pointer", what);
    NRS_REQUIRE_INIT();
    if (int rc = nrs::check_device(what)) return rc;
    const auto plan = nrs::plan_cross_backward(batch, heads, kv_heads, seq_q, seq_k, d_head,
                                               nrs::num_cus());
    float* scratch = nullptr;
    if (int rc = nrs::call_scratch(&scratch, plan.bytes(), work, work_bytes, what)) return rc;
    nrs::CrossArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.dout = dout;
    a.o = out;
    a.stats = const_cast<float*>(stats);  // only read here
    a.dq = dq;
    a.dk = dk;
    a.dv = dv;
    a.key_len = key_len;
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
    a.by_group = nrs::make_fastdiv((uint32_t)a.G);
    a.scale = scale;
    a.scale2 = scale * 1.4426950408889634f;  // as the forward computed it
    a.beta_q = beta_q;
    a.beta_kv = beta_kv;
    a.q_splits = plan.q_splits;
    a.kv_splits = plan.kv_splits;
    a.neg_lse = scratch;
    a.neg_delta = scratch + plan.rows;
    a.dq_part = scratch + plan.prepared;
    a.dk_part = a.dq_part + plan.q_part;
    a.dv_part = a.dk_part + plan.kv_part;
    if (!rows) a.dq = nullptr;
    if (!keys) a.dk = a.dv = nullptr;
    const bool is_short = plan.short_rows || plan.short_keys;
    nrs::cross_tile_backward(a, is_short);
    if (is_short && (a.dq || a.dk)) {
        nrs::for_width(a.D, [&](auto nj) {
            constexpr int NJ = decltype(nj)::value;
            (plan.short_rows ? nrs::launch_short<NJ, false> : nrs::launch_short<NJ, true>)(a);
        });
    }
    const int width = nrs::cross_row_width(a.D);
    const bool sum_q = a.dq && plan.q_splits > 1, sum_kv = a.dk && plan.kv_splits > 1;
    auto sums = width == 32   ? nrs::launch_sums<32>
                : width == 64 ? nrs::launch_sums<64>
                              : nrs::launch_sums<128>;
    sums(a, plan.rows, plan.keys, sum_q, sum_kv);
    NRS_LAUNCH_CHECK(what);
    return NRS_OK;
}

}  // extern "C"
