// Cross attention of many rows, forward and backward, on the bf16 matrix
// cores.
//
// A float is the exact sum of three bf16 pieces, and the six largest of the
// nine products of two floats' pieces give their product to 2^-24
// (gemm_split.hpp tells why that is as good as f32): 2.7 times the rate of the
// f32 matrix instructions.
//
// A workgroup of WAVES waves owns 32 * WAVES rows (or keys) of an item, 32 to
// a wave, held as split operands in registers, and walks the item's keys (or
// rows) in tiles through LDS. With "own" and "met" for the two sides, a wave
// computes met . own^T on v_mfma_f32_32x32x16_bf16: lane (c, h) = (lane % 32,
// lane / 32) gets 16 products of ONE of its own, c, with the met
// 8 (i / 4) + 4h + i % 4 of a block of 32. So
//   - the forward's softmax over the keys it meets is lane-local but for one
//     exchange with lane c ^ 32;
//   - registers 8u .. 8u + 7, split, are k-step u of the operand of
//     acc^T[d][own] += met^T[d][met] . w[met][own] as they lie: O += V^T P,
//     dQ += K^T dS (own rows), dV += dO^T P, dK += Q^T dS (own keys).
// met^T is read from the same LDS copy as met, by transposing reads.
//
// Tiles are split once per workgroup, on their way into LDS, as three planes
// of 16-byte units (one lane's operand): unit q of a row holds d = 4q .. 4q + 3
// and D/2 + 4q .. D/2 + 4q + 3, so that a row's lanes load whole segments. The
// next tile is loaded to registers while this one is multiplied, and stored to
// the other of two buffers.
//
// The forward's softmax is online in base 2, against a reference m that
// follows the running maximum only when that passes it by 2^8: sums of
// probabilities up to 256 lose nothing in f32, and most tiles need no
// rescaling of the accumulators. The products start from -m, so the exponent
// needs no subtraction. (The backward subtracts: -log2 of a row's sum is larger
// than the scores that matter, and every rounding on the way would be of its
// size. dout . out is small, and dout . v starts from its negative.)
//
// What bounds it is the SIMD's issue: a product's six matrix instructions take
// 32 cycles each, and the exponentials, splits and transposing reads between
// them about 5 an instruction, of which two waves to a SIMD hide a part.
//   rows x keys, heads of d          forward          backward
//   32 x 128 x 200, 8 of 32           12.7 us            27 us
//   4 x 1000 x 1500, 16 of 64          124 (198 TFLOP/s) 430 (143; 200 with the
//                                                        two products it repeats)
//   2 x 777 x 4096, 16 of 128, 4 key   233 (176)         869 (118; 165)
// (medians late in two hundred passes on the same inputs: after a pause the first dozen
// take 15 to 40% longer, as the clocks settle). In the last two backwards, of the time that a compute unit has work, matrix
// instructions run 53% and 49%, vector instructions issue 46% and 35%, and LDS is busy
// 45% and 42%; in the last, compute units have none for a fifth of the launch, as walks
// end at different times.
#include <algorithm>

#include "cross_attention.hpp"

namespace nrs {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The three pieces of 8 floats: an operand of the matrix instructions each.
__device__ __forceinline__ void split8(const float (&x)[8], u32x4 (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint32_t w = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
            p[n][i] = w;
            a -= __builtin_bit_cast(float, w << 16);
            b -= __builtin_bit_cast(float, w & 0xffff0000u);
        }
        p[2][i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b),
                                        __builtin_bit_cast(uint32_t, a), 0x07060302u);
    }
}

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// c += a . b from their pieces, the smallest products first.
__device__ __forceinline__ f32x16 mfma_split(const u32x4 (&a)[3], const u32x4 (&b)[3], f32x16 c) {
    c = mfma32(a[2], b[0], c);
    c = mfma32(a[1], b[1], c);
    c = mfma32(a[0], b[2], c);
    c = mfma32(a[1], b[0], c);
    c = mfma32(a[0], b[1], c);
    return mfma32(a[0], b[0], c);
}

__device__ __forceinline__ f32x16 all16(float x) {
    f32x16 v;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = x;
    return v;
}

// One wave to a SIMD when a wide head's operands fill its registers.
constexpr int waves_per_simd(int D, int waves) { return D > 96 && waves == 4 ? 1 : 2; }

template <int D_, int WAVES_>
struct TileCfg {
    static constexpr int D = D_, WAVES = WAVES_, NT = 64 * WAVES;
    static constexpr int KT = cross_tile_keys(D, WAVES);  // rows of a tile
    static constexpr int Q = D / 8;           // units of a row
    static constexpr int PLANE = KT * Q;      // units of a plane
    static constexpr int U = (PLANE + NT - 1) / NT;  // units a thread stages at most
    static constexpr int SET = 3 * PLANE;     // units of a tensor's tile
    static constexpr int NS = D / 16, NJ = D / 32, NB = KT / 32;
    static_assert(KT % 32 == 0 && D % 32 == 0, "blocks of 32");
    // Whether unit i is one of the tile (the last ones of a thread may not be).
    __device__ static constexpr bool has(int i) { return U * NT == PLANE || i < PLANE; }
};

// Unit q of row r in a plane: the 32 rows of a block are contiguous for the
// operand reads; the exclusive or sends the units of a row, which neighbouring
// lanes store, to different 16-byte columns, and units q and q + 2, which a
// transposing read takes together, to different 64-byte ones.
template <class C>
__device__ __forceinline__ constexpr int mix(int q) {
    return ((q ^ (q << 1)) * (C::Q < 8 ? 8 / C::Q : 1)) & 31;
}
template <class C>
__device__ __forceinline__ int unit_at(int r, int q) {
    return ((r >> 5) * C::Q + q) * 32 + ((r & 31) ^ mix<C>(q));
}

// A tile of a tensor on its way from global memory to LDS: thread t stages
// unit i % Q of row i / Q, i = t + NT u.
template <class C, bool FULL>
struct Stage {
    f32x4 x[C::U][2];

    // Rows r0 .. r0 + n - 1 of an item's keys, or (QUERY) of its rows.
    template <bool QUERY>
    __device__ __forceinline__ void load(const CrossArgs& a, const float* base, int ld, int b,
                                         int kv, int r0, int n) {
        int first = r0;
        int64_t at, floats;
        if (QUERY) {
            first = (int)fast_div((uint32_t)r0, a.by_group);
            const int last = (int)fast_div((uint32_t)(r0 + n - 1), a.by_group);
            at = ((int64_t)b * a.Sq + first) * ld + (int64_t)kv * a.G * a.D;
            floats = (int64_t)(last - first) * ld + a.G * a.D;
        } else {
            at = key_offset(a, b, kv, r0);
            floats = (int64_t)(n - 1) * ld + a.D;
        }
        const auto rs = buffer_rsrc(base + at, floats * 4);
#pragma unroll
        for (int u = 0; u < C::U; ++u) {
            const int i = threadIdx.x + C::NT * u, row = i / C::Q, q = i % C::Q;
            int off = row * ld;
            if (QUERY) {
                const int r = r0 + row, s = (int)fast_div((uint32_t)r, a.by_group);
                off = (s - first) * ld + (r - s * a.G) * a.D;
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int d = 4 * q + s * (C::D / 2);
                x[u][s] = buffer_load4(
                    rs, C::has(i) && row < n && (FULL || d < a.D) ? (off + d) * 4 : kOutOfRange);
            }
        }
    }

    __device__ __forceinline__ void store(const CrossArgs& a, u32x4* lds) const {
#pragma unroll
        for (int u = 0; u < C::U; ++u) {
            const int i = threadIdx.x + C::NT * u, row = i / C::Q, q = i % C::Q;
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = x[u][e / 4][e % 4];
                // what follows the head in its row is not part of it
                if (!FULL && 4 * q + e % 4 + (e / 4) * (C::D / 2) >= a.D) f[e] = 0.0f;
            }
            u32x4 p[3];
            split8(f, p);
#pragma unroll
            for (int n = 0; n < 3; ++n)
                if (C::has(i)) lds[n * C::PLANE + unit_at<C>(row, q)] = p[n];
        }
    }
};

// The lane's operands of its own row at `src` (zeros unless live), times f.
template <class C, bool FULL>
__device__ __forceinline__ void own_pieces(u32x4 (&own)[C::NS][3], const CrossArgs& a,
                                           const float* src, bool live, int h, float f) {
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = 4 * (2 * s + h) + e * (C::D / 2);
            f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (live) {
                if (FULL || d + 4 <= a.D) {
                    v = reinterpret_cast<const Quad*>(src + d)->v;
                } else {
                    for (int i = 0; i < 4; ++i)
                        if (d + i < a.D) v[i] = src[d + i];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * e + i] = v[i] * f;
        }
        split8(x, own[s]);
    }
}

// The operand of step s of the rows of block kb of a tile.
template <class C>
__device__ __forceinline__ u32x4 met_piece(const u32x4* set, int kb, int s, int p, int c, int h) {
    return set[p * C::PLANE + unit_at<C>(kb * 32 + c, 2 * s + h)];
}

// start + met . own^T of block kb of a tile.
template <class C>
__device__ __forceinline__ f32x16 products(const u32x4* set, const u32x4 (&own)[C::NS][3], int kb,
                                           f32x16 start, int c, int h) {
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
        u32x4 met[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) met[p] = met_piece<C>(set, kb, s, p, c, h);
        start = mfma_split(met, own[s], start);
    }
    return start;
}

// The same with fewer roundings: the five small products of all steps, then
// the large ones. An instruction rounds its sum twice, and the small ones'
// sum is 2^-7 of the whole, so that is rounded 2 NS times in place of 12 NS.
template <class C>
__device__ __forceinline__ f32x16 close_products(const u32x4* set, const u32x4 (&own)[C::NS][3],
                                                 int kb, f32x16 start, int c, int h) {
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
        u32x4 met[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) met[p] = met_piece<C>(set, kb, s, p, c, h);
        start = mfma32(met[2], own[s][0], start);
        start = mfma32(met[1], own[s][1], start);
        start = mfma32(met[0], own[s][2], start);
        start = mfma32(met[1], own[s][0], start);
        start = mfma32(met[0], own[s][1], start);
    }
    // (read again: the registers cannot hold the first pieces until now)
    asm volatile("" : "+v"(c));
#pragma unroll
    for (int s = 0; s < C::NS; ++s)
        start = mfma32(met_piece<C>(set, kb, s, 0, c, h), own[s][0], start);
    return start;
}

// A transposing read: lanes 4e + x of a group of 16 give the places of four
// 16-bit values each, x of row e; lane j gets values j of the four rows.
__device__ __forceinline__ u32x2 read_transposed(const u32x2* p) {
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    return __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (lds_ptr)(__attribute__((address_space(3))) void*)const_cast<u32x2*>(p)));
}

// acc[j] += met^T . w for k-step u of block kb, w split. Of the 32 places m of
// output block j, 16 tt + 4x + y is d = 4 (4j + 2 (x / 2) + tt) + (x % 2) D/2 + y:
// each x a half of one unit.
template <class C>
__device__ __forceinline__ void add_transposed(f32x16 (&acc)[C::NJ], const u32x4* set, int kb,
                                               int u, const u32x4 (&w)[3], int lane) {
    const int x = lane & 3, e = (lane >> 2) & 3, tt = (lane >> 4) & 1, h = lane >> 5;
    const int q0 = 2 * (x >> 1) + tt;
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) {
        u32x4 met[3];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int unit = unit_at<C>(kb * 32 + 16 * u + 8 * half + 4 * h + e, 4 * j + q0);
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const u32x2 v = read_transposed(
                    reinterpret_cast<const u32x2*>(set + p * C::PLANE + unit) + (x & 1));
                met[p][2 * half] = v[0];
                met[p][2 * half + 1] = v[1];
            }
        }
        acc[j] = mfma_split(met, w, acc[j]);
    }
}

// Stores a lane's acc * f (+ beta * old) into its own row of d_head floats.
template <class C, bool FULL>
__device__ __forceinline__ void store_own(float* dst, const f32x16 (&acc)[C::NJ], float f,
                                          float beta, int D, int h) {
#pragma unroll
    for (int j = 0; j < C::NJ; ++j)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = 4 * (4 * j + 2 * ((i / 4) % 2) + i / 8) + h * (C::D / 2);
            f32x4 v = f32x4{acc[j][i], acc[j][i + 1], acc[j][i + 2], acc[j][i + 3]} * f;
            if (FULL || d + 4 <= D) {
                Quad* const to = reinterpret_cast<Quad*>(dst + d);
                if (beta != 0.0f) v = v + beta * to->v;
                to->v = v;
            } else {
                for (int e = 0; e < 4; ++e)
                    if (d + e < D) dst[d + e] = beta != 0.0f ? v[e] + beta * dst[d + e] : v[e];
            }
        }
}

// The part of `count` that share number `no` of `shares` walks.
__device__ __forceinline__ void share(int count, int no, int shares, int& from, int& to) {
    from = (int)((int64_t)count * no / shares);
    to = (int)((int64_t)count * (no + 1) / shares);
}

// Key tiles t0 .. t1 - 1 of the rows of row tile `tile` of (b, kv), L live keys:
// all of them (slot < 0) or a part.
template <int D, int WAVES, bool FULL>
__device__ __forceinline__ void forward_walk(const CrossArgs& a,
                                             u32x4 (&lds)[2][2 * TileCfg<D, WAVES>::SET], int b,
                                             int kv, int tile, int L, int t0, int t1,
                                             int64_t slot) {
    using C = TileCfg<D, WAVES>;
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Sq * a.G, row = (tile * WAVES + w) * 32 + c;
    const bool wave_live = (tile * WAVES + w) * 32 < R, live = row < R;
    Stage<C, FULL> k, v;
    auto load = [&](int t) {
        const int n = min(C::KT, L - t * C::KT);
        k.template load<false>(a, a.k, a.ld_kv, b, kv, t * C::KT, n);
        v.template load<false>(a, a.v, a.ld_kv, b, kv, t * C::KT, n);
    };
    if (t0 < t1) load(t0);
    u32x4 qf[C::NS][3];
    own_pieces<C, FULL>(qf, a, a.q + (live ? query_offset(a, b, kv, row, a.ld_q) : 0), live, h,
                        a.scale2);
    f32x16 acc[C::NJ], start = all16(0.0f);  // start: -m, where the scores start
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc[j] = all16(0.0f);
    float m = 0.0f, l = 0.0f;
    if (t0 < t1) {
        k.store(a, lds[0]);
        v.store(a, lds[0] + C::SET);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        const u32x4* const kl = lds[(t - t0) & 1];
        const u32x4* const vl = kl + C::SET;
        if (wave_live) {
            const int n = L - t * C::KT;  // live keys of the tile, or more
            f32x16 s[C::NB];
#pragma unroll
            for (int kb = 0; kb < C::NB; ++kb) s[kb] = products<C>(kl, qf, kb, start, c, h);
            if (n < C::KT) {
#pragma unroll
                for (int kb = 0; kb < C::NB; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (kb * 32 + 8 * (i / 4) + 4 * h + i % 4 >= n) s[kb][i] = -INFINITY;
            }
            float top = s[0][0];
#pragma unroll
            for (int kb = 0; kb < C::NB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const bool first = t == t0;
            if (__any(first || top > 8.0f)) {
                const float shift = first || top > 8.0f ? top : 0.0f;
                const float alpha = first ? 0.0f : __builtin_amdgcn_exp2f(-shift);
                m += shift;
                l *= alpha;
                start = all16(-m);
#pragma unroll
                for (int kb = 0; kb < C::NB; ++kb) s[kb] = s[kb] - shift;
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
                        x[i] = __builtin_amdgcn_exp2f(s[kb][8 * u + i]);
                        l += x[i];
                    }
                    u32x4 p[3];
                    split8(x, p);
                    add_transposed<C>(acc, vl, kb, u, p, lane);
                }
        }
        if (t + 1 < t1) {
            // the other buffer was last read in step t - 1, which every wave
            // had left before the barrier that ended it
            k.store(a, lds[(t + 1 - t0) & 1]);
            v.store(a, lds[(t + 1 - t0) & 1] + C::SET);
            if (t + 2 < t1) load(t + 2);
            __syncthreads();
        }
    }
    l += __shfl_xor(l, 32, 64);
    if (!live) return;
    const bool whole = slot < 0;
    const int64_t at = slot * a.unit_rows + w * 32 + c;
    store_own<C, FULL>(whole ? a.out + query_offset(a, b, kv, row, a.ld_out) : a.part + at * a.D,
                       acc, !whole ? 1.0f : L > 0 ? 1.0f / l : 0.0f, 0.0f, a.D, h);
    if (h == 0 && (!whole || a.stats)) {
        float* st = whole ? row_stats(a, b, kv, row) : a.part_stats + 2 * at;
        st[0] = m;
        st[1] = l;
    }
}

template <int D, int WAVES, bool FULL>
__global__ __launch_bounds__(64 * WAVES, waves_per_simd(D, WAVES)) void cross_tile_fwd_kernel(
    CrossArgs a) {
    using C = TileCfg<D, WAVES>;
    __shared__ u32x4 lds[2][2 * C::SET];
    __shared__ int scan[WAVES], found[2];
    const int tiles = (a.Sq * a.G + 32 * WAVES - 1) / (32 * WAVES), per_item = a.KV * tiles;
    if (a.groups == 0) {
        const int unit = blockIdx.x, b = unit / per_item, sub = unit - b * per_item;
        const int L = live_keys(a, b);
        forward_walk<D, WAVES, FULL>(a, lds, b, sub / tiles, sub % tiles, L, 0,
                                     (L + C::KT - 1) / C::KT, -1);
        return;
    }
    LinePart<64 * WAVES> part;
    if (!part.begin(a, per_item, C::KT, scan, found)) return;
    while (part.next(a)) {
        forward_walk<D, WAVES, FULL>(a, lds, part.b, part.sub / tiles, part.sub % tiles, part.L,
                                     part.t0, part.t1, part.slot(a));
        __syncthreads();  // before the next piece's tiles take the place of this one's
    }
}

// What the backward starts its products from: per row -log2 of its sum of
// exponentials (-infinity where no key is live: no probability) and
// -dout . out. D / 4 lanes to a row, four columns each.
template <int D>
__global__ __launch_bounds__(256) void cross_rows_prepare_kernel(CrossArgs a) {
    constexpr int LANES = D / 4;
    const int R = a.Sq * a.G, x = threadIdx.x % LANES;
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
        a.neg_lse[at] = live_keys(a, b) > 0 ? -(st[0] + __builtin_amdgcn_logf(st[1])) : -INFINITY;
        a.neg_delta[at] = -dot;
    }
}

// dq of a workgroup's rows: P = 2^(k . q - lse), dS = P (v . dout - delta),
// dQ = scale * K^T dS.
template <int D, int WAVES, bool FULL>
__device__ __forceinline__ void dq_walk(const CrossArgs& a, u32x4* lds, int block) {
    using C = TileCfg<D, WAVES>;
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Sq * a.G, tiles = (R + 32 * WAVES - 1) / (32 * WAVES), items = a.B * a.KV;
    const int tile = block % tiles, item = block / tiles % items, no = block / tiles / items;
    const int b = item / a.KV, kv = item - b * a.KV, L = live_keys(a, b);
    const int row = (tile * WAVES + w) * 32 + c;
    const bool wave_live = (tile * WAVES + w) * 32 < R, live = row < R;
    int t0, t1;
    share((L + C::KT - 1) / C::KT, no, a.q_splits, t0, t1);
    Stage<C, FULL> k, v;
    auto load = [&](int t) {
        const int n = min(C::KT, L - t * C::KT);
        k.template load<false>(a, a.k, a.ld_kv, b, kv, t * C::KT, n);
        v.template load<false>(a, a.v, a.ld_kv, b, kv, t * C::KT, n);
    };
    if (t0 < t1) load(t0);
    u32x4 qf[C::NS][3], gf[C::NS][3];
    own_pieces<C, FULL>(qf, a, a.q + (live ? query_offset(a, b, kv, row, a.ld_q) : 0), live, h,
                        a.scale2);
    own_pieces<C, FULL>(gf, a, a.dout + (live ? query_offset(a, b, kv, row, a.ld_out) : 0), live, h,
                        1.0f);
    const float nl = live ? a.neg_lse[(int64_t)item * R + row] : -INFINITY;
    const float nd = live ? a.neg_delta[(int64_t)item * R + row] : 0.0f;
    f32x16 acc[C::NJ];
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc[j] = all16(0.0f);
    if (t0 < t1) {
        k.store(a, lds);
        v.store(a, lds + C::SET);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        u32x4* const kl = lds + ((t - t0) & 1) * 2 * C::SET;
        if (wave_live) {
            const int n = L - t * C::KT;
#pragma unroll
            for (int kb = 0; kb < C::NB; ++kb) {
                f32x16 s = close_products<C>(kl, qf, kb, all16(0.0f), c, h);
                const f32x16 dp = products<C>(kl + C::SET, gf, kb, all16(nd), c, h);
                if (n < C::KT) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (kb * 32 + 8 * (i / 4) + 4 * h + i % 4 >= n) s[i] = -INFINITY;
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        x[i] = __builtin_amdgcn_exp2f(s[8 * u + i] + nl) * dp[8 * u + i];
                    u32x4 p[3];
                    split8(x, p);
                    add_transposed<C>(acc, kl, kb, u, p, lane);
                }
            }
        }
        if (t + 1 < t1) {
            u32x4* const other = lds + ((t + 1 - t0) & 1) * 2 * C::SET;
            k.store(a, other);
            v.store(a, other + C::SET);
            if (t + 2 < t1) load(t + 2);
            __syncthreads();
        }
    }
    if (!live) return;
    if (a.q_splits > 1)
        store_own<C, FULL>(a.dq_part + (((int64_t)no * items + item) * R + row) * a.D, acc, 1.0f,
                           0.0f, a.D, h);
    else
        store_own<C, FULL>(a.dq + query_offset(a, b, kv, row, a.ld_q), acc, a.scale, a.beta_q, a.D,
                           h);
}

// dk and dv of a workgroup's keys: the same P and dS with the rows met,
// dV = dO^T P, dK = scale * Q^T dS.
template <int D, int WAVES, bool FULL>
__device__ __forceinline__ void dkv_walk(const CrossArgs& a, u32x4* lds, float* starts, int block) {
    using C = TileCfg<D, WAVES>;
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Sq * a.G, tiles = (a.Sk + 32 * WAVES - 1) / (32 * WAVES), items = a.B * a.KV;
    const int tile = block % tiles, item = block / tiles % items, no = block / tiles / items;
    const int b = item / a.KV, kv = item - b * a.KV, L = live_keys(a, b);
    const int key = (tile * WAVES + w) * 32 + c;
    const bool wave_live = (tile * WAVES + w) * 32 < L, live = key < L;
    int t0, t1;
    share((R + C::KT - 1) / C::KT, no, a.kv_splits, t0, t1);
    if (tile * WAVES * 32 >= L) t1 = t0;  // no live key here
    Stage<C, FULL> q, g;
    float start[2];  // of threads below KT: -lse and -delta of a row of the tile
    auto load = [&](int t) {
        const int r0 = t * C::KT, n = min(C::KT, R - r0);
        q.template load<true>(a, a.q, a.ld_q, b, kv, r0, n);
        g.template load<true>(a, a.dout, a.ld_out, b, kv, r0, n);
        start[0] = -INFINITY;
        start[1] = 0.0f;
        if ((int)threadIdx.x < n) {
            start[0] = a.neg_lse[(int64_t)item * R + r0 + threadIdx.x];
            start[1] = a.neg_delta[(int64_t)item * R + r0 + threadIdx.x];
        }
    };
    auto store = [&](int buf) {
        q.store(a, lds + buf * 2 * C::SET);
        g.store(a, lds + buf * 2 * C::SET + C::SET);
        if ((int)threadIdx.x < C::KT) {
            starts[buf * 2 * C::KT + threadIdx.x] = start[0];
            starts[buf * 2 * C::KT + C::KT + threadIdx.x] = start[1];
        }
    };
    if (t0 < t1) load(t0);
    u32x4 kf[C::NS][3], vf[C::NS][3];
    own_pieces<C, FULL>(kf, a, a.k + (live ? key_offset(a, b, kv, key) : 0), live, h, a.scale2);
    own_pieces<C, FULL>(vf, a, a.v + (live ? key_offset(a, b, kv, key) : 0), live, h, 1.0f);
    f32x16 acc_k[C::NJ], acc_v[C::NJ];
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc_k[j] = acc_v[j] = all16(0.0f);
    if (t0 < t1) {
        store(0);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        u32x4* const ql = lds + buf * 2 * C::SET;
        if (wave_live) {
#pragma unroll
            for (int rb = 0; rb < C::NB; ++rb) {
                // the 16 rows' -lse and -delta; the latter is where dp starts
                const float* const st = starts + buf * 2 * C::KT + rb * 32 + 4 * h;
                f32x16 dp;
#pragma unroll
                for (int i = 0; i < 16; i += 4)
#pragma unroll
                    for (int e = 0; e < 4; ++e) dp[i + e] = st[C::KT + 2 * i + e];
                f32x16 s = close_products<C>(ql, kf, rb, all16(0.0f), c, h);
                dp = products<C>(ql + C::SET, vf, rb, dp, c, h);
#pragma unroll
                for (int i = 0; i < 16; i += 4)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i + e] += st[2 * i + e];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float x[8], y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] = __builtin_amdgcn_exp2f(s[8 * u + i]);
                        y[i] = x[i] * dp[8 * u + i];
                    }
                    u32x4 p[3];
                    split8(x, p);
                    add_transposed<C>(acc_v, ql + C::SET, rb, u, p, lane);
                    split8(y, p);
                    add_transposed<C>(acc_k, ql, rb, u, p, lane);
                }
            }
        }
        if (t + 1 < t1) {
            store(buf ^ 1);
            if (t + 2 < t1) load(t + 2);
            __syncthreads();
        }
    }
    if (key >= a.Sk) return;
    if (a.kv_splits > 1) {
        if (!live) return;  // the sum takes dead keys as zeros
        const int64_t at = (((int64_t)no * items + item) * a.Sk + key) * a.D;
        store_own<C, FULL>(a.dk_part + at, acc_k, 1.0f, 0.0f, a.D, h);
        store_own<C, FULL>(a.dv_part + at, acc_v, 1.0f, 0.0f, a.D, h);
        return;
    }
    if (!live) {
        if (a.beta_kv == 1.0f) return;
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) acc_k[j] = acc_v[j] = all16(0.0f);
    }
    const int64_t at = key_offset(a, b, kv, key);
    store_own<C, FULL>(a.dk + at, acc_k, a.scale, a.beta_kv, a.D, h);
    store_own<C, FULL>(a.dv + at, acc_v, 1.0f, a.beta_kv, a.D, h);
}

// One launch for both: they need nothing of each other, and the workgroups of
// one fill the compute units that the other leaves idle.
template <int D, bool FULL>
__global__ __launch_bounds__(256, 2) void cross_tile_bwd_kernel(CrossArgs a) {
    constexpr int WAVES = 4;
    using C = TileCfg<D, WAVES>;
    __shared__ u32x4 lds[4 * C::SET];
    __shared__ float starts[4 * C::KT];
    if ((int)blockIdx.x < a.q_blocks)
        dq_walk<D, WAVES, FULL>(a, lds, blockIdx.x);
    else
        dkv_walk<D, WAVES, FULL>(a, lds, starts, blockIdx.x - a.q_blocks);
}

// The backward of heads past 32 columns, 16 rows or keys to a wave on
// v_mfma_f32_16x16x32_bf16 (rate and operands of the same size): a wave reads as
// much from LDS for half as many, but its operands and accumulators leave room for
// two waves on a SIMD, which hide each other's exponentials and splits. With 32 to a
// wave: 4 x 1000 x 1500, 16 heads of 64, 563 us and here 552; 4 x 512 x 1500 of 96,
// 539 and 440; 2 x 777 x 4096, 16 heads of 128 on 4, 1419 and 1162; but 32 x 128 x
// 200, 8 heads of 32, 33 and 39. A wave computes met . own^T in two blocks of 16:
// lane (c, g) = (lane % 16, lane / 16) gets its own c with the met 16 half + 4 g + r,
// which lie as the operand of the product over the 32 met rows: place 8 g + 4 half + r.
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The lane's operands of its own row at `src` (zeros unless live), times f: unit
// 4 s + g of it is step s.
template <class C, bool FULL>
__device__ __forceinline__ void own16(u32x4 (&own)[C::D / 32][3], const CrossArgs& a,
                                      const float* src, bool live, int g, float f) {
#pragma unroll
    for (int s = 0; s < C::D / 32; ++s) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = 4 * (4 * s + g) + e * (C::D / 2);
            f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (live) {
                if (FULL || d + 4 <= a.D) {
                    v = reinterpret_cast<const Quad*>(src + d)->v;
                } else {
                    for (int i = 0; i < 4; ++i)
                        if (d + i < a.D) v[i] = src[d + i];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * e + i] = v[i] * f;
        }
        split8(x, own[s]);
    }
}

// The operand of step s of 16 rows of a tile.
template <class C>
__device__ __forceinline__ u32x4 piece16(const u32x4* set, int row, int s, int p, int c, int g) {
    return set[p * C::PLANE + unit_at<C>(row + c, 4 * s + g)];
}

// out += met . own^T of block kb of a tile; CLOSE: the large products last, as in
// close_products.
template <class C, bool CLOSE>
__device__ __forceinline__ void products16(f32x4 (&out)[2], const u32x4* set,
                                           const u32x4 (&own)[C::D / 32][3], int kb, int c, int g) {
#pragma unroll
    for (int s = 0; s < C::D / 32; ++s) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            u32x4 met[3];
#pragma unroll
            for (int p = 0; p < 3; ++p) met[p] = piece16<C>(set, kb * 32 + 16 * half, s, p, c, g);
            f32x4& o = out[half];
            o = mfma16(met[2], own[s][0], o);
            o = mfma16(met[1], own[s][1], o);
            o = mfma16(met[0], own[s][2], o);
            o = mfma16(met[1], own[s][0], o);
            o = mfma16(met[0], own[s][1], o);
            if (!CLOSE) o = mfma16(met[0], own[s][0], o);
        }
    }
    if (CLOSE) {
        asm volatile("" : "+v"(c));  // read again, as there
#pragma unroll
        for (int s = 0; s < C::D / 32; ++s)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                out[half] = mfma16(piece16<C>(set, kb * 32 + 16 * half, s, 0, c, g), own[s][0], out[half]);
    }
}

// acc[j] += met^T . w over the 32 met rows of block kb, w split. Of the 16 places m of
// output block j, 4 x + y is d = 4 unit + (x % 2) D/2 + y, unit = 4 (j / 2) + j % 2 +
// 2 (x / 2): each x a half of one unit, as a transposing read takes them.
template <class C>
__device__ __forceinline__ void add16(f32x4 (&acc)[C::D / 16], const u32x4* set, int kb,
                                      const u32x4 (&w)[3], int lane) {
    const int x = lane & 3, e = (lane >> 2) & 3, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < C::D / 16; ++j) {
        u32x4 met[3];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int unit = unit_at<C>(kb * 32 + 16 * half + 4 * g + e,
                                        4 * (j >> 1) + (j & 1) + 2 * (x >> 1));
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const u32x2 v = read_transposed(
                    reinterpret_cast<const u32x2*>(set + p * C::PLANE + unit) + (x & 1));
                met[p][2 * half] = v[0];
                met[p][2 * half + 1] = v[1];
            }
        }
        f32x4& o = acc[j];
        o = mfma16(met[2], w[0], o);
        o = mfma16(met[1], w[1], o);
        o = mfma16(met[0], w[2], o);
        o = mfma16(met[1], w[0], o);
        o = mfma16(met[0], w[1], o);
        o = mfma16(met[0], w[0], o);
    }
}

// Stores a lane's acc * f (+ beta * old) into its own row of d_head floats.
template <class C, bool FULL>
__device__ __forceinline__ void store16(float* dst, const f32x4 (&acc)[C::D / 16], float f,
                                        float beta, int D, int g) {
#pragma unroll
    for (int j = 0; j < C::D / 16; ++j) {
        const int d = 4 * (4 * (j >> 1) + (j & 1) + 2 * (g >> 1)) + (g & 1) * (C::D / 2);
        f32x4 v = acc[j] * f;
        if (FULL || d + 4 <= D) {
            Quad* const to = reinterpret_cast<Quad*>(dst + d);
            if (beta != 0.0f) v = v + beta * to->v;
            to->v = v;
        } else {
            for (int e = 0; e < 4; ++e)
                if (d + e < D) dst[d + e] = beta != 0.0f ? v[e] + beta * dst[d + e] : v[e];
        }
    }
}

// dq_walk with 16 rows to a wave.
template <int D, bool FULL>
__device__ __forceinline__ void dq_walk16(const CrossArgs& a, u32x4* lds, int block) {
    using C = TileCfg<D, 8>;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Sq * a.G, tiles = (R + 127) / 128, items = a.B * a.KV;
    const int tile = block % tiles, item = block / tiles % items, no = block / tiles / items;
    const int b = item / a.KV, kv = item - b * a.KV, L = live_keys(a, b);
    const int row = (tile * 8 + w) * 16 + c;
    const bool wave_live = (tile * 8 + w) * 16 < R, live = row < R;
    int t0, t1;
    share((L + C::KT - 1) / C::KT, no, a.q_splits, t0, t1);
    Stage<C, FULL> k, v;
    auto load = [&](int t) {
        const int n = min(C::KT, L - t * C::KT);
        k.template load<false>(a, a.k, a.ld_kv, b, kv, t * C::KT, n);
        v.template load<false>(a, a.v, a.ld_kv, b, kv, t * C::KT, n);
    };
    if (t0 < t1) load(t0);
    u32x4 qf[D / 32][3], gf[D / 32][3];
    own16<C, FULL>(qf, a, a.q + (live ? query_offset(a, b, kv, row, a.ld_q) : 0), live, g, a.scale2);
    own16<C, FULL>(gf, a, a.dout + (live ? query_offset(a, b, kv, row, a.ld_out) : 0), live, g, 1.0f);
    const float nl = live ? a.neg_lse[(int64_t)item * R + row] : -INFINITY;
    const float nd = live ? a.neg_delta[(int64_t)item * R + row] : 0.0f;
    f32x4 acc[D / 16];
#pragma unroll
    for (int j = 0; j < D / 16; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (t0 < t1) {
        k.store(a, lds);
        v.store(a, lds + C::SET);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        u32x4* const kl = lds + ((t - t0) & 1) * 2 * C::SET;
        if (wave_live) {
            const int n = L - t * C::KT;
#pragma unroll
            for (int kb = 0; kb < C::NB; ++kb) {
                f32x4 s[2], dp[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    s[half] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    dp[half] = f32x4{nd, nd, nd, nd};
                }
                products16<C, true>(s, kl, qf, kb, c, g);
                products16<C, false>(dp, kl + C::SET, gf, kb, c, g);
                if (n < C::KT) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (kb * 32 + 16 * (i / 4) + 4 * g + i % 4 >= n) s[i / 4][i % 4] = -INFINITY;
                }
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = __builtin_amdgcn_exp2f(s[i / 4][i % 4] + nl) * dp[i / 4][i % 4];
                u32x4 p[3];
                split8(x, p);
                add16<C>(acc, kl, kb, p, lane);
            }
        }
        if (t + 1 < t1) {
            u32x4* const other = lds + ((t + 1 - t0) & 1) * 2 * C::SET;
            k.store(a, other);
            v.store(a, other + C::SET);
            if (t + 2 < t1) load(t + 2);
            __syncthreads();
        }
    }
    if (!live) return;
    if (a.q_splits > 1)
        store16<C, FULL>(a.dq_part + (((int64_t)no * items + item) * R + row) * a.D, acc, 1.0f, 0.0f,
                         a.D, g);
    else
        store16<C, FULL>(a.dq + query_offset(a, b, kv, row, a.ld_q), acc, a.scale, a.beta_q, a.D, g);
}

// dkv_walk with 16 keys to a wave.
template <int D, bool FULL>
__device__ __forceinline__ void dkv_walk16(const CrossArgs& a, u32x4* lds, f32x4* starts, int block) {
    using C = TileCfg<D, 8>;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Sq * a.G, tiles = (a.Sk + 127) / 128, items = a.B * a.KV;
    const int tile = block % tiles, item = block / tiles % items, no = block / tiles / items;
    const int b = item / a.KV, kv = item - b * a.KV, L = live_keys(a, b);
    const int key = (tile * 8 + w) * 16 + c;
    const bool wave_live = (tile * 8 + w) * 16 < L, live = key < L;
    int t0, t1;
    share((R + C::KT - 1) / C::KT, no, a.kv_splits, t0, t1);
    if (tile * 128 >= L) t1 = t0;  // no live key here
    Stage<C, FULL> q, go;
    float start[2];  // of threads below KT: -lse and -delta of a row of the tile
    auto load = [&](int t) {
        const int r0 = t * C::KT, n = min(C::KT, R - r0);
        q.template load<true>(a, a.q, a.ld_q, b, kv, r0, n);
        go.template load<true>(a, a.dout, a.ld_out, b, kv, r0, n);
        start[0] = -INFINITY;
        start[1] = 0.0f;
        if ((int)threadIdx.x < n) {
            start[0] = a.neg_lse[(int64_t)item * R + r0 + threadIdx.x];
            start[1] = a.neg_delta[(int64_t)item * R + r0 + threadIdx.x];
        }
    };
    auto store = [&](int buf) {
        q.store(a, lds + buf * 2 * C::SET);
        go.store(a, lds + buf * 2 * C::SET + C::SET);
        if ((int)threadIdx.x < C::KT) {
            float* const to = reinterpret_cast<float*>(starts) + buf * 2 * C::KT;
            to[threadIdx.x] = start[0];
            to[C::KT + threadIdx.x] = start[1];
        }
    };
    if (t0 < t1) load(t0);
    u32x4 kf[D / 32][3], vf[D / 32][3];
    own16<C, FULL>(kf, a, a.k + (live ? key_offset(a, b, kv, key) : 0), live, g, a.scale2);
    own16<C, FULL>(vf, a, a.v + (live ? key_offset(a, b, kv, key) : 0), live, g, 1.0f);
    f32x4 acc_k[D / 16], acc_v[D / 16];
#pragma unroll
    for (int j = 0; j < D / 16; ++j) acc_k[j] = acc_v[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (t0 < t1) {
        store(0);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        u32x4* const ql = lds + buf * 2 * C::SET;
        if (wave_live) {
#pragma unroll
            for (int rb = 0; rb < C::NB; ++rb) {
                const f32x4* const st = starts + (buf * 2 * C::KT + rb * 32) / 4 + g;
                f32x4 s[2], dp[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    s[half] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    dp[half] = st[C::KT / 4 + 4 * half];
                }
                products16<C, true>(s, ql, kf, rb, c, g);
                products16<C, false>(dp, ql + C::SET, vf, rb, c, g);
                float x[8], y[8];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const f32x4 nl = st[4 * half];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[4 * half + r] = __builtin_amdgcn_exp2f(s[half][r] + nl[r]);
                        y[4 * half + r] = x[4 * half + r] * dp[half][r];
                    }
                }
                u32x4 p[3];
                split8(x, p);
                add16<C>(acc_v, ql + C::SET, rb, p, lane);
                split8(y, p);
                add16<C>(acc_k, ql, rb, p, lane);
            }
        }
        if (t + 1 < t1) {
            store(buf ^ 1);
            if (t + 2 < t1) load(t + 2);
            __syncthreads();
        }
    }
    if (key >= a.Sk) return;
    if (a.kv_splits > 1) {
        if (!live) return;  // the sum takes dead keys as zeros
        const int64_t at = (((int64_t)no * items + item) * a.Sk + key) * a.D;
        store16<C, FULL>(a.dk_part + at, acc_k, 1.0f, 0.0f, a.D, g);
        store16<C, FULL>(a.dv_part + at, acc_v, 1.0f, 0.0f, a.D, g);
        return;
    }
    if (!live) {
        if (a.beta_kv == 1.0f) return;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) acc_k[j] = acc_v[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int64_t at = key_offset(a, b, kv, key);
    store16<C, FULL>(a.dk + at, acc_k, a.scale, a.beta_kv, a.D, g);
    store16<C, FULL>(a.dv + at, acc_v, 1.0f, a.beta_kv, a.D, g);
}

template <int D, bool FULL>
__global__ __launch_bounds__(512, 2) void cross_tile_bwd16_kernel(CrossArgs a) {
    using C = TileCfg<D, 8>;
    __shared__ u32x4 lds[4 * C::SET];
    __shared__ f32x4 starts[C::KT];
    const int kv_blocks = gridDim.x - a.q_blocks;  // (the longer walks begin first)
    if ((int)blockIdx.x >= kv_blocks)
        dq_walk16<D, FULL>(a, lds, blockIdx.x - kv_blocks);
    else
        dkv_walk16<D, FULL>(a, lds, starts, blockIdx.x);
}

template <int D>
void launch_forward(const CrossArgs& a, unsigned blocks) {
    const bool full = a.D == D;
    auto kernel = a.unit_rows == 256
                      ? (full ? cross_tile_fwd_kernel<D, 8, true> : cross_tile_fwd_kernel<D, 8, false>)
                      : (full ? cross_tile_fwd_kernel<D, 4, true> : cross_tile_fwd_kernel<D, 4, false>);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(2 * a.unit_rows), 0, stream(), a);
}

template <int D>
void launch_backward(CrossArgs a, bool only_rows) {
    const int R = a.Sq * a.G, own = kCrossBackwardRows;
    const int64_t items = (int64_t)a.B * a.KV, rows = items * R;
    if (rows > 0) {
        constexpr int WIDE = cross_row_width(D), PER = 1024 / WIDE;
        hipLaunchKernelGGL(cross_rows_prepare_kernel<WIDE>, dim3((unsigned)((rows + PER - 1) / PER)),
                           dim3(256), 0, stream(), a);
    }
    if (only_rows) return;
    a.q_blocks = a.dq ? (int)((R + own - 1) / own * items * a.q_splits) : 0;
    const int64_t kv_blocks = a.dk ? (a.Sk + own - 1) / own * items * a.kv_splits : 0;
    if (a.q_blocks + kv_blocks == 0) return;
    if constexpr (D > 32) {
        auto kernel =
            a.D == D ? cross_tile_bwd16_kernel<D, true> : cross_tile_bwd16_kernel<D, false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(a.q_blocks + kv_blocks)), dim3(512), 0, stream(),
                           a);
    } else {
        auto kernel = a.D == D ? cross_tile_bwd_kernel<D, true> : cross_tile_bwd_kernel<D, false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(a.q_blocks + kv_blocks)), dim3(256), 0, stream(), a);
    }
}

}  // namespace

void cross_tile_forward(const CrossArgs& a, unsigned blocks) {
    if (a.D <= 32)
        launch_forward<32>(a, blocks);
    else if (a.D <= 64)
        launch_forward<64>(a, blocks);
    else if (a.D <= 96)
        launch_forward<96>(a, blocks);
    else
        launch_forward<128>(a, blocks);
}

void cross_tile_backward(const CrossArgs& a, bool only_rows) {
    if (a.D <= 32)
        launch_backward<32>(a, only_rows);
    else if (a.D <= 64)
        launch_backward<64>(a, only_rows);
    else if (a.D <= 96)
        launch_backward<96>(a, only_rows);
    else
        launch_backward<128>(a, only_rows);
}

}  // namespace nrs
