// Tiles of split floats on the bf16 matrix cores, for the attention kernels of many
// rows (cross_attention_tile.hip tells the layout): operands of a wave's own rows in
// registers, tiles of the other side in LDS, products of both kinds, stores.
#pragma once

#include "cross_attention.hpp"

namespace nrs {

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

// ---- 16 rows to a wave, on v_mfma_f32_16x16x32_bf16. A wave computes met . own^T in
// two blocks of 16: lane (c, g) = (lane % 16, lane / 16) gets its own c with the met
// 16 half + 4 g + r, which lie as the operand of the product over the 32 met rows:
// place 8 g + 4 half + r.
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

}  // namespace nrs
