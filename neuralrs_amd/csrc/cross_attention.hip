// Attention of a decoder's rows over an encoder's states: queries and keys of
// different lengths, several query heads to a key head, a length of live keys
// for each batch item. Forward and backward, all f32.
//
// The query heads of one key head are further rows of the same product: with
// group = heads / kv_heads, row r of (item, key head) is query r / group of
// head kv_head * group + r % group, R = seq_q * group rows in all. Keys past
// the item's length are never read (they stand for nothing, and may hold
// anything); an item without live keys gets zeros.
#include <algorithm>

#include "buffer_ops.hpp"

namespace nrs {
namespace {

struct CrossArgs {
    const float *q, *k, *v, *dout, *o;
    float *out, *stats;  // stats: [batch][heads][seq_q][2], base-2 max and sum
    float *dq, *dk, *dv;
    const int32_t* key_len;  // per item, null: all keys
    int B, H, KV, G, Sq, Sk, D, ld_q, ld_kv, ld_out;
    float scale, scale2;  // scale2 = scale * log2(e)
    float beta_q, beta_kv;
};

__device__ __forceinline__ f32x4 mfma16(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ int live_keys(const CrossArgs& a, int b) {
    return a.key_len ? max(0, min(a.key_len[b], a.Sk)) : a.Sk;
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

// acc[j][d'][n] += sum over the tile's 16 rows of x[row][d] w[row][n]: w as
// dot_rows leaves it, lane (c, g) of acc[j] gets d = (4g + r) * NJ + j of n = c.
template <int NJ, class R>
__device__ __forceinline__ void add_rows(f32x4 (&acc)[NJ], const R& x, f32x4 w, int c, int g) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float f[NJ];
        x.template across<NJ>(f, 4 * g + r, c);
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j] = mfma16(f[j], w[r], acc[j]);
    }
}

// Stores acc (as add_rows leaves it) times `f` into a row of d_head floats.
template <int NJ>
__device__ __forceinline__ void store_row(float* dst, const f32x4 (&acc)[NJ], float f, float beta,
                                          int D, int g) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int d = (4 * g + r) * NJ + j;
            if (d < D) dst[d] = beta != 0.0f ? acc[j][r] * f + beta * dst[d] : acc[j][r] * f;
        }
}

__device__ __forceinline__ int64_t query_offset(const CrossArgs& a, int b, int kv, int r, int ld) {
    return ((int64_t)b * a.Sq + r / a.G) * ld + (int64_t)(kv * a.G + r % a.G) * a.D;
}

__device__ __forceinline__ float* row_stats(const CrossArgs& a, int b, int kv, int r) {
    return a.stats + (((int64_t)b * a.H + kv * a.G + r % a.G) * a.Sq + r / a.G) * 2;
}

__device__ __forceinline__ float across_groups(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

// One wave per 16 rows of an (item, key head), its keys 16 at a time.
template <int NJ>
__global__ __launch_bounds__(64) void cross_fwd_kernel(CrossArgs a) {
    const int lane = threadIdx.x, c = lane & 15, g = lane >> 4;
    const int R = a.Sq * a.G, tiles = (R + 15) / 16;
    const int item = blockIdx.x / tiles, r0 = (blockIdx.x - item * tiles) * 16;
    const int b = item / a.KV, kv = item - b * a.KV, L = live_keys(a, b);
    f32x4 qf[NJ], acc[NJ];
    Rows<true>(a, a.q, b, kv, a.ld_q, r0, min(16, R - r0)).template along<NJ>(qf, c, g);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        qf[j] = qf[j] * a.scale2;
        acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    float m = -INFINITY, l = 0.0f;
    for (int k0 = 0; k0 < L; k0 += 16) {
        const int n = min(16, L - k0);
        f32x4 kf[NJ];
        Rows<false>(a, a.k, b, kv, a.ld_kv, k0, n).template along<NJ>(kf, c, g);
        f32x4 p = dot_rows<NJ>(kf, qf);
        float mt = -INFINITY;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (4 * g + r >= n) p[r] = -INFINITY;
            mt = fmaxf(mt, p[r]);
        }
        mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        const float top = fmaxf(m, mt);
        const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= alpha;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            p[r] = 4 * g + r < n ? __builtin_amdgcn_exp2f(p[r] - m) : 0.0f;
            l += p[r];
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j] = acc[j] * alpha;
        add_rows<NJ>(acc, Rows<false>(a, a.v, b, kv, a.ld_kv, k0, n), p, c, g);
    }
    l = across_groups(l);
    if (r0 + c >= R) return;
    store_row<NJ>(a.out + query_offset(a, b, kv, r0 + c, a.ld_out), acc, L > 0 ? 1.0f / l : 0.0f,
                  0.0f, a.D, g);
    if (a.stats && g == 0) {
        float* st = row_stats(a, b, kv, r0 + c);
        st[0] = L > 0 ? m : 0.0f;
        st[1] = l;
    }
}

// The gradient of the queries: the forward's walk over the keys again.
template <int NJ>
__global__ __launch_bounds__(64) void cross_dq_kernel(CrossArgs a) {
    const int lane = threadIdx.x, c = lane & 15, g = lane >> 4;
    const int R = a.Sq * a.G, tiles = (R + 15) / 16;
    const int item = blockIdx.x / tiles, r0 = (blockIdx.x - item * tiles) * 16;
    const int b = item / a.KV, kv = item - b * a.KV, L = live_keys(a, b), nr = min(16, R - r0);
    f32x4 qf[NJ], gf[NJ], of[NJ], acc[NJ];
    Rows<true>(a, a.q, b, kv, a.ld_q, r0, nr).template along<NJ>(qf, c, g);
    Rows<true>(a, a.dout, b, kv, a.ld_out, r0, nr).template along<NJ>(gf, c, g);
    Rows<true>(a, a.o, b, kv, a.ld_out, r0, nr).template along<NJ>(of, c, g);
    float delta = 0.0f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        qf[j] = qf[j] * a.scale2;
        acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 4; ++e) delta = fmaf(gf[j][e], of[j][e], delta);
    }
    delta = across_groups(delta);
    float m = 0.0f, rl = 0.0f;
    if (c < nr && L > 0) {
        const float* st = row_stats(a, b, kv, r0 + c);
        m = st[0];
        rl = 1.0f / st[1];
    }
    for (int k0 = 0; k0 < L; k0 += 16) {
        const int n = min(16, L - k0);
        const Rows<false> keys(a, a.k, b, kv, a.ld_kv, k0, n);
        f32x4 kf[NJ], vf[NJ];
        keys.template along<NJ>(kf, c, g);
        Rows<false>(a, a.v, b, kv, a.ld_kv, k0, n).template along<NJ>(vf, c, g);
        f32x4 p = dot_rows<NJ>(kf, qf), dp = dot_rows<NJ>(vf, gf);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float w = 4 * g + r < n ? __builtin_amdgcn_exp2f(p[r] - m) * rl : 0.0f;
            dp[r] = w * (dp[r] - delta) * a.scale;
        }
        add_rows<NJ>(acc, keys, dp, c, g);
    }
    if (c < nr)
        store_row<NJ>(a.dq + query_offset(a, b, kv, r0 + c, a.ld_q), acc, 1.0f, a.beta_q, a.D, g);
}

// The gradients of 16 keys and values: one wave walks the rows of all heads
// that share them.
template <int NJ>
__global__ __launch_bounds__(64) void cross_dkv_kernel(CrossArgs a) {
    const int lane = threadIdx.x, c = lane & 15, g = lane >> 4;
    const int tiles = (a.Sk + 15) / 16;
    const int item = blockIdx.x / tiles, k0 = (blockIdx.x - item * tiles) * 16;
    const int b = item / a.KV, kv = item - b * a.KV, L = live_keys(a, b);
    const int n = min(16, L - k0), R = n > 0 ? a.Sq * a.G : 0;  // dead keys: zeros
    f32x4 kf[NJ], vf[NJ], acc_k[NJ], acc_v[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc_k[j] = acc_v[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (n > 0) {
        Rows<false>(a, a.k, b, kv, a.ld_kv, k0, n).template along<NJ>(kf, c, g);
        Rows<false>(a, a.v, b, kv, a.ld_kv, k0, n).template along<NJ>(vf, c, g);
#pragma unroll
        for (int j = 0; j < NJ; ++j) kf[j] = kf[j] * a.scale2;
    }
    for (int r0 = 0; r0 < R; r0 += 16) {
        const int nr = min(16, R - r0);
        const Rows<true> qs(a, a.q, b, kv, a.ld_q, r0, nr), gs(a, a.dout, b, kv, a.ld_out, r0, nr);
        f32x4 qf[NJ], gf[NJ], of[NJ];
        qs.template along<NJ>(qf, c, g);
        gs.template along<NJ>(gf, c, g);
        Rows<true>(a, a.o, b, kv, a.ld_out, r0, nr).template along<NJ>(of, c, g);
        float delta = 0.0f, m = 0.0f, rl = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) delta = fmaf(gf[j][e], of[j][e], delta);
        delta = across_groups(delta);
        if (c < nr) {
            const float* st = row_stats(a, b, kv, r0 + c);
            m = st[0];
            rl = 1.0f / st[1];
        }
        f32x4 p = dot_rows<NJ>(qf, kf), dp = dot_rows<NJ>(gf, vf);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            // the row of register r is 4g + r, whose values lane 4g + r holds
            const float mr = __shfl(m, 4 * g + r, 64), lr = __shfl(rl, 4 * g + r, 64),
                        dr = __shfl(delta, 4 * g + r, 64);
            const bool live = 4 * g + r < nr && c < n;
            p[r] = live ? __builtin_amdgcn_exp2f(p[r] - mr) * lr : 0.0f;
            dp[r] = p[r] * (dp[r] - dr) * a.scale;
        }
        add_rows<NJ>(acc_v, gs, p, c, g);
        add_rows<NJ>(acc_k, qs, dp, c, g);
    }
    if (k0 + c >= a.Sk) return;
    const int64_t at = ((int64_t)b * a.Sk + k0 + c) * a.ld_kv + (int64_t)kv * a.D;
    store_row<NJ>(a.dk + at, acc_k, 1.0f, a.beta_kv, a.D, g);
    store_row<NJ>(a.dv + at, acc_v, 1.0f, a.beta_kv, a.D, g);
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

constexpr int64_t kMaxLd = 1 << 20, kMaxLen = 1 << 26;

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
    const int64_t rows = (seq_q * (heads / kv_heads) + 15) / 16, keys = (seq_k + 15) / 16;
    if (seq_q * (heads / kv_heads) > INT32_MAX / 2 || batch > INT32_MAX / kv_heads ||
        batch * kv_heads * std::max<int64_t>({rows, keys, 1}) > INT32_MAX)
        return "too many rows for one launch";
    return nullptr;
}

int check_shape(const char* what, int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q,
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

}  // namespace
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
    if (int rc = nrs::check_shape("cross attention workspace", batch, heads, kv_heads, seq_q,
                                  seq_k, d_head, heads * d_head, kv_heads * d_head,
                                  heads * d_head))
        return rc;
    (void)backward;
    *bytes = 0;
    return NRS_OK;
}

int nrs_cross_attention_forward(float* out, float* stats, const float* q, const float* k,
                                const float* v, const int32_t* key_len, int64_t batch,
                                int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_k,
                                int64_t d_head, int64_t ld_q, int64_t ld_kv, int64_t ld_out,
                                float scale, void* work, size_t work_bytes) {
    const char* what = "cross attention forward";
    if (int rc = nrs::check_shape(what, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                                  ld_out))
        return rc;
    if (batch == 0 || seq_q == 0) return NRS_OK;
    NRS_ARG_CHECK(out && q && ((k && v) || seq_k == 0), "%s: null pointer", what);
    NRS_REQUIRE_INIT();
    if (int rc = nrs::check_device(what)) return rc;
    float* scratch = nullptr;
    if (int rc = nrs::call_scratch(&scratch, 0, work, work_bytes, what)) return rc;
    nrs::CrossArgs a{};
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
    a.scale = scale;
    a.scale2 = scale * 1.4426950408889634f;
    const int64_t tiles = (seq_q * a.G + 15) / 16;
    nrs::for_width(a.D, [&](auto nj) {
        hipLaunchKernelGGL(nrs::cross_fwd_kernel<decltype(nj)::value>,
                           dim3((unsigned)(batch * kv_heads * tiles)), dim3(64), 0, nrs::stream(),
                           a);
    });
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
    if (int rc = nrs::check_shape(what, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                                  ld_out))
        return rc;
    NRS_ARG_CHECK((dk == nullptr) == (dv == nullptr), "%s: dk and dv go together", what);
    if (batch == 0) return NRS_OK;
    const bool rows = seq_q > 0, keys = seq_k > 0;
    NRS_ARG_CHECK((!rows || (dout && out && q && stats)) && (!keys || (k && v)),
                  "%s: null pointer", what);
    NRS_REQUIRE_INIT();
    if (int rc = nrs::check_device(what)) return rc;
    float* scratch = nullptr;
    if (int rc = nrs::call_scratch(&scratch, 0, work, work_bytes, what)) return rc;
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
    a.scale = scale;
    a.scale2 = scale * 1.4426950408889634f;  // as the forward computed it
    a.beta_q = beta_q;
    a.beta_kv = beta_kv;
    const int64_t row_tiles = (seq_q * a.G + 15) / 16, key_tiles = (seq_k + 15) / 16;
    nrs::for_width(a.D, [&](auto nj) {
        if (dq && rows)
            hipLaunchKernelGGL(nrs::cross_dq_kernel<decltype(nj)::value>,
                               dim3((unsigned)(batch * kv_heads * row_tiles)), dim3(64), 0,
                               nrs::stream(), a);
        if (dk && keys)
            hipLaunchKernelGGL(nrs::cross_dkv_kernel<decltype(nj)::value>,
                               dim3((unsigned)(batch * kv_heads * key_tiles)), dim3(64), 0,
                               nrs::stream(), a);
    });
    NRS_LAUNCH_CHECK(what);
    return NRS_OK;
}

}  // extern "C"
