// Attention whose rows see ranges of keys, with capped scores and a bias by
// distance, forward and backward, all f32.
#include "masked_attention.hpp"

#include <cmath>

namespace nrs {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// A row's score of a key from their product, in base 2; `inner` is the cap's
// derivative.
struct Scores {
    float scale, cap, slope;
    int64_t at, near;

    __device__ __forceinline__ Scores(const MaskedArgs& a, const RowRange& r, int head)
        : scale(a.scale), cap(a.cap), slope(a.slopes ? a.slopes[head] : 0.0f), at(r.at),
          near(nearest(r)) {}
    __device__ __forceinline__ float of(float dot, int key, float& inner) const {
        float u = dot * scale;
        inner = 1.0f;
        if (cap > 0.0f) {
            const float t = tanhf(u / cap);
            inner = 1.0f - t * t;
            u = cap * t;
        }
        const int64_t far = at < key ? key - at : at - key;
        return (u - slope * (float)(far - near)) * kLog2e;
    }
};

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) x += __shfl_xor(x, i, 64);
    return x;
}

// Columns lane and lane + 64 of a row of d_head floats.
__device__ __forceinline__ void row2(float (&x)[2], const float* p, int lane, int D) {
    x[0] = lane < D ? p[lane] : 0.0f;
    x[1] = lane + 64 < D ? p[lane + 64] : 0.0f;
}

// A wave to a row.
__global__ __launch_bounds__(256) void masked_fwd_kernel(MaskedArgs a) {
    const int lane = threadIdx.x & 63, R = a.Sq * a.G;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (int64_t)a.B * a.KV * R) return;
    const int item = (int)(row / R), r = (int)(row - (int64_t)item * R);
    const int b = item / a.KV, kv = item - b * a.KV;
    const RowRange range = row_range(a, b, r / a.G);
    const Scores scores(a, range, kv * a.G + r % a.G);
    float q[2], acc[2] = {0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
    row2(q, a.q + query_offset(a, b, kv, r, a.ld_q), lane, a.D);
    for (int t = range.lo; t < range.hi; ++t) {
        float k[2], v[2], inner;
        const int64_t at = key_offset(a, b, kv, t);
        row2(k, a.k + at, lane, a.D);
        row2(v, a.v + at, lane, a.D);
        const float u = scores.of(wave_sum(q[0] * k[0] + q[1] * k[1]), t, inner);
        const float top = fmaxf(m, u);
        const float old = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        const float p = __builtin_amdgcn_exp2f(u - top);
        m = top;
        l = l * old + p;
        acc[0] = acc[0] * old + p * v[0];
        acc[1] = acc[1] * old + p * v[1];
    }
    const bool any = range.hi > range.lo;
    const float f = any ? 1.0f / l : 0.0f;
    float* const out = a.out + query_offset(a, b, kv, r, a.ld_out);
    if (lane < a.D) out[lane] = acc[0] * f;
    if (lane + 64 < a.D) out[lane + 64] = acc[1] * f;
    if (a.stats && lane == 0) {
        float* const st = row_stats(a, b, kv, r);
        st[0] = any ? m : 0.0f;
        st[1] = l;
    }
}

// P and dS of a row and a key; all lanes get them.
__device__ __forceinline__ void weights(const MaskedArgs& a, const Scores& scores, int t,
                                        const float (&q)[2], const float (&g)[2],
                                        const float (&k)[2], const float (&v)[2], float lse,
                                        float delta, float& p, float& ds) {
    float inner;
    const float u = scores.of(wave_sum(q[0] * k[0] + q[1] * k[1]), t, inner);
    p = __builtin_amdgcn_exp2f(u - lse);
    ds = p * (wave_sum(g[0] * v[0] + g[1] * v[1]) - delta) * inner * a.scale;
}

__device__ __forceinline__ void add_to(float* dst, const float (&x)[2], float beta, int lane, int D) {
    if (lane < D) dst[lane] = beta != 0.0f ? x[0] + beta * dst[lane] : x[0];
    if (lane + 64 < D) dst[lane + 64] = beta != 0.0f ? x[1] + beta * dst[lane + 64] : x[1];
}

__device__ __forceinline__ void row_start(const MaskedArgs& a, int b, int kv, int r,
                                          const float (&g)[2], int lane, float& lse, float& delta) {
    float o[2];
    row2(o, a.o + query_offset(a, b, kv, r, a.ld_out), lane, a.D);
    const float* const st = row_stats(a, b, kv, r);
    lse = st[0] + __builtin_amdgcn_logf(st[1]);
    delta = wave_sum(g[0] * o[0] + g[1] * o[1]);
}

// dq, a wave to a row.
__global__ __launch_bounds__(256) void masked_dq_kernel(MaskedArgs a) {
    const int lane = threadIdx.x & 63, R = a.Sq * a.G;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (int64_t)a.B * a.KV * R) return;
    const int item = (int)(row / R), r = (int)(row - (int64_t)item * R);
    const int b = item / a.KV, kv = item - b * a.KV;
    const RowRange range = row_range(a, b, r / a.G);
    const Scores scores(a, range, kv * a.G + r % a.G);
    float q[2], g[2], acc[2] = {0.0f, 0.0f}, lse, delta;
    row2(q, a.q + query_offset(a, b, kv, r, a.ld_q), lane, a.D);
    row2(g, a.dout + query_offset(a, b, kv, r, a.ld_out), lane, a.D);
    row_start(a, b, kv, r, g, lane, lse, delta);
    for (int t = range.lo; t < range.hi; ++t) {
        float k[2], v[2], p, ds;
        const int64_t at = key_offset(a, b, kv, t);
        row2(k, a.k + at, lane, a.D);
        row2(v, a.v + at, lane, a.D);
        weights(a, scores, t, q, g, k, v, lse, delta, p, ds);
        acc[0] += ds * k[0];
        acc[1] += ds * k[1];
    }
    add_to(a.dq + query_offset(a, b, kv, r, a.ld_q), acc, a.beta_q, lane, a.D);
}

// dk and dv, a wave to a key.
__global__ __launch_bounds__(256) void masked_dkv_kernel(MaskedArgs a) {
    const int lane = threadIdx.x & 63, R = a.Sq * a.G;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= (int64_t)a.B * a.KV * a.Sk) return;
    const int item = (int)(at / a.Sk), t = (int)(at - (int64_t)item * a.Sk);
    const int b = item / a.KV, kv = item - b * a.KV;
    const int64_t key = key_offset(a, b, kv, t);
    float k[2] = {0.0f, 0.0f}, v[2] = {0.0f, 0.0f}, dk[2] = {0.0f, 0.0f}, dv[2] = {0.0f, 0.0f};
    bool seen = false;
    for (int r = 0; r < R; ++r) {
        const RowRange range = row_range(a, b, r / a.G);
        if (t < range.lo || t >= range.hi) continue;
        if (!seen) {
            row2(k, a.k + key, lane, a.D);
            row2(v, a.v + key, lane, a.D);
            seen = true;
        }
        const Scores scores(a, range, kv * a.G + r % a.G);
        float q[2], g[2], lse, delta, p, ds;
        row2(q, a.q + query_offset(a, b, kv, r, a.ld_q), lane, a.D);
        row2(g, a.dout + query_offset(a, b, kv, r, a.ld_out), lane, a.D);
        row_start(a, b, kv, r, g, lane, lse, delta);
        weights(a, scores, t, q, g, k, v, lse, delta, p, ds);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            dk[e] += ds * q[e];
            dv[e] += p * g[e];
        }
    }
    if (!seen && a.beta_kv == 1.0f) return;
    add_to(a.dk + key, dk, a.beta_kv, lane, a.D);
    add_to(a.dv + key, dv, a.beta_kv, lane, a.D);
}

int check(const char* what, const nrs_attention_mask* mask, int64_t batch, int64_t heads,
          int64_t kv_heads, int64_t seq_q, int64_t seq_k, int64_t d_head, int64_t ld_q,
          int64_t ld_kv, int64_t ld_out) {
    if (int rc = cross_check_shape(what, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q,
                                   ld_kv, ld_out))
        return rc;
    if (!mask) return NRS_OK;
    NRS_ARG_CHECK(mask->cap >= 0.0f && std::isfinite(mask->cap),
                  "%s: cap must be 0 (none) or a positive number, is %g", what, (double)mask->cap);
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
        a.cap = mask->cap;
    }
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
    (void)backward;
    *bytes = 0;
    return NRS_OK;
}

int nrs_masked_attention_forward(float* out, float* stats, const float* q, const float* k,
                                 const float* v, const nrs_attention_mask* mask, int64_t batch,
                                 int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_k,
                                 int64_t d_head, int64_t ld_q, int64_t ld_kv, int64_t ld_out,
                                 float scale, void* work, size_t work_bytes) {
    const char* what = "masked attention forward";
    if (int rc = nrs::check(what, mask, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                            ld_out))
        return rc;
    if (batch == 0 || seq_q == 0) return NRS_OK;
    NRS_ARG_CHECK(out && q && ((k && v) || seq_k == 0), "%s: null pointer", what);
    NRS_REQUIRE_INIT();
    if (int rc = nrs::check_device(what)) return rc;
    float* scratch = nullptr;
    if (int rc = nrs::call_scratch(&scratch, 0, work, work_bytes, what)) return rc;
    auto a = nrs::arguments(mask, batch, heads, kv_heads, seq_q, seq_k, d_head, ld_q, ld_kv,
                            ld_out, scale);
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.stats = stats;
    const int64_t rows = batch * heads * seq_q;
    hipLaunchKernelGGL(nrs::masked_fwd_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0,
                       nrs::stream(), a);
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
    const int64_t all_rows = batch * heads * seq_q, all_keys = batch * kv_heads * seq_k;
    if (a.dq)
        hipLaunchKernelGGL(nrs::masked_dq_kernel, dim3((unsigned)((all_rows + 3) / 4)), dim3(256),
                           0, nrs::stream(), a);
    if (a.dk)
        hipLaunchKernelGGL(nrs::masked_dkv_kernel, dim3((unsigned)((all_keys + 3) / 4)), dim3(256),
                           0, nrs::stream(), a);
    NRS_LAUNCH_CHECK(what);
    return NRS_OK;
}

}  // extern "C"
