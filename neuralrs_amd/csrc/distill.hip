// The loss of a student's logits against a teacher's top logits, mixed with
// cross-entropy against a label, and its gradient.
//
// Per row, with p = softmax(top / T) over the teacher's tokens, q = softmax(z / T)
// and r = softmax(z) over the vocabulary:
//   loss = (1 - hard) T^2 sum_k p_k (log p_k - log q_{id_k}) + hard (-log r_label)
//   dz   = (1 - hard) T (q - sum_{id_k = v} p_k) + hard (r - [v = label])
// A workgroup has a row: its maximum and sums, then the gradient from the row read
// again, then the few columns that the teacher or the label change.
#include <algorithm>

#include "buffer_ops.hpp"

namespace nrs {
namespace {

constexpr int kMaxTop = 1024, kWaves = 8, kThreads = 64 * kWaves;
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
    float *grad, *row_loss;
    const float *row_grad, *logits, *top;
    const int32_t *ids, *labels;
    int64_t ld, vocab;
    int k;
    float temperature, hard, mean;  // mean: a row's gradient without row_grad
};

// f over a wave's lanes, then over the waves, in an order of their places alone.
// `part` is shared memory that nothing else uses between two calls' barriers.
template <class F>
__device__ __forceinline__ float all_threads(float x, float (&part)[kWaves], F f) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) x = f(x, __shfl_xor(x, i, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = part[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) x = f(x, part[w]);
    return x;
}

struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// The running maximum of a thread's logits and the sums of exp((z - m) / T) and
// (TWO) exp(z - m).
template <bool TWO>
struct Sums {
    float m = -INFINITY, soft = 0.0f, one = 0.0f;

    __device__ __forceinline__ void rise(float to, float by_t) {
        const float old = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - to) * by_t);
        soft *= old;
        if (TWO) one *= m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - to) * kLog2e);
        m = to;
    }
    __device__ __forceinline__ void add(f32x4 z, float by_t) {
        const float top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
        if (top > m) rise(top, by_t);
        if (m == -INFINITY) {
            // (only minus infinities so far, or NaN, which has to come through)
#pragma unroll
            for (int e = 0; e < 4; ++e) soft += z[e] == -INFINITY ? 0.0f : z[e];
            if (TWO) one = soft;
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            soft += __builtin_amdgcn_exp2f((z[e] - m) * by_t);
            if (TWO) one += __builtin_amdgcn_exp2f((z[e] - m) * kLog2e);
        }
    }
};

template <bool GRAD, bool TWO>
__global__ __launch_bounds__(kThreads) void distill_kernel(DistillArgs a) {
    __shared__ float part[kWaves];
    __shared__ float tops[kMaxTop];   // the teacher's weights, 0 where there is no token
    __shared__ int ids[kMaxTop];      // -1 where there is none
    const int64_t row = blockIdx.x;
    const float* const z = a.logits + row * a.ld;
    const int t = threadIdx.x;
    const float by_t = kLog2e / a.temperature, inv_t = 1.0f / a.temperature;

    // the teacher
    float most = -INFINITY;
    for (int i = t; i < a.k; i += kThreads) {
        const int id = a.ids[row * a.k + i];
        const bool live = id >= 0 && id < a.vocab;
        const float v = live ? a.top[row * a.k + i] : -INFINITY;
        ids[i] = live ? id : -1;
        tops[i] = v;
        most = fmaxf(most, v);
    }
    most = all_threads(most, part, Max());
    float mass = 0.0f;
    for (int i = t; i < a.k; i += kThreads)
        if (most > -INFINITY) mass += __builtin_amdgcn_exp2f((tops[i] - most) * by_t);
    mass = all_threads(mass, part, Add());
    const bool taught = a.hard < 1.0f && most > -INFINITY;
    const int label = a.labels ? a.labels[row] : -1;
    const bool labelled = a.hard > 0.0f && label >= 0 && label < a.vocab;

    // the row's maximum and sums
    Sums<TWO> s;
    for (int64_t v = 4 * t; v < a.vocab; v += 4 * kThreads) {
        f32x4 x = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (v + 4 <= a.vocab)
            x = reinterpret_cast<const Quad*>(z + v)->v;
        else
            for (int e = 0; v + e < a.vocab; ++e) x[e] = z[v + e];
        s.add(x, by_t);
    }
    const float m = all_threads(s.m, part, Max());
    if (s.m != -INFINITY) s.rise(m, by_t);
    const float soft = all_threads(s.soft, part, Add());
    const float one = TWO ? all_threads(s.one, part, Add()) : soft;

    // the loss: log p - log q = (top - most) / T - log mass - (z - m) / T + log sum
    const float log_soft = logf(soft), log_mass = logf(mass);
    float loss = 0.0f;
    for (int i = t; i < a.k; i += kThreads) {
        const float p = taught ? __builtin_amdgcn_exp2f((tops[i] - most) * by_t) / mass : 0.0f;
        if (p > 0.0f || p != p)
            loss += p * (((tops[i] - most) - (z[ids[i]] - m)) * inv_t + (log_soft - log_mass));
        tops[i] = p;  // this thread's own
    }
    loss = all_threads(loss, part, Add()) * (1.0f - a.hard) * a.temperature * a.temperature;
    float z_label = 0.0f;
    if (labelled) {
        z_label = z[label];
        loss += a.hard * (logf(one) - (z_label - m));
    }
    if (t == 0 && a.row_loss) a.row_loss[row] = loss;
    if (!GRAD) return;

    const float w = a.row_grad ? a.row_grad[row] : a.mean;
    const float of_soft = taught ? w * (1.0f - a.hard) * a.temperature : 0.0f;
    const float of_one = labelled ? w * a.hard : 0.0f;
    const float by_soft = of_soft / soft, by_one = of_one / one;
    auto dense = [&](float x) {
        // one exponential serves both where they are the same
        const float e = __builtin_amdgcn_exp2f((x - m) * by_t);
        if (!TWO) return e * (by_soft + by_one);
        return e * by_soft + __builtin_amdgcn_exp2f((x - m) * kLog2e) * by_one;
    };
    // what the teacher's tokens get, before the gradient may take the logits' place
    float own[kMaxTop / kThreads];
    bool label_met = false;
#pragma unroll
    for (int n = 0; n < kMaxTop / kThreads; ++n) {
        const int i = t + n * kThreads;
        own[n] = 0.0f;
        if (i >= a.k || ids[i] < 0) continue;
        float p = 0.0f;
        bool first = true;
        for (int j = 0; j < a.k; ++j)
            if (ids[j] == ids[i]) {
                p += tops[j];
                first = first && j >= i;
            }
        if (!first) continue;  // another place of the same token
        own[n] = dense(z[ids[i]]) - of_soft * p - (labelled && ids[i] == label ? of_one : 0.0f);
    }
    float* const g = a.grad + row * a.ld;
    __syncthreads();
    for (int64_t v = 4 * t; v < a.vocab; v += 4 * kThreads) {
        if (v + 4 <= a.vocab) {
            f32x4 x = reinterpret_cast<const Quad*>(z + v)->v;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = dense(x[e]);
            reinterpret_cast<Quad*>(g + v)->v = x;
        } else {
            for (int e = 0; v + e < a.vocab; ++e) g[v + e] = dense(z[v + e]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kMaxTop / kThreads; ++n) {
        const int i = t + n * kThreads;
        if (i >= a.k || ids[i] < 0) continue;
        bool first = true;
        for (int j = 0; j < i; ++j) first = first && ids[j] != ids[i];
        if (first) g[ids[i]] = own[n];
        label_met = label_met || ids[i] == label;
    }
    if (labelled && !__syncthreads_or(label_met) && t == 0) g[label] = dense(z_label) - of_one;
}

int check(const char* what, const float* logits, const float* top, const int32_t* ids,
          const int32_t* labels, int64_t rows, int64_t vocab, int64_t k, int64_t ld,
          float temperature, float hard) {
    NRS_ARG_CHECK(rows >= 0 && vocab >= 1 && k >= 0, "%s: a size is negative or there is no "
                  "vocabulary (rows %lld, vocab %lld, k %lld)", what, (long long)rows,
                  (long long)vocab, (long long)k);
    NRS_ARG_CHECK(k <= kMaxTop, "%s: k is %lld, at most %d are taken", what, (long long)k, kMaxTop);
    NRS_ARG_CHECK(ld >= vocab, "%s: row stride %lld is shorter than the vocabulary of %lld", what,
                  (long long)ld, (long long)vocab);
    // a row is a workgroup of 512 threads, of fewer than 2^32 in all
    NRS_ARG_CHECK(rows < (int64_t(1) << 23) && ld < (int64_t(1) << 31),
                  "%s: more than 2^23 - 1 rows or 2^31 - 1 columns (rows %lld, stride %lld)", what,
                  (long long)rows, (long long)ld);
    NRS_ARG_CHECK(temperature > 0.0f && temperature <= 1e6f && temperature >= 1e-6f,
                  "%s: temperature must be in [1e-6, 1e6], is %g", what, (double)temperature);
    NRS_ARG_CHECK(hard >= 0.0f && hard <= 1.0f, "%s: hard must be in [0, 1], is %g", what,
                  (double)hard);
    if (rows == 0) return NRS_OK;
    NRS_ARG_CHECK(hard == 0.0f || labels, "%s: hard is %g but there are no labels", what,
                  (double)hard);
    NRS_ARG_CHECK(logits && (k == 0 || (top && ids)), "%s: null pointer", what);
    return NRS_OK;
}

template <bool GRAD>
int launch(const char* what, const DistillArgs& a, int64_t rows) {
    NRS_REQUIRE_INIT();
    if (int rc = check_device(what)) return rc;
    const bool two = a.hard > 0.0f && a.temperature != 1.0f;
    auto kernel = two ? distill_kernel<GRAD, true> : distill_kernel<GRAD, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(kThreads), 0, stream(), a);
    NRS_LAUNCH_CHECK(what);
    return NRS_OK;
}

}  // namespace
}  // namespace nrs

extern "C" {

int nrs_distill_forward(float* row_loss, const float* logits, const float* top,
                        const int32_t* top_ids, const int32_t* labels, int64_t rows, int64_t vocab,
                        int64_t k, int64_t ld, float temperature, float hard) {
    const char* what = "distill forward";
    if (int rc = nrs::check(what, logits, top, top_ids, labels, rows, vocab, k, ld, temperature,
                            hard))
        return rc;
    if (rows == 0) return NRS_OK;
    NRS_ARG_CHECK(row_loss, "%s: null pointer", what);
    nrs::DistillArgs a{};
    a.row_loss = row_loss;
    a.logits = logits;
    a.top = top;
    a.ids = top_ids;
    a.labels = labels;
    a.ld = ld;
    a.vocab = vocab;
    a.k = (int)k;
    a.temperature = temperature;
    a.hard = hard;
    return nrs::launch<false>(what, a, rows);
}

int nrs_distill_backward(float* grad, float* row_loss, const float* row_grad, const float* logits,
                         const float* top, const int32_t* top_ids, const int32_t* labels,
                         int64_t rows, int64_t vocab, int64_t k, int64_t ld, float temperature,
                         float hard) {
    const char* what = "distill backward";
    if (int rc = nrs::check(what, logits, top, top_ids, labels, rows, vocab, k, ld, temperature,
                            hard))
        return rc;
    if (rows == 0) return NRS_OK;
    NRS_ARG_CHECK(grad, "%s: null pointer", what);
    nrs::DistillArgs a{};
    a.grad = grad;
    a.row_loss = row_loss;
    a.row_grad = row_grad;
    a.logits = logits;
    a.top = top;
    a.ids = top_ids;
    a.labels = labels;
    a.ld = ld;
    a.vocab = vocab;
    a.k = (int)k;
    a.temperature = temperature;
    a.hard = hard;
    a.mean = (float)(1.0 / (double)rows);
    return nrs::launch<true>(what, a, rows);
}

}  // extern "C"
