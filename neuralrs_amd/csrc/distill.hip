// The loss of a student's logits against a teacher's top logits, mixed with
// cross-entropy against a label, and its gradient.
//
// Per row, with p = softmax(top / T) over the teacher's tokens, q = softmax(z / T)
// and r = softmax(z) over the vocabulary:
//   loss = (1 - hard) T^2 sum_k p_k (log p_k - log q_{id_k}) + hard (-log r_label)
//   dz   = (1 - hard) T (q - sum_{id_k = v} p_k) + hard (r - [v = label])
// A workgroup has a row. The gradient needs the row twice, so that its first part stays
// in registers, and only what is past that is read again. The few columns that
// the teacher or the label change are written last. Where rows are few, several
// workgroups go over one row, which the caches hold, and write a part of its gradient
// each.
//
// Memory is the bound: 4096 x 32000 (64 tokens, two temperatures) takes 203 us, 5.2 TB/s
// of what is read and written once, 20000 x 2000 68 us, 4.8 TB/s; 1021 x 128003, of which
// half is read again, 238 us, 4.4 TB/s (223 with 128000, whose rows are aligned). A
// row by itself, 160000 logits, takes 23 us: one compute unit's exponentials.
#include <algorithm>

#include "buffer_ops.hpp"

namespace nrs {
namespace {

constexpr int kMaxTop = 1024;
constexpr int kSlots = 2 * kMaxTop;  // of the table that finds repeated tokens
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
    float *grad, *row_loss;
    const float *row_grad, *logits, *top;
    const int32_t *ids, *labels;
    int64_t ld, vocab;
    int k, shares;  // shares: workgroups that write a row's gradient
    int rows;
    float temperature, hard, mean;  // mean: a row's gradient without row_grad
};

// f over the lanes of a wave, then over the waves, in an order of their places alone,
// of N values at once. `part` is shared memory that nothing else uses.
template <int N, int WAVES, class F>
__device__ __forceinline__ void all_threads(float (&x)[N], float (&part)[WAVES][2], F f) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 1; i < 64; i *= 2) x[n] = f(x[n], __shfl_xor(x[n], i, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int n = 0; n < N; ++n) part[threadIdx.x >> 6][n] = x[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        x[n] = part[0][n];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) x[n] = f(x[n], part[w][n]);
    }
}

struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
// (NaN if either is)
struct MaxOrNan {
    __device__ __forceinline__ float operator()(float a, float b) const {
        return __builtin_elementwise_maximum(a, b);
    }
};

__device__ __forceinline__ float most_of(f32x4 z) {
    return fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
}

// The running maximum of a thread's logits and the sums of exp((z - m) / T) and
// (TWO) exp(z - m).
template <bool TWO>
struct Sums {
    float m = -INFINITY, soft = 0.0f, one = 0.0f;

    __device__ __forceinline__ void rise(float to, float by_t) {
        if (m != -INFINITY) {
            soft *= __builtin_amdgcn_exp2f((m - to) * by_t);
            if (TWO) one *= __builtin_amdgcn_exp2f((m - to) * kLog2e);
        }
        m = to;
    }
    // (m is at least the largest of them)
    __device__ __forceinline__ void add(float z, float by_t) {
        // only minus infinities so far, or NaN, which has to come through
        const float d = m == -INFINITY ? z : z - m;
        soft += __builtin_amdgcn_exp2f(d * by_t);
        if (TWO) one += __builtin_amdgcn_exp2f(d * kLog2e);
    }
    __device__ __forceinline__ void add(f32x4 z, float by_t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) add(z[e], by_t);
    }
};

// Of a row, each thread keeps QUADS times four logits.
template <int WAVES, int QUADS, bool GRAD, bool TWO>
__global__ __launch_bounds__(64 * WAVES, 4) void distill_kernel(DistillArgs a) {
    constexpr int kThreads = 64 * WAVES, kOwn = kMaxTop / kThreads;  // kOwn: teacher tokens
    __shared__ float part[WAVES][2];
    __shared__ int slots[kSlots], repeated, label_met;
    // where a token is repeated, in the place of the table: tokens and their weights
    int* const ids = slots;
    float* const weights = reinterpret_cast<float*>(slots + kMaxTop);
    const int64_t row = blockIdx.x % (uint32_t)a.rows;
    const int share = blockIdx.x / (uint32_t)a.rows;
    const float* const z = a.logits + row * a.ld;
    const int t = threadIdx.x;
    const float by_t = kLog2e / a.temperature, inv_t = 1.0f / a.temperature;
    // four logits at a time, and the last one to three by a thread each
    const int64_t quads = a.vocab / 4;
    const bool has_tail = 4 * quads + t < a.vocab && t < 3;
    auto quad = [&](int64_t i) { return reinterpret_cast<const Quad*>(z + 4 * i)->v; };
    f32x4 held[QUADS];
#pragma unroll
    for (int n = 0; n < QUADS; ++n) {
        const int64_t i = t + n * kThreads;
        held[n] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (i < quads) held[n] = quad(i);
    }
    const float tail = has_tail ? z[4 * quads + t] : -INFINITY;

    // the teacher: a thread's tokens, their weights and the student's logits of them
    const int label = a.labels ? a.labels[row] : -1;
    const bool labelled = a.hard > 0.0f && label >= 0 && label < a.vocab;
    const float z_label = labelled ? z[label] : 0.0f;
    int id[kOwn];
    float top[kOwn], own_z[kOwn], most[1] = {-INFINITY}, mass[1] = {0.0f};
    if (a.k > 0) {
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
            const int i = t + n * kThreads;
            id[n] = i < a.k ? a.ids[row * a.k + i] : -1;
            top[n] = i < a.k ? a.top[row * a.k + i] : 0.0f;
        }
        if (GRAD) {
            for (int i = t; i < kSlots; i += kThreads) slots[i] = -1;
            if (t == 0) repeated = label_met = 0;
        }
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
            if (id[n] < 0 || id[n] >= a.vocab) {
                id[n] = -1;
                top[n] = -INFINITY;
            }
            own_z[n] = id[n] >= 0 ? z[id[n]] : 0.0f;
            most[0] = MaxOrNan()(most[0], top[n]);
        }
        // (a teacher of NaN alone has a weight, too, which is not the absence of one)
        all_threads(most, part, MaxOrNan());
#pragma unroll
        for (int n = 0; n < kOwn; ++n)
            if (most[0] != -INFINITY) mass[0] += __builtin_amdgcn_exp2f((top[n] - most[0]) * by_t);
        if (GRAD)  // the barrier of the sum stands between this and the look at `repeated`
#pragma unroll
            for (int n = 0; n < kOwn; ++n) {
                if (id[n] < 0) continue;
                if (labelled && id[n] == label) label_met = 1;
                uint32_t at = (uint32_t)id[n] * 2654435761u >> 21;  // (a table of 2^11)
                for (;;) {  // fewer tokens than slots: an empty one or the same token ends it
                    const int was = atomicCAS(&slots[at], -1, id[n]);
                    if (was == id[n]) repeated = 1;
                    if (was == -1 || was == id[n]) break;
                    at = (at + 1) & (kSlots - 1);
                }
            }
        all_threads(mass, part, Add());
    }
    const bool taught = a.hard < 1.0f && most[0] != -INFINITY;

    // the row's maximum and sums
    Sums<TWO> s;
    s.m = tail;
    s.add(tail, by_t);
    constexpr int kAhead = 4;
    auto take = [&](const f32x4* x) {  // (as they arrive: the rest is on its way)
        float to = s.m;
#pragma unroll
        for (int n = 0; n < kAhead; ++n) to = fmaxf(to, most_of(x[n]));
        if (to > s.m) s.rise(to, by_t);
#pragma unroll
        for (int n = 0; n < kAhead; ++n) s.add(x[n], by_t);
    };
#pragma unroll
    for (int n = 0; n < QUADS; n += kAhead) take(held + n);
    for (int64_t i0 = QUADS * kThreads + t; i0 < quads; i0 += kAhead * kThreads) {
        f32x4 x[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            const int64_t i = i0 + n * kThreads;
            x[n] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (i < quads) x[n] = quad(i);
        }
        take(x);
    }
    float m[1] = {s.m};
    all_threads(m, part, Max());
    s.rise(m[0], by_t);
    float sums[TWO ? 2 : 1];
    sums[0] = s.soft;
    if (TWO) sums[TWO ? 1 : 0] = s.one;
    all_threads(sums, part, Add());
    const float soft = sums[0], one = sums[TWO ? 1 : 0];

    // the loss: log p - log q = (top - most) / T - log mass - (z - m) / T + log sum
    const float log_ratio = logf(soft) - logf(mass[0]);
    float loss[1] = {0.0f}, p[kOwn];
#pragma unroll
    for (int n = 0; n < kOwn; ++n) {
        p[n] = 0.0f;
        if (!taught || id[n] < 0) continue;
        const float far = top[n] - most[0];
        p[n] = __builtin_amdgcn_exp2f(far * by_t) / mass[0];
        if (p[n] != 0.0f) loss[0] += p[n] * ((far - (own_z[n] - m[0])) * inv_t + log_ratio);
    }
    if (a.row_loss) {
        all_threads(loss, part, Add());
        loss[0] *= (1.0f - a.hard) * a.temperature * a.temperature;
        if (labelled) loss[0] += a.hard * (logf(one) - (z_label - m[0]));
        if (t == 0 && share == 0) a.row_loss[row] = loss[0];
    }
    if (!GRAD) return;

    const float w = a.row_grad ? a.row_grad[row] : a.mean;
    const float of_soft = taught ? w * (1.0f - a.hard) * a.temperature : 0.0f;
    const float of_one = labelled ? w * a.hard : 0.0f;
    const float by_soft = of_soft / soft, by_one = of_one / one;
    // (padding may hold any numbers: a row that learns from nothing gets zeros)
    const bool learns = taught || labelled;
    auto dense = [&](float x) {
        // one exponential serves both where they are the same
        const float e = __builtin_amdgcn_exp2f((x - m[0]) * by_t);
        if (!TWO) return e * (by_soft + by_one);
        return e * by_soft + __builtin_amdgcn_exp2f((x - m[0]) * kLog2e) * by_one;
    };
    auto dense4 = [&](f32x4 x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = dense(x[e]);
        return x;
    };
    // (the teacher's logits of the student are in registers: the gradient may take the
    // logits' place)
    float* const g = a.grad + row * a.ld;
    // the workgroups that share a row take turns at runs of a quad to each thread
    auto mine = [&](int64_t run) { return (uint32_t)run % (uint32_t)a.shares == (uint32_t)share; };
    auto put = [&](int64_t i, f32x4 x) {
        if (i >= quads) return;
        x = learns ? dense4(x) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (WAVES <= 8) {
            reinterpret_cast<Quad*>(g + 4 * i)->v = x;
        } else {  // past the caches, which hold what is read again (1021 x 128003: 259 us if not)
#pragma unroll
            for (int e = 0; e < 4; ++e) __builtin_nontemporal_store(x[e], g + 4 * i + e);
        }
    };
#pragma unroll
    for (int n = 0; n < QUADS; ++n)
        if (mine(n)) put(t + n * kThreads, held[n]);
    if (has_tail && mine(quads / kThreads)) g[4 * quads + t] = learns ? dense(tail) : 0.0f;
    for (int64_t run = QUADS; run * kThreads < quads; run += kAhead) {
        f32x4 x[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            const int64_t i = t + (run + n) * kThreads;
            if (mine(run + n) && i < quads) x[n] = quad(i);
        }
#pragma unroll
        for (int n = 0; n < kAhead; ++n)
            if (mine(run + n)) put(t + (run + n) * kThreads, x[n]);
    }
    bool first[kOwn];
    if (a.k > 0) {
#pragma unroll
        for (int n = 0; n < kOwn; ++n) first[n] = id[n] >= 0;
        if (repeated) {  // the first place of a token takes the sum of all, in order
            // (the barriers of the row's sums stand between the table and this)
#pragma unroll
            for (int n = 0; n < kOwn; ++n) {
                ids[t + n * kThreads] = id[n];
                weights[t + n * kThreads] = p[n];
            }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < kOwn; ++n) {
                if (!first[n]) continue;
                p[n] = 0.0f;
                for (int j = 0; j < a.k; ++j)
                    if (ids[j] == id[n]) {
                        p[n] += weights[j];
                        if (j < t + n * kThreads) first[n] = false;
                    }
            }
        }
    }
    __syncthreads();  // the row is written: its few other columns can follow
    if (a.k > 0) {
#pragma unroll
        for (int n = 0; n < kOwn; ++n)
            if (learns && first[n] && mine(id[n] / 4 / kThreads))
                g[id[n]] = dense(own_z[n]) - of_soft * p[n] -
                           (labelled && id[n] == label ? of_one : 0.0f);
    }
    if (labelled && t == 0 && !(a.k > 0 && label_met) && mine(label / 4 / kThreads))
        g[label] = dense(z_label) - of_one;
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
    // a row is a workgroup of 512 threads, of fewer than 2^32 in all (1024 past 32768
    // columns, of which no memory holds 2^22 rows)
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

template <int WAVES, int QUADS, bool GRAD>
void launch_rows(const DistillArgs& a) {
    const bool two = a.hard > 0.0f && a.temperature != 1.0f;
    auto kernel = two ? distill_kernel<WAVES, QUADS, GRAD, true>
                      : distill_kernel<WAVES, QUADS, GRAD, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.rows * a.shares)), dim3(64 * WAVES), 0, stream(), a);
}

template <bool GRAD>
int launch(const char* what, DistillArgs a) {
    NRS_REQUIRE_INIT();
    if (int rc = check_device(what)) return rc;
    // A row is shared while that leaves every workgroup a compute unit, 8192 logits each at
    // least; not in place, where one would write what another still reads.
    const int64_t cus = num_cus();
    a.shares = 1;
    if (GRAD && a.grad != a.logits)
        a.shares = (int)std::max<int64_t>(1, std::min<int64_t>(cus / a.rows, a.vocab / 8192));
    // Waves to a row by what they hold of it: 2000 logits in two waves 68 us for 20000
    // rows, in eight 122; 128003 in 16 waves that hold 65536 259 us for 1021 rows, in eight
    // that hold 81920 271, in eight that hold 32768 (two rows to a compute unit) 324, all
    // with plain stores. The forward sums as the backward does: one loss, to the bit.
    if (a.vocab <= 2048)
        launch_rows<2, 4, GRAD>(a);
    else if (a.vocab <= 8192)
        launch_rows<8, 4, GRAD>(a);
    else if (a.vocab <= 32768)
        launch_rows<8, 16, GRAD>(a);
    else
        launch_rows<16, 16, GRAD>(a);
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
    a.rows = (int)rows;
    a.k = (int)k;
    a.temperature = temperature;
    a.hard = hard;
    return nrs::launch<false>(what, a);
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
    a.rows = (int)rows;
    a.k = (int)k;
    a.temperature = temperature;
    a.hard = hard;
    a.mean = (float)(1.0 / (double)rows);
    return nrs::launch<true>(what, a);
}

}  // extern "C"
