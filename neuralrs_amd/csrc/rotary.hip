// Rotary positions: pair j of every head of a row is turned by the angle
// positions[axis[j]][row] * freq[j], forward by it and backward by its negative.
//
// The angle is taken in 64 bits and reduced to a part of a whole turn before it
// is rounded to a float: at position 100000 a float angle would be off by 0.004.
//
// Memory is the bound: 16001 rows of 20 heads of 128 take 69 us, 4.8 TB/s of what is read
// and written once (with one head's columns on the way at a time, in place of four, 90);
// 32 rows 3.6 us, a launch, two round trips and the functions.
#include <algorithm>

#include "buffer_ops.hpp"
#include "fastdiv.hpp"

namespace nrs {
namespace {

struct RotaryArgs {
    float* out;
    const float* x;
    const int32_t *positions, *axis;
    const float* freq;
    int64_t rows, ld_x, ld_out;
    int heads, d, pairs, axes;
    int units;       // of a head: four pairs each, then eight columns that are not turned
    int turned;      // units of pairs
    int slots;       // threads that share a row's heads
    FastDiv by_units, by_row;
    bool interleaved;
    float sign, beta;
};

__device__ __forceinline__ f32x4 load4(const float* p, int n) {
    if (n >= 4) return reinterpret_cast<const Quad*>(p)->v;
    f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int e = 0; e < n; ++e) v[e] = p[e];
    return v;
}

__device__ __forceinline__ void store4(float* p, int n, f32x4 v, float beta) {
    if (n >= 4) {
        Quad* const to = reinterpret_cast<Quad*>(p);
        if (beta != 0.0f) v = v + beta * to->v;
        to->v = v;
    } else {
        for (int e = 0; e < n; ++e) p[e] = beta != 0.0f ? v[e] + beta * p[e] : v[e];
    }
}

// A thread has a unit of a row, the sines and cosines of its four pairs, and every
// slots-th head, of which it has kAhead on the way at a time.
template <bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    constexpr int kAhead = 4;
    const uint32_t per_row = (uint32_t)(a.units * a.slots);
    // (a workgroup's first row by one division, its threads' by small ones)
    const uint64_t id0 = (uint64_t)blockIdx.x * 256;
    const uint32_t in0 = (uint32_t)(id0 % per_row) + threadIdx.x;
    const uint32_t over = fast_div(in0, a.by_row);
    const int64_t row = (int64_t)(id0 / per_row) + over;
    if (row >= a.rows) return;
    const uint32_t in_row = in0 - over * per_row;
    const int slot = (int)fast_div(in_row, a.by_units), unit = (int)in_row - slot * a.units;
    const bool turn = unit < a.turned;
    const int j0 = 4 * unit, n = min(4, a.pairs - j0);  // pairs of a unit that is turned
    int c0 = 2 * a.pairs + 8 * (unit - a.turned), c1 = c0 + 4, n0 = a.d - c0, n1 = a.d - c1;
    if (turn) {
        c0 = INTERLEAVED ? 2 * j0 : j0;
        c1 = INTERLEAVED ? c0 + 4 : a.pairs + j0;
        n0 = INTERLEAVED ? 2 * n : n;
        n1 = INTERLEAVED ? 2 * n - 4 : n;
    }
    const float* const src = a.x + row * a.ld_x;
    float* const dst = a.out + row * a.ld_out;
    f32x4 p[kAhead], q[kAhead];
    auto load = [&](int h0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int h = h0 + i * a.slots;
            if (h >= a.heads) break;
            p[i] = load4(src + (int64_t)h * a.d + c0, n0);
            q[i] = load4(src + (int64_t)h * a.d + c1, n1);
        }
    };
    load(slot);
    f32x4 cos, sin;
    if (turn) {
        int axis[4];
        double place[4];
        float freq[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = j0 + min(e, n - 1);
            axis[e] = a.axis ? a.axis[j] : 0;
            freq[e] = a.freq[j];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool any = axis[e] >= 0 && axis[e] < a.axes;
            place[e] = any ? (double)a.positions[axis[e] * a.rows + row] : 0.0;
            freq[e] = any ? freq[e] : 0.0f;  // an angle of zero
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double turns = place[e] * (double)freq[e] * 0.15915494309189535;
            float s, c;
            sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
            cos[e] = c;
            sin[e] = s * a.sign;
        }
    }
    for (int h0 = slot; h0 < a.heads; h0 += kAhead * a.slots) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int h = h0 + i * a.slots;
            if (h >= a.heads) break;
            f32x4 x = p[i], y = q[i];
            if (turn) {
                if (INTERLEAVED) {
                    x = f32x4{p[i][0] * cos[0] - p[i][1] * sin[0], p[i][1] * cos[0] + p[i][0] * sin[0],
                              p[i][2] * cos[1] - p[i][3] * sin[1], p[i][3] * cos[1] + p[i][2] * sin[1]};
                    y = f32x4{q[i][0] * cos[2] - q[i][1] * sin[2], q[i][1] * cos[2] + q[i][0] * sin[2],
                              q[i][2] * cos[3] - q[i][3] * sin[3], q[i][3] * cos[3] + q[i][2] * sin[3]};
                } else {
                    x = p[i] * cos - q[i] * sin;
                    y = q[i] * cos + p[i] * sin;
                }
            }
            store4(dst + (int64_t)h * a.d + c0, n0, x, a.beta);
            store4(dst + (int64_t)h * a.d + c1, n1, y, a.beta);
        }
        if (h0 + kAhead * a.slots < a.heads) load(h0 + kAhead * a.slots);
    }
}

constexpr int64_t kMaxLd = 1 << 20, kMaxRows = int64_t(1) << 30;

int launch(const char* what, RotaryArgs a) {
    NRS_REQUIRE_INIT();
    if (int rc = check_device(what)) return rc;
    a.turned = (a.pairs + 3) / 4;
    // in place, what is not turned is there already
    const bool copied = a.out != a.x;
    a.units = a.turned + (copied ? (a.d - 2 * a.pairs + 7) / 8 : 0);
    if (a.units == 0) return NRS_OK;
    // Heads to a thread, which has their angles once: up to 16, as long as there are 512
    // threads to a compute unit.
    const int64_t each = std::min<int64_t>(
        16, std::max<int64_t>(1, a.rows * a.units * a.heads / (512 * (int64_t)num_cus())));
    a.slots = (int)((a.heads + each - 1) / each);
    a.by_units = make_fastdiv((uint32_t)a.units);
    a.by_row = make_fastdiv((uint32_t)(a.units * a.slots));
    const int64_t threads = a.rows * a.units * a.slots;
    hipLaunchKernelGGL(a.interleaved ? rotary_kernel<true> : rotary_kernel<false>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0,
                       stream(), a);
    NRS_LAUNCH_CHECK(what);
    return NRS_OK;
}

int check(const char* what, const RotaryArgs& a, int64_t rows, int64_t heads, int64_t d_head,
          int64_t pairs, int64_t axes, int64_t ld_x, int64_t ld_out) {
    const char* why = nullptr;
    if (rows < 0 || heads < 1 || d_head < 1 || pairs < 0 || axes < 1)
        why = "a size is negative or there are no heads, columns or axes";
    else if (pairs > d_head / 2)
        why = "more pairs than half of d_head";
    else if (heads > kMaxLd / d_head || ld_x < heads * d_head || ld_out < heads * d_head)
        why = "a row stride is shorter than its heads";
    else if (ld_x > kMaxLd || ld_out > kMaxLd)
        why = "a row stride is past 2^20";
    // a thread has eight columns, or what is left of a head, and a launch has fewer
    // than 2^32 threads
    else if (rows > kMaxRows || axes > kMaxRows ||
             rows > (int64_t(1) << 31) / (heads * ((d_head + 15) / 8)))
        why = "more than 2^30 rows or axes, or 2^31 pieces of eight columns";
    NRS_ARG_CHECK(!why, "%s: %s (rows %lld, heads %lld, d_head %lld, pairs %lld, axes %lld, "
                  "strides %lld and %lld)", what, why, (long long)rows, (long long)heads,
                  (long long)d_head, (long long)pairs, (long long)axes, (long long)ld_x,
                  (long long)ld_out);
    if (rows == 0) return NRS_OK;
    NRS_ARG_CHECK(a.out && a.x && (pairs == 0 || (a.positions && a.freq)), "%s: null pointer",
                  what);
    NRS_ARG_CHECK(a.out != a.x || ld_x == ld_out, "%s: in place with two row strides", what);
    return NRS_OK;
}

}  // namespace
}  // namespace nrs

extern "C" {

int nrs_rotary_forward(float* out, const float* x, const int32_t* positions, const float* freq,
                       const int32_t* axis, int64_t rows, int64_t heads, int64_t d_head,
                       int64_t pairs, int64_t axes, int64_t ld_x, int64_t ld_out,
                       int interleaved) {
    nrs::RotaryArgs a{};
    a.out = out;
    a.x = x;
    a.positions = positions;
    a.freq = freq;
    a.axis = axis;
    if (int rc = nrs::check("rotary forward", a, rows, heads, d_head, pairs, axes, ld_x, ld_out))
        return rc;
    if (rows == 0) return NRS_OK;
    a.rows = rows;
    a.ld_x = ld_x;
    a.ld_out = ld_out;
    a.heads = (int)heads;
    a.d = (int)d_head;
    a.pairs = (int)pairs;
    a.axes = (int)axes;
    a.interleaved = interleaved != 0;
    a.sign = 1.0f;
    return nrs::launch("rotary forward", a);
}

int nrs_rotary_backward(float* gin, const float* grad, const int32_t* positions, const float* freq,
                        const int32_t* axis, int64_t rows, int64_t heads, int64_t d_head,
                        int64_t pairs, int64_t axes, int64_t ld_gin, int64_t ld_grad,
                        int interleaved, float beta) {
    const char* what = "rotary backward";
    nrs::RotaryArgs a{};
    a.out = gin;
    a.x = grad;
    a.positions = positions;
    a.freq = freq;
    a.axis = axis;
    if (int rc = nrs::check(what, a, rows, heads, d_head, pairs, axes, ld_grad, ld_gin)) return rc;
    if (rows == 0) return NRS_OK;
    NRS_ARG_CHECK(gin != grad || beta == 0.0f, "%s: in place with a beta of %g", what,
                  (double)beta);
    a.rows = rows;
    a.ld_x = ld_grad;
    a.ld_out = ld_gin;
    a.heads = (int)heads;
    a.d = (int)d_head;
    a.pairs = (int)pairs;
    a.axes = (int)axes;
    a.interleaved = interleaved != 0;
    a.sign = -1.0f;
    a.beta = beta;
    return nrs::launch(what, a);
}

}  // extern "C"
