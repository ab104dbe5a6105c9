// Rotary positions: pair j of every head of a row is turned by the angle
// positions[axis[j]][row] * freq[j], forward by it and backward by its negative.
//
// The angle is taken in 64 bits and reduced to a part of a whole turn before it
// is rounded to a float: at position 100000 a float angle would be off by 0.004.
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
    FastDiv by_units, by_slots;
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

// A thread has a unit of a row, the sines and cosines of its four pairs, and
// every slots-th head.
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    const int64_t per_row = (int64_t)a.units * a.slots;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = id / per_row;
    if (row >= a.rows) return;
    const uint32_t in_row = (uint32_t)(id - row * per_row);
    const int slot = (int)fast_div(in_row, a.by_units), unit = (int)in_row - slot * a.units;
    int c0, c1, n0, n1;
    f32x4 cos = f32x4{1.0f, 1.0f, 1.0f, 1.0f}, sin = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const bool turn = unit < a.turned;
    if (turn) {
        const int j0 = 4 * unit, n = min(4, a.pairs - j0);
        if (a.interleaved) {
            c0 = 2 * j0;
            c1 = c0 + 4;
            n0 = min(4, 2 * n);
            n1 = 2 * n - 4;
        } else {
            c0 = j0;
            c1 = a.pairs + j0;
            n0 = n1 = n;
        }
        for (int e = 0; e < n; ++e) {
            const int axis = a.axis ? a.axis[j0 + e] : 0;
            if (axis < 0 || axis >= a.axes) continue;
            const double turns = (double)a.positions[axis * a.rows + row] * (double)a.freq[j0 + e] *
                                 0.15915494309189535;
            float s, c;
            sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
            cos[e] = c;
            sin[e] = s * a.sign;
        }
    } else {
        c0 = 2 * a.pairs + 8 * (unit - a.turned);
        c1 = c0 + 4;
        n0 = a.d - c0;
        n1 = a.d - c1;
    }
    for (int h = slot; h < a.heads; h += a.slots) {
        const float* const src = a.x + row * a.ld_x + (int64_t)h * a.d;
        float* const dst = a.out + row * a.ld_out + (int64_t)h * a.d;
        f32x4 p = load4(src + c0, n0), q = load4(src + c1, n1);
        if (turn) {
            if (a.interleaved) {
                const f32x4 x = p, y = q;
                p = f32x4{x[0] * cos[0] - x[1] * sin[0], x[1] * cos[0] + x[0] * sin[0],
                          x[2] * cos[1] - x[3] * sin[1], x[3] * cos[1] + x[2] * sin[1]};
                q = f32x4{y[0] * cos[2] - y[1] * sin[2], y[1] * cos[2] + y[0] * sin[2],
                          y[2] * cos[3] - y[3] * sin[3], y[3] * cos[3] + y[2] * sin[3]};
            } else {
                const f32x4 x = p, y = q;
                p = x * cos - y * sin;
                q = y * cos + x * sin;
            }
        }
        store4(dst + c0, n0, p, a.beta);
        store4(dst + c1, n1, q, a.beta);
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
    // up to eight heads to a thread, as long as there are 512 threads to a compute unit
    const int64_t each = std::min<int64_t>(
        8, std::max<int64_t>(1, a.rows * a.units * a.heads / (512 * (int64_t)num_cus())));
    a.slots = (int)((a.heads + each - 1) / each);
    a.by_units = make_fastdiv((uint32_t)a.units);
    const int64_t threads = a.rows * a.units * a.slots;
    hipLaunchKernelGGL(rotary_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0,
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
