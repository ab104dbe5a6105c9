// Dropout whose mask is recomputed wherever it is needed and never stored.
//
// Element i is kept when word i % 4 of the Philox4x32-10 block with counter
// (i / 4, call) and key `seed` (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011) is at least round(p * 2^32): the mask
// is a function of the element's index and two numbers, so the backward makes
// the same one and it does not depend on how a launch divides the elements.
// A thread makes one block of four words at a time for four neighbouring
// elements. Memory is the bound: 16.8 M floats take 21.6 us, 6.2 TB/s of what is
// read and written, with the blocks' 20 wide products apiece behind it; 8192
// floats take 2.6 us, a launch and a round trip.
#include <algorithm>

#include "nrs_internal.hpp"

namespace nrs {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct DropoutArgs {
    float* out;
    const float* x;
    const float* add;  // added to the result: the residual, or the old gradient
    const uint64_t* step;
    int64_t n;
    uint64_t seed, call, threshold;  // kept: word >= threshold (2^32 keeps none)
    float inv;                       // 1 / (1 - p)
    float add_scale;                 // 0 leaves `add` unread
};

// Ten rounds; each multiplies two words by a constant into 64-bit products.
__device__ __forceinline__ u32x4 philox(uint64_t block, uint64_t call, uint64_t seed) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)call,
             c3 = (uint32_t)(call >> 32), k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}

// x times the rounded 1 / (1 - p) (a product, where a quotient would take ten
// instructions) is rounded by itself before anything is added, so that dropout with
// a residual has the bits of dropout followed by nrs_vadd. A dropped
// element is a zero whatever x holds there.
__device__ __forceinline__ float drop(float x, uint32_t word, const DropoutArgs& a) {
#pragma clang fp contract(off)
    const float v = x * a.inv;
    return word >= a.threshold ? v : 0.0f;
}

template <bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
    const uint64_t call = a.call + (a.step ? *a.step : 0);
    const int64_t blocks = (a.n + 3) / 4, stride = (int64_t)gridDim.x * 256;
    for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < blocks; b += stride) {
        const u32x4 w = philox((uint64_t)b, call, a.seed);
        if (VEC && 4 * b + 4 <= a.n) {
            const f32x4 x = reinterpret_cast<const f32x4*>(a.x)[b];
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = drop(x[e], w[e], a);
            if (a.add_scale != 0.0f)
                v = v + a.add_scale * reinterpret_cast<const f32x4*>(a.add)[b];
            reinterpret_cast<f32x4*>(a.out)[b] = v;
        } else {
            for (int e = 0; e < 4 && 4 * b + e < a.n; ++e) {
                float v = drop(a.x[4 * b + e], w[e], a);
                if (a.add_scale != 0.0f) v = v + a.add_scale * a.add[4 * b + e];
                a.out[4 * b + e] = v;
            }
        }
    }
}

int launch(const char* what, DropoutArgs a, float p) {
    if (int rc = check_device(what)) return rc;
    a.threshold = (uint64_t)((double)p * 4294967296.0 + 0.5);
    a.inv = p < 1.0f ? (float)(1.0 / (1.0 - (double)p)) : 0.0f;
    const bool vec = (((uintptr_t)a.out | (uintptr_t)a.x |
                       (a.add_scale != 0.0f ? (uintptr_t)a.add : 0)) & 15) == 0;
    const int64_t groups = ((a.n + 3) / 4 + 255) / 256;
    const dim3 grid((unsigned)std::min<int64_t>(groups, 8 * (int64_t)num_cus()));
    auto kernel = vec ? dropout_kernel<true> : dropout_kernel<false>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream(), a);
    NRS_LAUNCH_CHECK(what);
    return NRS_OK;
}

}  // namespace
}  // namespace nrs

extern "C" {

int nrs_dropout_forward(float* out, const float* x, const float* residual, int64_t n, float p,
                        uint64_t seed, uint64_t call, const uint64_t* step) {
    NRS_ARG_CHECK(n >= 0, "dropout: negative size %lld", (long long)n);
    NRS_ARG_CHECK(p >= 0.0f && p <= 1.0f, "dropout: p must be in [0, 1], is %g", (double)p);
    if (n == 0) return NRS_OK;
    NRS_ARG_CHECK(out && x, "dropout: null pointer");
    NRS_REQUIRE_INIT();
    nrs::DropoutArgs a{};
    a.out = out;
    a.x = x;
    a.add = residual;
    a.add_scale = residual ? 1.0f : 0.0f;
    a.n = n;
    a.seed = seed;
    a.call = call;
    a.step = step;
    return nrs::launch("dropout forward", a, p);
}

int nrs_dropout_backward(float* gin, const float* grad, int64_t n, float p, uint64_t seed,
                         uint64_t call, const uint64_t* step, float beta) {
    NRS_ARG_CHECK(n >= 0, "dropout backward: negative size %lld", (long long)n);
    NRS_ARG_CHECK(p >= 0.0f && p <= 1.0f, "dropout backward: p must be in [0, 1], is %g",
                  (double)p);
    if (n == 0) return NRS_OK;
    NRS_ARG_CHECK(gin && grad, "dropout backward: null pointer");
    NRS_REQUIRE_INIT();
    nrs::DropoutArgs a{};
    a.out = gin;
    a.x = grad;
    a.add = gin;
    a.add_scale = beta;
    a.n = n;
    a.seed = seed;
    a.call = call;
    a.step = step;
    return nrs::launch("dropout backward", a, p);
}

}  // extern "C"
