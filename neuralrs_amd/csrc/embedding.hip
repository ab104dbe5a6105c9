// Embedding lookup with scaling, and its gradient.
//
//   out[i] = scale * table[ids[i]]                          (a zero row for an id
//   dtable[t] = scale * sum over ids[i] = t of grad[i] + beta * dtable[t]
//                                              outside the table, no gradient)
//
// The gradient adds a token's rows in the order of their positions, by no
// atomics: the same call gives the same bits.
#include <algorithm>

#include "nrs_internal.hpp"

namespace nrs {
namespace {

// Rows need not be 16-byte aligned: gfx950 loads 128 bits from any dword.
typedef float f32x4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(4))) Quad {
    f32x4 v;
};

constexpr int kThreads = 256;

// `lanes` threads (a power of two) share a row, four columns each at a time;
// a row's last columns go one by one when dim is no multiple of four.
__global__ __launch_bounds__(kThreads) void embedding_forward_kernel(
    float* out, const float* table, const int32_t* ids, int64_t count, int vocab, int dim,
    int lanes, float scale) {
    const int rows = kThreads / lanes, r = threadIdx.x / lanes, c = threadIdx.x % lanes;
    const int64_t stride = (int64_t)gridDim.x * rows;
    for (int64_t i = (int64_t)blockIdx.x * rows + r; i < count; i += stride) {
        const int id = ids[i];
        const bool live = (uint32_t)id < (uint32_t)vocab;
        const float* src = table + (int64_t)(live ? id : 0) * dim;
        float* dst = out + i * dim;
        for (int d = 4 * c; d < dim; d += 4 * lanes) {
            if (d + 4 <= dim) {
                f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (live) v = reinterpret_cast<const Quad*>(src + d)->v * scale;
                reinterpret_cast<Quad*>(dst + d)->v = v;
            } else {
                for (int e = d; e < dim; ++e) dst[e] = live ? src[e] * scale : 0.0f;
            }
        }
    }
}

// One wave per table row and 256 columns: it looks through all ids and adds
// the rows that are its token's.
__global__ __launch_bounds__(64) void embedding_backward_kernel(
    float* dtable, const float* grad, const int32_t* ids, int64_t count, int vocab, int dim,
    float scale, float beta) {
    const int t = blockIdx.x, d = blockIdx.y * 256 + threadIdx.x * 4;
    const int live = max(0, min(4, dim - d));
    float sum[4] = {};
    bool any = false;
    for (int64_t i0 = 0; i0 < count; i0 += 64) {
        const int64_t i = i0 + threadIdx.x;
        uint64_t hits = __ballot(i < count && ids[i] == t);
        any |= hits != 0;
        while (hits) {
            const int64_t row = i0 + __builtin_ctzll(hits);
            hits &= hits - 1;
            for (int e = 0; e < live; ++e) sum[e] += grad[row * dim + d + e];
        }
    }
    float* dst = dtable + (int64_t)t * dim + d;
    for (int e = 0; e < live; ++e) {
        if (beta == 0.0f)
            dst[e] = scale * sum[e];
        else if (any || beta != 1.0f)
            dst[e] = scale * sum[e] + beta * dst[e];
    }
}

int check_shape(const char* what, int64_t count, int64_t vocab, int64_t dim) {
    NRS_ARG_CHECK(count >= 0 && count < INT32_MAX && vocab >= 1 && vocab < INT32_MAX && dim >= 1 &&
                      dim <= (1 << 20),
                  "%s: unsupported sizes (count %lld, vocab %lld, dim %lld): count and vocab are "
                  "below 2^31 - 1, vocab and dim at least 1, dim at most 2^20",
                  what, (long long)count, (long long)vocab, (long long)dim);
    return NRS_OK;
}

}  // namespace
}  // namespace nrs

extern "C" {

int nrs_embedding_forward(float* out, const float* table, const int32_t* ids, int64_t count,
                          int64_t vocab, int64_t dim, float scale) {
    if (int rc = nrs::check_shape("embedding forward", count, vocab, dim)) return rc;
    if (count == 0) return NRS_OK;
    NRS_ARG_CHECK(out && table && ids, "embedding forward: null pointer");
    NRS_REQUIRE_INIT();
    if (int rc = nrs::check_device("embedding forward")) return rc;
    int lanes = 1;
    while (lanes < nrs::kThreads && 4 * lanes < dim) lanes *= 2;
    const int64_t rows = nrs::kThreads / lanes;
    const dim3 grid((unsigned)std::min<int64_t>((count + rows - 1) / rows,
                                                16 * (int64_t)nrs::num_cus()));
    hipLaunchKernelGGL(nrs::embedding_forward_kernel, grid, dim3(nrs::kThreads), 0, nrs::stream(),
                       out, table, ids, count, (int)vocab, (int)dim, lanes, scale);
    NRS_LAUNCH_CHECK("embedding forward");
    return NRS_OK;
}

int nrs_embedding_workspace(size_t* bytes, int64_t count, int64_t vocab, int64_t dim) {
    NRS_ARG_CHECK(bytes, "embedding workspace: null pointer");
    if (int rc = nrs::check_shape("embedding workspace", count, vocab, dim)) return rc;
    *bytes = 0;
    return NRS_OK;
}

int nrs_embedding_backward(float* dtable, const float* grad, const int32_t* ids, int64_t count,
                           int64_t vocab, int64_t dim, float scale, float beta, void* work,
                           size_t work_bytes) {
    if (int rc = nrs::check_shape("embedding backward", count, vocab, dim)) return rc;
    NRS_ARG_CHECK(dtable && ((grad && ids) || count == 0), "embedding backward: null pointer");
    NRS_REQUIRE_INIT();
    if (int rc = nrs::check_device("embedding backward")) return rc;
    float* scratch = nullptr;
    if (int rc = nrs::call_scratch(&scratch, 0, work, work_bytes, "embedding backward")) return rc;
    const dim3 grid((unsigned)vocab, (unsigned)((dim + 255) / 256));
    hipLaunchKernelGGL(nrs::embedding_backward_kernel, grid, dim3(64), 0, nrs::stream(), dtable,
                       grad, ids, count, (int)vocab, (int)dim, scale, beta);
    NRS_LAUNCH_CHECK("embedding backward");
    return NRS_OK;
}

}  // extern "C"
