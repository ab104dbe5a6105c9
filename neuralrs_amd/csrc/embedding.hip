// Embedding lookup with scaling, and its gradient.
//
//   out[i] = scale * table[ids[i]]                          (a zero row for an id
//   dtable[t] = scale * sum over ids[i] = t of grad[i] + beta * dtable[t]
//                                              outside the table, no gradient)
//
// The gradient of more than 256 positions takes three launches:
//  1. sort: every workgroup owns a range of tokens, looks through all ids twice
//     (they stay in the caches) and places its own tokens' positions, in order,
//     behind those of lower tokens: a counting sort without a pass between
//     workgroups. Beside it, with beta 0, other workgroups clear the table.
//  2. sum: the sorted positions are cut into tiles of equal length, so that a
//     token that holds a sixth of all places (a space, say) is as even as any.
//     A wave adds a tile's rows, 256 columns of them, and writes the sums of
//     the tokens that begin and end in it; the sum of a run that crosses the
//     tile's beginning or end goes to scratch.
//  3. join: adds the parts of every run that crosses tiles, in order.
// No floating-point atomics: the order of a sum depends on the ids alone.
// Memory bounds the large calls, round trips and launches the small ones:
//                                       lookup    sort    sum   join (us)
//   4096 ids of 32000 tokens, 256 wide       3.8    10.3    6.6    4.0
//   49999 of 50021, 1000 wide               60      46     73      6.3
//   65536 of 259, 512 wide                  24      26     23     10
// In the second, whose ids are of some 13000 tokens, the lookup moves 4.2 TB/s and the
// sum 3.4; the 200 MB of the table's gradient are cleared beside the sort, in its 46
// us (4.3). In the third the lookup moves 5.6 and the sum 5.8.
#include <algorithm>

#include "buffer_ops.hpp"

namespace nrs {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 4;  // rows a thread of the lookup has in flight

// `lanes` threads (a power of two) share a row, four columns each at a time;
// a row's last columns go one by one when dim is no multiple of four. The
// rows' tokens, then the rows, are asked for together: a row by itself waits
// for two loads, one after the other.
__global__ __launch_bounds__(kThreads) void embedding_forward_kernel(
    float* out, const float* table, const int32_t* ids, int64_t count, int vocab, int dim,
    int lanes, float scale) {
    const int rows = kThreads / lanes, r = threadIdx.x / lanes, c = threadIdx.x % lanes;
    const int64_t stride = (int64_t)gridDim.x * rows;
    for (int64_t i0 = (int64_t)blockIdx.x * rows + r; i0 < count; i0 += kRows * stride) {
        int id[kRows];
#pragma unroll
        for (int k = 0; k < kRows; ++k) id[k] = i0 + k * stride < count ? ids[i0 + k * stride] : -1;
        for (int d = 4 * c; d < dim; d += 4 * lanes) {
            const int live = min(4, dim - d);
            f32x4 v[kRows];
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                v[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if ((uint32_t)id[k] >= (uint32_t)vocab) continue;
                const float* src = table + (int64_t)id[k] * dim + d;
                if (live == 4)
                    v[k] = reinterpret_cast<const Quad*>(src)->v;
                else
                    for (int e = 0; e < live; ++e) v[k][e] = src[e];
            }
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                const int64_t i = i0 + k * stride;
                if (i >= count) break;
                const f32x4 x = (uint32_t)id[k] < (uint32_t)vocab ? v[k] * scale : v[k];
                float* dst = out + i * dim + d;
                if (live == 4)
                    reinterpret_cast<Quad*>(dst)->v = x;
                else
                    for (int e = 0; e < live; ++e) dst[e] = x[e];
            }
        }
    }
}

constexpr int kSortWaves = 16, kSortThreads = 64 * kSortWaves;
constexpr int kMaxBins = 1024;  // tokens of a sorting workgroup
constexpr int kIds = 16;        // ids a lane has in flight
constexpr int kBatch = 8;       // rows a wave has in flight
constexpr int kFew = 256;       // positions up to which one launch does it

struct BackwardArgs {
    float* dtable;
    const float* grad;
    const int32_t* ids;
    int count, vocab, dim, bins, tile, blocks;  // blocks: of 256 columns
    int groups;  // sorting workgroups; any after them clear the table
    float scale, beta;
    int32_t* sorted;  // [count] positions by token, then by position
    int32_t* start;   // [vocab + 1] where each token's begin
    float* part;      // [tiles][2][dim] sums of runs from before, and into after, a tile
    int32_t* crossing;  // [tiles][2] the run that begins in a tile and goes on past
                        // it: its token (-1: none) and its last tile
};

// Zeros over workgroup `no` of `shares`' part of the table.
__device__ __forceinline__ void clear_table(const BackwardArgs& a, int no, int shares) {
    const int64_t n = (int64_t)a.vocab * a.dim, quads = n / 4;
    Quad* const to = reinterpret_cast<Quad*>(a.dtable);
    const int64_t step = (int64_t)shares * kSortThreads;
    int64_t i = (int64_t)no * kSortThreads + threadIdx.x;
    for (; i + 3 * step < quads; i += 4 * step)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            __builtin_nontemporal_store(f32x4{0.0f, 0.0f, 0.0f, 0.0f}, &to[i + k * step].v);
    for (; i < quads; i += step) to[i].v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (no == 0 && threadIdx.x < n - 4 * quads) a.dtable[4 * quads + threadIdx.x] = 0.0f;
}

// Ids base + 64 e + lane, -1 past the end: all asked for before any is used.
__device__ __forceinline__ void load_ids(int (&id)[kIds], const int32_t* ids, int base, int end,
                                         int lane) {
    const int n = min(64 * kIds, end - base);
    const auto rs = buffer_rsrc(reinterpret_cast<const float*>(ids) + base, 4 * n);
#pragma unroll
    for (int e = 0; e < kIds; ++e)
        id[e] = __builtin_bit_cast(int, buffer_load1(rs, 4 * lane + 256 * e));
    if (n < 64 * kIds) {
#pragma unroll
        for (int e = 0; e < kIds; ++e)
            if (64 * e + lane >= n) id[e] = -1;
    }
}

__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(BackwardArgs a) {
    __shared__ int hist[kSortWaves][kMaxBins];
    __shared__ int totals[kMaxBins];
    __shared__ int below[kSortWaves];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((int)blockIdx.x >= a.groups) {
        clear_table(a, blockIdx.x - a.groups, gridDim.x - a.groups);
        return;
    }
    const int lo = blockIdx.x * a.bins, bins = min(a.bins, a.vocab - lo);
    // the wave's part of the ids
    const int per = ((a.count + kSortWaves - 1) / kSortWaves + 63) & ~63;
    const int i0 = (int)min((int64_t)a.count, (int64_t)w * per), i1 = (int)min((int64_t)a.count, (int64_t)i0 + per);
    for (int i = threadIdx.x; i < kSortWaves * a.bins; i += kSortThreads)
        hist[i / a.bins][i % a.bins] = 0;
    __syncthreads();
    int less = 0;  // this lane's ids of lower tokens
    for (int base = i0; base < i1; base += 64 * kIds) {
        int id[kIds];
        load_ids(id, a.ids, base, i1, lane);
#pragma unroll
        for (int e = 0; e < kIds; ++e) {
            less += (uint32_t)id[e] < (uint32_t)lo;
            const uint32_t bin = (uint32_t)id[e] - (uint32_t)lo;
            // (whole numbers: the order does not matter)
            if (__ballot(bin < (uint32_t)bins) != 0 && bin < (uint32_t)bins)
                atomicAdd(&hist[w][bin], 1);
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) less += __shfl_xor(less, d, 64);
    if (lane == 0) below[w] = less;
    __syncthreads();
    // a bin's total, then where each wave's places of each bin begin
    const int t = threadIdx.x;
    int total = 0;
    if (t < bins)
#pragma unroll
        for (int i = 0; i < kSortWaves; ++i) total += hist[i][t];
    int upto = total;  // inclusive over the bins of the wave
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(upto, d, 64);
        if (lane >= d) upto += v;
    }
    if (t < kMaxBins) totals[t] = total;
    __shared__ int wave_sum[kSortWaves];
    if (lane == 63) wave_sum[w] = upto;
    __syncthreads();
    int at = upto - total;
    for (int i = 0; i < kSortWaves; ++i) at += below[i] + (i < w ? wave_sum[i] : 0);
    if (t < bins) {
        a.start[lo + t] = at;
#pragma unroll
        for (int i = 0; i < kSortWaves; ++i) {
            const int n = hist[i][t];
            hist[i][t] = at;
            at += n;
        }
        if (lo + t == a.vocab - 1) a.start[a.vocab] = at;
    }
    __syncthreads();
    // the rows of absent tokens (beta 0: cleared by other workgroups)
    if (a.beta != 1.0f && a.beta != 0.0f) {
        for (int bin = w; bin < bins; bin += kSortWaves) {
            if (totals[bin] != 0) continue;
            float* const row = a.dtable + (int64_t)(lo + bin) * a.dim;
            for (int d = 4 * lane; d < a.dim; d += 256) {
                if (d + 4 <= a.dim) {
                    Quad* const to = reinterpret_cast<Quad*>(row + d);
                    to->v = a.beta * to->v;
                } else {
                    for (int e = d; e < a.dim; ++e) row[e] = a.beta * row[e];
                }
            }
        }
    }
    // place the positions: 64 ids at a time, in order. Only this wave uses its
    // row of `hist` now. Up to 64 bins stay in registers, bin b's next place in
    // lane b (a turn through LDS takes 250 cycles, and few bins mean that most
    // steps hold some of them); past that one lane writes what all read in the
    // next turn.
    volatile int* const places = hist[w];
    const bool few = bins <= 64;
    int place = lane < bins ? hist[w][lane] : 0;
    for (int base = i0; base < i1; base += 64 * kIds) {
        int id[kIds];
        load_ids(id, a.ids, base, i1, lane);
#pragma unroll
        for (int e = 0; e < kIds; ++e) {
            const uint32_t bin = (uint32_t)id[e] - (uint32_t)lo;
            uint64_t mine = __ballot(bin < (uint32_t)bins);
            while (mine) {
                const uint32_t one = __builtin_amdgcn_readlane(bin, __builtin_ctzll(mine));
                const uint64_t same = __ballot(bin == one);
                const int first = few ? __builtin_amdgcn_readlane(place, one) : places[one];
                if (bin == one)
                    a.sorted[first + __popcll(same & ((1ull << lane) - 1))] = base + 64 * e + lane;
                if (few)
                    place += lane == (int)one ? __popcll(same) : 0;
                else if (lane == 0)
                    places[one] = first + __popcll(same);
                mine &= ~same;
            }
        }
    }
}

// One wave per tile of sorted positions and 256 columns, a row's columns one
// after the other: their loads come to a page of memory together.
__global__ __launch_bounds__(64) void embedding_sum_kernel(BackwardArgs a) {
    const int lane = threadIdx.x, tile = blockIdx.x / a.blocks;
    const int d0 = (blockIdx.x - tile * a.blocks) * 256, d = d0 + 4 * lane;
    const int total = a.start[a.vocab];
    const int64_t e0 = (int64_t)tile * a.tile;
    if (e0 >= total) {
        if (d == 0) a.crossing[2 * tile] = -1;
        return;
    }
    const int e1 = (int)min((int64_t)total, e0 + a.tile);
    const bool whole = d + 4 <= a.dim;
    const int live = max(0, min(4, a.dim - d));
    f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = (int)e0; c0 < e1; c0 += 64) {
        // lane j looks up entry c0 + j: its position, its token and that one's run
        const int n = min(64, e1 - c0);
        int pos = 0, token = 0, begin = 0, end = 0;
        if (lane < n) {
            pos = a.sorted[c0 + lane];
            token = a.ids[pos];
            begin = a.start[token];
            end = a.start[token + 1];
        }
        const uint64_t ends = __ballot(lane < n && (c0 + lane + 1 == end || c0 + lane + 1 == e1));
        for (int i0 = 0; i0 < n; i0 += kBatch) {
            f32x4 rows[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                // past the row, and past the chunk, a load gives zeros
                const int64_t row = __builtin_amdgcn_readlane(pos, min(i0 + i, 63));
                rows[i] = buffer_load4(buffer_rsrc(a.grad + row * a.dim + d0,
                                                   i0 + i < n ? (int64_t)(a.dim - d0) * 4 : 0),
                                       16 * lane);
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                sum = sum + rows[i];
                if (i0 + i >= n || !((ends >> (i0 + i)) & 1)) continue;
                // the end of a run, or of the tile
                const int e = c0 + i0 + i + 1, t = __builtin_amdgcn_readlane(token, i0 + i);
                const bool head = __builtin_amdgcn_readlane(begin, i0 + i) < e0,
                           tail = __builtin_amdgcn_readlane(end, i0 + i) > e;
                const bool inside = !head && !tail;
                if (e == e1 && d == 0) {
                    a.crossing[2 * tile] = tail && !head ? t : -1;
                    a.crossing[2 * tile + 1] =
                        (__builtin_amdgcn_readlane(end, i0 + i) - 1) / a.tile;
                }
                float* dst = inside ? a.dtable + (int64_t)t * a.dim + d
                                    : a.part + ((int64_t)tile * 2 + (head ? 0 : 1)) * a.dim + d;
                f32x4 v = sum;
                sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (inside) v = v * a.scale;
                const bool add = inside && a.beta != 0.0f;
                if (whole) {
                    Quad* const to = reinterpret_cast<Quad*>(dst);
                    if (add) v = v + a.beta * to->v;
                    to->v = v;
                } else {
                    for (int k = 0; k < live; ++k) dst[k] = add ? v[k] + a.beta * dst[k] : v[k];
                }
            }
        }
    }
}

// One workgroup per tile and 256 columns: the run that begins in the tile and
// goes on past it, if there is one. Its waves add a quarter of the run's parts
// each, in order, and the quarters are added in order. Of a run of more than
// kFewParts, what each addition rounds off is added up beside it (the two-sum of
// Knuth, TAOCP vol. 2, 4.2.2): a run may have millions of parts, and equal ones
// round in one direction. 2^24 gradients of 1.1 were off by 1.7e-4 of their sum and
// are by 2.5e-6, the tiles' own error, in 20.0 ms for 19.4. (For runs of fewer, 1 us
// in 86 at 65536 positions of 259 tokens, 512 wide, for at most the error of a tile.)
constexpr int kFewParts = 1024;  // 256 additions in a wave, as in a tile

__global__ __launch_bounds__(256) void embedding_join_kernel(BackwardArgs a) {
    __shared__ f32x4 quarter[4][64];
    const int tile = blockIdx.x / a.blocks, token = a.crossing[2 * tile];
    if (token < 0) return;
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int d0 = (blockIdx.x - tile * a.blocks) * 256, d = d0 + 4 * lane, live = max(0, min(4, a.dim - d));
    // part 0 is the tile's own, part i the beginning of tile + i
    const int n = a.crossing[2 * tile + 1] - tile + 1;
    const int p0 = (int)((int64_t)n * w / 4), p1 = (int)((int64_t)n * (w + 1) / 4);
    f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f}, lost = sum;
    for (int p = p0; p < p1; p += kBatch) {
        f32x4 rows[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const float* src =
                a.part + ((int64_t)(tile + p + k) * 2 + (p + k == 0)) * a.dim + d0;
            rows[k] = buffer_load4(
                buffer_rsrc(src, p + k < p1 ? (int64_t)(a.dim - d0) * 4 : 0), 16 * lane);
        }
        if (n <= kFewParts) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) sum = sum + rows[k];
            continue;
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const f32x4 next = sum + rows[k], added = next - sum;
            lost = lost + ((sum - (next - added)) + (rows[k] - added));
            sum = next;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)  // (an infinite sum has no such rest)
        quarter[w][lane][e] = lost[e] - lost[e] == 0.0f ? sum[e] + lost[e] : sum[e];
    __syncthreads();
    if (w != 0) return;
    sum = (quarter[0][lane] + quarter[1][lane]) + (quarter[2][lane] + quarter[3][lane]);
    float* dst = a.dtable + (int64_t)token * a.dim + d;
    for (int e = 0; e < live; ++e)
        dst[e] = a.beta != 0.0f ? a.scale * sum[e] + a.beta * dst[e] : a.scale * sum[e];
}

// The gradient of few positions in one launch: a workgroup owns a range of
// tokens and 256 columns of them, finds its own among the ids (one to a thread),
// sorts them in LDS, clears its rows (beta 0) and adds. Its waves share a run, or
// take a run each where there are several short ones. The three launches for the
// same: 16 ids of 15 tokens, 704 wide, 4.3 us and 11.1; 256 of 32000, 256 wide, 9.2
// and 16.3 (half of them one token: 12.5 and 16.7). Past 256 positions, in groups
// of 1024 threads, it was 1.7 times as fast or 2 times as slow.
__global__ __launch_bounds__(kFew) void embedding_few_kernel(BackwardArgs a) {
    constexpr int WAVES = kFew / 64;
    __shared__ int token[kFew], position[kFew], runs[kFew], sums[2][WAVES];
    __shared__ f32x4 part[2][WAVES][64];
    const int t = threadIdx.x, lane = t & 63;
    const int w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int range = blockIdx.x / a.blocks, d0 = (blockIdx.x - range * a.blocks) * 256;
    const int lo = range * a.bins, bins = min(a.bins, a.vocab - lo);
    const int cols = min(256, a.dim - d0);
    const int id = t < a.count ? a.ids[t] : -1;
    const bool mine = id >= lo && id - lo < bins;
    if (a.beta == 0.0f) {
        int lanes = 1;
        while (4 * lanes < cols) lanes *= 2;
        const int c = 4 * (t & (lanes - 1));
        for (int row = t / lanes; row < bins; row += kFew / lanes) {
            float* const to = a.dtable + (int64_t)(lo + row) * a.dim + d0 + c;
            if (c + 4 <= cols)
                reinterpret_cast<Quad*>(to)->v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            else
                for (int e = 0; c + e < cols; ++e) to[e] = 0.0f;
        }
    }
    // the range's own positions, in order
    const uint64_t before = (1ull << lane) - 1;
    auto place = [&](bool one, int (&counts)[WAVES], int& n) {
        const uint64_t all = __ballot(one);
        if (lane == 0) counts[w] = __popcll(all);
        __syncthreads();
        int at = __popcll(all & before);
        n = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            at += i < w ? counts[i] : 0;
            n += counts[i];
        }
        return at;
    };
    int n, n_runs;
    const int at = place(mine, sums[0], n);
    if (n == 0) return;
    if (mine) runs[at] = id;  // (the tokens, until they are sorted)
    __syncthreads();
    if (mine) {
        int rank = at;
        if (bins > 1) {
            rank = 0;
            for (int j = 0; j < n; ++j) rank += runs[j] < id || (runs[j] == id && j < at);
        }
        token[rank] = id;
        position[rank] = t;
    }
    __syncthreads();
    const bool begins = t < n && (t == 0 || token[t] != token[t - 1]);
    const int run = place(begins, sums[1], n_runs);
    if (begins) runs[run] = t;
    __syncthreads();
    // entries p0 .. p1 - 1, in order
    auto add = [&](int p0, int p1) {
        f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int p = p0; p < p1; p += kBatch) {
            f32x4 rows[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int64_t row = __builtin_amdgcn_readfirstlane(position[min(p + k, p1 - 1)]);
                rows[k] = buffer_load4(
                    buffer_rsrc(a.grad + row * a.dim + d0, p + k < p1 ? (int64_t)cols * 4 : 0),
                    16 * lane);
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) sum = sum + rows[k];
        }
        return sum;
    };
    auto store = [&](int one, f32x4 sum) {
        float* const dst = a.dtable + (int64_t)one * a.dim + d0 + 4 * lane;
        const int live = min(4, cols - 4 * lane);
        for (int e = 0; e < live; ++e)
            dst[e] = a.beta != 0.0f ? a.scale * sum[e] + a.beta * dst[e] : a.scale * sum[e];
    };
    const bool together = n_runs < WAVES || n > 4 * n_runs;
    for (int i = together ? 0 : w; i < n_runs; i += together ? 1 : WAVES) {
        const int p0 = runs[i], p1 = i + 1 < n_runs ? runs[i + 1] : n;
        const int one = __builtin_amdgcn_readfirstlane(token[p0]);
        if (!together) {
            store(one, add(p0, p1));
            continue;
        }
        part[i & 1][w][lane] = add(p0 + (p1 - p0) * w / WAVES, p0 + (p1 - p0) * (w + 1) / WAVES);
        __syncthreads();
        if (w == 0) {
            f32x4 sum = part[i & 1][0][lane];
#pragma unroll
            for (int k = 1; k < WAVES; ++k) sum = sum + part[i & 1][k][lane];
            store(one, sum);
        }
    }
}

struct BackwardPlan {
    int bins, tile;
    int64_t groups, tiles;
    size_t sorted, start, part, crossing;  // scratch, in 4-byte words
    size_t bytes() const { return 4 * (sorted + start + part + crossing); }
};

BackwardPlan plan_backward(int64_t count, int64_t vocab, int64_t dim) {
    BackwardPlan p;
    const int64_t cus = num_cus();
    p.bins = (int)std::min<int64_t>(kMaxBins, (vocab + cus - 1) / cus);
    p.groups = (vocab + p.bins - 1) / p.bins;
    // about 16 waves to a compute unit, a column block each; tiles of at least 16
    const int64_t blocks = (dim + 255) / 256;
    const int64_t even = count * blocks / (16 * cus);
    p.tile = (int)std::max<int64_t>(16, std::min<int64_t>(256, (even + 15) / 16 * 16));
    p.tiles = (count + p.tile - 1) / p.tile;
    auto round4 = [](int64_t n) { return (size_t)((n + 3) / 4 * 4); };
    p.sorted = round4(count);
    p.start = round4(vocab + 1);
    p.part = round4(p.tiles * 2 * dim);
    p.crossing = (size_t)(2 * p.tiles);
    return p;
}

int check_shape(const char* what, int64_t count, int64_t vocab, int64_t dim) {
    NRS_ARG_CHECK(count >= 0 && count <= (1 << 30) && vocab >= 1 && vocab < INT32_MAX &&
                      dim >= 1 && dim <= (1 << 20) && count * dim <= (1ll << 39),
                  "%s: unsupported sizes (count %lld, vocab %lld, dim %lld): count is at most 2^30, "
                  "vocab below 2^31 - 1, dim at most 2^20, count * dim at most 2^39, vocab and dim "
                  "at least 1",
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
    *bytes = nrs::plan_backward(count, vocab, dim).bytes();
    return NRS_OK;
}

int nrs_embedding_backward(float* dtable, const float* grad, const int32_t* ids, int64_t count,
                           int64_t vocab, int64_t dim, float scale, float beta, void* work,
                           size_t work_bytes) {
    if (int rc = nrs::check_shape("embedding backward", count, vocab, dim)) return rc;
    NRS_ARG_CHECK(dtable && ((grad && ids) || count == 0), "embedding backward: null pointer");
    NRS_REQUIRE_INIT();
    if (int rc = nrs::check_device("embedding backward")) return rc;
    const auto plan = nrs::plan_backward(count, vocab, dim);
    const int64_t blocks = (dim + 255) / 256;
    // (a wide table, or one whose absent rows change, too, has the three launches)
    const bool few = count <= nrs::kFew && blocks <= 16 && (beta == 0.0f || beta == 1.0f);
    float* scratch = nullptr;
    if (int rc = nrs::call_scratch(&scratch, plan.bytes(), work, work_bytes, "embedding backward",
                                   !few))
        return rc;
    nrs::BackwardArgs a{};
    a.dtable = dtable;
    a.grad = grad;
    a.ids = ids;
    a.count = (int)count;
    a.vocab = (int)vocab;
    a.dim = (int)dim;
    a.bins = plan.bins;
    a.tile = plan.tile;
    a.blocks = (int)blocks;
    a.groups = (int)plan.groups;
    a.scale = scale;
    a.beta = beta;
    if (few) {
        const int64_t ranges = std::min<int64_t>(vocab, 4 * (int64_t)nrs::num_cus() / a.blocks);
        a.bins = (int)((vocab + ranges - 1) / ranges);
        const int64_t used = (vocab + a.bins - 1) / a.bins;
        hipLaunchKernelGGL(nrs::embedding_few_kernel, dim3((unsigned)(used * a.blocks)),
                           dim3(nrs::kFew), 0, nrs::stream(), a);
        NRS_LAUNCH_CHECK("embedding backward");
        return NRS_OK;
    }
    a.sorted = reinterpret_cast<int32_t*>(scratch);
    a.start = a.sorted + plan.sorted;
    a.part = scratch + plan.sorted + plan.start;
    a.crossing = reinterpret_cast<int32_t*>(a.part + plan.part);
    const int64_t clear =
        beta != 0.0f ? 0 : std::min<int64_t>((vocab * dim + 16383) / 16384, nrs::num_cus());
    hipLaunchKernelGGL(nrs::embedding_sort_kernel, dim3((unsigned)(plan.groups + clear)),
                       dim3(nrs::kSortThreads), 0, nrs::stream(), a);
    if (count > 0) {
        const dim3 grid((unsigned)(plan.tiles * a.blocks));
        hipLaunchKernelGGL(nrs::embedding_sum_kernel, grid, dim3(64), 0, nrs::stream(), a);
        hipLaunchKernelGGL(nrs::embedding_join_kernel, grid, dim3(256), 0, nrs::stream(), a);
    }
    NRS_LAUNCH_CHECK("embedding backward");
    return NRS_OK;
}

}  // extern "C"
