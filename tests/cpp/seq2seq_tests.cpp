// The operators of an encoder-decoder model through the C++ host layer, alone
// and as a run: token embedding, dropout, attention over states of another
// length. The other side is the same algebra in double on the host; the sizes
// and the absolute tolerance, 1e-3, are those of the reference's attention
// twins (tests/cuda_composite_test.rs:16-82).
//
// Usage: seq2seq_tests [name-substring]. Prints one "PASS <name>" or
// "FAIL <name>: <reason>" line per test; exit status 1 if any failed.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <random>
#include <sstream>
#include <string>
#include <vector>

#include "neuralrs.hpp"

using namespace neuralrs;
namespace gpu = neuralrs::hip::runtime;
namespace nn = neuralrs::hip::nn;
using Vec = std::vector<float>;
using Dbl = std::vector<double>;
using Ids = std::vector<int32_t>;

struct Failure : std::runtime_error {
    explicit Failure(const std::string& m) : std::runtime_error(m) {}
};

void close(const Vec& g, const Dbl& c, double tol, const std::string& what) {
    if (g.size() != c.size()) throw Failure(what + ": length mismatch");
    for (size_t i = 0; i < g.size(); ++i)
        if (!(std::fabs(g[i] - c[i]) < tol)) {
            std::ostringstream m;
            m << what << " [" << i << "]: gpu " << g[i] << " cpu " << c[i] << " (tol " << tol << ")";
            throw Failure(m.str());
        }
}

void same(const Vec& a, const Vec& b, const std::string& what) {
    if (a.size() != b.size() || std::memcmp(a.data(), b.data(), a.size() * sizeof(float)) != 0)
        throw Failure(what + ": bits differ");
}

template <class F>
void panics(F f, const std::string& part) {
    try {
        f();
    } catch (const Panic& p) {
        if (std::string(p.what()).find(part) == std::string::npos)
            throw Failure("panic says \"" + std::string(p.what()) + "\", not \"" + part + "\"");
        return;
    }
    throw Failure("no panic about \"" + part + "\"");
}

Vec values(size_t n, unsigned seed, float scale = 1.0f) {
    std::mt19937 rng(seed);
    std::uniform_real_distribution<float> u(-1.0f, 1.0f);
    Vec v(n);
    for (float& x : v) x = scale * u(rng);
    return v;
}

NodeRef resident(const Vec& d, std::vector<size_t> shape) {
    NodeRef n = Node::create(d, std::move(shape));
    gpu::to_cuda(n);
    return n;
}

Dbl wide(const Vec& v) { return Dbl(v.begin(), v.end()); }

// ------------------------------------------------------------ host algebra
// c [m,n] = op(a) . op(b)
Dbl mm(const Dbl& a, const Dbl& b, size_t m, size_t k, size_t n, bool ta = false, bool tb = false) {
    Dbl c(m * n, 0.0);
    for (size_t i = 0; i < m; ++i)
        for (size_t j = 0; j < n; ++j)
            for (size_t p = 0; p < k; ++p)
                c[i * n + j] += (ta ? a[p * m + i] : a[i * k + p]) * (tb ? b[j * k + p] : b[p * n + j]);
    return c;
}

void add_to(Dbl& a, const Dbl& b) {
    for (size_t i = 0; i < a.size(); ++i) a[i] += b[i];
}

// Philox4x32-10 (Salmon et al., SC 2011): the factor of element i of a dropout.
double kept(size_t i, float p, uint64_t seed, uint64_t call) {
    const uint64_t block = i / 4;
    uint32_t c[4] = {(uint32_t)block, (uint32_t)(block >> 32), (uint32_t)call, (uint32_t)(call >> 32)};
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
        const uint32_t n[4] = {(uint32_t)(b >> 32) ^ c[1] ^ k0, (uint32_t)b,
                               (uint32_t)(a >> 32) ^ c[3] ^ k1, (uint32_t)a};
        std::memcpy(c, n, sizeof c);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c[i % 4] >= (uint64_t)((double)p * 4294967296.0 + 0.5) ? 1.0 / (1.0 - (double)p) : 0.0;
}

Dbl drop(const Dbl& x, float p, uint64_t seed, uint64_t call) {
    Dbl y(x.size());
    for (size_t i = 0; i < x.size(); ++i) y[i] = x[i] * kept(i, p, seed, call);
    return y;
}

// Attention of [batch*sq, h*d] over [batch*sk, kv*d], and its gradients.
struct HostCross {
    Dbl out, dq, dk, dv;
    HostCross(const Dbl& q, const Dbl& k, const Dbl& v, const Ids* lens, size_t batch, size_t h,
              size_t kv, size_t sq, size_t sk, size_t d, const Dbl* g)
        : out(q.size(), 0.0), dq(q.size(), 0.0), dk(k.size(), 0.0), dv(v.size(), 0.0) {
        const double s = 1.0 / std::sqrt((double)d);
        for (size_t b = 0; b < batch; ++b)
            for (size_t hh = 0; hh < h; ++hh)
                for (size_t i = 0; i < sq; ++i) {
                    const size_t n = lens ? (size_t)(*lens)[b] : sk, kh = hh / (h / kv);
                    const size_t qa = ((b * sq + i) * h + hh) * d;
                    auto at = [&](size_t j) { return ((b * sk + j) * kv + kh) * d; };
                    Dbl p(n);
                    double top = -INFINITY, sum = 0.0;
                    for (size_t j = 0; j < n; ++j) {
                        for (size_t e = 0; e < d; ++e) p[j] += q[qa + e] * k[at(j) + e] * s;
                        top = std::max(top, p[j]);
                    }
                    for (double& x : p) sum += x = std::exp(x - top);
                    for (size_t j = 0; j < n; ++j) {
                        p[j] /= sum;
                        for (size_t e = 0; e < d; ++e) out[qa + e] += p[j] * v[at(j) + e];
                    }
                    if (!g) continue;
                    Dbl dp(n, 0.0);
                    double dot = 0.0;
                    for (size_t j = 0; j < n; ++j) {
                        for (size_t e = 0; e < d; ++e) dp[j] += (*g)[qa + e] * v[at(j) + e];
                        dot += p[j] * dp[j];
                    }
                    for (size_t j = 0; j < n; ++j) {
                        const double ds = p[j] * (dp[j] - dot) * s;
                        for (size_t e = 0; e < d; ++e) {
                            dq[qa + e] += ds * k[at(j) + e];
                            dk[at(j) + e] += ds * q[qa + e];
                            dv[at(j) + e] += p[j] * (*g)[qa + e];
                        }
                    }
                }
    }
};

// ---------------------------------------------------------------- the tests
void embedding_rows_and_gradient() {
    const size_t vocab = 11, dim = 6;
    const Ids ids = {3, 0, -1, 3, 10, 3, 7, 11};
    const Vec table = values(vocab * dim, 1), seed = values(ids.size() * dim, 2);
    nn::Embedding layer{resident(table, {vocab, dim}), 2.5f};
    NodeRef out = layer.forward(ids, {2, 4});
    if (out->shape != std::vector<size_t>{2, 4, dim}) throw Failure("shape");
    Dbl want(ids.size() * dim, 0.0), grad(vocab * dim, 0.0);
    for (size_t i = 0; i < ids.size(); ++i)
        for (size_t e = 0; e < dim; ++e)
            if (ids[i] >= 0 && ids[i] < (int)vocab) {
                want[i * dim + e] = 2.5 * table[ids[i] * dim + e];
                grad[ids[i] * dim + e] += 2.5 * seed[i * dim + e];
            }
    close(gpu::to_host(out), want, 1e-6, "rows");
    gpu::set_grad(out, seed);
    backward_graph(out);
    close(gpu::read_grad(layer.table), grad, 1e-5, "table gradient");
    // a second use of the same table adds to its gradient
    NodeRef again = layer.forward(ids, {8});
    gpu::set_grad(again, seed);
    backward_graph(again);
    for (double& x : grad) x *= 2.0;
    close(gpu::read_grad(layer.table), grad, 1e-5, "table gradient, added");
    panics([&] { layer.forward(ids, {7}); }, "shape does not match");
}

void dropout_masks() {
    const size_t n = 1003;
    const Vec x = values(n, 3), r = values(n, 4), seed = values(n, 5);
    NodeRef xn = resident(x, {n}), rn = resident(r, {n});
    NodeRef out = nn::dropout(xn, 0.3f, 77, 5, rn);
    Dbl want = drop(wide(x), 0.3f, 77, 5);
    add_to(want, wide(r));
    close(gpu::to_host(out), want, 1e-6, "with a residual");
    gpu::set_grad(out, seed);
    backward_graph(out);
    close(gpu::read_grad(xn), drop(wide(seed), 0.3f, 77, 5), 1e-6, "input gradient");
    close(gpu::read_grad(rn), wide(seed), 1e-9, "residual gradient");
    // x as its own residual: both gradients in one buffer
    gpu::zero_grad({xn});
    NodeRef twice = nn::dropout(xn, 0.3f, 77, 6, xn);
    gpu::set_grad(twice, seed);
    backward_graph(twice);
    Dbl g = drop(wide(seed), 0.3f, 77, 6);
    add_to(g, wide(seed));
    close(gpu::read_grad(xn), g, 1e-6, "gradient of both");

    nn::Dropout layer(0.3f, 77);
    const Vec a = gpu::to_host(layer.forward(xn)), b = gpu::to_host(layer.forward(xn));
    close(a, drop(wide(x), 0.3f, 77, 0), 1e-6, "call 0");
    close(b, drop(wide(x), 0.3f, 77, 1), 1e-6, "call 1");
    layer.training = false;
    if (layer.forward(xn) != xn) throw Failure("not training: the input itself");
    panics([&] { nn::dropout(xn, 0.1f, 1, 1, resident(r, {1, n})); }, "shape mismatch");
    panics([&] { nn::dropout(xn, 1.5f, 1, 1); }, "p must be in");
}

void cross_attention_nodes() {
    const size_t batch = 2, h = 4, kv = 2, sq = 5, sk = 9, d = 8;
    const Ids lens = {9, 4};
    const Vec q = values(batch * sq * h * d, 6), k = values(batch * sk * kv * d, 7),
              v = values(batch * sk * kv * d, 8), seed = values(batch * sq * h * d, 9);
    NodeRef qn = resident(q, {batch, sq, h * d}), kn = resident(k, {batch, sk, kv * d}),
            vn = resident(v, {batch, sk, kv * d});
    for (const Ids* l : {(const Ids*)nullptr, &lens}) {
        gpu::zero_grad({qn, kn, vn});
        NodeRef out = nn::cross_attention(qn, kn, vn, h, kv, l ? device_ints(*l) : nullptr);
        gpu::set_grad(out, seed);
        backward_graph(out);
        const Dbl g = wide(seed);
        const HostCross want(wide(q), wide(k), wide(v), l, batch, h, kv, sq, sk, d, &g);
        close(gpu::to_host(out), want.out, 1e-3, "out");
        close(gpu::read_grad(qn), want.dq, 1e-3, "dq");
        close(gpu::read_grad(kn), want.dk, 1e-3, "dk");
        close(gpu::read_grad(vn), want.dv, 1e-3, "dv");
    }
    // keys that are the values: both gradients in one buffer
    gpu::zero_grad({qn, kn});
    NodeRef out = nn::cross_attention(qn, kn, kn, h, kv);
    gpu::set_grad(out, seed);
    backward_graph(out);
    const Dbl g = wide(seed);
    HostCross want(wide(q), wide(k), wide(k), nullptr, batch, h, kv, sq, sk, d, &g);
    add_to(want.dk, want.dv);
    close(gpu::read_grad(kn), want.dk, 1e-3, "dk + dv");
    panics([&] { nn::cross_attention(qn, kn, vn, h, kv, device_ints({1})); }, "one length per item");
    panics([&] { nn::cross_attention(qn, kn, vn, h, 3); }, "shape mismatch");
    panics([&] { nn::cross_attention(qn, kn, vn, 5, kv); }, "width % heads");
    panics([&] { nn::cross_attention(resident(Vec(260), {1, 1, 260}), resident(Vec(260), {1, 1, 260}),
                                     resident(Vec(260), {1, 1, 260}), 1, 1); },
           "d_head must be 1 to 128");
}

// One step of a small translation model: source and target tokens through one
// embedding table, dropout on both, the target's attention to the source with a
// length per sentence, dropout and the residual, the vocabulary's logits,
// cross-entropy. Every parameter's gradient against the host's.
void a_run_of_them() {
    const size_t B = 3, Sq = 6, Sk = 10, D = 16, H = 4, V = 13;
    const Ids lens = {10, 0, 7};
    Ids src(B * Sk), tgt(B * Sq);
    std::mt19937 rng(11);
    for (size_t b = 0; b < B; ++b)
        for (size_t i = 0; i < Sk; ++i)
            src[b * Sk + i] = (int)i < lens[b] ? (int)(rng() % V) : -1;
    for (int32_t& t : tgt) t = (int)(rng() % V);
    const float scale = 2.0f, p = 0.25f;
    const Vec table = values(V * D, 12, 0.5f), wq = values(D * D, 13, 0.4f), wk = values(D * D, 14, 0.4f),
              wv = values(D * D, 15, 0.4f), wo = values(D * D, 16, 0.4f), wl = values(D * V, 17, 0.4f),
              bl = values(V, 18, 0.1f);
    Vec target(B * Sq * V, 0.0f);
    for (size_t i = 0; i < B * Sq; ++i) target[i * V + rng() % V] = 1.0f;

    NodeRef tn = resident(table, {V, D});
    nn::Embedding embed{tn, scale};
    nn::MultiHeadAttention mha(resident(wq, {D, D}), resident(wk, {D, D}), resident(wv, {D, D}),
                               resident(wo, {D, D}), D, H);
    nn::Linear head(resident(wl, {D, V}), resident(bl, {V}));
    nn::Dropout drop_src(p, 100), drop_tgt(p, 200), drop_out(p, 300);
    const std::vector<NodeRef> params = {tn, mha.w_q, mha.w_k, mha.w_v, mha.w_o, head.weights, head.bias};
    const IntsRef lengths = device_ints(lens);
    float loss = 0.0f;
    auto step = [&] {
        gpu::zero_grad(params);
        drop_src.calls = drop_tgt.calls = drop_out.calls = 0;
        NodeRef memory = drop_src.forward(embed.forward(src, {B, Sk}));
        NodeRef x = drop_tgt.forward(embed.forward(tgt, {B, Sq}));
        NodeRef z = drop_out.forward(mha.forward_cross(x, memory, lengths), x);
        NodeRef logits = head.forward(hip::graph::reshape(z, {B * Sq, D}));
        NodeRef want = resident(target, {B * Sq, V});
        loss = hip::loss::cross_entropy(logits, want);
        hip::loss::cross_entropy_backward(logits, want);
        backward_graph(logits);
        std::vector<Vec> g;
        for (const NodeRef& n : params) g.push_back(gpu::read_grad(n));
        return g;
    };
    const std::vector<Vec> got = step();

    // the host's side
    auto rows = [&](const Ids& ids) {
        Dbl r(ids.size() * D, 0.0);
        for (size_t i = 0; i < ids.size(); ++i)
            for (size_t e = 0; e < D; ++e)
                if (ids[i] >= 0) r[i * D + e] = (double)scale * table[ids[i] * D + e];
        return r;
    };
    const size_t N = B * Sq, M = B * Sk;
    const Dbl mem = drop(rows(src), p, 100, 0), x = drop(rows(tgt), p, 200, 0);
    const Dbl q = mm(x, wide(wq), N, D, D), k = mm(mem, wide(wk), M, D, D), v = mm(mem, wide(wv), M, D, D);
    const HostCross att(q, k, v, &lens, B, H, H, Sq, Sk, D / H, nullptr);
    Dbl z = drop(mm(att.out, wide(wo), N, D, D), p, 300, 0);
    add_to(z, x);
    Dbl logits = mm(z, wide(wl), N, D, V), gl(N * V);
    double host_loss = 0.0;
    for (size_t i = 0; i < N; ++i) {
        double top = -INFINITY, sum = 0.0;
        for (size_t c = 0; c < V; ++c) top = std::max(top, logits[i * V + c] += bl[c]);
        for (size_t c = 0; c < V; ++c) sum += std::exp(logits[i * V + c] - top);
        for (size_t c = 0; c < V; ++c) {
            gl[i * V + c] = (std::exp(logits[i * V + c] - top) / sum - target[i * V + c]) / N;
            if (target[i * V + c] > 0) host_loss -= (logits[i * V + c] - top - std::log(sum)) / N;
        }
    }
    if (!(std::fabs(loss - host_loss) < 1e-3)) throw Failure("loss");
    Dbl gb(V, 0.0);
    for (size_t i = 0; i < N * V; ++i) gb[i % V] += gl[i];
    const Dbl gwl = mm(z, gl, D, N, V, true), gz = mm(gl, wide(wl), N, V, D, false, true);
    const Dbl gy = drop(gz, p, 300, 0), gwo = mm(att.out, gy, D, N, D, true),
              go = mm(gy, wide(wo), N, D, D, false, true);
    const HostCross back(q, k, v, &lens, B, H, H, Sq, Sk, D / H, &go);
    Dbl gx = mm(back.dq, wide(wq), N, D, D, false, true);
    add_to(gx, gz);
    Dbl gm = mm(back.dk, wide(wk), M, D, D, false, true);
    add_to(gm, mm(back.dv, wide(wv), M, D, D, false, true));
    Dbl gt(V * D, 0.0);
    auto scatter = [&](const Ids& ids, const Dbl& g) {
        for (size_t i = 0; i < ids.size(); ++i)
            for (size_t e = 0; e < D; ++e)
                if (ids[i] >= 0) gt[ids[i] * D + e] += scale * g[i * D + e];
    };
    scatter(src, drop(gm, p, 100, 0));
    scatter(tgt, drop(gx, p, 200, 0));
    close(got[0], gt, 1e-3, "table");
    close(got[1], mm(x, back.dq, D, N, D, true), 1e-3, "w_q");
    close(got[2], mm(mem, back.dk, D, M, D, true), 1e-3, "w_k");
    close(got[3], mm(mem, back.dv, D, M, D, true), 1e-3, "w_v");
    close(got[4], gwo, 1e-3, "w_o");
    close(got[5], gwl, 1e-3, "logit weights");
    close(got[6], gb, 1e-3, "logit bias");
    // the same step again: the same bits
    const std::vector<Vec> again = step();
    for (size_t i = 0; i < got.size(); ++i) same(again[i], got[i], "second step");
}

struct Case {
    const char* name;
    void (*fn)();
};

const Case kCases[] = {
    {"embedding_rows_and_gradient", embedding_rows_and_gradient},
    {"dropout_masks", dropout_masks},
    {"cross_attention_nodes", cross_attention_nodes},
    {"a_run_of_them", a_run_of_them},
};

int main(int argc, char** argv) {
    const char* filter = argc > 1 ? argv[1] : "";
    int failed = 0;
    for (const Case& c : kCases) {
        if (!std::strstr(c.name, filter)) continue;
        std::printf("RUN  %s\n", c.name);
        std::fflush(stdout);
        try {
            c.fn();
            gpu::synchronize();
            std::printf("PASS %s\n", c.name);
        } catch (const std::exception& e) {
            ++failed;
            std::printf("FAIL %s: %s\n", c.name, e.what());
        }
        std::fflush(stdout);
    }
    return failed ? 1 : 0;
}
