// The operators of a decoder through the C++ host layer, alone and as a run: masked
// self-attention, rotary positions, distillation from a teacher's top logits. The other
// side is the same algebra in double on the host; its gradients are central differences
// of the host's loss, whose step of 1e-5 leaves some 1e-9 of the values involved. The
// tolerance, 1e-3, is that of the reference's attention twins
// (tests/cuda_composite_test.rs:16-82).
//
// Usage: decoder_tests [name-substring]. Prints one "PASS <name>" or
// "FAIL <name>: <reason>" line per test; exit status 1 if any failed.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>
#include <random>
#include <sstream>
#include <string>
#include <vector>

#include "neuralrs.hpp"

using namespace neuralrs;
namespace gpu = neuralrs::hip::runtime;
namespace nn = neuralrs::hip::nn;
namespace loss = neuralrs::hip::loss;
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
// c [m,n] = a . b
Dbl mm(const Dbl& a, const Dbl& b, size_t m, size_t k, size_t n) {
    Dbl c(m * n, 0.0);
    for (size_t i = 0; i < m; ++i)
        for (size_t j = 0; j < n; ++j)
            for (size_t p = 0; p < k; ++p) c[i * n + j] += a[i * k + p] * b[p * n + j];
    return c;
}

// The mask of a test, on the host.
struct HostMask {
    bool causal = true;
    Ids q_start, key_len, prefix_len, key_begin, key_end;  // empty: not given
    Vec slopes;
    double cap = 0.0;

    bool sees(size_t b, size_t i, size_t t, size_t sq, size_t sk) const {
        const long at = place(b, i, sq, sk);
        if (!key_len.empty() && (long)t >= key_len[b]) return false;
        if (causal && (long)t > at && (prefix_len.empty() || (long)t >= prefix_len[b])) return false;
        if (!key_begin.empty() && (long)t < key_begin[b * sq + i]) return false;
        return key_end.empty() || (long)t < key_end[b * sq + i];
    }
    long place(size_t b, size_t i, size_t sq, size_t sk) const {
        return (q_start.empty() ? (long)sk - (long)sq : (long)q_start[b]) + (long)i;
    }
    nn::AttentionMask device() const {
        auto ints = [](const Ids& x) { return x.empty() ? nullptr : device_ints(x); };
        nn::AttentionMask m;
        m.causal = causal;
        m.q_start = ints(q_start);
        m.key_len = ints(key_len);
        m.prefix_len = ints(prefix_len);
        m.key_begin = ints(key_begin);
        m.key_end = ints(key_end);
        if (!slopes.empty()) m.slopes = resident(slopes, {slopes.size()});
        m.cap = (float)cap;
        return m;
    }
};

// Attention of [batch*sq, h*d] over [batch*sk, kv*d].
Dbl attend(const Dbl& q, const Dbl& k, const Dbl& v, const HostMask& m, size_t batch, size_t h,
           size_t kv, size_t sq, size_t sk, size_t d) {
    Dbl out(q.size(), 0.0);
    const double s = 1.0 / std::sqrt((double)d);
    for (size_t b = 0; b < batch; ++b)
        for (size_t hh = 0; hh < h; ++hh)
            for (size_t i = 0; i < sq; ++i) {
                const size_t qa = ((b * sq + i) * h + hh) * d;
                auto at = [&](size_t t) { return ((b * sk + t) * kv + hh / (h / kv)) * d; };
                Dbl u(sk, -INFINITY);
                double top = -INFINITY, sum = 0.0;
                for (size_t t = 0; t < sk; ++t) {
                    if (!m.sees(b, i, t, sq, sk)) continue;
                    double x = 0.0;
                    for (size_t e = 0; e < d; ++e) x += q[qa + e] * k[at(t) + e] * s;
                    if (m.cap > 0.0) x = m.cap * std::tanh(x / m.cap);
                    if (!m.slopes.empty())
                        x -= m.slopes[hh] * std::fabs((double)(m.place(b, i, sq, sk) - (long)t));
                    u[t] = x;
                    top = std::max(top, x);
                }
                if (top == -INFINITY) continue;
                for (double& x : u) sum += x = std::exp(x - top);
                for (size_t t = 0; t < sk; ++t)
                    if (u[t] > 0.0)
                        for (size_t e = 0; e < d; ++e) out[qa + e] += u[t] / sum * v[at(t) + e];
            }
    return out;
}

// Each row's heads with their pairs turned.
Dbl turned(const Dbl& x, size_t rows, size_t heads, size_t d, const Ids& positions, const Vec& freq,
           const Ids& axis, bool interleaved) {
    Dbl y = x;
    const size_t pairs = freq.size();
    for (size_t r = 0; r < rows; ++r)
        for (size_t h = 0; h < heads; ++h)
            for (size_t j = 0; j < pairs; ++j) {
                const size_t a = axis.empty() ? 0 : axis[j];
                const double angle = (double)positions[a * rows + r] * (double)freq[j];
                const size_t at = (r * heads + h) * d;
                const size_t c0 = at + (interleaved ? 2 * j : j), c1 = at + (interleaved ? 2 * j + 1 : pairs + j);
                y[c0] = x[c0] * std::cos(angle) - x[c1] * std::sin(angle);
                y[c1] = x[c1] * std::cos(angle) + x[c0] * std::sin(angle);
            }
    return y;
}

double distilled(const Dbl& z, size_t rows, size_t vocab, size_t k, const Vec& top, const Ids& ids,
                 const Ids& labels, double temp, double hard) {
    double total = 0.0;
    for (size_t r = 0; r < rows; ++r) {
        auto log_sum = [&](double by) {
            double m = -INFINITY, s = 0.0;
            for (size_t c = 0; c < vocab; ++c) m = std::max(m, z[r * vocab + c] / by);
            for (size_t c = 0; c < vocab; ++c) s += std::exp(z[r * vocab + c] / by - m);
            return m + std::log(s);
        };
        double m = -INFINITY, s = 0.0;
        auto live = [&](size_t j) { return ids[r * k + j] >= 0 && ids[r * k + j] < (int)vocab; };
        for (size_t j = 0; j < k; ++j)
            if (live(j)) m = std::max(m, top[r * k + j] / temp);
        for (size_t j = 0; j < k; ++j)
            if (live(j)) s += std::exp(top[r * k + j] / temp - m);
        const double ls = log_sum(temp);
        for (size_t j = 0; j < k; ++j) {
            if (!live(j)) continue;
            const double lp = top[r * k + j] / temp - m - std::log(s);
            const double lq = z[r * vocab + ids[r * k + j]] / temp - ls;
            total += (1.0 - hard) * temp * temp * std::exp(lp) * (lp - lq);
        }
        if (hard > 0.0 && labels[r] >= 0 && labels[r] < (int)vocab)
            total -= hard * (z[r * vocab + labels[r]] - log_sum(1.0));
    }
    return total / rows;
}

// d f / d x by central differences.
Dbl differences(Dbl& x, const std::function<double()>& f) {
    const double h = 1e-5;
    Dbl g(x.size());
    for (size_t i = 0; i < x.size(); ++i) {
        const double was = x[i];
        x[i] = was + h;
        const double up = f();
        x[i] = was - h;
        g[i] = (up - f()) / (2 * h);
        x[i] = was;
    }
    return g;
}

double dot(const Dbl& a, const Vec& b) {
    double s = 0.0;
    for (size_t i = 0; i < a.size(); ++i) s += a[i] * b[i];
    return s;
}

// ---------------------------------------------------------------- the tests
void masked_attention_nodes() {
    const size_t batch = 2, h = 4, kv = 2, sq = 5, sk = 7, d = 8;
    Dbl q = wide(values(batch * sq * h * d, 6)), k = wide(values(batch * sk * kv * d, 7)),
        v = wide(values(batch * sk * kv * d, 8));
    const Vec seed = values(batch * sq * h * d, 9);
    auto f32 = [](const Dbl& x) { return Vec(x.begin(), x.end()); };
    NodeRef qn = resident(f32(q), {batch, sq, h * d}), kn = resident(f32(k), {batch, sk, kv * d}),
            vn = resident(f32(v), {batch, sk, kv * d});
    std::vector<HostMask> masks(6);
    masks[1].key_len = {6, 3};
    masks[1].cap = 0.5;
    masks[2].prefix_len = {6, 0};
    masks[2].slopes = {0.5f, 0.25f, 0.125f, 0.0f};
    masks[3].key_begin = {0, 1, 1, 5, 5, 2, 2, 2, 7, 6};
    masks[3].q_start = {2, 1};
    masks[4].causal = false;
    masks[4].key_begin = {0, 3, 0, 6, 7, 1, 1, 1, 1, 1};
    masks[4].key_end = {2, 5, 0, 7, 9, 2, 3, 4, 5, 6};
    masks[4].slopes = {1.0f, 0.5f, 0.25f, 0.125f};
    masks[4].cap = 1.0;
    masks[5].causal = false;
    for (const HostMask& m : masks) {
        gpu::zero_grad({qn, kn, vn});
        NodeRef out = nn::masked_attention(qn, kn, vn, h, kv, m.device());
        gpu::set_grad(out, seed);
        backward_graph(out);
        auto run = [&] { return attend(q, k, v, m, batch, h, kv, sq, sk, d); };
        close(gpu::to_host(out), run(), 1e-3, "out");
        auto f = [&] { return dot(run(), seed); };
        close(gpu::read_grad(qn), differences(q, f), 1e-3, "dq");
        close(gpu::read_grad(kn), differences(k, f), 1e-3, "dk");
        close(gpu::read_grad(vn), differences(v, f), 1e-3, "dv");
    }
    // keys that are the values: both gradients in one buffer
    gpu::zero_grad({qn, kn});
    NodeRef out = nn::masked_attention(qn, kn, kn, h, kv, masks[0].device());
    gpu::set_grad(out, seed);
    backward_graph(out);
    close(gpu::read_grad(kn),
          differences(k, [&] { return dot(attend(q, k, k, masks[0], batch, h, kv, sq, sk, d), seed); }),
          1e-3, "dk + dv");
    auto with = [&](const std::function<void(nn::AttentionMask&)>& change) {
        nn::AttentionMask m;
        change(m);
        return [=] { nn::masked_attention(qn, kn, vn, h, kv, m); };
    };
    panics(with([](auto& m) { m.key_len = device_ints({1}); }), "one number per item");
    panics(with([](auto& m) { m.key_begin = device_ints({1, 2}); }), "one number per query");
    panics(with([](auto& m) { m.slopes = resident({1.0f}, {1}); }), "one slope per head");
    panics(with([](auto& m) { m.cap = -1.0f; }), "cap must be");
    panics(with([](auto& m) {
               m.causal = false;
               m.prefix_len = device_ints({1, 2});
           }),
           "prefix");
    panics([&] { nn::masked_attention(qn, kn, vn, h, 3, {}); }, "shape mismatch");
    panics([&] { nn::masked_attention(qn, kn, vn, 5, kv, {}); }, "width % heads");
}

void rotary_nodes() {
    const size_t batch = 2, seq = 3, rows = batch * seq, heads = 3, d = 10, pairs = 4;
    const Vec x = values(rows * heads * d, 20), seed = values(rows * heads * d, 21);
    const Ids positions = {0, 1, 2, 100, -7, 5000, 9, 8, 7, 6, 5, 4}, axis = {0, 1, 1, 0};
    const Vec freq = {1.0f, 0.3f, 0.1f, 0.01f};
    for (bool interleaved : {false, true}) {
        NodeRef xn = resident(x, {batch, seq, heads * d});
        nn::Rotary turn{device_ints(positions), resident(freq, {pairs}), device_ints(axis), interleaved};
        NodeRef out = nn::rotary(xn, heads, turn);
        Dbl xd = wide(x);
        auto run = [&] { return turned(xd, rows, heads, d, positions, freq, axis, interleaved); };
        close(gpu::to_host(out), run(), 1e-5, "out");
        gpu::set_grad(out, seed);
        backward_graph(out);
        Dbl want = differences(xd, [&] { return dot(run(), seed); });
        close(gpu::read_grad(xn), want, 1e-5, "gradient");
        // a second use adds to the gradient
        NodeRef again = nn::rotary(xn, heads, turn);
        gpu::set_grad(again, seed);
        backward_graph(again);
        for (double& g : want) g *= 2.0;
        close(gpu::read_grad(xn), want, 1e-5, "gradient, added");
        panics([&] { nn::rotary(xn, 7, turn); }, "width % heads");
        panics([&] { nn::rotary(xn, heads, {device_ints({1, 2}), turn.freq, nullptr, false}); },
               "one position per row");
        panics([&] { nn::rotary(xn, heads, {turn.positions, turn.freq, device_ints({0}), false}); },
               "one axis per pair");
        panics([&] { nn::rotary(xn, 15, turn); }, "more pairs than half");
    }
}

void distillation_loss() {
    const size_t rows = 5, vocab = 19, k = 4;
    const Vec z = values(rows * vocab, 30, 3.0f), top = values(rows * k, 31, 3.0f);
    const Ids ids = {1, 4, 18, -1, 0, 0, 7, 3, -1, -1, -1, -1, 5, 6, 19, 8, 2, 17, 9, 11},
              labels = {4, -1, 6, 18, 0};
    for (float hard : {0.0f, 0.3f, 1.0f})
        for (float temp : {1.0f, 2.0f}) {
            NodeRef zn = resident(z, {rows, vocab});
            const loss::Teacher teacher{resident(top, {rows, k}), device_ints(ids), device_ints(labels),
                                        temp, hard};
            Dbl zd = wide(z);
            auto f = [&] { return distilled(zd, rows, vocab, k, top, ids, labels, temp, hard); };
            const float forward = loss::distillation(zn, teacher);
            if (!(std::fabs(forward - f()) < 1e-5)) throw Failure("loss");
            if (loss::distillation_backward(zn, teacher) != forward) throw Failure("the backward's loss");
            close(gpu::read_grad(zn), differences(zd, f), 1e-6, "gradient");
        }
    NodeRef zn = resident(z, {rows, vocab}), tn = resident(top, {rows, k});
    panics([&] { loss::distillation(zn, {tn, device_ints({1}), nullptr}); }, "[rows, k]");
    panics([&] { loss::distillation(zn, {tn, device_ints(ids), device_ints({1}), 1.0f, 0.5f}); },
           "one label per row");
    panics([&] { loss::distillation(zn, {tn, device_ints(ids), nullptr, 1.0f, 0.5f}); }, "no labels");
    panics([&] { loss::distillation(zn, {tn, device_ints(ids), nullptr, 0.0f}); }, "temperature");
}

// One training step of a small decoder: tokens of packed documents through the
// embedding, self-attention that sees its own document up to itself, with rotary
// positions that begin anew in each document, capped scores and a bias by distance, the
// residual, the vocabulary's logits, and the loss against a teacher. Every parameter's
// gradient against the host's differences.
void a_run_of_them() {
    const size_t B = 2, S = 6, D = 8, H = 2, V = 9, K = 3, N = B * S, d = D / H;
    const Ids tokens = {1, 5, 8, 0, 2, 2, 3, 4, 4, 7, 6, -1};
    const Ids begin = {0, 0, 0, 3, 3, 3, 0, 0, 2, 2, 2, 2}, positions = {0, 1, 2, 0, 1, 2, 0, 1, 0, 1, 2, 3};
    const Vec freq = {1.0f, 0.1f};
    HostMask mask;
    mask.key_begin = begin;
    mask.slopes = {0.5f, 0.0625f};
    mask.cap = 2.0;
    const Vec top = values(N * K, 40, 2.0f);
    Ids ids(N * K), labels(N);
    std::mt19937 rng(41);
    for (size_t i = 0; i < N; ++i) {
        labels[i] = (int)(rng() % V);
        for (size_t j = 0; j < K; ++j) ids[i * K + j] = (int)((i + 3 * j) % V);
    }
    const float temp = 2.0f, hard = 0.25f;
    Dbl table = wide(values(V * D, 42, 0.5f)), wq = wide(values(D * D, 43, 0.4f)),
        wk = wide(values(D * D, 44, 0.4f)), wv = wide(values(D * D, 45, 0.4f)),
        wo = wide(values(D * D, 46, 0.4f)), wl = wide(values(D * V, 47, 0.4f)), bl = wide(values(V, 48, 0.1f));
    auto f32 = [](const Dbl& x) { return Vec(x.begin(), x.end()); };

    NodeRef tn = resident(f32(table), {V, D});
    nn::Embedding embed{tn, 1.5f};
    nn::MultiHeadAttention mha(resident(f32(wq), {D, D}), resident(f32(wk), {D, D}),
                               resident(f32(wv), {D, D}), resident(f32(wo), {D, D}), D, H);
    nn::Linear head(resident(f32(wl), {D, V}), resident(f32(bl), {V}));
    const nn::Rotary turn{device_ints(positions), resident(freq, {2}), nullptr, false};
    const nn::AttentionMask device_mask = mask.device();
    const loss::Teacher teacher{resident(top, {N, K}), device_ints(ids), device_ints(labels), temp, hard};
    const std::vector<NodeRef> params = {tn, mha.w_q, mha.w_k, mha.w_v, mha.w_o, head.weights, head.bias};
    float got_loss = 0.0f;
    auto step = [&] {
        gpu::zero_grad(params);
        NodeRef x = embed.forward(tokens, {B, S});
        NodeRef z = hip::graph::add(mha.forward_masked(x, device_mask, &turn), x);
        NodeRef logits = head.forward(hip::graph::reshape(z, {N, D}));
        got_loss = loss::distillation_backward(logits, teacher);
        backward_graph(logits);
        std::vector<Vec> g;
        for (const NodeRef& n : params) g.push_back(gpu::read_grad(n));
        return g;
    };
    const std::vector<Vec> got = step();

    auto host = [&] {
        Dbl x(N * D, 0.0);
        for (size_t i = 0; i < N; ++i)
            for (size_t e = 0; e < D; ++e)
                if (tokens[i] >= 0) x[i * D + e] = 1.5 * table[tokens[i] * D + e];
        const Dbl q = turned(mm(x, wq, N, D, D), N, H, d, positions, freq, {}, false),
                  k = turned(mm(x, wk, N, D, D), N, H, d, positions, freq, {}, false);
        Dbl z = mm(attend(q, k, mm(x, wv, N, D, D), mask, B, H, H, S, S, d), wo, N, D, D);
        for (size_t i = 0; i < z.size(); ++i) z[i] += x[i];
        Dbl logits = mm(z, wl, N, D, V);
        for (size_t i = 0; i < logits.size(); ++i) logits[i] += bl[i % V];
        return distilled(logits, N, V, K, top, ids, labels, temp, hard);
    };
    if (!(std::fabs(got_loss - host()) < 1e-4)) throw Failure("loss");
    const char* names[] = {"table", "w_q", "w_k", "w_v", "w_o", "logit weights", "logit bias"};
    Dbl* host_params[] = {&table, &wq, &wk, &wv, &wo, &wl, &bl};
    for (size_t i = 0; i < params.size(); ++i)
        close(got[i], differences(*host_params[i], host), 1e-5, names[i]);
    // the same step again: the same bits
    const std::vector<Vec> again = step();
    for (size_t i = 0; i < got.size(); ++i)
        if (std::memcmp(again[i].data(), got[i].data(), got[i].size() * sizeof(float)) != 0)
            throw Failure(std::string(names[i]) + ": second step's bits differ");
    panics([&] { mha.forward_masked(tn, device_mask); }, "[batch, seq, d_model]");
}

struct Case {
    const char* name;
    void (*fn)();
};

const Case kCases[] = {
    {"masked_attention_nodes", masked_attention_nodes},
    {"rotary_nodes", rotary_nodes},
    {"distillation_loss", distillation_loss},
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
