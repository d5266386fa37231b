// test_student_amd.cpp — the operators of a language-model student through the C++ host layer: embedding, the gated pair of
// Linear layers, the distillation loss, checked against plain host loops in double precision.
#include "mini_test.h"

#include <cmath>

using namespace tt_amd;

namespace {
template <typename T>
std::vector<T> wave(int n, double step, double scale) {
    std::vector<T> v;
    for (int i = 0; i < n; ++i) v.push_back(static_cast<T>(scale * std::sin(step * i + 0.3)));
    return v;
}
// within `steps` rounding steps of the type, relative to `size`
template <typename T>
bool near(T got, double want, double size, double steps) {
    return std::abs(static_cast<double>(got) - want) <= steps * std::numeric_limits<T>::epsilon() * size + 1e-300;
}
}  // namespace

TEST_CASE("Embedding and its gradient") {
    auto test = []<typename T>(Device device) {
        const int V = 23, D = 13, N = 300;
        const auto table = wave<T>(V * D, 0.7, 2.0), dy = wave<T>(N * D, 0.31, 1.0);
        std::vector<int32_t> ids;
        for (int i = 0; i < N; ++i) ids.push_back(i % 11 == 0 ? -1 : (i * i) % V);
        const Tensor t(table, {V, D}, device), idx(ids, {N}, device), g(dy, {N, D}, device);
        const auto out = nn::embedding(idx, t, 2.0).template to_vec<T>();
        std::vector<double> want(static_cast<std::size_t>(V * D), 0.0), mag = want;
        bool same = true;
        for (int i = 0; i < N; ++i)
            for (int d = 0; d < D; ++d) {
                const int v = ids[static_cast<std::size_t>(i)];
                same = same && out[static_cast<std::size_t>(i * D + d)] == (v < 0 ? T(0) : static_cast<T>(table[static_cast<std::size_t>(v * D + d)] * T(2)));
                if (v >= 0) {
                    want[static_cast<std::size_t>(v * D + d)] += 2.0 * dy[static_cast<std::size_t>(i * D + d)];
                    mag[static_cast<std::size_t>(v * D + d)] += 2.0 * std::abs(dy[static_cast<std::size_t>(i * D + d)]);
                }
            }
        CHECK(same);
        const Tensor grad = nn::embedding_backward(g, idx, V, 2.0);
        const auto got = grad.template to_vec<T>();
        (void)nn::embedding_backward(g, idx, V, 2.0, &grad);  // once more on top
        const auto twice = grad.template to_vec<T>();
        bool close = true;
        for (std::size_t i = 0; i < want.size(); ++i)
            close = close && near(got[i], want[i], mag[i], 64) && near(twice[i], 2 * want[i], 2 * mag[i], 64);
        CHECK(close);
        // a transposed view as the table, read in place
        const auto turned = nn::embedding(Tensor(std::vector<int32_t>{3, 0}, {2}, device), t.permute({1, 0})).template to_vec<T>();
        bool right = true;
        for (int v = 0; v < V; ++v)
            right = right && turned[static_cast<std::size_t>(v)] == table[static_cast<std::size_t>(v * D + 3)] && turned[static_cast<std::size_t>(V + v)] == table[static_cast<std::size_t>(v * D)];
        CHECK(right);
    };
    test.operator()<float>(kAMD);
    test.operator()<double>(kAMD);
}

TEST_CASE("Gated linear layers forward and backward") {
    auto test = []<typename T>(Device device) {
        for (const int R : {1, 5, 70}) {
            const int I = 18, H = 21;
            const auto x = wave<T>(R * I, 0.9, 1.0), wg = wave<T>(I * H, 0.37, 0.5), wu = wave<T>(I * H, 0.53, 0.5), bg = wave<T>(H, 0.2, 0.1), dh = wave<T>(R * H, 0.77, 1.0);
            const Tensor tx(x, {R, I}, device), tg(wg, {I, H}, device), tu(wu, {I, H}, device), tb(bg, {H}, device), td(dh, {R, H}, device);
            const nn::GatedResult f = nn::gated_linear(tx, tg, tu, &tb, nullptr, "silu", true);
            const nn::GatedGrads b = nn::gated_linear_backward(td, tx, tg, tu, *f.gate, *f.up, "silu", true);
            const auto h = f.output.template to_vec<T>();
            std::vector<double> dx(static_cast<std::size_t>(R * I)), dwg(static_cast<std::size_t>(I * H)), dwu = dwg, dbg(static_cast<std::size_t>(H)), dbu = dbg;
            bool close = true;
            for (int r = 0; r < R; ++r)
                for (int c = 0; c < H; ++c) {
                    double g = bg[static_cast<std::size_t>(c)], u = 0;
                    for (int k = 0; k < I; ++k) {
                        g += static_cast<double>(x[static_cast<std::size_t>(r * I + k)]) * wg[static_cast<std::size_t>(k * H + c)];
                        u += static_cast<double>(x[static_cast<std::size_t>(r * I + k)]) * wu[static_cast<std::size_t>(k * H + c)];
                    }
                    const double s = 1 / (1 + std::exp(-g)), d = dh[static_cast<std::size_t>(r * H + c)];
                    const double pg = d * u * s * (1 + g * (1 - s)), pu = d * g * s;
                    close = close && near(h[static_cast<std::size_t>(r * H + c)], g * s * u, 20.0, 40);
                    dbg[static_cast<std::size_t>(c)] += pg;
                    dbu[static_cast<std::size_t>(c)] += pu;
                    for (int k = 0; k < I; ++k) {
                        dx[static_cast<std::size_t>(r * I + k)] += pg * wg[static_cast<std::size_t>(k * H + c)] + pu * wu[static_cast<std::size_t>(k * H + c)];
                        dwg[static_cast<std::size_t>(k * H + c)] += pg * x[static_cast<std::size_t>(r * I + k)];
                        dwu[static_cast<std::size_t>(k * H + c)] += pu * x[static_cast<std::size_t>(r * I + k)];
                    }
                }
            const auto all = [&](const Tensor &got, const std::vector<double> &want) {
                const auto v = got.template to_vec<T>();
                bool ok = v.size() == want.size();
                for (std::size_t i = 0; ok && i < v.size(); ++i) ok = near(v[i], want[i], 20.0 * (R + H), 40);  // (terms of at most 20)
                return ok;
            };
            CHECK(close);
            CHECK(all(b.dx, dx));
            CHECK(all(b.dw_gate, dwg));
            CHECK(all(b.dw_up, dwu));
            CHECK(all(*b.db_gate, dbg));
            CHECK(all(*b.db_up, dbu));
            CHECK(nn::gated_linear(tx, tg, tu, &tb).output.template to_vec<T>() == h);
        }
        CHECK_THROWS_AS(nn::gated_linear(Tensor(std::vector<T>(6), {2, 3}, device), Tensor(std::vector<T>(8), {4, 2}, device), Tensor(std::vector<T>(8), {4, 2}, device)), TTException);
        CHECK_THROWS_AS(nn::gated_linear(Tensor(std::vector<T>(8), {2, 4}, device), Tensor(std::vector<T>(8), {4, 2}, device), Tensor(std::vector<T>(8), {4, 2}, device), nullptr, nullptr, "tanh"), TTException);
    };
    test.operator()<float>(kAMD);
    test.operator()<double>(kAMD);
}

TEST_CASE("Distillation loss and its gradient") {
    auto test = []<typename T>(Device device) {
        for (const int C : {10, 700, 5000, 20001}) {
            const int R = 4, K = 3;
            const double temp = 2.0;
            const auto z = wave<T>(R * C, 0.61, 3.0), t = wave<T>(R * K, 1.1, 2.0), w = std::vector<T>{T(0.5), T(0), T(1), T(0.25)};
            const std::vector<int64_t> ids = {1, 7, 3, 0, 1, 2, 9, 9, 4, 5, -1, 8};
            const nn::DistillLoss r = nn::distill_loss(Tensor(z, {R, C}, device), Tensor(ids, {R, K}, device), Tensor(t, {R, K}, device), temp, nullptr);
            const Tensor tw(w, {R}, device);
            const nn::DistillLoss rw = nn::distill_loss(Tensor(z, {R, C}, device), Tensor(ids, {R, K}, device), Tensor(t, {R, K}, device), temp, &tw);
            for (const bool weighted : {false, true}) {
                const auto grad = (weighted ? rw : r).grad_input.template to_vec<T>();
                const auto loss = (weighted ? rw : r).loss.template to_vec<T>()[0];
                double want = 0;
                bool close = true;
                for (int i = 0; i < R; ++i) {
                    const double wt = weighted ? static_cast<double>(w[static_cast<std::size_t>(i)]) : 1.0 / R;
                    double zs = 0, ts = 0;
                    for (int c = 0; c < C; ++c) zs += std::exp(z[static_cast<std::size_t>(i * C + c)] / temp);
                    for (int k = 0; k < K; ++k)
                        if (ids[static_cast<std::size_t>(i * K + k)] >= 0) ts += std::exp(t[static_cast<std::size_t>(i * K + k)] / temp);
                    std::vector<double> g(static_cast<std::size_t>(C));
                    for (int c = 0; c < C; ++c) g[static_cast<std::size_t>(c)] = wt * temp * std::exp(z[static_cast<std::size_t>(i * C + c)] / temp) / zs;
                    for (int k = 0; k < K; ++k) {
                        const auto id = ids[static_cast<std::size_t>(i * K + k)];
                        if (id < 0) continue;
                        const double p = std::exp(t[static_cast<std::size_t>(i * K + k)] / temp) / ts;
                        want += wt * temp * temp * p * (std::log(p) - (z[static_cast<std::size_t>(i * C + id)] / temp - std::log(zs)));
                        g[static_cast<std::size_t>(id)] -= wt * temp * p;
                    }
                    for (int c = 0; c < C; ++c) close = close && near(grad[static_cast<std::size_t>(i * C + c)], g[static_cast<std::size_t>(c)], wt * temp, 60);
                }
                CHECK(close);
                CHECK(near(loss, want, 50.0, 60));
            }
        }
    };
    test.operator()<float>(kAMD);
    test.operator()<double>(kAMD);
}

int main(int argc, char **argv) { return mini::run_all(argc, argv); }
