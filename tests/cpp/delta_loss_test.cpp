// C++ test of DeviceDeltaRule and DeviceCrossEntropy: refusals (made-up addresses, no GPU needed) with the argument
// "refusals"; without one, both operators against plain loops in double.  Exit code 0 = all checks passed.
#include <lcpp/parallel_primitive.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

using namespace luisa;
using namespace luisa::compute;
using namespace luisa::parallel_primitive;

static int g_failures = 0;
static void near(const char* what, double got, double want, double tol) {
    if (!(std::abs(got - want) <= tol)) {
        if (++g_failures < 10) std::printf("FAIL %s: got %.9g want %.9g\n", what, got, want);
    }
}
template <typename T>
static BufferView<T> made_up(size_t i, size_t n) { return {reinterpret_cast<T*>(i << 40), n}; }
static void refused(const char* what, CommandList& cmdlist) {
    CommitCommand c = cmdlist.commit();
    for (auto& cmd : c.cmds)
        if (const int status = cmd(nullptr); status != LCPP_ERR_INVALID_ARG) ++g_failures, std::printf("FAIL %s: status %d\n", what, status);
}

static int refusals() {
    Device device;
    CommandList c;
    DeviceDeltaRule delta;
    delta.create(device);
    const DeltaHeads heads{4, 2, 64, 32};
    const size_t R = 100;
    const auto temp = made_up<uint>(1, 1 << 24), saved = made_up<uint>(2, 1 << 24);
    const auto q = made_up<float>(3, R * 128), k = made_up<float>(4, R * 128), v = made_up<float>(5, R * 128), out = made_up<float>(6, R * 128);
    const auto decay = made_up<float>(7, R * 4), beta = made_up<float>(8, R * 4);
    const auto all = Sequences::of_length(1, R);
    delta.Forward<float>(c, temp, q, k, v, decay, made_up<float>(8, R * 4 - 1), out, R, heads, all, 1);
    refused("Forward: beta too short", c);
    delta.Forward<float>(c, temp, q, k, v, decay, beta, out, R, heads, {4, 0, made_up<uint>(9, 4)}, 1);
    refused("Forward: fewer offsets than sequences", c);
    delta.Forward<float>(c, temp, q, k, v, decay, beta, out, R, heads, all, 1, made_up<float>(10, 4 * 32 * 64 - 1));
    refused("Forward: states too short", c);
    delta.Forward<float>(c, temp, q, k, v, decay, beta, out, R, heads, all, 1, {}, {}, made_up<uint>(2, 10));
    refused("Forward: saved too short", c);
    delta.Backward<float>(c, temp, q, k, v, decay, beta, made_up<uint>(2, 10), out, q, k, v, {}, decay, R, heads, all, 1);
    refused("Backward: saved too short", c);
    delta.Step<float>(c, q, k, v, decay, beta, {}, made_up<float>(11, 5), out, R, heads, 1);
    refused("Step: states too short", c);
    DeviceCrossEntropy loss;
    loss.create(device);
    const auto t = made_up<int32_t>(12, R);
    loss.Forward<float>(c, temp, q, k, made_up<int32_t>(12, R - 1), beta, {}, R, 128, 100);
    refused("Forward: fewer targets than rows", c);
    loss.Forward<float>(c, temp, q, k, t, beta, {}, R, 128, 101);
    refused("Forward: weight too short", c);
    loss.Backward<float>(c, temp, q, k, t, beta, made_up<float>(13, 2), out, {}, R, 128, 100);
    refused("Backward: two gradients for a hundred rows", c);
    std::printf("%d failure(s)\n", g_failures);
    return g_failures != 0;
}

int main(int argc, char* argv[]) {
    if (argc > 1 && !std::strcmp(argv[1], "refusals")) return refusals();
    Context context{argv[0]};
    Device device = context.create_device("cuda");
    Stream stream = device.create_stream();
    std::mt19937 rng(7);
    std::normal_distribution<float> normal;
    auto random = [&](size_t n, float by = 1) {
        std::vector<float> v(n);
        for (auto& x : v) x = by * normal(rng);
        return v;
    };
    auto upload = [&](const std::vector<float>& v) {
        auto b = device.create_buffer<float>(v.size());
        stream << b.copy_from(v.data()) << synchronize();
        return b;
    };
    {  // two sequences of 90 tokens, a key head for two heads; then a token more, and the gradients of the values
        const size_t S = 2, T = 90, R = S * T;
        const DeltaHeads h{2, 1, 16, 24};
        auto q = random(R * 16, 0.25f), k = random(R * 16, 0.25f), v = random(R * 48), d = random(R * 2), b = random(R * 2), go = random(R * 48);
        for (auto& x : d) x = -std::abs(x) * 0.1f;
        for (auto& x : b) x = 1 / (1 + std::exp(-x));
        for (size_t r = 0; r < R; ++r) {
            double n = 0;
            for (int i = 0; i < 16; ++i) n += k[r * 16 + i] * k[r * 16 + i];
            for (int i = 0; i < 16; ++i) k[r * 16 + i] /= std::sqrt(n);
        }
        auto dq = upload(q), dk = upload(k), dv = upload(v), dd = upload(d), db = upload(b), dgo = upload(go);
        auto out = device.create_buffer<float>(R * 48), last = device.create_buffer<float>(S * h.state());
        auto gq = device.create_buffer<float>(R * 16), gk = device.create_buffer<float>(R * 16), gv = device.create_buffer<float>(R * 48),
             gb = device.create_buffer<float>(R * 2);
        auto temp = device.create_buffer<uint>(bytes_to_uint_count(DeviceDeltaRule::GetTempStorageBytes<float>(R, S, h)));
        auto saved = device.create_buffer<uint>(bytes_to_uint_count(DeviceDeltaRule::GetSavedStateBytes(R, S, h)));
        DeviceDeltaRule rule;
        rule.create(device, &stream);
        CommandList c;
        const auto seqs = Sequences::of_length(S, T);
        rule.Forward<float>(c, temp.view(), dq.view(), dk.view(), dv.view(), dd.view(), db.view(), out.view(), R, h, seqs, 0.5f, {},
                            last.view(), saved.view());
        rule.Backward<float>(c, temp.view(), dq.view(), dk.view(), dv.view(), dd.view(), db.view(), saved.view(), dgo.view(), gq.view(),
                             gk.view(), gv.view(), {}, gb.view(), R, h, seqs, 0.5f);
        std::vector<float> ho(R * 48), hl(S * h.state()), hgv(R * 48);
        stream << c.commit() << out.copy_to(ho.data()) << last.copy_to(hl.data()) << gv.copy_to(hgv.data()) << synchronize();
        for (size_t s = 0; s < S; ++s)
            for (size_t n = 0; n < 2; ++n) {
                std::vector<double> state(24 * 16), x(24 * 16);
                for (size_t t = 0; t < T; ++t) {
                    const size_t r = s * T + t;
                    for (int i = 0; i < 24; ++i) {
                        double sk = 0, o = 0;
                        for (int j = 0; j < 16; ++j) state[i * 16 + j] *= std::exp((double)d[r * 2 + n]), sk += state[i * 16 + j] * k[r * 16 + j];
                        const double u = b[r * 2 + n] * (v[(r * 2 + n) * 24 + i] - sk);
                        for (int j = 0; j < 16; ++j) state[i * 16 + j] += u * k[r * 16 + j], o += 0.5 * state[i * 16 + j] * q[r * 16 + j];
                        near("out", ho[(r * 2 + n) * 24 + i], o, 2e-4);
                    }
                }
                for (size_t i = 0; i < state.size(); ++i) near("last", hl[(s * 2 + n) * h.state() / 2 + i], state[i], 2e-4);
                for (size_t t = T; t-- > 0;) {
                    const size_t r = s * T + t;
                    for (int i = 0; i < 24; ++i) {
                        double du = 0;
                        for (int j = 0; j < 16; ++j) x[i * 16 + j] += 0.5 * go[(r * 2 + n) * 24 + i] * q[r * 16 + j], du += x[i * 16 + j] * k[r * 16 + j];
                        const double y = b[r * 2 + n] * du;
                        near("grad_v", hgv[(r * 2 + n) * 24 + i], y, 2e-4);
                        for (int j = 0; j < 16; ++j) x[i * 16 + j] = (x[i * 16 + j] - y * k[r * 16 + j]) * std::exp((double)d[r * 2 + n]);
                    }
                }
            }
        // a token more for each sequence, in place
        rule.Step<float>(c, dq.view(0, S * 16), dk.view(0, S * 16), dv.view(0, S * 48), dd.view(0, S * 2), db.view(0, S * 2), last.view(),
                         last.view(), out.view(0, S * 48), S, h, 0.5f);
        std::vector<float> after(S * h.state());
        stream << c.commit() << last.copy_to(after.data()) << synchronize();
        for (size_t s = 0; s < S; ++s)
            for (size_t n = 0; n < 2; ++n)
                for (int i = 0; i < 24; ++i) {
                    const float* from = &hl[((s * 2 + n) * 24 + i) * 16];
                    double sk = 0;
                    const double a = std::exp((double)d[s * 2 + n]);
                    for (int j = 0; j < 16; ++j) sk += a * from[j] * k[s * 16 + j];
                    const double u = b[s * 2 + n] * (v[(s * 2 + n) * 24 + i] - sk);
                    for (int j = 0; j < 16; ++j) near("step", after[((s * 2 + n) * 24 + i) * 16 + j], a * from[j] + u * k[s * 16 + j], 1e-5);
                }
    }
    {  // 50 rows, one of which takes no part, over 70 tokens; one gradient of the loss for all
        const size_t R = 50, D = 20, V = 70;
        const auto x = random(R * D), w = random(V * D, 0.5f);
        std::vector<int32_t> t(R);
        for (size_t i = 0; i < R; ++i) t[i] = i == 3 ? -1 : (int32_t)(i * 7 % V);
        auto dx = upload(x), dw = upload(w), one = upload({0.1f});
        auto dt = device.create_buffer<int32_t>(R);
        stream << dt.copy_from(t.data()) << synchronize();
        auto loss = device.create_buffer<float>(R), logsum = device.create_buffer<float>(R);
        auto gx = device.create_buffer<float>(R * D), gw = device.create_buffer<float>(V * D);
        auto temp = device.create_buffer<uint>(bytes_to_uint_count(DeviceCrossEntropy::GetTempStorageBytes<float>(R, D, V)));
        DeviceCrossEntropy ce;
        ce.create(device, &stream);
        CommandList c;
        ce.Forward<float>(c, temp.view(), dx.view(), dw.view(), dt.view(), loss.view(), logsum.view(), R, D, V);
        ce.Backward<float>(c, temp.view(), dx.view(), dw.view(), dt.view(), logsum.view(), one.view(), gx.view(), gw.view(), R, D, V);
        std::vector<float> hl(R), hgx(R * D), hgw(V * D);
        stream << c.commit() << loss.copy_to(hl.data()) << gx.copy_to(hgx.data()) << gw.copy_to(hgw.data()) << synchronize();
        std::vector<double> want(V * D);
        for (size_t i = 0; i < R; ++i) {
            std::vector<double> z(V), g(D);
            double sum = 0;
            for (size_t v = 0; v < V; ++v) {
                for (size_t j = 0; j < D; ++j) z[v] += (double)x[i * D + j] * w[v * D + j];
                sum += std::exp(z[v]);
            }
            if (t[i] >= 0)
                for (size_t v = 0; v < V; ++v) {
                    const double p = 0.1 * (std::exp(z[v]) / sum - ((int32_t)v == t[i]));
                    for (size_t j = 0; j < D; ++j) g[j] += p * w[v * D + j], want[v * D + j] += p * x[i * D + j];
                }
            near("loss", hl[i], t[i] < 0 ? 0 : std::log(sum) - z[t[i]], 1e-4);
            for (size_t j = 0; j < D; ++j) near("grad_hidden", hgx[i * D + j], g[j], 1e-5);
        }
        for (size_t i = 0; i < V * D; ++i) near("grad_weight", hgw[i], want[i], 1e-5);
    }
    std::printf("OK: %d failure(s)\n", g_failures);
    return g_failures != 0;
}
