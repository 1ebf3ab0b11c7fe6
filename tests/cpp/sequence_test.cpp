// C++ test of the sequence operators' public headers: a recurrence forward, backward and step by step, and a beam
// selection with reordering, against plain loops in double.  Exit code 0 = all checks passed.
#include <lcpp/parallel_primitive.h>

#include <cmath>
#include <cstdio>
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

int main(int, char* argv[]) {
    Context context{argv[0]};
    Device device = context.create_device("cuda");
    Stream stream = device.create_stream();
    std::mt19937 rng(7);
    std::normal_distribution<float> normal;
    auto random = [&](size_t n) {
        std::vector<float> v(n);
        for (auto& x : v) x = normal(rng);
        return v;
    };
    auto upload = [&](auto& b, const auto& v) { stream << b.copy_from(v.data()) << synchronize(); };

    {  // two sequences of 200 tokens, 33 channels, float
        const size_t S = 2, T = 200, R = S * T, D = 33;
        const auto g = random(R * D), x = random(R * D), h0 = random(S * D), go = random(R * D), gl = random(S * D);
        auto dg = device.create_buffer<float>(R * D), dx = device.create_buffer<float>(R * D);
        auto out = device.create_buffer<float>(R * D), dgo = device.create_buffer<float>(R * D);
        auto gg = device.create_buffer<float>(R * D), gi = device.create_buffer<float>(R * D);
        auto init = device.create_buffer<float>(S * D), last = device.create_buffer<float>(S * D);
        auto dgl = device.create_buffer<float>(S * D), g0 = device.create_buffer<float>(S * D);
        upload(dg, g), upload(dx, x), upload(init, h0), upload(dgo, go), upload(dgl, gl);
        auto temp = device.create_buffer<uint>(bytes_to_uint_count(DeviceLinearRecurrence::GetTempStorageBytes(R, D)));
        auto saved = device.create_buffer<uint>(bytes_to_uint_count(DeviceLinearRecurrence::GetSavedStateBytes(R, D)));
        DeviceLinearRecurrence rec;
        rec.create(device, &stream);
        CommandList cmdlist;
        const auto seqs = Sequences::of_length(S, T);
        rec.Forward<SigmoidGate, float>(cmdlist, temp.view(), dg.view(), dx.view(), out.view(), R, D, seqs, {}, init.view(),
                                        last.view(), saved.view());
        rec.Backward<SigmoidGate, float>(cmdlist, temp.view(), dg.view(), dx.view(), saved.view(), dgo.view(), gg.view(),
                                         gi.view(), R, D, seqs, {}, init.view(), dgl.view(), g0.view());
        std::vector<float> ho(R * D), hl(S * D), hgg(R * D), hgi(R * D), hg0(S * D);
        stream << cmdlist.commit() << out.copy_to(ho.data()) << last.copy_to(hl.data()) << gg.copy_to(hgg.data())
               << gi.copy_to(hgi.data()) << g0.copy_to(hg0.data()) << synchronize();
        for (size_t s = 0; s < S; ++s)
            for (size_t c = 0; c < D; ++c) {
                std::vector<double> h(T + 1);
                h[0] = h0[s * D + c];
                auto at = [&](size_t t) { return (s * T + t) * D + c; };
                for (size_t t = 0; t < T; ++t) {
                    const double a = 1 / (1 + std::exp(-(double)g[at(t)]));
                    h[t + 1] = a * h[t] + (1 - a) * x[at(t)];
                    near("out", ho[at(t)], h[t + 1], 2e-5);
                }
                near("last", hl[s * D + c], h[T], 2e-5);
                double mu = gl[s * D + c];
                for (size_t t = T; t-- > 0;) {
                    const double a = 1 / (1 + std::exp(-(double)g[at(t)])), lam = go[at(t)] + mu;
                    near("grad_gate", hgg[at(t)], lam * (h[t] - x[at(t)]) * a * (1 - a), 1e-4);
                    near("grad_in", hgi[at(t)], lam * (1 - a), 1e-4);
                    mu = a * lam;
                }
                near("grad_init", hg0[s * D + c], mu, 1e-4);
            }
        // a token more, in place
        rec.Step<SigmoidGate, float>(cmdlist, dg.view(0, S * D), dx.view(0, S * D), last.view(), last.view(),
                                     BufferView<float>{}, S, D, {});
        std::vector<float> after(S * D);
        stream << cmdlist.commit() << last.copy_to(after.data()) << synchronize();
        for (size_t i = 0; i < S * D; ++i) {
            const double a = 1 / (1 + std::exp(-(double)g[i]));
            near("step", after[i], a * hl[i] + (1 - a) * x[i], 2e-5);
        }
        // a temp buffer that is too small is a status, not a fault
        CommandList bad;
        DeviceLinearRecurrence quiet;
        quiet.create(device);
        quiet.Forward<LinearGate, float>(bad, BufferView<uint>{}, dg.view(), dx.view(), out.view(), R, D, seqs, {});
        Stream other = device.create_stream();
        other << bad.commit() << synchronize();
        if (other.last_status() != LCPP_ERR_TEMP_TOO_SMALL) ++g_failures, std::printf("FAIL status %d\n", other.last_status());
    }

    {  // one entry, two beams, five tokens; the states follow
        const std::vector<float> z = {0, 1, 2, 3, 4, 4, 3, 2, 1, 0}, scores = {0, -1};
        auto dz = device.create_buffer<float>(10), ds = device.create_buffer<float>(2), so = device.create_buffer<float>(2);
        auto tok = device.create_buffer<int32_t>(2), par = device.create_buffer<int32_t>(2);
        auto fin = device.create_buffer<uint8_t>(2);
        upload(dz, z), upload(ds, scores);
        auto temp = device.create_buffer<uint>(bytes_to_uint_count(DeviceBeamSearch::GetTempStorageBytes(1, 2, 5)));
        auto in = device.create_buffer<float>(2 * 2 * 3), out = device.create_buffer<float>(2 * 2 * 3);
        const std::vector<float> states = {0, 1, 2, 10, 11, 12, 20, 21, 22, 30, 31, 32};
        upload(in, states);
        DeviceBeamSearch beams;
        beams.create(device, &stream);
        CommandList cmdlist;
        beams.Select<float>(cmdlist, temp.view(), dz.view(), ds.view(), {}, so.view(), tok.view(), par.view(), fin.view(), 1, 2,
                            5, 3);
        beams.Reorder<float>(cmdlist, in.view(), out.view(), par.view(), 2, 2, 2, 3);
        std::vector<float> hs(2), ho(12);
        std::vector<int32_t> ht(2), hp(2);
        std::vector<uint8_t> hf(2);
        stream << cmdlist.commit() << so.copy_to(hs.data()) << tok.copy_to(ht.data()) << par.copy_to(hp.data())
               << fin.copy_to(hf.data()) << out.copy_to(ho.data()) << synchronize();
        const double log_sum = std::log(1 + std::exp(-1.) + std::exp(-2.) + std::exp(-3.) + std::exp(-4.));
        near("score 0", hs[0], -log_sum, 1e-5);
        near("score 1", hs[1], -1 - log_sum, 1e-5);  // ties: token 3 of beam 0 and token 0 of beam 1; beam 0 first
        if (ht[0] != 4 || ht[1] != 3 || hp[0] != 0 || hp[1] != 0 || hf[0] != 0 || hf[1] != 1)
            ++g_failures, std::printf("FAIL tokens %d %d parents %d %d\n", ht[0], ht[1], hp[0], hp[1]);
        for (int l = 0; l < 2; ++l)
            for (int i = 0; i < 2; ++i)
                for (int w = 0; w < 3; ++w) near("states", ho[(l * 2 + i) * 3 + w], states[(l * 2 + hp[i]) * 3 + w], 0);
    }
    std::printf("OK: %d failure(s)\n", g_failures);
    return g_failures != 0;
}
