// What the C++ classes of the sequence operators refuse before anything is launched (made-up addresses, no GPU needed).
// Exit code 0 = all refused.
#include <lcpp/parallel_primitive.h>

#include <cstdio>

using namespace luisa;
using namespace luisa::compute;
using namespace luisa::parallel_primitive;

template <typename T>
static BufferView<T> made_up(size_t i, size_t n) { return {reinterpret_cast<T*>(i << 40), n}; }

static int g_failures = 0;
static void refused(const char* what, CommandList& cmdlist) {
    CommitCommand c = cmdlist.commit();
    for (auto& cmd : c.cmds)
        if (const int status = cmd(nullptr); status != LCPP_ERR_INVALID_ARG)
            ++g_failures, std::printf("FAIL %s: status %d\n", what, status);
}

int main() {
    Device device;
    DeviceLinearRecurrence rec;
    rec.create(device);
    CommandList cmdlist;
    const size_t R = 300, D = 64;
    const auto temp = made_up<uint>(1, 1 << 20), saved = made_up<uint>(2, 1 << 20);
    const auto gate = made_up<float>(3, R * D), in = made_up<float>(4, R * D), out = made_up<float>(5, R * D);
    const auto gg = made_up<float>(6, R * D), gi = made_up<float>(7, R * D);
    Sequences more{4, 0, made_up<uint>(8, 4)};  // four sequences need five offsets
    rec.Forward<SigmoidGate, float>(cmdlist, temp, gate, in, out, R, D, more, {});
    refused("Forward: fewer offsets than sequences", cmdlist);
    rec.Backward<SigmoidGate, float>(cmdlist, temp, gate, in, saved, out, gg, gi, R, D, more, {});
    refused("Backward: fewer offsets than sequences", cmdlist);
    std::printf("%d failure(s)\n", g_failures);
    return g_failures != 0;
}
