// shrike::MicroscaledBlocks, the C++ mirror of the operators over microscaled blocks. Without an argument: what a call refuses, on the host. With
// "gpu": each of them on numbers whose result is known. Exit code 0 = all passed.
// Build: g++ -std=c++17 -I include tests/cpp/mx_harness.cpp -L shrike_amd -lshrikehip
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "shrike.hpp"

using namespace shrike;

static int failures = 0;
#define EXPECT(cond)                                                      \
    do {                                                                  \
        if (!(cond)) {                                                    \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            ++failures;                                                   \
        }                                                                 \
    } while (0)

template <typename Call>
static int codeOf(Call call) {
    try {
        call();
    } catch (const Error &e) {
        return e.code;
    }
    return 0;
}

static void host() {
    void *p = reinterpret_cast<void *>(uintptr_t(0x10000));  // an address that is only ever looked at
    // numbers of rows that 32 bits do not hold arrive whole: as many as 2^40 are refused, not taken for none
    for (uint64_t rows : {uint64_t(1) << 40, uint64_t(1) << 50, (uint64_t(1) << 40) + 1}) {
        EXPECT(codeOf([&] { MicroscaledBlocks::quantize(nullptr, p, SHRIKE_ELEM_F16, 64, SHRIKE_MX_E4M3, p, p, rows, 64); }) == EINVAL);
        EXPECT(codeOf([&] { MicroscaledBlocks::dequantize(nullptr, p, p, SHRIKE_MX_E4M3, p, SHRIKE_ELEM_F16, 64, rows, 64); }) == EINVAL);
    }
    EXPECT(codeOf([&] { MicroscaledBlocks::quantize(nullptr, p, SHRIKE_ELEM_F16, 64, SHRIKE_MX_E4M3, p, p, 0, 64); }) == 0);
    EXPECT(codeOf([&] { MicroscaledBlocks::product(nullptr, p, p, SHRIKE_MX_E4M3, p, p, nullptr, p, SHRIKE_ELEM_F32, 16, 1, 16, 64); }) == EINVAL);
    EXPECT(codeOf([&] { MicroscaledBlocks::residualAddRMSNorm(nullptr, p, p, p, nullptr, p, p, p, 64, 0.0f, 1); }) == EINVAL);
    shrike_expert_offsets off;
    EXPECT(MicroscaledBlocks::expertOffsets(128, 64, false, off) == 3u * 128u * 64u * 17u / 32u);
    EXPECT(codeOf([&] { MicroscaledBlocks::expertOffsets(128, 65, false, off); }) == EINVAL);
    EXPECT(MicroscaledBlocks::groupedWorkspaceBytes(3, 64) >= 3u * 64u * (64u + 2u));
    EXPECT(MicroscaledBlocks::decodeWorkspaceBytes(3, 4, 64) >= 3u * 4u * (64u + 2u));
}

struct Device {  // a device allocation with host copies in and out
    void *p;
    uint64_t bytes;
    explicit Device(uint64_t n) : p(shrike_hip_malloc(n)), bytes(n) {
        if (!p) throw Error(ENOMEM, shrike_hip_last_error());
    }
    template <typename T>
    explicit Device(const std::vector<T> &host) : Device(uint64_t(host.size() * sizeof(T))) {
        check(shrike_hip_memcpy_h2d(p, host.data(), bytes));
    }
    ~Device() { shrike_hip_free(p); }
    Device(const Device &) = delete;
    template <typename T>
    bool all(T value) const {
        std::vector<T> out(bytes / sizeof(T));
        check(shrike_hip_memcpy_d2h(out.data(), p, bytes));
        for (T v : out)
            if (v != value) return false;
        return true;
    }
    template <typename T>
    T *as() const { return static_cast<T *>(p); }
};

// Every row of x is ones. gate: weights of 1 / d, so sums of 1; up: of 0.5 / d, 0.5. silu(1) / 2 = 0.3655 lies nearest to 0.375 of E4M3 at the
// scale of its block; down: weights of 1 / f, so 0.375 comes out, and of eight experts at an eighth each.
static void device() {
    const uint32_t d = 128, f = 64, experts = 8, k = 8, t = 5;
    const uint16_t one = 0x3C00, half = 0x3800, eighth = 0x3000, three8ths = 0x3600, seven8ths = 0x3B00;  // fp16
    check(shrike_hip_init(0));

    // the norm of (1/2 + 1/2) is ones, in E4M3 blocks 256 * 2^-8
    Device hidden(std::vector<uint16_t>(t * d, half)), delta(std::vector<uint16_t>(t * d, half)), weight(std::vector<uint16_t>(d, 0x3F80));
    Device sum(uint64_t(2) * t * d), out(uint64_t(2) * t * d), codes(uint64_t(t) * d), scales(uint64_t(t) * d / 32);
    MicroscaledBlocks::residualAddRMSNorm(nullptr, hidden.p, delta.p, weight.p, sum.p, out.p, codes.p, scales.p, d, 0.0f, t);
    check(shrike_hip_device_synchronize());
    EXPECT(sum.all<uint16_t>(one) && out.all<uint16_t>(one) && codes.all<uint8_t>(0x78) && scales.all<uint8_t>(127 - 8));

    // the same rows by the quantiser, and back
    Device codes2(uint64_t(t) * d), scales2(uint64_t(t) * d / 32), back(uint64_t(2) * t * d);
    MicroscaledBlocks::quantize(nullptr, out.p, SHRIKE_ELEM_F16, d, SHRIKE_MX_E4M3, codes2.p, scales2.p, t, d);
    MicroscaledBlocks::dequantize(nullptr, codes2.p, scales2.p, SHRIKE_MX_E4M3, back.p, SHRIKE_ELEM_F16, d, t, d);
    check(shrike_hip_device_synchronize());
    EXPECT(codes2.all<uint8_t>(0x78) && scales2.all<uint8_t>(127 - 8) && back.all<uint16_t>(one));

    // 128 ones by weights of 1 / 128, and a bias of 2
    const uint32_t n = 24;
    Device w(std::vector<uint8_t>(n * d / 2, 0x22)), ws(std::vector<uint8_t>(n * d / 32, 127 - 7)), bias(std::vector<uint16_t>(n, 0x4000));
    Device product(uint64_t(2) * t * n);
    MicroscaledBlocks::product(nullptr, codes.p, scales.p, SHRIKE_MX_E4M3, w.p, ws.p, bias.p, product.p, SHRIKE_ELEM_F16, n, t, n, d);
    check(shrike_hip_device_synchronize());
    EXPECT(product.all<uint16_t>(0x4200));

    shrike_expert_offsets off;
    const uint64_t size = MicroscaledBlocks::expertOffsets(d, f, false, off);
    std::vector<uint8_t> blob(size, 0);
    auto fill = [&](uint32_t at, uint32_t count, uint8_t byte) { std::memset(&blob[at], byte, count); };
    fill(off.gate_w_off, d * f / 2, 0x22); fill(off.gate_s_off, d * f / 32, 127 - 7);
    fill(off.up_w_off, d * f / 2, 0x11); fill(off.up_s_off, d * f / 32, 127 - 7);
    fill(off.down_w_off, d * f / 2, 0x22); fill(off.down_s_off, d * f / 32, 127 - 6);
    shrike_moe_desc desc{};
    desc.d = d; desc.f = f; desc.num_experts = experts; desc.top_k = k;
    desc.routed_weight_bits = 4; desc.meta_dtype = SHRIKE_META_F16; desc.activation = SHRIKE_ACT_SILU;
    MoE moe(desc);
    ExpertPool pool(experts, size, experts);
    for (uint32_t e = 0; e < experts; ++e) {
        pool.upload(e, blob.data(), size, nullptr);
        pool.publish(e, e, SHRIKE_RESIDENCY_RESIDENT, nullptr);
    }
    check(shrike_hip_device_synchronize());
    {
        const uint32_t tokens = 2;
        std::vector<uint32_t> slots(tokens * k);
        for (uint32_t i = 0; i < tokens * k; ++i) slots[i] = i * 3u % experts;
        Device resolved(slots), weights(std::vector<uint16_t>(tokens * k, eighth)), residual(std::vector<uint16_t>(tokens * d, 0));
        Device y(uint64_t(2) * tokens * d), stream(std::vector<uint16_t>(tokens * d, half)), workspace(MicroscaledBlocks::decodeWorkspaceBytes(tokens, k, f));
        MicroscaledBlocks::encodeDecodeFFN(moe, nullptr, pool, resolved.as<uint32_t>(), off, codes.p, scales.p, weights.p, residual.p, y.p, stream.p,
                                           workspace.p, workspace.bytes, d, f, k, tokens);
        check(shrike_hip_device_synchronize());
        EXPECT(y.all<uint16_t>(three8ths) && stream.all<uint16_t>(seven8ths));
    }
    {
        std::vector<uint32_t> indices(t * k);
        for (uint32_t i = 0; i < t * k; ++i) indices[i] = (i + i / k) % experts;
        Device idx(indices), weights(std::vector<uint16_t>(t * k, eighth));
        const uint32_t maxTiles = shrike_hip_group_max_row_tiles(t * k, experts);
        Device sorted(uint64_t(16) * t * k), offsets(4 * experts), counts(4 * experts), tiles(uint64_t(16) * maxTiles), tileCount(4);
        const shrike_hip_grouped_routes routes{sorted.p, offsets.as<uint32_t>(), counts.as<uint32_t>(), tiles.as<shrike_row_tile>(), tileCount.as<uint32_t>()};
        PrefillMoEGrouping::encodeGroupPairs(nullptr, idx.as<uint32_t>(), weights.p, t, k, experts, nullptr, pool.residencyTable(), routes);
        Device partials(uint64_t(2) * t * k * d), workspace(MicroscaledBlocks::groupedWorkspaceBytes(maxTiles, f));
        MicroscaledBlocks::encodeGroupedExpertGEMMs(moe, nullptr, pool, off, routes, maxTiles, codes.p, scales.p, partials.p, workspace.p, workspace.bytes, t,
                                                    d, f, k);
        check(shrike_hip_device_synchronize());
        EXPECT(partials.all<uint16_t>(three8ths));
    }
}

int main(int argc, char **argv) {
    if (argc > 1 && std::string(argv[1]) == "gpu") device();
    else host();
    std::printf(failures ? "%d checks failed\n" : "all checks passed\n", failures);
    return failures ? 1 : 0;
}
