// shrike::LogitRouter and shrike::AffineProduct, the C++ mirrors of routing from logits and of products with 4-bit weights. Without an argument: what a
// call refuses, on the host. With "gpu": each of them on numbers whose result is known. Exit code 0 = all passed.
// Build: g++ -std=c++17 -I include tests/cpp/logit_routing_harness.cpp -L shrike_amd -lshrikehip
#include <cstdio>
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
    uint32_t *u = static_cast<uint32_t *>(p);
    auto route = [&](shrike_route_desc d, uint64_t stride, uint32_t rows) {
        return codeOf([&] { LogitRouter::encode(nullptr, d, p, SHRIKE_ELEM_F32, stride, nullptr, SHRIKE_ELEM_F32, u, p, SHRIKE_ELEM_F16, rows); });
    };
    shrike_route_desc d = LogitRouter::description(64, 8, SHRIKE_SCORES_SIGMOID, true);
    EXPECT(d.groups == 1 && d.kept_groups == 1 && d.group_top == 1 && d.renormalize == 1 && d.scaling == 1.0f);
    EXPECT(route(d, 64, 0) == 0);
    EXPECT(route(d, 63, 1) == EINVAL);
    d.groups = 5;
    EXPECT(route(d, 64, 1) == EINVAL);
    EXPECT(route(LogitRouter::description(64, 33, SHRIKE_SCORES_SOFTMAX, false), 64, 1) == EINVAL);
    const shrike_projection w{p, p, nullptr}, none{p, nullptr, nullptr};
    auto product = [&](const shrike_projection &of, uint64_t xStride, uint32_t rows, uint32_t k) {
        return codeOf([&] {
            AffineProduct::encode(nullptr, p, SHRIKE_ELEM_F16, xStride, of, SHRIKE_META_BF16, 64, nullptr, p, SHRIKE_ELEM_F32, 16, rows, 16, k);
        });
    };
    EXPECT(product(w, 64, 0, 64) == 0);
    EXPECT(product(none, 64, 1, 64) == EINVAL);
    EXPECT(product(w, 100, 1, 96) == EINVAL);
    EXPECT(product(w, 68, 1, 64) == EINVAL);
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
    std::vector<T> host() const {
        std::vector<T> out(bytes / sizeof(T));
        check(shrike_hip_memcpy_d2h(out.data(), p, bytes));
        return out;
    }
};

// Rows of ones by codes of 3 at a scale of 1/128 and a bias of 1/64 a group: k = 128 of them are 5, and i on top for output i;
// symmetric ones (3 - 8) / 128 each, -5.
static void device() {
    const uint32_t d = 128, experts = 16, k = 4;
    check(shrike_hip_init(0));
    for (uint32_t t : {1u, 5u, 70u}) {
        std::vector<uint16_t> scale(experts * d / 64, 0x2000), bias(experts * d / 64, 0x2400);  // fp16 2^-7, 2^-6
        Device x(std::vector<uint16_t>(t * d, 0x3C00)), codes(std::vector<uint8_t>(experts * d / 2, 0x33)), scales(scale), biases(bias);
        std::vector<uint16_t> own(experts);
        for (uint32_t i = 0; i < experts; ++i) own[i] = uint16_t(i == 0 ? 0 : i < 2 ? 0x3C00 : i < 4 ? 0x4000 + (i - 2) * 0x200 : i < 8 ? 0x4400 + (i - 4) * 0x100 : 0x4800 + (i - 8) * 0x80);
        Device addend(own), logits(uint64_t(4) * t * experts), plain(uint64_t(4) * t * experts);  // addend: i as fp16
        AffineProduct::encode(nullptr, x.p, SHRIKE_ELEM_F16, d, {codes.p, scales.p, biases.p}, SHRIKE_META_F16, 64, addend.p, logits.p, SHRIKE_ELEM_F32, experts, t,
                              experts, d);
        AffineProduct::encode(nullptr, x.p, SHRIKE_ELEM_F16, d, {codes.p, scales.p, nullptr}, SHRIKE_META_F16, 64, nullptr, plain.p, SHRIKE_ELEM_F32, experts, t,
                              experts, d);
        check(shrike_hip_device_synchronize());
        const std::vector<float> got = logits.host<float>(), symmetric = plain.host<float>();
        for (uint32_t i = 0; i < t * experts; ++i) EXPECT(got[i] == 5.0f + float(i % experts) && symmetric[i] == -5.0f);
        // equal logits: the first of each kept group's, and equal weights
        shrike_route_desc desc = LogitRouter::description(experts, k, SHRIKE_SCORES_SOFTMAX, true, 2.0f);
        desc.groups = 4;
        desc.kept_groups = 2;
        Device indices(uint64_t(4) * t * k), weights(uint64_t(4) * t * k);
        LogitRouter::encode(nullptr, desc, plain.p, SHRIKE_ELEM_F32, experts, nullptr, SHRIKE_ELEM_F32, static_cast<uint32_t *>(indices.p), weights.p,
                            SHRIKE_ELEM_F32, t);
        check(shrike_hip_device_synchronize());
        const std::vector<uint32_t> equal = indices.host<uint32_t>();
        const std::vector<float> halves = weights.host<float>();
        for (uint32_t i = 0; i < t * k; ++i) EXPECT(equal[i] == i % k && halves[i] == 0.5f);
        // rising logits: the last experts, the largest first
        LogitRouter::encode(nullptr, LogitRouter::description(experts, k, SHRIKE_SCORES_SIGMOID, true), logits.p, SHRIKE_ELEM_F32, experts, nullptr,
                            SHRIKE_ELEM_F32, static_cast<uint32_t *>(indices.p), weights.p, SHRIKE_ELEM_F32, t);
        check(shrike_hip_device_synchronize());
        const std::vector<uint32_t> last = indices.host<uint32_t>();
        for (uint32_t i = 0; i < t * k; ++i) EXPECT(last[i] == experts - 1u - i % k);
    }
}

int main(int argc, char **argv) {
    if (argc > 1 && std::string(argv[1]) == "gpu") device();
    else host();
    std::printf(failures ? "%d checks failed\n" : "all checks passed\n", failures);
    return failures ? 1 : 0;
}
