// Routes from logits: scores, a bias on the choice, groups, the top k and their weights.
//
// A wave takes a row. Order is decided in 64 bits: a choice is an unsigned key that rises with it, 1 for an expert out of service, 0 for
// what must not be taken (experts past the last, experts of groups that were not kept, what has been taken already).
#include "gemv_common.h"

#include <cmath>

namespace shrike {

struct RouteArgs {
    const void *logits;
    uint64_t stride;  // elements
    const void *bias;
    uint32_t *indices;
    void *weights;
    uint32_t rows, experts, top_k, groups, kept, group_size;
    uint32_t logits_type, bias_type, weights_type, group_top, sigmoid, renormalize;
    float scaling;
};

__device__ __forceinline__ float route_load(const void *p, uint64_t i, uint32_t type) {
    if (type == SHRIKE_ELEM_F32) return static_cast<const float *>(p)[i];
    const uint16_t h = static_cast<const uint16_t *>(p)[i];
    return type == SHRIKE_ELEM_F16 ? f16_to_f32(h) : bf16_to_f32(h);
}
// NaN stands for -inf, +inf for the largest finite value
__device__ __forceinline__ float in_service(float v) { return v != v ? -INFINITY : fminf(v, 3.4028234663852886e38f); }

__device__ __forceinline__ uint64_t order_key(double v) {
    const uint64_t u = uint64_t(__double_as_longlong(v + 0.0));  // -0 and +0 tie
    return u >> 63 ? ~u : u | uint64_t(1) << 63;
}
constexpr uint64_t kOutOfService = 1;

__device__ __forceinline__ double shfl_xor(double v, uint32_t o) { return __shfl_xor(v, int(o)); }
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (uint32_t o = 32; o; o >>= 1) v += shfl_xor(v, o);
    return v;
}

__device__ __forceinline__ void route_store_weight(const RouteArgs &a, uint64_t at, double w) {
    const float v = float(w);
    if (a.weights_type == SHRIKE_ELEM_F32) {
        static_cast<float *>(a.weights)[at] = v;
    } else if (a.weights_type == SHRIKE_ELEM_F16) {
        static_cast<uint16_t *>(a.weights)[at] = f32_to_f16(v);
    } else {
        const uint32_t u = __float_as_uint(v);
        static_cast<uint16_t *>(a.weights)[at] = uint16_t(v != v ? 0x7fc0u : (u + 0x7fffu + (u >> 16 & 1u)) >> 16);
    }
}

// One row by one wave; lane l holds experts l, l + 64, ... `s_value` (a double an expert) is the wave's own.
template <int NPL>
__device__ void route_row(const RouteArgs &a, uint32_t row, double *s_value) {
    const uint32_t lane = threadIdx.x & 63u;
    float l[NPL];
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const uint32_t e = lane + 64u * j;
        l[j] = e < a.experts ? in_service(route_load(a.logits, uint64_t(row) * a.stride + e, a.logits_type)) : -INFINITY;
        top = fmaxf(top, l[j]);
    }
    top = wave_max_f32(top);
    const double base = top == -INFINITY ? 0.0 : double(top);
    double total = 0.0;
    if (!a.sigmoid) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) total += exp(double(l[j]) - base);
        total = wave_sum_f64(total);
        total = total > 0.0 ? total : 1.0;
    }
    auto score = [&](float v) -> double { return v == -INFINITY ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-double(v))) : exp(double(v) - base) / total; };
    const bool by_value = a.bias != nullptr, values = by_value || (a.groups > 1u && a.group_top == 2u);
    uint64_t key[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const uint32_t e = lane + 64u * j;
        const bool there = e < a.experts;
        double v = values ? score(l[j]) : 0.0;
        bool out = l[j] == -INFINITY;
        if (by_value && there) {
            const float b = in_service(route_load(a.bias, e, a.bias_type));
            out |= b == -INFINITY;
            v += double(b);
        }
        key[j] = !there ? 0 : out ? kOutOfService : order_key(by_value ? v : double(l[j]));
        if (a.groups > 1u && there) s_value[e] = out ? -INFINITY : a.group_top == 2u || by_value ? v : double(l[j]);
    }
    if (a.groups > 1u) {
        __builtin_amdgcn_wave_barrier();
        // lane g has group g
        uint64_t mark = 0;
        if (lane < a.groups) {
            double first = -INFINITY, second = -INFINITY;
            for (uint32_t i = 0; i < a.group_size; ++i) {
                const double v = s_value[lane * a.group_size + i];
                if (v > first) {
                    second = first;
                    first = v;
                } else if (v > second) {
                    second = v;
                }
            }
            const double sum = a.group_top == 2u && first != -INFINITY ? first + (second == -INFINITY ? 0.0 : second) : first;
            mark = first == -INFINITY ? kOutOfService : order_key(sum);
        }
        uint64_t kept = 0;
        for (uint32_t r = 0; r < a.kept; ++r) {
            const uint64_t best = wave_max_u64(mark);
            const uint32_t g = uint32_t(__builtin_ctzll(__ballot(mark == best)));
            kept |= uint64_t(1) << g;
            if (lane == g) mark = 0;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            const uint32_t e = lane + 64u * j;
            if (e < a.experts && !(kept >> (e / a.group_size) & 1u)) key[j] = 0;
        }
    }
    uint32_t mine = 0;
    uint64_t my_key = kOutOfService;
    float my_logit = -INFINITY;
    for (uint32_t r = 0; r < a.top_k; ++r) {
        uint64_t best = 0;
        uint32_t e = 0;
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            if (key[j] > best) {  // strictly: of equals the lower index stays
                best = key[j];
                e = lane + 64u * j;
                v = l[j];
            }
        }
        const uint64_t most = wave_max_u64(best);
        const uint32_t win = wave_min_u32(best == most ? e : 0xffffffffu);
        const float logit = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), int(win & 63u)));
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (lane + 64u * j == win) key[j] = 0;
        if (lane == r) {
            mine = win;
            my_key = most;
            my_logit = logit;
        }
    }
    const bool on = lane < a.top_k, served = on && my_key != kOutOfService;
    double w = 0.0;
    if (a.renormalize && !a.sigmoid) {  // the softmax of the chosen ones: nothing underflows that counts
        const float most = wave_max_f32(served ? my_logit : -INFINITY);
        w = served ? exp(double(my_logit) - double(most)) : 0.0;
    } else {
        w = served ? score(my_logit) : 0.0;
    }
    if (a.renormalize) {
        const double sum = wave_sum_f64(w);
        w = sum > 0.0 ? w / sum : 0.0;
    }
    if (on) {
        const uint64_t at = uint64_t(row) * a.top_k + lane;
        a.indices[at] = mine;
        route_store_weight(a, at, w * double(a.scaling));
    }
}

template <int NPL>
__global__ __launch_bounds__(256) void k_route_rows(RouteArgs a) {
    __shared__ double s_value[4][64 * NPL];
    const uint32_t wave = wave_index();
    for (uint64_t row = uint64_t(blockIdx.x) * 4u + wave; row < a.rows; row += uint64_t(gridDim.x) * 4u) route_row<NPL>(a, uint32_t(row), s_value[wave]);
}

}  // namespace shrike

using namespace shrike;

extern "C" int shrike_hip_route_rows(void *stream, const shrike_route_desc *desc, const void *d_logits, uint32_t logits_dtype,
                                     uint64_t logits_stride_elements, const void *d_bias, uint32_t bias_dtype, uint32_t *d_out_indices,
                                     void *d_out_weights, uint32_t weights_dtype, uint32_t rows) {
    SHRIKE_REQUIRE(desc && d_logits && d_out_indices && d_out_weights, "route: NULL argument");
    SHRIKE_REQUIRE(logits_dtype <= SHRIKE_ELEM_F32 && weights_dtype <= SHRIKE_ELEM_F32 && (!d_bias || bias_dtype <= SHRIKE_ELEM_F32),
                   "route: an element type of %u, %u, %u (logits, bias, weights) is not a known value", logits_dtype, bias_dtype, weights_dtype);
    SHRIKE_REQUIRE(desc->num_experts >= 1 && desc->num_experts <= SHRIKE_ROUTE_MAX_EXPERTS, "route: numExperts=%u not in 1...%u", desc->num_experts,
                   SHRIKE_ROUTE_MAX_EXPERTS);
    SHRIKE_REQUIRE(desc->scores <= SHRIKE_SCORES_SIGMOID, "route: scores %u are not a known value", desc->scores);
    SHRIKE_REQUIRE(desc->groups >= 1 && desc->groups <= SHRIKE_ROUTE_MAX_GROUPS && desc->num_experts % desc->groups == 0,
                   "route: %u groups do not divide %u experts, or are not in 1...%u", desc->groups, desc->num_experts, SHRIKE_ROUTE_MAX_GROUPS);
    SHRIKE_REQUIRE(desc->kept_groups >= 1 && desc->kept_groups <= desc->groups, "route: keptGroups=%u not in 1...%u", desc->kept_groups, desc->groups);
    SHRIKE_REQUIRE(desc->group_top == 1 || desc->group_top == 2, "route: groupTop=%u is neither 1 nor 2", desc->group_top);
    const uint32_t size = desc->num_experts / desc->groups;
    SHRIKE_REQUIRE(desc->top_k >= 1 && desc->top_k <= SHRIKE_ROUTE_MAX_TOP_K && desc->top_k <= desc->kept_groups * size,
                   "route: topK=%u not in 1...%u, or more than the %u experts of the kept groups", desc->top_k, SHRIKE_ROUTE_MAX_TOP_K,
                   desc->kept_groups * size);
    SHRIKE_REQUIRE(std::isfinite(desc->scaling), "route: the scaling is not finite");
    SHRIKE_REQUIRE(logits_stride_elements >= desc->num_experts && logits_stride_elements <= uint64_t(1) << 28,
                   "route: a stride of %llu does not fit %u experts", (unsigned long long)logits_stride_elements, desc->num_experts);
    auto aligned = [](const void *p, uint32_t type) { return reinterpret_cast<uintptr_t>(p) % (type == SHRIKE_ELEM_F32 ? 4u : 2u) == 0; };
    SHRIKE_REQUIRE(aligned(d_logits, logits_dtype) && aligned(d_out_weights, weights_dtype) && (!d_bias || aligned(d_bias, bias_dtype))
                       && reinterpret_cast<uintptr_t>(d_out_indices) % 4u == 0,
                   "route: a buffer is not aligned to its elements' size");
    if (rows == 0) return 0;
    RouteArgs a = {};
    a.logits = d_logits;
    a.stride = logits_stride_elements;
    a.bias = d_bias;
    a.indices = d_out_indices;
    a.weights = d_out_weights;
    a.rows = rows;
    a.experts = desc->num_experts;
    a.top_k = desc->top_k;
    a.groups = desc->kept_groups == desc->groups ? 1u : desc->groups;  // all of them kept: as if there were none
    a.kept = desc->kept_groups;
    a.group_size = size;
    a.logits_type = logits_dtype;
    a.bias_type = bias_dtype;
    a.weights_type = weights_dtype;
    a.group_top = desc->group_top;
    a.sigmoid = desc->scores == SHRIKE_SCORES_SIGMOID;
    a.renormalize = desc->renormalize != 0;
    a.scaling = desc->scaling;
    const uint32_t blocks = std::min((rows - 1u) / 4u + 1u, 65536u);
    const hipStream_t s = as_stream(stream);
    const uint32_t per_lane = (a.experts + 63u) / 64u;
    if (per_lane <= 1) hipLaunchKernelGGL((k_route_rows<1>), dim3(blocks), dim3(256), 0, s, a);
    else if (per_lane <= 2) hipLaunchKernelGGL((k_route_rows<2>), dim3(blocks), dim3(256), 0, s, a);
    else if (per_lane <= 4) hipLaunchKernelGGL((k_route_rows<4>), dim3(blocks), dim3(256), 0, s, a);
    else if (per_lane <= 8) hipLaunchKernelGGL((k_route_rows<8>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_route_rows<16>), dim3(blocks), dim3(256), 0, s, a);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}
