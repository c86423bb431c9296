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
    uint32_t group_shift;        // 2^i lanes have a group
    float levels;                // of the additions of a row's experts in pairs
    uint32_t whole, whole_bias;  // rows (the bias) and their groups start at multiples of 16 bytes and are multiples of 16 bytes long
};

__device__ __forceinline__ float route_load(const void *p, uint64_t i, uint32_t type) {
    if (type == SHRIKE_ELEM_F32) return static_cast<const float *>(p)[i];
    const uint16_t h = static_cast<const uint16_t *>(p)[i];
    return type == SHRIKE_ELEM_F16 ? f16_to_f32(h) : bf16_to_f32(h);
}
// NaN stands for -inf, +inf for the largest finite value
__device__ __forceinline__ float in_service(float v) { return fminf(fmaxf(v, -INFINITY), 3.4028234663852886e38f); }  // (fmaxf takes the number of a number and a NaN)

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

// ------------------------------------------------------------------ many rows at once
//
// 64 bits are needed where two choices lie close together, and that is seldom: here a choice is a 32-bit word, its value in fixed point below the row's
// largest (22 bits) over the expert's number (10, so that the lower one is the larger word), from fp32 arithmetic whose error has a
// bound. The words' order is the choices' order where neighbours in it, the last one taken and the first one left among them, are as far
// apart as both may be off. Where some of them are not, the words next in order are taken too, up to a gap, and the scores of those alone are formed and
// put into order in 64 bits; a row without a gap in 32, or whose groups lie too close, is routed again by route_row. Where the logits themselves
// decide and have 16 bits, the word is all of them over the number, and exact.
//
// Both sums, of all scores and of the chosen ones, are formed in pairs of neighbours, pairs of these and so on, an order that does not depend on the lanes
// a row has: its weights are the same bits in a call of any size.
//
// LANES lanes have a row, each up to NPL neighbouring experts of one group: 64 for few rows, which takes the fewest steps, 16 for many, where four rows
// share every step between lanes. A step of the selection is the largest of a lane's words below the last one taken, and then of the row's lanes. The
// vector unit bounds it, busy 99 % of the time: 16,384 rows of 512, top 10, take 21 us where their bytes take 7 (in 64 bits alone 75; every close row again in 64 bits 33; words with a test of range each 30). One row takes 3.2 us on the GPU, and
// a call from the host 8.

enum class RouteWord { kValue, kLogit, kLogit16 };
constexpr float kUnits = 4194296.0f;  // 2^22 - 8
// How far a score in fp32 may be off, in 2^-24. exp_fast of -x: its argument has two or three roundings and the constant's, which count x times, and the
// instruction 2 (one place), (2.25 x + 2) of it: for a softmax up to 2.1 of the largest term, which is 1. The softmax's sum, of 2^i experts: what its terms
// are off, under i + 2 of the sum (11.7 where 1,023 of them lie near x = 5 beside the 1), its additions in pairs i, its reciprocal 2. That factor is one for the
// whole row and moves a choice against another, as the bias is not scaled with it, by 2 i + 4 of the scores' difference. Two choices of a softmax: 2 * 2.1 + 2 i + 4
// of the largest score at most; of sigmoids, s (1 - s) (1.25 x + 2) + 3 s each, under 3.2.
__device__ __forceinline__ float softmax_off(float levels) { return (levels + 4.25f) * 0x1p-24f; }
__device__ __forceinline__ float softmax_sum_off(float levels) { return (2.0f * levels + 5.0f) * 0x1p-24f; }
constexpr float kSigmoidOff = 0x1p-22f;

template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    if constexpr (LANES == 64) return wave_max_u32(v);
    v = max(v, dpp_keep_u32<0xB1>(v));   // quad_perm [1,0,3,2]
    v = max(v, dpp_keep_u32<0x4E>(v));   // quad_perm [2,3,0,1]
    v = max(v, dpp_keep_u32<0x141>(v));  // row_half_mirror
    return max(v, dpp_keep_u32<0x140>(v));  // row_mirror
}
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
    if constexpr (LANES == 64) return wave_max_f32(v);
    v = fmaxf(v, dpp_keep_f32<0xB1>(v));
    v = fmaxf(v, dpp_keep_f32<0x4E>(v));
    v = fmaxf(v, dpp_keep_f32<0x141>(v));
    return fmaxf(v, dpp_keep_f32<0x140>(v));
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (LANES == 64) return wave_sum(v);
    v += dpp_f32<0xB1>(v);
    v += dpp_f32<0x4E>(v);
    v += dpp_f32<0x141>(v);
    return v + dpp_f32<0x140>(v);
}
__device__ __forceinline__ float exp_fast(float v) { return __builtin_amdgcn_exp2f(1.4426950408889634f * v); }

// NPL neighbouring values, from the expert `first` of the row at `at` on, and their 16 bits where they have 16; past the last expert something. `whole`: from
// 16-byte aligned addresses, in whole loads.
template <int NPL>
__device__ __forceinline__ void load_experts(const void *from, uint64_t at, uint32_t type, uint32_t whole, uint32_t first, uint32_t experts, float (&v)[NPL],
                                             uint16_t (&bits)[NPL]) {
    if (type == SHRIKE_ELEM_F32) {
        const float *p = static_cast<const float *>(from) + at;
        if (NPL % 4 == 0 && whole) {
#pragma unroll
            for (int j = 0; j < NPL; j += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(p + (first + j < experts ? first + j : 0u));
                const float w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) v[(j + i) % NPL] = w[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < NPL; ++j) v[j] = p[min(first + j, experts - 1u)];
        }
        return;
    }
    const uint16_t *p = static_cast<const uint16_t *>(from) + at;
    if (NPL % 8 == 0 && whole) {
#pragma unroll
        for (int j = 0; j < NPL; j += 8) {
            const uint4 f = *reinterpret_cast<const uint4 *>(p + (first + j < experts ? first + j : 0u));
            const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) bits[(j + i) % NPL] = uint16_t(w[i / 2] >> 16 * (i % 2));
        }
    } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j) bits[j] = p[min(first + j, experts - 1u)];
    }
    if (type == SHRIKE_ELEM_F16) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) v[j] = f16_to_f32(bits[j]);
    } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j) v[j] = bf16_to_f32(bits[j]);
    }
}

template <int LANES, int NPL, RouteWord WORD>
__global__ __launch_bounds__(256) void k_route_rows_fast(RouteArgs a) {
    constexpr int kWide = LANES * NPL < 64 ? 1 : LANES * NPL / 64;  // experts a lane where a wave has the row
    constexpr uint32_t kIndexBits = WORD == RouteWord::kLogit16 ? 16 : 10, kRows = 64 / LANES, kSlots = LANES == 16 ? 2 : 1;
    constexpr uint32_t kOutWord = WORD == RouteWord::kLogit16 ? 0 : 1;  // what an expert out of service has above its number
    constexpr int kDoubles = 64 * kWide < int(kRows) * 64 ? int(kRows) * 64 : 64 * kWide;
    __shared__ double s_value[4][kDoubles];
    const uint32_t lane = threadIdx.x & 63u, wave = wave_index(), sub = lane % LANES;
    const uint64_t first_row = (uint64_t(blockIdx.x) * 4u + wave) * kRows;
    if (first_row >= a.rows) return;
    const bool real = first_row + lane / LANES < a.rows;
    const uint64_t row = real ? first_row + lane / LANES : a.rows - 1u, at = row * a.stride;

    // ---- the row: of 2^group_shift lanes a group's experts, up to NPL of them a lane
    const uint32_t group = sub >> a.group_shift, within = (sub & ((1u << a.group_shift) - 1u)) * NPL, first = group * a.group_size + within;
    const uint32_t have = group < a.groups && within < a.group_size ? a.group_size - within : 0u;  // (NPL or more: all of a lane's)
    float l[NPL], b[NPL];
    uint16_t bits[NPL];  // 16-bit logits as they are
    load_experts<NPL>(a.logits, at, a.logits_type, a.whole, first, a.experts, l, bits);
    if (WORD == RouteWord::kValue) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) b[j] = 0.0f;
        uint16_t unused[NPL];
        if (a.bias) load_experts<NPL>(a.bias, 0, a.bias_type, a.whole_bias, first, a.experts, b, unused);
    }
    const bool full = a.experts == uint32_t(LANES * NPL);  // every lane's experts are there
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NPL; ++j) l[j] = in_service(l[j]);
    if (!full)
#pragma unroll
        for (uint32_t j = 0; j < NPL; ++j) l[j] = j < have ? l[j] : -INFINITY;
#pragma unroll
    for (int j = 0; j < NPL; ++j) top = fmaxf(top, l[j]);
    top = lanes_max<LANES>(top);
    const float base = top == -INFINITY ? 0.0f : top;
    float inverse = 0.0f;  // of the softmax's sum, where it is wanted
    float v[NPL];
    if (!a.sigmoid && (WORD == RouteWord::kValue || !a.renormalize)) {
        // (in pairs of neighbours, pairs of these, and so on: log2 of the experts' number roundings, where one after the other are as many as a lane has)
        float part[6];  // part[i]: 2^i of them
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            v[j] = exp_fast(l[j] - base);
            float sum = v[j];
            int i = 0;
#pragma unroll
            for (; j >> i & 1; ++i) sum = part[i] + sum;
            part[i] = sum;
        }
        const float total = lanes_sum<LANES>(part[__builtin_ctz(NPL)]);
        inverse = total > 0.0f ? __builtin_amdgcn_rcpf(total) : 0.0f;
    }
    auto score = [&](float v) { return a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + exp_fast(-v)) : exp_fast(v - base) * inverse; };

    // ---- the words
    uint32_t key[NPL], apart = 3;  // units that two choices have to be apart
    bool certain = true;
    if constexpr (WORD == RouteWord::kLogit16) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            const uint32_t e = first + j, as_is = bits[j] == 0x8000u ? 0u : bits[j], order = (as_is & 0x8000u ? ~as_is : as_is | 0x8000u) & 0xffffu;
            key[j] = j >= have ? 0u : (l[j] == -INFINITY ? 0u : order << 16) | (1024u - e);
        }
    } else {
        float most = -INFINITY, least = INFINITY;
        if (WORD == RouteWord::kValue && a.sigmoid)
#pragma unroll
            for (int j = 0; j < NPL; ++j) v[j] = score(l[j]);
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            if constexpr (WORD == RouteWord::kLogit) v[j] = l[j];
            if constexpr (WORD == RouteWord::kValue) {
                float value = fmaf(v[j], a.sigmoid ? 1.0f : inverse, in_service(b[j]));
                asm volatile("" : "+v"(value));  // (or the compiler branches round it, lane by lane)
                v[j] = l[j] == -INFINITY ? -INFINITY : value;
            }
            most = fmaxf(most, v[j]);
            if (WORD == RouteWord::kValue) least = fminf(least, v[j] == -INFINITY ? INFINITY : v[j]);
        }
        most = lanes_max<LANES>(most);
        float span = 32.0f;
        if constexpr (WORD == RouteWord::kValue) {
            // all the row's choices, or as far down as 2; a choice is off by the score's few last places and by half a one of its own
            span = fminf(fmaxf(most + lanes_max<LANES>(-least), 0x1p-10f), 2.0f);
            certain = most == -INFINITY || fabsf(most) <= 4.0f;  // (further off, an fp32 is too coarse)
            const float off = (a.sigmoid ? kSigmoidOff : inverse * softmax_off(a.levels)) + (fabsf(most) + span) * 0x1p-24f;
            apart = 3u + uint32_t(2.0f * off * (kUnits / span));
        }
        const float per_unit = kUnits / span, from = -(most - span) * per_unit;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            const uint32_t e = first + j;
            // 2: as far below the largest as the word reaches, or further
            const uint32_t q = v[j] == -INFINITY ? kOutWord : uint32_t(__builtin_amdgcn_fmed3f(fmaf(v[j], per_unit, from), 2.0f, 4194303.0f));
            key[j] = q << 10 | (1023u - e);
        }
        if (!full)
#pragma unroll
            for (int j = 0; j < NPL; ++j) key[j] = j < have ? key[j] : 0u;
    }
    // a ahead of b for certain, by the parts above their numbers
    auto ahead = [&](uint32_t a_, uint32_t b_, uint32_t by) { return WORD == RouteWord::kLogit16 || b_ <= kOutWord || a_ >= b_ + by; };

    // ---- groups
    if (a.groups > 1u) {
        const uint32_t lanes = 1u << a.group_shift;
        uint32_t best = 0, second = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            const uint32_t q = key[j] >> kIndexBits;
            second = max(second, min(best, q));
            best = max(best, q);
        }
        auto merge = [&](uint32_t o1, uint32_t o2) {
            second = max(max(second, o2), min(best, o1));
            best = max(best, o1);
        };
        if (lanes >= 2u) merge(dpp_keep_u32<0xB1>(best), dpp_keep_u32<0xB1>(second));
        if (lanes >= 4u) merge(dpp_keep_u32<0x4E>(best), dpp_keep_u32<0x4E>(second));
        if (lanes >= 8u) merge(dpp_keep_u32<0x141>(best), dpp_keep_u32<0x141>(second));
        if (lanes >= 16u) merge(dpp_keep_u32<0x140>(best), dpp_keep_u32<0x140>(second));
        if (lanes >= 32u) merge(__shfl_xor(best, 16), __shfl_xor(second, 16));
        // (the same in every lane, also of groups out of service and past the last: the row is certain in all of its lanes or in none)
        const uint32_t by = WORD != RouteWord::kLogit16 && a.group_top == 2u ? 2u * apart : apart;
        uint32_t mark = best;
        bool known = true;
        if (WORD != RouteWord::kLogit16 && a.group_top == 2u && best > kOutWord) {
            known = second > 2u && best > 2u;  // (what is missing counts 0, and what lies too low is not known: both by route_row)
            mark = best + second;
        }
        if (WORD != RouteWord::kLogit16) known &= best != 2u;
        const bool counts = group < a.groups;
        uint32_t word = counts ? (mark + 1u) << 6 | (63u - group) : 0u, last = 0;
        bool kept = false;
        for (uint32_t r = 0; r < a.kept; ++r) {
            last = lanes_max<LANES>(word);
            const bool mine = word == last;
            kept |= mine;
            word = mine ? 0u : word;
        }
        const uint32_t left = lanes_max<LANES>(word);
        certain &= ahead((last >> 6) - 1u, (left >> 6) - 1u, by);
        certain &= lanes_max<LANES>(counts && !known ? 1u : 0u) == 0u;
#pragma unroll
        for (int j = 0; j < NPL; ++j) key[j] = kept ? key[j] : 0u;
    }

    // ---- the top k
    uint32_t won[kSlots] = {};  // of rank sub, and sub + 16
    uint32_t before = 0;
    // the largest word below `taken` (0: of all): less `taken`, what lies below it wraps round above what does not, in its order
    auto largest_below = [&](uint32_t taken) {
        uint32_t best = key[0] - taken;
#pragma unroll
        for (int j = 1; j < NPL; ++j) best = max(best, key[j] - taken);
        return lanes_max<LANES>(best) + taken;
    };
    bool apart_all = true;
    for (uint32_t r = 0; r < a.top_k; ++r) {
        const uint32_t most = largest_below(before);
        if (r) apart_all &= ahead(before >> kIndexBits, most >> kIndexBits, apart);
        before = most;
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i) won[i] = sub + i * LANES == r ? most : won[i];
    }
    uint32_t place[kSlots];  // in the route
#pragma unroll
    for (uint32_t i = 0; i < kSlots; ++i) place[i] = sub + i * LANES;
    if constexpr (WORD != RouteWord::kLogit16) {
        // Where words lie too close together, those that come next are taken too, up to a gap, and 64 bits put all that were taken into order: their
        // scores alone, not the row's. (A softmax's sum stays the fp32 one: two choices whose difference it could turn, or hide, are left to route_row.)
        uint32_t left = largest_below(before), taken = a.top_k;
        auto gap = [&] { return left >= before || ahead(before >> kIndexBits, left >> kIndexBits, apart); };  // (not below: nothing is left)
        bool open = certain && !gap();
        const bool closer = certain && (open || !apart_all);
        if (__ballot(closer) != 0) {
            while (__ballot(open) != 0) {
                if (open && taken == 32u) {
                    certain = open = false;
                }
#pragma unroll
                for (uint32_t i = 0; i < kSlots; ++i) won[i] = open && sub + i * LANES == taken ? left : won[i];
                before = open ? left : before;
                taken += open ? 1u : 0u;
                left = largest_below(before);
                open &= !gap();
            }
            double *const values = s_value[wave] + lane / LANES * 64u, *const scores = values + 32;
            double mine[kSlots], my_score[kSlots];
            uint32_t number[kSlots];
#pragma unroll
            for (uint32_t i = 0; i < kSlots; ++i) {
                const uint32_t slot = sub + i * LANES;
                number[i] = min(1023u - (won[i] & 0x3ffu), a.experts - 1u);
                const float logit = in_service(route_load(a.logits, at + number[i], a.logits_type));
                my_score[i] = !a.bias || logit == -INFINITY ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-double(logit))) : exp(double(logit) - double(base)) * double(inverse);
                mine[i] = a.bias ? my_score[i] + double(in_service(route_load(a.bias, number[i], a.bias_type))) : double(logit);
                if ((won[i] >> kIndexBits) <= kOutWord) mine[i] = -INFINITY;
                if (slot < 32u) {
                    values[slot] = mine[i];
                    scores[slot] = my_score[i];
                }
            }
            __builtin_amdgcn_wave_barrier();
            uint32_t rank[kSlots] = {};
            bool known = true;
            for (uint32_t c = 0; c < 32u && __ballot(c < taken) != 0; ++c) {
                const double v = values[c], of = scores[c];
                const uint32_t e = 1023u - (__shfl(won[0], int(lane / LANES * LANES + c % LANES)) & 0x3ffu);
                const uint32_t e2 = kSlots == 2 ? 1023u - (__shfl(won[kSlots - 1], int(lane / LANES * LANES + c % LANES)) & 0x3ffu) : e;
                const uint32_t other = c < LANES ? e : e2;
                if (c < taken)
#pragma unroll
                    for (uint32_t i = 0; i < kSlots; ++i) {
                        rank[i] += v > mine[i] || (v == mine[i] && other < number[i]) ? 1u : 0u;
                        if (!a.sigmoid && a.bias && sub + i * LANES < taken && of != my_score[i] && v > -INFINITY && mine[i] > -INFINITY)
                            known &= fabs(v - mine[i]) > fabs(of - my_score[i]) * double(softmax_sum_off(a.levels));
                    }
            }
            __builtin_amdgcn_wave_barrier();
            if (closer) {
                certain &= lanes_max<LANES>(known ? 0u : 1u) == 0u;
#pragma unroll
                for (uint32_t i = 0; i < kSlots; ++i) place[i] = sub + i * LANES < taken ? rank[i] : ~0u;
            }
        }
    }

    // ---- the weights
    uint32_t index[kSlots];
    float w[kSlots], most = -INFINITY;
    bool served[kSlots];
#pragma unroll
    for (uint32_t i = 0; i < kSlots; ++i) {
        const bool on = place[i] < a.top_k;
        index[i] = on ? (WORD == RouteWord::kLogit16 ? 1024u - (won[i] & 0xffffu) : 1023u - (won[i] & 0x3ffu)) : 0u;
        served[i] = on && (won[i] >> kIndexBits) > kOutWord;
        w[i] = in_service(route_load(a.logits, at + min(index[i], a.experts - 1u), a.logits_type));
        most = fmaxf(most, served[i] ? w[i] : -INFINITY);
    }
    const bool among = a.renormalize && !a.sigmoid;  // the softmax of the chosen ones
    most = among ? lanes_max<LANES>(most) : 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kSlots; ++i) w[i] = !served[i] ? 0.0f : among ? exp_fast(w[i] - most) : score(w[i]);
    if (a.renormalize) {
        // (in the same order whatever the lanes: of neighbours, of pairs of these, and so on)
        float sum = lanes_sum<LANES>(w[0]);
        if constexpr (kSlots == 2) sum += lanes_sum<LANES>(w[1]);
        // (scores that fp32 does not hold well are 64 bits' again; none in service leaves zeros)
        if (a.sigmoid) certain &= sum > 1e-30f || lanes_max<LANES>(served[0] || served[kSlots - 1] ? 1u : 0u) == 0u;
        const float of_sum = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
        for (int i = 0; i < kSlots; ++i) w[i] *= of_sum;  // (first: the scaling over a small sum may leave fp32)
    }
#pragma unroll
    for (int i = 0; i < kSlots; ++i) w[i] *= a.scaling;
    if (real && certain)
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i)
            if (place[i] < a.top_k) {
                a.indices[row * a.top_k + place[i]] = index[i];
                route_store_weight(a, row * a.top_k + place[i], double(w[i]));
            }
    // ---- rows that are not certain, one by one by the whole wave
    for (uint64_t again = __ballot(real && !certain && sub == 0); again; again &= again - 1u)
        route_row<kWide>(a, uint32_t(first_row + __builtin_ctzll(again) / LANES), s_value[wave]);
}

template <int LANES, int NPL>
static void launch_route_fast(const RouteArgs &a, hipStream_t s) {
    const uint32_t per = 4u * (64u / LANES), blocks = uint32_t((uint64_t(a.rows) + per - 1u) / per);
    const bool by_value = a.bias || (a.groups > 1u && a.group_top == 2u);
    if (by_value) hipLaunchKernelGGL((k_route_rows_fast<LANES, NPL, RouteWord::kValue>), dim3(blocks), dim3(256), 0, s, a);
    else if (a.logits_type == SHRIKE_ELEM_F32) hipLaunchKernelGGL((k_route_rows_fast<LANES, NPL, RouteWord::kLogit>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_route_rows_fast<LANES, NPL, RouteWord::kLogit16>), dim3(blocks), dim3(256), 0, s, a);
}
// 16 lanes a row against 64: 2,048 rows of 512 11 us against 7.5, 8,192 16.6 against 15.8 (of 256 in groups 12.0 against 12.8, of 64 6.5 against 7.0),
// 16,384 22 against 27 (18 against 22, 7.7 against 10.8).
constexpr uint32_t kRowsForNarrow = 8192;
static uint32_t levels_of(uint32_t n) {
    uint32_t l = 0;
    while ((1u << l) < n) ++l;
    return l;
}
// How a row's experts lie in `lanes` lanes: 2^shift lanes a group (of one group: all), `each` experts a lane, also 2^i. each > 32: they do not.
struct RouteLanes {
    uint32_t shift = 0, each = 64;
};
static RouteLanes lanes_of(const RouteArgs &a, uint32_t lanes) {
    RouteLanes l;
    uint32_t groups = 1;
    while (groups < a.groups) groups *= 2u;
    if (groups > lanes) return l;
    while ((lanes / groups) >> (l.shift + 1u)) ++l.shift;
    l.each = 1;
    while ((l.each << l.shift) < a.group_size) l.each *= 2u;
    return l;
}

static void launch_route(RouteArgs a, hipStream_t s) {
    const RouteLanes narrow = lanes_of(a, 16), wide = lanes_of(a, 64);
    if (a.rows >= kRowsForNarrow && narrow.each <= 32u) {
        a.group_shift = narrow.shift;
        if (narrow.each == 1u) launch_route_fast<16, 1>(a, s);
        else if (narrow.each == 2u) launch_route_fast<16, 2>(a, s);
        else if (narrow.each == 4u) launch_route_fast<16, 4>(a, s);
        else if (narrow.each == 8u) launch_route_fast<16, 8>(a, s);
        else if (narrow.each == 16u) launch_route_fast<16, 16>(a, s);
        else launch_route_fast<16, 32>(a, s);
    } else if (wide.each <= 16u) {
        a.group_shift = wide.shift;
        if (wide.each == 1u) launch_route_fast<64, 1>(a, s);
        else if (wide.each == 2u) launch_route_fast<64, 2>(a, s);
        else if (wide.each == 4u) launch_route_fast<64, 4>(a, s);
        else if (wide.each == 8u) launch_route_fast<64, 8>(a, s);
        else launch_route_fast<64, 16>(a, s);
    } else {
        const dim3 blocks(std::min((a.rows - 1u) / 4u + 1u, 65536u)), threads(256);
        if (a.experts <= 64u) hipLaunchKernelGGL((k_route_rows<1>), blocks, threads, 0, s, a);
        else if (a.experts <= 128u) hipLaunchKernelGGL((k_route_rows<2>), blocks, threads, 0, s, a);
        else if (a.experts <= 256u) hipLaunchKernelGGL((k_route_rows<4>), blocks, threads, 0, s, a);
        else if (a.experts <= 512u) hipLaunchKernelGGL((k_route_rows<8>), blocks, threads, 0, s, a);
        else hipLaunchKernelGGL((k_route_rows<16>), blocks, threads, 0, s, a);
    }
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
    a.group_size = a.groups == 1u ? a.experts : size;
    a.levels = float(levels_of(a.groups) + levels_of(a.group_size));
    a.logits_type = logits_dtype;
    a.bias_type = bias_dtype;
    a.weights_type = weights_dtype;
    a.group_top = desc->group_top;
    a.sigmoid = desc->scores == SHRIKE_SCORES_SIGMOID;
    a.renormalize = desc->renormalize != 0;
    a.scaling = desc->scaling;
    const uint64_t size_of = logits_dtype == SHRIKE_ELEM_F32 ? 4u : 2u;
    a.whole = reinterpret_cast<uintptr_t>(d_logits) % 16u == 0 && (rows == 1u || logits_stride_elements * size_of % 16u == 0) && a.group_size * size_of % 16u == 0;
    a.whole_bias = d_bias && reinterpret_cast<uintptr_t>(d_bias) % 16u == 0 && a.group_size * (bias_dtype == SHRIKE_ELEM_F32 ? 4u : 2u) % 16u == 0;
    constexpr uint32_t kMostRows = 1u << 24;  // of a launch, which holds fewer than 2^32 threads
    for (uint32_t done = 0; done < rows; done += kMostRows) {
        RouteArgs part = a;
        part.rows = std::min(rows - done, kMostRows);
        part.logits = static_cast<const uint8_t *>(d_logits) + uint64_t(done) * logits_stride_elements * size_of;
        part.indices = d_out_indices + uint64_t(done) * a.top_k;
        part.weights = static_cast<uint8_t *>(d_out_weights) + uint64_t(done) * a.top_k * (weights_dtype == SHRIKE_ELEM_F32 ? 4u : 2u);
        launch_route(part, as_stream(stream));
        SHRIKE_HIP(hipGetLastError());
        if (rows - done <= kMostRows) break;
    }
    return 0;
}
