// Products with 4-bit weights and a scale (and a bias) a group:
//
//   out[r, i] = sum_g scale[i, g] (sum_{k in g} x[r, k] code[i, k]) + sum_g bias[i, g] (sum_{k in g} x[r, k]) + bias[i]
//
// A wave takes an output of up to four rows; its lanes take eight k each, which never cross a group.
#include "gemv_common.h"

namespace shrike {

struct Affine4Args {
    const uint16_t *x;
    uint64_t x_stride;  // elements
    const uint8_t *codes;
    const uint16_t *scales, *biases, *bias;
    void *out;
    uint64_t out_stride;  // elements
    uint32_t rows, n, k, group, x_type, meta, out_type;
};

__device__ __forceinline__ float affine4_value(uint32_t h, uint32_t type) { return type == SHRIKE_ELEM_F16 ? f16_to_f32(uint16_t(h)) : bf16_to_f32(uint16_t(h)); }

__device__ __forceinline__ void affine4_store(const Affine4Args &a, uint32_t r, uint32_t i, float v) {
    const uint64_t at = uint64_t(r) * a.out_stride + i;
    if (a.out_type == SHRIKE_ELEM_F32) {
        static_cast<float *>(a.out)[at] = v;
    } else if (a.out_type == SHRIKE_ELEM_F16) {
        static_cast<uint16_t *>(a.out)[at] = f32_to_f16(v);
    } else {
        const uint32_t u = __float_as_uint(v);
        static_cast<uint16_t *>(a.out)[at] = uint16_t(v != v ? 0x7fc0u : (u + 0x7fffu + (u >> 16 & 1u)) >> 16);
    }
}

__global__ __launch_bounds__(256) void k_affine4_simple(Affine4Args a) {
    const uint32_t lane = threadIdx.x & 63u, i = blockIdx.x * 4u + wave_index(), r0 = blockIdx.y * 4u;
    if (i >= a.n) return;
    const uint32_t groups = a.k / a.group;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t k = 8u * lane; k < a.k; k += 512u) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(a.codes + (uint64_t(i) * a.k + k) / 2u);
        const uint64_t g = uint64_t(i) * groups + k / a.group;
        const float scale = affine4_value(a.scales[g], a.meta);
        const float bias = a.biases ? affine4_value(a.biases[g], a.meta) : -8.0f * scale;
        for (uint32_t r = 0; r < 4u && r0 + r < a.rows; ++r) {
            const uint4 v = *reinterpret_cast<const uint4 *>(a.x + uint64_t(r0 + r) * a.x_stride + k);
            const uint32_t words[4] = {v.x, v.y, v.z, v.w};
            float sum = 0.0f, all = 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                const float xv = affine4_value(words[j / 2u] >> 16u * (j % 2u) & 0xffffu, a.x_type);
                sum = fmaf(xv, float(w >> 4u * j & 15u), sum);
                all += xv;
            }
            acc[r] = fmaf(scale, sum, fmaf(bias, all, acc[r]));
        }
    }
    for (uint32_t r = 0; r < 4u && r0 + r < a.rows; ++r) {
        const float v = wave_sum(acc[r]);
        if (lane == 0) affine4_store(a, r0 + r, i, a.bias ? v + affine4_value(a.bias[i], a.meta) : v);
    }
}

}  // namespace shrike

using namespace shrike;

extern "C" int shrike_hip_affine4_product(void *stream, const void *d_x, uint32_t x_dtype, uint64_t x_stride_elements, const shrike_projection *w,
                                          uint32_t meta_dtype, uint32_t group_size, const void *d_bias, void *d_out, uint32_t out_dtype,
                                          uint64_t out_stride_elements, uint32_t rows, uint32_t n, uint32_t k) {
    SHRIKE_REQUIRE(d_x && w && w->weights && w->scales && d_out, "affine4 product: NULL buffer");
    SHRIKE_REQUIRE(x_dtype == SHRIKE_ELEM_F16 || x_dtype == SHRIKE_ELEM_BF16, "affine4 product: rows are fp16 or bf16, not type %u", x_dtype);
    SHRIKE_REQUIRE(meta_dtype <= SHRIKE_META_F16, "affine4 product: metadata type %u is not a known value", meta_dtype);
    SHRIKE_REQUIRE(out_dtype <= SHRIKE_ELEM_F32, "affine4 product: element type %u is not a known value", out_dtype);
    SHRIKE_REQUIRE(group_size == 32 || group_size == 64 || group_size == 128, "affine4 product: groups of %u are not 32, 64 or 128", group_size);
    SHRIKE_REQUIRE(k > 0 && k % group_size == 0 && k <= SHRIKE_AFFINE4_MAX_K, "affine4 product: k=%u must be a multiple of %u up to %u", k, group_size,
                   SHRIKE_AFFINE4_MAX_K);
    SHRIKE_REQUIRE(n > 0 && n <= 1u << 24, "affine4 product: n=%u not in 1...%u", n, 1u << 24);
    SHRIKE_REQUIRE(rows <= 1u << 22, "affine4 product: %u rows are too many", rows);
    SHRIKE_REQUIRE(x_stride_elements >= k && x_stride_elements % 8u == 0 && x_stride_elements <= uint64_t(1) << 36,
                   "affine4 product: a stride of %llu does not fit rows of %u, or is not a multiple of 8", (unsigned long long)x_stride_elements, k);
    SHRIKE_REQUIRE(out_stride_elements >= n && out_stride_elements <= uint64_t(1) << 36, "affine4 product: a stride of %llu does not fit %u outputs",
                   (unsigned long long)out_stride_elements, n);
    SHRIKE_REQUIRE((reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(w->weights)) % 16u == 0,
                   "affine4 product: rows and codes must be 16-byte aligned");
    SHRIKE_REQUIRE((reinterpret_cast<uintptr_t>(w->scales) | reinterpret_cast<uintptr_t>(w->biases) | reinterpret_cast<uintptr_t>(d_bias)) % 2u == 0
                       && reinterpret_cast<uintptr_t>(d_out) % (out_dtype == SHRIKE_ELEM_F32 ? 4u : 2u) == 0,
                   "affine4 product: scales, biases or out are not aligned to their elements' size");
    if (rows == 0) return 0;
    Affine4Args a = {};
    a.x = static_cast<const uint16_t *>(d_x);
    a.x_stride = x_stride_elements;
    a.codes = static_cast<const uint8_t *>(w->weights);
    a.scales = static_cast<const uint16_t *>(w->scales);
    a.biases = static_cast<const uint16_t *>(w->biases);
    a.bias = static_cast<const uint16_t *>(d_bias);
    a.out = d_out;
    a.out_stride = out_stride_elements;
    a.rows = rows;
    a.n = n;
    a.k = k;
    a.group = group_size;
    a.x_type = x_dtype;
    a.meta = meta_dtype;
    a.out_type = out_dtype;
    for (uint32_t first = 0; first < rows; first += 4u * 65535u) {  // (a grid's second dimension ends at 65,535)
        Affine4Args part = a;
        part.x += uint64_t(first) * a.x_stride;
        part.out = static_cast<uint8_t *>(a.out) + uint64_t(first) * a.out_stride * (out_dtype == SHRIKE_ELEM_F32 ? 4u : 2u);
        part.rows = std::min(rows - first, 4u * 65535u);
        hipLaunchKernelGGL(k_affine4_simple, dim3((n + 3u) / 4u, (part.rows + 3u) / 4u), dim3(256), 0, as_stream(stream), part);
        SHRIKE_HIP(hipGetLastError());
    }
    return 0;
}
