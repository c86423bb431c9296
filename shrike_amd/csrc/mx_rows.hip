// Rows into MX blocks and back, and the RMS norm that leaves its rows as such blocks: streaming kernels, bound by memory. A quad of
// lanes holds a block, eight elements a lane, so that a block's largest magnitude takes two lane exchanges, a lane's fp16 values are
// one 16-byte load and its codes one store.
#include "mx_common.h"
#include "rmsnorm_row.h"

namespace shrike {

template <int TYPE>
__device__ __forceinline__ float elem_to_f32(uint16_t b) {
    return TYPE == SHRIKE_ELEM_F16 ? f16_to_f32(b) : bf16_to_f32(b);
}

// Eight elements from `src`; WIDE: 16-byte loads (the row starts at a multiple of 16 bytes).
template <int TYPE, bool WIDE>
__device__ __forceinline__ void load_eight(const void *src, float (&v)[8]) {
    if constexpr (TYPE == SHRIKE_ELEM_F32) {
        const float *p = static_cast<const float *>(src);
        if constexpr (WIDE) {
            const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = p[i];
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(src);
        if constexpr (WIDE) {
            const uint4 a = *reinterpret_cast<const uint4 *>(p);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = elem_to_f32<TYPE>(uint16_t(w[i]));
                v[2 * i + 1] = elem_to_f32<TYPE>(uint16_t(w[i] >> 16));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = elem_to_f32<TYPE>(p[i]);
        }
    }
}

// 16 bits of an fp32 value, rounded to nearest even (NaN stays NaN).
template <int TYPE>
__device__ __forceinline__ uint16_t f32_to_elem(float v) {
    if constexpr (TYPE == SHRIKE_ELEM_F16) return f32_to_f16(v);
    const uint32_t u = __float_as_uint(v);
    return uint16_t(v != v ? 0x7fc0u : (u + 0x7fffu + (u >> 16 & 1u)) >> 16);
}

struct MxRowsArgs {
    const void *src;
    uint64_t src_stride;  // elements
    uint8_t *codes, *scales;
    void *dst;
    uint64_t dst_stride;  // elements
    uint64_t eighths;     // rows * d / 8
    uint32_t per_row;     // d / 8
};

// Codes and scales lie row behind row without a gap, so an eighth's index names them; only the source has a stride.
template <int TYPE, int FORMAT, bool WIDE>
__global__ __launch_bounds__(256) void k_mx_quantize(MxRowsArgs a) {
    for (uint64_t i = uint64_t(blockIdx.x) * 256u + threadIdx.x; i < a.eighths; i += uint64_t(gridDim.x) * 256u) {
        const uint64_t row = i / a.per_row, at = row * a.src_stride + (i - row * a.per_row) * 8u;
        float v[8];
        load_eight<TYPE, WIDE>(static_cast<const uint8_t *>(a.src) + at * (TYPE == SHRIKE_ELEM_F32 ? 4u : 2u), v);
        const MxEighths<FORMAT> q = mx_quantize_quad<FORMAT>(v);
        if constexpr (FORMAT == SHRIKE_MX_E4M3) reinterpret_cast<uint2 *>(a.codes)[i] = make_uint2(q.codes[0], q.codes[1]);
        else reinterpret_cast<uint32_t *>(a.codes)[i] = q.codes[0];
        if ((i & 3u) == 0) a.scales[i >> 2] = uint8_t(q.scale);
    }
}

template <int TYPE, int FORMAT, bool WIDE>
__global__ __launch_bounds__(256) void k_mx_dequantize(MxRowsArgs a) {
    for (uint64_t i = uint64_t(blockIdx.x) * 256u + threadIdx.x; i < a.eighths; i += uint64_t(gridDim.x) * 256u) {
        float v[8];
        if constexpr (FORMAT == SHRIKE_MX_E4M3) {
            const uint2 c = reinterpret_cast<const uint2 *>(a.codes)[i];
            const uint32_t w[2] = {c.x, c.y};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[j]), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[j]), true);
                v[4 * j] = lo[0]; v[4 * j + 1] = lo[1]; v[4 * j + 2] = hi[0]; v[4 * j + 3] = hi[1];
            }
        } else {
            const uint32_t w = reinterpret_cast<const uint32_t *>(a.codes)[i];
            const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
            const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
            v[0] = p0[0]; v[1] = p0[1]; v[2] = p1[0]; v[3] = p1[1]; v[4] = p2[0]; v[5] = p2[1]; v[6] = p3[0]; v[7] = p3[1];
        }
        const float scale = mx_scale(a.scales[i >> 2]);
        const uint64_t row = i / a.per_row, at = row * a.dst_stride + (i - row * a.per_row) * 8u;
        if constexpr (TYPE == SHRIKE_ELEM_F32) {
            float *to = static_cast<float *>(a.dst) + at;
            if constexpr (WIDE) {
                reinterpret_cast<float4 *>(to)[0] = make_float4(v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale);
                reinterpret_cast<float4 *>(to)[1] = make_float4(v[4] * scale, v[5] * scale, v[6] * scale, v[7] * scale);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) to[j] = v[j] * scale;
            }
        } else {
            uint16_t h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = f32_to_elem<TYPE>(__fmul_rn(v[j], scale));
            uint16_t *to = static_cast<uint16_t *>(a.dst) + at;
            if constexpr (WIDE) {
                *reinterpret_cast<uint4 *>(to) = make_uint4(h[0] | uint32_t(h[1]) << 16, h[2] | uint32_t(h[3]) << 16,
                                                            h[4] | uint32_t(h[5]) << 16, h[6] | uint32_t(h[7]) << 16);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) to[j] = h[j];
            }
        }
    }
}

struct MxNormArgs {
    const uint16_t *hidden, *delta, *weight;
    uint16_t *sum, *out;
    uint8_t *codes, *scales;
    uint32_t d, rows;
    float eps;
};

// The norm's arithmetic is rmsnorm_row_each's: `sum` and `out` are the bits of k_residual_add_rmsnorm, and the codes those of
// k_mx_quantize over `out`. A workgroup a row.
__global__ __launch_bounds__(256) void k_residual_add_rmsnorm_mx8(MxNormArgs a) {
    __shared__ float s_partial[4];
    const size_t row = size_t(blockIdx.x) * a.d;
    rmsnorm_row_each(a.hidden + row, a.delta ? a.delta + row : nullptr, a.delta ? a.sum + row : nullptr, a.weight, a.d, a.eps, s_partial,
                     [&](uint32_t c, uint4 o) {
                         if (a.out) reinterpret_cast<uint4 *>(a.out + row)[c] = o;
                         const uint32_t w[4] = {o.x, o.y, o.z, o.w};
                         float v[8];
#pragma unroll
                         for (int j = 0; j < 4; ++j) {
                             v[2 * j] = f16_to_f32(uint16_t(w[j]));
                             v[2 * j + 1] = f16_to_f32(uint16_t(w[j] >> 16));
                         }
                         const MxEighths<SHRIKE_MX_E4M3> q = mx_quantize_quad<SHRIKE_MX_E4M3>(v);
                         const size_t i = row / 8u + c;
                         reinterpret_cast<uint2 *>(a.codes)[i] = make_uint2(q.codes[0], q.codes[1]);
                         if ((c & 3u) == 0) a.scales[i >> 2] = uint8_t(q.scale);
                     });
}

// Workgroups of a streaming launch: enough to fill the device several times over, each walking on from there.
static uint32_t stream_workgroups(uint64_t eighths) { return uint32_t(std::min<uint64_t>((eighths + 255u) / 256u, 16384u)); }

template <int TYPE, int FORMAT>
static int launch_rows(bool quantize, bool wide, const MxRowsArgs &a, hipStream_t s) {
    const dim3 grid(stream_workgroups(a.eighths)), block(256);
    if (quantize) {
        if (wide) hipLaunchKernelGGL((k_mx_quantize<TYPE, FORMAT, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((k_mx_quantize<TYPE, FORMAT, false>), grid, block, 0, s, a);
    } else {
        if (wide) hipLaunchKernelGGL((k_mx_dequantize<TYPE, FORMAT, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((k_mx_dequantize<TYPE, FORMAT, false>), grid, block, 0, s, a);
    }
    SHRIKE_HIP(hipGetLastError());
    return 0;
}
template <int FORMAT>
static int launch_rows_type(bool quantize, bool wide, uint32_t dtype, const MxRowsArgs &a, hipStream_t s) {
    if (dtype == SHRIKE_ELEM_F32) return launch_rows<SHRIKE_ELEM_F32, FORMAT>(quantize, wide, a, s);
    if (dtype == SHRIKE_ELEM_F16) return launch_rows<SHRIKE_ELEM_F16, FORMAT>(quantize, wide, a, s);
    return launch_rows<SHRIKE_ELEM_BF16, FORMAT>(quantize, wide, a, s);
}

static int mx_rows(bool quantize, void *stream, const void *plain, uint32_t dtype, uint64_t stride, uint32_t format, const void *codes,
                   const void *scales, uint64_t rows, uint32_t d) {
    const char *what = quantize ? "mx quantize" : "mx dequantize";
    SHRIKE_REQUIRE(plain && codes && scales, "%s: NULL buffer", what);
    SHRIKE_REQUIRE(dtype <= SHRIKE_ELEM_F32, "%s: element type %u is not a known value", what, dtype);
    SHRIKE_REQUIRE(format <= SHRIKE_MX_E2M1, "%s: format %u is not a known value", what, format);
    SHRIKE_REQUIRE(d > 0 && d % kMxBlock == 0, "%s: d=%u must be a positive multiple of %u", what, d, kMxBlock);
    SHRIKE_REQUIRE(stride >= d, "%s: a stride of %llu elements is too small for rows of %u", what, (unsigned long long)stride, d);
    SHRIKE_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16u == 0, "%s: codes must be 16-byte aligned", what);
    const uint64_t size = dtype == SHRIKE_ELEM_F32 ? 4u : 2u;
    SHRIKE_REQUIRE(reinterpret_cast<uintptr_t>(plain) % size == 0, "%s: the elements are not aligned to their own size", what);
    SHRIKE_REQUIRE(rows <= (uint64_t(1) << 40) / d && stride <= (uint64_t(1) << 40) && (rows == 0 || stride <= (uint64_t(1) << 60) / rows),
                   "%s: %llu rows of %u elements, %llu apart, are too many", what, (unsigned long long)rows, d, (unsigned long long)stride);
    if (rows == 0) return 0;
    MxRowsArgs a = {};
    a.src = plain;
    a.dst = const_cast<void *>(plain);
    a.src_stride = a.dst_stride = stride;
    a.codes = static_cast<uint8_t *>(const_cast<void *>(codes));
    a.scales = static_cast<uint8_t *>(const_cast<void *>(scales));
    a.per_row = d / 8u;
    a.eighths = rows * a.per_row;
    const bool wide = reinterpret_cast<uintptr_t>(plain) % 16u == 0 && (rows == 1 || stride * size % 16u == 0);
    if (format == SHRIKE_MX_E4M3) return launch_rows_type<SHRIKE_MX_E4M3>(quantize, wide, dtype, a, as_stream(stream));
    return launch_rows_type<SHRIKE_MX_E2M1>(quantize, wide, dtype, a, as_stream(stream));
}

}  // namespace shrike

using namespace shrike;

extern "C" {

int shrike_hip_mx_quantize(void *stream, const void *d_src, uint32_t src_dtype, uint64_t src_stride_elements, uint32_t format,
                           void *d_codes, void *d_scales, uint64_t rows, uint32_t d) {
    return mx_rows(true, stream, d_src, src_dtype, src_stride_elements, format, d_codes, d_scales, rows, d);
}

int shrike_hip_mx_dequantize(void *stream, const void *d_codes, const void *d_scales, uint32_t format, void *d_out, uint32_t out_dtype,
                             uint64_t out_stride_elements, uint64_t rows, uint32_t d) {
    return mx_rows(false, stream, d_out, out_dtype, out_stride_elements, format, d_codes, d_scales, rows, d);
}

int shrike_hip_residual_add_rmsnorm_bf16w_mx8(void *stream, const void *d_hidden, const void *d_delta, const void *d_weight, void *d_sum,
                                              void *d_out, void *d_codes, void *d_scales, uint32_t d, float eps, uint32_t rows) {
    SHRIKE_REQUIRE(d_hidden && d_weight && d_codes && d_scales, "rmsnorm mx8: hidden, weight, codes and scales must be bound");
    SHRIKE_REQUIRE((d_delta == nullptr) == (d_sum == nullptr), "rmsnorm mx8: delta and sum must be bound together");
    SHRIKE_REQUIRE(d > 0 && d % kMxBlock == 0 && d <= SHRIKE_MAX_HIDDEN, "rmsnorm mx8: d=%u must be a multiple of %u up to %u", d, kMxBlock,
                   SHRIKE_MAX_HIDDEN);
    SHRIKE_REQUIRE(((reinterpret_cast<uintptr_t>(d_hidden) | reinterpret_cast<uintptr_t>(d_delta) | reinterpret_cast<uintptr_t>(d_weight)
                     | reinterpret_cast<uintptr_t>(d_sum) | reinterpret_cast<uintptr_t>(d_out) | reinterpret_cast<uintptr_t>(d_codes)) & 15u) == 0,
                   "rmsnorm mx8: buffers must be 16-byte aligned");
    SHRIKE_REQUIRE(rows <= kMaxNormRows, "rmsnorm mx8: %u rows are too many, %u at most", rows, kMaxNormRows);
    if (rows == 0) return 0;
    MxNormArgs a = {static_cast<const uint16_t *>(d_hidden), static_cast<const uint16_t *>(d_delta), static_cast<const uint16_t *>(d_weight),
                    static_cast<uint16_t *>(d_sum), static_cast<uint16_t *>(d_out), static_cast<uint8_t *>(d_codes),
                    static_cast<uint8_t *>(d_scales), d, rows, eps};
    hipLaunchKernelGGL(k_residual_add_rmsnorm_mx8, dim3(rows), dim3(256), 0, as_stream(stream), a);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
