// Products over microscaled blocks on the scaled matrix instruction of gfx950, and the routed experts' gated FFN made of them.
//
//   out[r, n] = sum_k x[r, k] w[n, k],   x = E4M3 or E2M1 blocks, w = E2M1 blocks
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes the codes and the blocks' E8M0 scales as they lie in memory: in a step of 128 k lane l holds row
// l % 16 of its operand; of E2M1 codes the 16 bytes of block l / 16, of E4M3 codes the 16 bytes from k = 16 (l / 16) and those from
// k = 64 + 16 (l / 16); and the scale of block l / 16. Nothing is converted on the way. The weights are the first operand, so a lane's four
// sums are four neighbouring outputs n = 4 (l / 16) + 0..3 of row r = l % 16.
//
// What the instruction keeps of a sum (measured): E4M3 times E2M1 products are added in groups of eight neighbouring k, whose addends
// below 2^-13 of the group's largest are cut off, and the groups and the fp32 accumulator in a window of about 24 bits. E2M1 by E2M1 is
// exact there. With N(0, 1) rows that is 5e-6 of the result, with rows of outliers a hundred times the rest 6e-5: under the outputs'
// rounding to 16 bits (2^-11 and 2^-8 a half step), which is why no output is 32 bits wide. Sums over the steps are fp32 throughout.
//
// Two kernels. k_mx_few: up to 16 rows, everything straight from memory into the operands' registers, k split over the waves. k_mx_tile:
// 64 rows, staged through LDS by asynchronous loads and shared by four waves of 64 weight rows each.
#include "decode_launch.h"
#include "mx_common.h"
#include "prefill_common.h"

namespace shrike {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// where lanes past the end of a row load their codes: zeros
__device__ const uint32_t g_mx_zeros[4] = {0, 0, 0, 0};

// A row operand of a lane, for one step: two 16-byte pieces of E4M3 codes, one of E2M1.
template <int XF>
struct MxFragment {
    uint4 piece[XF == SHRIKE_MX_E4M3 ? 2 : 1];
};

template <int XF>
__device__ __forceinline__ f32x4 mx_multiply(u32x4 w, const MxFragment<XF> &x, f32x4 c, uint32_t w_scale, uint32_t x_scale) {
    const i32x8 a = {int(w[0]), int(w[1]), int(w[2]), int(w[3]), 0, 0, 0, 0};
    const uint4 p = x.piece[0];
    if constexpr (XF == SHRIKE_MX_E4M3) {
        const uint4 p2 = x.piece[1];
        const i32x8 b = {int(p.x), int(p.y), int(p.z), int(p.w), int(p2.x), int(p2.y), int(p2.z), int(p2.w)};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, int(w_scale), 0, int(x_scale));
    } else {
        const i32x8 b = {int(p.x), int(p.y), int(p.z), int(p.w), 0, 0, 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, 0, int(w_scale), 0, int(x_scale));
    }
}

__device__ __forceinline__ uint32_t max_xor16(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(r[0], r[1]);
}
__device__ __forceinline__ uint32_t max_xor32(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(r[0], r[1]);
}

// The activation of four neighbouring gate and up sums in each of two tiles: one MX block of 32 over the four lanes l, l ^ 16, l ^ 32,
// l ^ 48. The activation goes to eight bits from fp32, without a rounding to fp16 between. (fminf and fmaxf drop a NaN: it is put back.)
struct MxActBlock {
    uint32_t codes[2];  // of the lane's four values in either tile
    uint32_t scale;
};
__device__ __forceinline__ MxActBlock mx_activate(const f32x4 (&gate)[2], const f32x4 (&up)[2], uint32_t act_kind) {
    float v[8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float g = gate[i / 4][i % 4], u = up[i / 4][i % 4];
        v[i] = __builtin_isunordered(g, u) ? __uint_as_float(0x7fc00000u) : glu_rt_fast(g, u, act_kind);
        top = max(top, magnitude_bits(v[i]));
    }
    top = max_xor32(max_xor16(top));
    MxActBlock b;
    b.scale = mx_scale_byte<SHRIKE_MX_E4M3>(top);
    const float inverse = mx_inverse_scale(b.scale);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = b.scale == 255u ? 0.0f : __fmul_rn(v[i], inverse);
    b.codes[0] = mx_e4m3_x4(v[0], v[1], v[2], v[3]);
    b.codes[1] = mx_e4m3_x4(v[4], v[5], v[6], v[7]);
    return b;
}

// bf16 biases n..n+3 (nothing past `rows`), or zeros
typedef uint16_t u16x4_by2 __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ f32x4 mx_bias4(const uint16_t *bias, uint32_t n, uint32_t rows) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!bias) return v;
    if (n + 4u <= rows) {
        const u16x4_by2 b = *reinterpret_cast<const u16x4_by2 *>(bias + n);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = bf16_to_f32(b[i]);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (n + i < rows) v[i] = bf16_to_f32(bias[n + i]);
    }
    return v;
}

__device__ __forceinline__ uint16_t mx_out16(float v, uint32_t dtype) {
    if (dtype == SHRIKE_ELEM_F16) return f32_to_f16(v);
    const uint32_t u = __float_as_uint(v);
    return uint16_t(v != v ? 0x7fc0u : (u + 0x7fffu + (u >> 16 & 1u)) >> 16);
}
// four neighbouring outputs; `whole`: rows start at multiples of 8 bytes, so that four in a row are one store
__device__ __forceinline__ void mx_store4(uint16_t *row, uint32_t n, uint32_t outputs, f32x4 v, uint32_t dtype, bool whole) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = mx_out16(v[i], dtype);
    if (whole && n + 4u <= outputs) {
        *reinterpret_cast<uint2 *>(row + n) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (n + i < outputs) row[n + i] = uint16_t(h[i]);
    }
}

enum class MxWork { kDense, kGateUp, kDown };

struct MxArgs {
    const uint8_t *x, *x_scales;  // rows of k codes
    uint32_t rows, n, k;          // n outputs a row
    // dense
    const uint8_t *w, *w_scales;
    const uint16_t *bias;
    uint16_t *out;
    uint64_t out_stride;
    uint32_t out_dtype, out_whole;
    // routed: the experts' cells
    PoolArg pool;
    uint64_t stride;
    shrike_expert_offsets off;
    uint32_t ebias, act_kind, top_k;
    uint8_t *act, *act_scales;
    // ... of a chunk
    const shrike_row_tile *tiles;
    const uint32_t *tile_count;
    const shrike_token_expert_pair *pairs;
    // ... of single tokens
    const uint32_t *slots;
    const uint16_t *weights, *residual;
    uint16_t *y, *hidden;
};

// ------------------------------------------------------------------ few rows

// Loads from an address that the wave shares, a lane's 32-bit offset and one that moves with the loop. As buffer loads: from pointers the
// compiler makes a 64-bit address a load and lane of them, which are more registers than there are.
typedef __amdgpu_buffer_rsrc_t buffer_t;
__device__ __forceinline__ buffer_t buffer_of(const uint8_t *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p), 0, 0xffffffffu, 0x00020000);
}
__device__ __forceinline__ u32x4 load16(buffer_t b, uint32_t at, uint32_t moving) { return __builtin_amdgcn_raw_buffer_load_b128(b, at, moving, 0); }
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x2 load8(buffer_t b, uint32_t at, uint32_t moving) { return __builtin_amdgcn_raw_buffer_load_b64(b, at, moving, 0); }

// The weight rows of a wave: an address that the whole wave shares and, for each tile of 16, where a lane's row and its 16 bytes of a step
// lie from there.
template <int NT>
struct MxWeights {
    const uint8_t *codes[2], *scales[2];  // of the first and the second half of the tiles
    uint32_t at[NT], scale_at[NT];
};
template <int NT>
__device__ __forceinline__ void mx_weights(MxWeights<NT> &w, const uint8_t *codes, const uint8_t *scales, uint32_t n0, uint32_t n, uint32_t blocks) {
    const uint32_t lane = threadIdx.x & 63u, q = lane >> 4;
    const uint32_t first = min(n0, n - 1u);
    w.codes[0] = w.codes[1] = codes + size_t(first) * blocks * 16u;
    w.scales[0] = w.scales[1] = scales + size_t(first) * blocks;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const uint32_t r = min(n0 + 16u * i + (lane & 15u), n - 1u) - first;  // (rows past the last are the last again: nobody stores them)
        w.at[i] = r * blocks * 16u + 16u * q;
        w.scale_at[i] = r * blocks;
    }
}
// the same for as many gate as up rows from f0 on
template <int NT>
__device__ __forceinline__ void mx_gate_up_weights(MxWeights<NT> &w, const uint8_t *base, const shrike_expert_offsets &off, uint32_t f0, uint32_t f, uint32_t blocks) {
    MxWeights<NT / 2> half;
    mx_weights<NT / 2>(half, base + off.gate_w_off, base + off.gate_s_off, f0, f, blocks);
    const size_t first = min(f0, f - 1u);
    w.codes[0] = half.codes[0];
    w.scales[0] = half.scales[0];
    w.codes[1] = base + off.up_w_off + first * blocks * 16u;
    w.scales[1] = base + off.up_s_off + first * blocks;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        w.at[i] = half.at[i % (NT / 2)];
        w.scale_at[i] = half.scale_at[i % (NT / 2)];
    }
}

// Steps [from, to) of a wave's weight rows against MT tiles of rows of x, `blocks` blocks long. x_at, x_scale_at: where a lane's rows start.
template <int XF, int MT, int NT>
__device__ __forceinline__ void few_steps(f32x4 (&acc)[MT][NT], const MxWeights<NT> &w, const uint8_t *x, const uint8_t *xs, const uint32_t (&x_at)[MT],
                                          const uint32_t (&x_scale_at)[MT], uint32_t from, uint32_t to, uint32_t blocks) {
    const uint32_t q = (threadIdx.x & 63u) >> 4;
    constexpr uint32_t kStep = XF == SHRIKE_MX_E4M3 ? 128u : 64u;  // bytes of x
    struct Step {
        u32x4 w[NT];
        uint32_t ws[NT], xs[MT];
        MxFragment<XF> x[MT];
    };
    auto load = [&](Step &t, uint32_t s) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            t.w[i] = *reinterpret_cast<const u32x4 *>(w.codes[i * 2 / NT] + 64u * s + w.at[i]);
            t.ws[i] = (w.scales[i * 2 / NT] + 4u * s)[w.scale_at[i] + q];
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            t.x[j].piece[0] = *reinterpret_cast<const uint4 *>(x + kStep * s + (x_at[j] + 16u * q));
            if constexpr (XF == SHRIKE_MX_E4M3) t.x[j].piece[1] = *reinterpret_cast<const uint4 *>(x + kStep * s + 64u + (x_at[j] + 16u * q));
            t.xs[j] = (xs + 4u * s)[x_scale_at[j] + q];
        }
    };
    auto multiply = [&](const Step &t) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[j][i] = mx_multiply<XF>(t.w[i], t.x[j], acc[j][i], t.ws[i], t.xs[j]);
    };
    const uint32_t whole = min(to, blocks / 4u);
    uint32_t s = from;
    constexpr uint32_t kAhead = MT == 1 ? 4 : 2;
    for (; s + kAhead <= whole; s += kAhead) {
        Step t[kAhead];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) load(t[i], s + i);
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) multiply(t[i]);
    }
    for (; s < whole; ++s) {
        Step t;
        load(t, s);
        multiply(t);
    }
    if (s < to) {  // the last step of rows that end inside it: what lies past their blocks is zeros
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const bool mine = 4u * s + q < blocks;
        Step t;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            t.w[i] = u32x4{0, 0, 0, 0};
            t.ws[i] = 0;
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            t.x[j].piece[0] = zero;
            if constexpr (XF == SHRIKE_MX_E4M3) t.x[j].piece[1] = zero;
            t.xs[j] = 0;
        }
        if (mine) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                t.w[i] = *reinterpret_cast<const u32x4 *>(w.codes[i * 2 / NT] + 64u * s + w.at[i]);
                t.ws[i] = (w.scales[i * 2 / NT] + 4u * s)[w.scale_at[i] + q];
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) t.xs[j] = (xs + 4u * s)[x_scale_at[j] + q];
        }
        if (XF == SHRIKE_MX_E4M3 ? 4u * s + q / 2u < blocks : mine)
#pragma unroll
            for (int j = 0; j < MT; ++j) t.x[j].piece[0] = *reinterpret_cast<const uint4 *>(x + kStep * s + (x_at[j] + 16u * q));
        if constexpr (XF == SHRIKE_MX_E4M3)
            if (4u * s + 2u + q / 2u < blocks)
#pragma unroll
                for (int j = 0; j < MT; ++j) t.x[j].piece[1] = *reinterpret_cast<const uint4 *>(x + kStep * s + 64u + (x_at[j] + 16u * q));
        multiply(t);
    }
}

// A workgroup takes 16 MT rows of x against 16 NT weight rows (gate and up: NT / 2 tiles of each), its WAVES waves a part of k each; the
// partial sums meet in LDS. Routed work takes one row, which every column of the instruction then holds.
template <int XF, int MT, int NT, int WAVES, MxWork WORK>
__global__ __launch_bounds__(64 * WAVES) void k_mx_few(MxArgs a) {
    __shared__ f32x4 s_part[WAVES][MT * NT][64];
    const uint32_t wave = wave_index(), lane = threadIdx.x & 63u, m = lane & 15u, q = lane >> 4;
    const uint32_t blocks = a.k / kMxBlock, steps = (blocks + 3u) / 4u;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT * NT; ++i) acc[i / NT][i % NT] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint8_t *base = nullptr;
    uint32_t n0 = blockIdx.x * 16u * NT;
    MxWeights<NT> w;
    uint32_t x_at[MT], x_scale_at[MT];

    if constexpr (WORK == MxWork::kDense) {
        mx_weights<NT>(w, a.w, a.w_scales, n0, a.n, blocks);
        const uint32_t row0 = blockIdx.y * 16u * MT;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const uint32_t r = min(row0 + 16u * j + m, a.rows - 1u) - row0;
            x_at[j] = r * mx_code_bytes<XF>(a.k);
            x_scale_at[j] = r * blocks;
        }
        few_steps<XF, MT, NT>(acc, w, a.x + size_t(row0) * mx_code_bytes<XF>(a.k), a.x_scales + size_t(row0) * blocks, x_at, x_scale_at,
                              steps * wave / WAVES, steps * (wave + 1u) / WAVES, blocks);
    } else if constexpr (WORK == MxWork::kGateUp) {
        n0 = blockIdx.x * 8u * NT;
        const uint32_t cell = a.slots[blockIdx.y];
        if (cell == kSentinel) return;
        base = cell_base_uniform(a.pool, cell, a.stride);
        const size_t row = blockIdx.y / a.top_k;
        mx_gate_up_weights<NT>(w, base, a.off, n0, a.n, blocks);
        x_at[0] = x_scale_at[0] = 0;
        few_steps<XF, MT, NT>(acc, w, a.x + row * a.k, a.x_scales + row * blocks, x_at, x_scale_at, steps * wave / WAVES, steps * (wave + 1u) / WAVES, blocks);
    } else {
        // the positions' steps one behind the other, an equal part of them a wave; a position's sum is weighted when its steps end
        const uint32_t all = steps * a.top_k, to = all * (wave + 1u) / WAVES;
        uint32_t at = all * wave / WAVES;
        x_at[0] = x_scale_at[0] = 0;
        while (at < to) {
            const uint32_t position = at / steps, from = at - position * steps, until = min(steps, from + (to - at));
            at += until - from;
            const size_t pair = size_t(blockIdx.y) * a.top_k + position;
            const uint32_t cell = a.slots[pair];
            if (cell == kSentinel) continue;
            base = cell_base_uniform(a.pool, cell, a.stride);
            mx_weights<NT>(w, base + a.off.down_w_off, base + a.off.down_s_off, n0, a.n, blocks);
            f32x4 sum[1][NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) sum[0][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            few_steps<XF, 1, NT>(sum, w, a.x + pair * a.k, a.x_scales + pair * blocks, x_at, x_scale_at, from, until, blocks);
            const float weight = f16_to_f32(a.weights[pair]);
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[0][i] += weight * sum[0][i];
        }
    }
#pragma unroll
    for (int i = 0; i < MT * NT; ++i) s_part[wave][i][lane] = acc[i / NT][i % NT];
    __syncthreads();
    auto total = [&](uint32_t i) {
        f32x4 v = s_part[0][i][lane];
#pragma unroll
        for (int p = 1; p < WAVES; ++p) v += s_part[p][i][lane];
        return v;
    };

    if constexpr (WORK == MxWork::kGateUp) {
        constexpr uint32_t kBlocks = NT / 4;  // MX blocks of activations
        if (wave >= kBlocks) return;
        const uint32_t f0 = n0 + 32u * wave;
        f32x4 gate[2], up[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            gate[i] = total(2u * wave + i);
            up[i] = total(NT / 2 + 2u * wave + i);
            if (a.ebias) {
                gate[i] += mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.gate_ab_off), f0 + 16u * i + 4u * q, a.n);
                up[i] += mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.up_ab_off), f0 + 16u * i + 4u * q, a.n);
            }
        }
        const MxActBlock b = mx_activate(gate, up, a.act_kind);
        if (m == 0) {
            uint8_t *to = a.act + size_t(blockIdx.y) * a.n + f0 + 4u * q;
            *reinterpret_cast<uint32_t *>(to) = b.codes[0];
            *reinterpret_cast<uint32_t *>(to + 16) = b.codes[1];
            if (q == 0) a.act_scales[size_t(blockIdx.y) * (a.n / kMxBlock) + f0 / kMxBlock] = uint8_t(b.scale);
        }
    } else if constexpr (WORK == MxWork::kDense) {
        for (uint32_t i = wave; i < uint32_t(MT * NT); i += WAVES) {
            const uint32_t row = (blockIdx.y * MT + i / NT) * 16u + m, n = n0 + 16u * (i % NT) + 4u * q;
            const f32x4 v = total(i) + mx_bias4(a.bias, n, a.n);
            if (row < a.rows) mx_store4(a.out + row * a.out_stride, n, a.n, v, a.out_dtype, a.out_whole);
        }
    } else {
        if (wave >= uint32_t(NT)) return;
        const uint32_t n = n0 + 16u * wave + 4u * q;
        f32x4 v = total(wave);
        if (m != 0 || n >= a.n) return;  // (n and a.n are multiples of four)
        if (a.ebias)
            for (uint32_t p = 0; p < a.top_k; ++p) {
                const size_t pair = size_t(blockIdx.y) * a.top_k + p;
                const uint32_t cell = a.slots[pair];
                if (cell == kSentinel) continue;
                const uint8_t *at = cell_base(a.pool, cell, a.stride) + a.off.down_ab_off;
                v += f16_to_f32(a.weights[pair]) * mx_bias4(reinterpret_cast<const uint16_t *>(at), n, a.n);
            }
        const size_t at = size_t(blockIdx.y) * a.n + n;
        uint32_t out[4], sum[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float r = a.residual ? f16_to_f32(a.residual[at + i]) : 0.0f;
            out[i] = f32_to_f16(__fadd_rn(r, v[i]));
            if (a.hidden) sum[i] = f32_to_f16(__fadd_rn(f16_to_f32(a.hidden[at + i]), f16_to_f32(uint16_t(out[i]))));
        }
        *reinterpret_cast<uint2 *>(a.y + at) = make_uint2(out[0] | out[1] << 16, out[2] | out[3] << 16);
        if (a.hidden) *reinterpret_cast<uint2 *>(a.hidden + at) = make_uint2(sum[0] | sum[1] << 16, sum[2] | sum[3] << 16);
    }
}

// ------------------------------------------------------------------ tiles of rows

// A tile of up to 16 MT rows against four waves of NT tiles of 16 weight rows (gate and up: NT / 2 of each). A chunk of 256 k at a time:
// the rows by asynchronous loads into one of two places in LDS, 16-byte pieces swapped about within a row so that 16 rows' same piece
// lies in 64 different banks; the weights straight into registers, as no other wave wants them; all of it asked for while the chunk
// before is multiplied. What a row has behind its last whole chunk goes first, so that its wait is the first chunk's too.
template <int XF, int MT>
struct MxTileLds {
    static constexpr uint32_t kRows = 16u * MT;
    static constexpr uint32_t kRowBytes = XF == SHRIKE_MX_E4M3 ? 256u : 128u;  // of a chunk
    static constexpr uint32_t kPlace = kRows * kRowBytes, kScales = 2u * kPlace, kBytes = kScales + 2u * 256u * 8u;  // (every thread puts eight scale bytes down, its row's or the last one's: no branch)
};

template <int XF, int MT, int NT>
struct MxTile {
    using L = MxTileLds<XF, MT>;
    static constexpr uint32_t kPieces = L::kRowBytes / 16u;
    static constexpr uint32_t kLoads = L::kRows * kPieces / 256u;  // a thread
    static_assert(L::kRows * kPieces % 256u == 0);
    struct Chunk {
        u32x4 w[2][NT];
        u32x2 ws[NT];
    };
    f32x4 acc[MT][NT];

    // x, xs: where the rows that `row(r)` numbers start
    template <typename Row>
    __device__ __forceinline__ void run(uint8_t *lds, const MxWeights<NT> &w, const uint8_t *x, const uint8_t *xs, uint32_t blocks, Row row) {
        const uint32_t wave = wave_index(), lane = threadIdx.x & 63u, m = lane & 15u, q = lane >> 4;
        const uint32_t whole = blocks / 8u, left = blocks % 8u;
        const uint32_t place0 = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds));
        uint32_t x_at[kLoads];
        uint32_t x_piece = 0;  // (the same for all of a thread's loads: they lie a multiple of 16 rows apart)
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t at = (i * 4u + wave) * 64u + lane, r = at / kPieces;
            x_piece = 16u * (((at % kPieces) ^ (XF == SHRIKE_MX_E4M3 ? r : r >> 1)) % kPieces);
            x_at[i] = row(r) * (blocks * (XF == SHRIKE_MX_E4M3 ? 32u : 16u)) + x_piece;
        }
        const uint32_t xs_at = row(threadIdx.x) * blocks;
        u32x2 x_scales;
        const buffer_t codes[2] = {buffer_of(w.codes[0]), buffer_of(w.codes[1])}, scales[2] = {buffer_of(w.scales[0]), buffer_of(w.scales[1])};
        const buffer_t x_scales_from = buffer_of(xs);
        auto lds_of = [&](uint32_t place, uint32_t i) { return place0 + place * L::kPlace + (i * 4u + wave) * 1024u; };
        auto load = [&](uint32_t c, Chunk &to, uint32_t place) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) lds_load16(lds_of(place, i), x + c * L::kRowBytes, x_at[i]);
            x_scales = load8(x_scales_from, xs_at, 8u * c);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                to.w[0][i] = load16(codes[i * 2 / NT], w.at[i], 128u * c);
                to.w[1][i] = load16(codes[i * 2 / NT], w.at[i] + 64u, 128u * c);
                to.ws[i] = load8(scales[i * 2 / NT], w.scale_at[i], 8u * c);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        auto load_left = [&](Chunk &to, uint32_t place) {  // past the row: zeros
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const void *from = x + whole * L::kRowBytes + x_at[i];
                if (x_piece >= left * (L::kRowBytes / 8u)) from = g_mx_zeros;
                lds_load16(lds_of(place, i), from);
            }
            x_scales = u32x2{0, 0};
            for (uint32_t b = 0; b < left; ++b) x_scales[b / 4u] |= uint32_t((xs + 8u * whole)[xs_at + b]) << 8u * (b % 4u);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                to.ws[i] = u32x2{0, 0};
#pragma unroll
                for (uint32_t s = 0; s < 2; ++s) {
                    to.w[s][i] = u32x4{0, 0, 0, 0};
                    if (4u * s + q < left) {
                        to.w[s][i] = *reinterpret_cast<const u32x4 *>(w.codes[i * 2 / NT] + 128u * whole + 64u * s + w.at[i]);
                        to.ws[i][s] = uint32_t((w.scales[i * 2 / NT] + 8u * whole)[w.scale_at[i] + 4u * s + q]) << 8u * q;
                    }
                }
            }
        };
        auto landed = [&](uint32_t place) {
            __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0) in the compiler's own count: it need not wait for the next chunk's loads before it uses this one's
            reinterpret_cast<uint2 *>(lds + L::kScales)[place * 256u + threadIdx.x] = make_uint2(x_scales[0], x_scales[1]);
            wait_loads_and_sync<0>();
        };
        // 16 rows' 128 k at a time, those of the next on their way from LDS meanwhile: no more, or they would take the registers of all
        auto multiply = [&](const Chunk &now, uint32_t place) {
            const uint8_t *rows = lds + place * L::kPlace;
            const uint2 *scales = reinterpret_cast<const uint2 *>(lds + L::kScales) + place * 256u;
            struct Operand {
                MxFragment<XF> f;
                uint32_t scale;
            };
            auto fetch = [&](int k) {
                const uint32_t r = 16u * (k / 2) + m, s = k % 2;
                Operand o;
                if constexpr (XF == SHRIKE_MX_E4M3) {
                    o.f.piece[0] = *reinterpret_cast<const uint4 *>(rows + r * 256u + 16u * ((8u * s + q) ^ m));
                    o.f.piece[1] = *reinterpret_cast<const uint4 *>(rows + r * 256u + 16u * ((8u * s + 4u + q) ^ m));
                } else {
                    o.f.piece[0] = *reinterpret_cast<const uint4 *>(rows + r * 128u + 16u * ((4u * s + q) ^ (m >> 1)));
                }
                o.scale = reinterpret_cast<const uint8_t *>(scales + r)[4u * s + q];
                return o;
            };
#pragma unroll
            for (int k = 0; k < 2 * MT; ++k) {
                const Operand o = fetch(k);
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[k / 2][i] = mx_multiply<XF>(now.w[k % 2][i], o.f, acc[k / 2][i], now.ws[i][k % 2] >> 8u * q, o.scale);
            }
            // (the products stay in this block: they have no effect that would keep the compiler from moving them past the next wait)
#pragma unroll
            for (int i = 0; i < MT * NT; ++i) asm volatile("" : "+v"(acc[i / NT][i % NT]));
            constexpr int kReads = XF == SHRIKE_MX_E4M3 ? 3 : 2;
            __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);  // LDS reads
#pragma unroll
            for (int k = 0; k < 2 * MT; ++k) {
                if (k + 1 < 2 * MT) __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, NT, 0);  // matrix instructions
            }
        };
#pragma unroll
        for (int i = 0; i < MT * NT; ++i) acc[i / NT][i % NT] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        Chunk even, odd;
        if (left) {
            load_left(odd, 1);
            landed(1);
            if (whole) load(0, even, 0);
            multiply(odd, 1);
        } else {
            load(0, even, 0);
        }
        uint32_t c = 0;
        for (; c + 2u <= whole; c += 2u) {
            landed(0);
            load(c + 1u, odd, 1);
            multiply(even, 0);
            landed(1);
            if (c + 2u < whole) load(c + 2u, even, 0);
            multiply(odd, 1);
        }
        if (c < whole) {
            landed(0);
            multiply(even, 0);
        }
    }
};

template <int XF, int MT, int NT, MxWork WORK>
__device__ __forceinline__ void mx_tile(const MxArgs &a, uint8_t *lds, uint32_t number, uint32_t row0, uint32_t rows, uint32_t pair0, const uint8_t *base) {
    const uint32_t wave = wave_index(), m = threadIdx.x & 15u, q = (threadIdx.x & 63u) >> 4;
    const uint32_t blocks = a.k / kMxBlock, n0 = (number * 4u + wave) * (WORK == MxWork::kGateUp ? 8u : 16u) * NT;
    MxWeights<NT> w;
    if constexpr (WORK == MxWork::kDense) mx_weights<NT>(w, a.w, a.w_scales, n0, a.n, blocks);
    else if constexpr (WORK == MxWork::kGateUp) mx_gate_up_weights<NT>(w, base, a.off, n0, a.n, blocks);
    else mx_weights<NT>(w, base + a.off.down_w_off, base + a.off.down_s_off, n0, a.n, blocks);
    MxTile<XF, MT, NT> tile;
    // the rows past the tile's are its last one again; gate and up take a pair's token's row of the chunk
    if constexpr (WORK == MxWork::kGateUp)
        tile.run(lds, w, a.x, a.x_scales, blocks, [&](uint32_t r) -> uint32_t { return a.pairs[pair0 + min(r, rows - 1u)].token; });
    else
        tile.run(lds, w, a.x + size_t(row0) * mx_code_bytes<XF>(a.k), a.x_scales + size_t(row0) * blocks, blocks, [&](uint32_t r) { return min(r, rows - 1u); });

    if constexpr (WORK == MxWork::kGateUp) {
        if (n0 >= a.n) return;
#pragma unroll
        for (int b = 0; b < NT / 4; ++b) {
            const uint32_t f0 = n0 + 32u * b;
            if (f0 >= a.n) break;
            f32x4 bias[4] = {};
            if (a.ebias)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    bias[i] = mx_bias4(reinterpret_cast<const uint16_t *>(base + (i < 2u ? a.off.gate_ab_off : a.off.up_ab_off)), f0 + 16u * (i % 2u) + 4u * q, a.n);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const uint32_t r = 16u * t + m;
                const f32x4 gate[2] = {tile.acc[t][2 * b] + bias[0], tile.acc[t][2 * b + 1] + bias[1]};
                const f32x4 up[2] = {tile.acc[t][NT / 2 + 2 * b] + bias[2], tile.acc[t][NT / 2 + 2 * b + 1] + bias[3]};
                const MxActBlock q8 = mx_activate(gate, up, a.act_kind);
                if (r < rows) {
                    uint8_t *to = a.act + size_t(row0 + r) * a.n + f0 + 4u * q;
                    *reinterpret_cast<uint32_t *>(to) = q8.codes[0];
                    *reinterpret_cast<uint32_t *>(to + 16) = q8.codes[1];
                    if (q == 0) a.act_scales[size_t(row0 + r) * (a.n / kMxBlock) + f0 / kMxBlock] = uint8_t(q8.scale);
                }
            }
        }
    } else {
        f32x4 bias[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint16_t *from = a.bias;
            if constexpr (WORK == MxWork::kDown) from = a.ebias ? reinterpret_cast<const uint16_t *>(base + a.off.down_ab_off) : nullptr;
            bias[i] = mx_bias4(from, n0 + 16u * i + 4u * q, a.n);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const uint32_t r = 16u * t + m;
            if (r >= rows) continue;
            uint16_t *to;
            if constexpr (WORK == MxWork::kDense) {
                to = a.out + (row0 + r) * a.out_stride;
            } else {
                const shrike_token_expert_pair p = a.pairs[pair0 + r];
                to = a.out + (size_t(p.token) * a.top_k + p.rank) * a.n;
            }
#pragma unroll
            for (int i = 0; i < NT; ++i)
                mx_store4(to, n0 + 16u * i + 4u * q, a.n, tile.acc[t][i] + bias[i], WORK == MxWork::kDense ? a.out_dtype : uint32_t(SHRIKE_ELEM_F16),
                          WORK != MxWork::kDense || a.out_whole);
        }
    }
}

template <int XF, int MT, int NT>
__global__ __launch_bounds__(256, 2) void k_mx_product(MxArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[MxTileLds<XF, MT>::kBytes];
    const uint32_t row0 = blockIdx.y * 16u * MT;
    mx_tile<XF, MT, NT, MxWork::kDense>(a, lds, blockIdx.x, row0, min(16u * MT, a.rows - row0), 0, nullptr);
}

// A row tile of one expert; as few of its 16-row tiles as hold its rows are multiplied.
template <int NT, MxWork WORK>
__global__ __launch_bounds__(256, 2) void k_mx_expert_rows(MxArgs a) {
    constexpr int XF = SHRIKE_MX_E4M3;
    __shared__ __attribute__((aligned(16))) uint8_t lds[MxTileLds<XF, 4>::kBytes];
    if (blockIdx.y >= *a.tile_count) return;
    const shrike_row_tile tile = a.tiles[blockIdx.y];
    if (tile.cell == kSentinel || tile.rows == 0) return;
    const uint8_t *base = cell_base_uniform(a.pool, tile.cell, a.stride);
    const uint32_t rows = min(uint32_t(__builtin_amdgcn_readfirstlane(int(tile.rows))), kRowTile);
    const uint32_t pair0 = uint32_t(__builtin_amdgcn_readfirstlane(int(tile.pair_start))), row0 = blockIdx.y * kRowTile;
    if (rows > 32u) mx_tile<XF, 4, NT, WORK>(a, lds, blockIdx.x, row0, rows, pair0, base);
    else if (rows > 16u) mx_tile<XF, 2, NT, WORK>(a, lds, blockIdx.x, row0, rows, pair0, base);
    else mx_tile<XF, 1, NT, WORK>(a, lds, blockIdx.x, row0, rows, pair0, base);
}

template <int XF>
static int launch_product(const MxArgs &a, hipStream_t s) {
    if (a.rows <= 16u) {
        hipLaunchKernelGGL((k_mx_few<XF, 1, 2, 4, MxWork::kDense>), dim3((a.n + 31u) / 32u, 1), dim3(256), 0, s, a);
    } else if (a.rows <= 64u) {
        hipLaunchKernelGGL((k_mx_few<XF, 4, 2, 4, MxWork::kDense>), dim3((a.n + 31u) / 32u, 1), dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL((k_mx_product<XF, 4, 4>), dim3((a.n + 255u) / 256u, (a.rows + 63u) / 64u), dim3(256), 0, s, a);
    }
    SHRIKE_HIP(hipGetLastError());
    return 0;
}

static bool mx_aligned(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16u == 0; }

// An expert's blob in a cell: what the codes' 16-byte loads and the cell's size allow.
static int check_mx_offsets(const shrike_expert_offsets *o, uint64_t stride, uint32_t d, uint32_t f, bool biases) {
    const uint64_t codes = uint64_t(d) * f / 2u, scales = uint64_t(d) * f / kMxBlock;
    SHRIKE_REQUIRE(o->gate_w_off % 16u == 0 && o->up_w_off % 16u == 0 && o->down_w_off % 16u == 0, "mx experts: code offsets must be multiples of 16");
    SHRIKE_REQUIRE(o->gate_w_off + codes <= stride && o->up_w_off + codes <= stride && o->down_w_off + codes <= stride
                       && o->gate_s_off + scales <= stride && o->up_s_off + scales <= stride && o->down_s_off + scales <= stride,
                   "mx experts: a projection of %u x %u does not fit a cell of %llu bytes", d, f, (unsigned long long)stride);
    if (biases) {
        SHRIKE_REQUIRE(o->gate_ab_off % 2u == 0 && o->up_ab_off % 2u == 0 && o->down_ab_off % 2u == 0, "mx experts: bias offsets must be even");
        SHRIKE_REQUIRE(o->gate_ab_off + 2ull * f <= stride && o->up_ab_off + 2ull * f <= stride && o->down_ab_off + 2ull * d <= stride,
                       "mx experts: the biases do not fit a cell of %llu bytes", (unsigned long long)stride);
    }
    return 0;
}

static int check_mx_experts(const shrike_hip_moe *moe, const shrike_pool_bases *pool, uint64_t stride, const shrike_expert_offsets *offsets, uint32_t d,
                            uint32_t f, uint32_t top_k) {
    SHRIKE_REQUIRE(moe && pool && offsets, "mx experts: NULL argument");
    SHRIKE_REQUIRE(d == moe->desc.d && f == moe->desc.f, "mx experts: shape %ux%u differs from the handle's %ux%u", d, f, moe->desc.d, moe->desc.f);
    SHRIKE_REQUIRE(top_k >= 1 && top_k <= SHRIKE_MAX_TOP_K, "mx experts: topK=%u not in 1...%u", top_k, SHRIKE_MAX_TOP_K);
    SHRIKE_REQUIRE(pool->cells_per_chunk > 0 && stride % 16u == 0, "mx experts: bad pool geometry");
    for (const void *base : pool->base) SHRIKE_REQUIRE(mx_aligned(base), "mx experts: the pool's bases must be 16-byte aligned");
    return check_mx_offsets(offsets, stride, d, f, moe->desc.expert_additive_biases != 0);
}

static void fill_mx_experts(MxArgs &a, const shrike_hip_moe *moe, const shrike_pool_bases *pool, uint64_t stride, const shrike_expert_offsets *offsets) {
    fill_pool(a.pool, pool);
    a.stride = stride;
    a.off = *offsets;
    a.ebias = moe->desc.expert_additive_biases;
    a.act_kind = moe->desc.activation;
}

// The activations between the two launches: codes of `rows` rows, then their scales.
struct MxActs {
    size_t scales, total;
};
static MxActs mx_acts(uint64_t rows, uint32_t f) {
    const size_t codes = (size_t(rows) * f + 255u) & ~size_t(255);
    return {codes, codes + ((size_t(rows) * (f / kMxBlock) + 255u) & ~size_t(255))};
}

}  // namespace shrike

using namespace shrike;

extern "C" {

uint64_t shrike_mx_expert_offsets_make(uint32_t d, uint32_t f, int additive_biases, shrike_expert_offsets *out) {
    const uint64_t codes = uint64_t(d) * f / 2u, scales = uint64_t(d) * f / kMxBlock;
    if (!out || d == 0 || f == 0 || d % SHRIKE_GROUP_SIZE || f % SHRIKE_GROUP_SIZE || 3u * (codes + scales) + 4u * uint64_t(f) + 2u * uint64_t(d) > 0xffffffffull) {
        set_error("mx offsets: d=%u and f=%u must be positive multiples of %u, and the blob below 4 GiB", d, f, SHRIKE_GROUP_SIZE);
        return 0;
    }
    uint64_t at = 0;
    auto take = [&at](uint64_t size) { const uint64_t here = at; at += size; return uint32_t(here); };
    *out = shrike_expert_offsets{};
    out->gate_w_off = take(codes); out->gate_s_off = take(scales);
    out->up_w_off = take(codes); out->up_s_off = take(scales);
    out->down_w_off = take(codes); out->down_s_off = take(scales);
    if (additive_biases) {
        out->gate_ab_off = take(uint64_t(f) * 2u); out->up_ab_off = take(uint64_t(f) * 2u);
        out->down_ab_off = take(uint64_t(d) * 2u);
    }
    return at;
}

int shrike_hip_mx_product(void *stream, const void *d_x_codes, const void *d_x_scales, uint32_t x_format, const void *d_w_codes,
                          const void *d_w_scales, const void *d_bias, void *d_out, uint32_t out_dtype, uint64_t out_stride_elements,
                          uint32_t rows, uint32_t n, uint32_t k) {
    SHRIKE_REQUIRE(d_x_codes && d_x_scales && d_w_codes && d_w_scales && d_out, "mx product: NULL buffer");
    SHRIKE_REQUIRE(x_format <= SHRIKE_MX_E2M1, "mx product: format %u is not a known value", x_format);
    SHRIKE_REQUIRE(out_dtype == SHRIKE_ELEM_F16 || out_dtype == SHRIKE_ELEM_BF16, "mx product: outputs are fp16 or bf16, not type %u", out_dtype);
    SHRIKE_REQUIRE(k > 0 && k % kMxBlock == 0 && k <= SHRIKE_MX_MAX_K, "mx product: k=%u must be a multiple of %u up to %u", k, kMxBlock, SHRIKE_MX_MAX_K);
    SHRIKE_REQUIRE(n > 0 && n <= 1u << 24, "mx product: n=%u not in 1...%u", n, 1u << 24);
    SHRIKE_REQUIRE(rows <= 1u << 22, "mx product: %u rows is too many", rows);
    SHRIKE_REQUIRE(out_stride_elements >= n && out_stride_elements <= uint64_t(1) << 36, "mx product: a stride of %llu does not fit %u outputs",
                   (unsigned long long)out_stride_elements, n);
    SHRIKE_REQUIRE(mx_aligned(d_x_codes) && mx_aligned(d_w_codes), "mx product: codes must be 16-byte aligned");
    SHRIKE_REQUIRE((reinterpret_cast<uintptr_t>(d_out) | reinterpret_cast<uintptr_t>(d_bias)) % 2u == 0, "mx product: out and bias must be 2-byte aligned");
    if (rows == 0) return 0;
    MxArgs a = {};
    a.x = static_cast<const uint8_t *>(d_x_codes);
    a.x_scales = static_cast<const uint8_t *>(d_x_scales);
    a.rows = rows; a.n = n; a.k = k;
    a.w = static_cast<const uint8_t *>(d_w_codes);
    a.w_scales = static_cast<const uint8_t *>(d_w_scales);
    a.bias = static_cast<const uint16_t *>(d_bias);
    a.out = static_cast<uint16_t *>(d_out);
    a.out_stride = out_stride_elements;
    a.out_dtype = out_dtype;
    a.out_whole = reinterpret_cast<uintptr_t>(d_out) % 8u == 0 && (rows == 1u || out_stride_elements % 4u == 0);
    return x_format == SHRIKE_MX_E4M3 ? launch_product<SHRIKE_MX_E4M3>(a, as_stream(stream)) : launch_product<SHRIKE_MX_E2M1>(a, as_stream(stream));
}

size_t shrike_hip_mx_ffn_workspace_bytes(uint32_t max_row_tiles, uint32_t f) { return mx_acts(uint64_t(max_row_tiles) * kRowTile, f).total; }

int shrike_hip_mx_grouped_ffn(shrike_hip_moe *moe, void *stream, const shrike_pool_bases *pool, uint64_t pool_slot_stride,
                              const shrike_expert_offsets *offsets, const shrike_hip_grouped_routes *routes, uint32_t max_row_tiles,
                              const void *d_x_codes, const void *d_x_scales, void *d_route_partials, void *d_workspace, size_t workspace_bytes,
                              uint32_t query_count, uint32_t d, uint32_t f, uint32_t top_k) {
    if (int rc = check_mx_experts(moe, pool, pool_slot_stride, offsets, d, f, top_k)) return rc;
    SHRIKE_REQUIRE(routes && routes->sorted_pairs && routes->row_tiles && routes->row_tile_count, "mx grouped FFN: routes are not bound");
    SHRIKE_REQUIRE(d_x_codes && d_x_scales && d_route_partials && d_workspace, "mx grouped FFN: NULL buffer");
    SHRIKE_REQUIRE(mx_aligned(d_x_codes) && mx_aligned(d_route_partials), "mx grouped FFN: codes and partials must be 16-byte aligned");
    SHRIKE_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 256u == 0, "mx grouped FFN: workspace must be 256-byte aligned");
    SHRIKE_REQUIRE(uint64_t(query_count) * d <= 0xffffffffull, "mx grouped FFN: %u rows of %u are more than 4 GiB of codes", query_count, d);
    if (query_count == 0 || max_row_tiles == 0) return 0;
    // (an expert's last tile may be partly filled: more tiles than this there cannot be)
    const uint32_t tiles = readable_records(max_row_tiles, uint64_t(query_count) * top_k, moe->desc.num_experts);
    SHRIKE_REQUIRE(tiles <= 65535u, "mx grouped FFN: %u row tiles are too many", tiles);
    const MxActs acts = mx_acts(uint64_t(max_row_tiles) * kRowTile, f);
    SHRIKE_REQUIRE(workspace_bytes >= acts.total, "mx grouped FFN: workspace of %zu bytes, %zu needed", workspace_bytes, acts.total);
    MxArgs a = {};
    fill_mx_experts(a, moe, pool, pool_slot_stride, offsets);
    a.x = static_cast<const uint8_t *>(d_x_codes);
    a.x_scales = static_cast<const uint8_t *>(d_x_scales);
    a.rows = query_count; a.n = f; a.k = d; a.top_k = top_k;
    a.act = static_cast<uint8_t *>(d_workspace);
    a.act_scales = a.act + acts.scales;
    a.tiles = routes->row_tiles;
    a.tile_count = routes->row_tile_count;
    a.pairs = static_cast<const shrike_token_expert_pair *>(routes->sorted_pairs);
    hipStream_t s = as_stream(stream);
    hipLaunchKernelGGL((k_mx_expert_rows<4, MxWork::kGateUp>), dim3((f + 127u) / 128u, tiles), dim3(256), 0, s, a);
    SHRIKE_HIP(hipGetLastError());
    a.x = a.act;
    a.x_scales = a.act_scales;
    a.n = d; a.k = f;
    a.out = static_cast<uint16_t *>(d_route_partials);
    hipLaunchKernelGGL((k_mx_expert_rows<4, MxWork::kDown>), dim3((d + 255u) / 256u, tiles), dim3(256), 0, s, a);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}

size_t shrike_hip_mx_decode_workspace_bytes(uint32_t tokens, uint32_t top_k, uint32_t f) { return mx_acts(uint64_t(tokens) * top_k, f).total; }

int shrike_hip_mx_decode_ffn(shrike_hip_moe *moe, void *stream, const shrike_pool_bases *pool, uint64_t pool_slot_stride,
                             const uint32_t *d_resolved_slots, const shrike_expert_offsets *offsets, const void *d_x_codes,
                             const void *d_x_scales, const void *d_routing_weights, const void *d_residual, void *d_y, void *d_hidden,
                             void *d_workspace, size_t workspace_bytes, uint32_t d, uint32_t f, uint32_t top_k, uint32_t tokens) {
    if (int rc = check_mx_experts(moe, pool, pool_slot_stride, offsets, d, f, top_k)) return rc;
    SHRIKE_REQUIRE(d_resolved_slots && d_x_codes && d_x_scales && d_routing_weights && d_y && d_workspace, "mx decode FFN: NULL buffer");
    SHRIKE_REQUIRE(mx_aligned(d_x_codes) && mx_aligned(d_y) && mx_aligned(d_hidden), "mx decode FFN: codes, y and hidden must be 16-byte aligned");
    SHRIKE_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 256u == 0, "mx decode FFN: workspace must be 256-byte aligned");
    SHRIKE_REQUIRE(tokens <= 65535u / SHRIKE_MAX_TOP_K, "mx decode FFN: %u tokens are too many", tokens);
    const MxActs acts = mx_acts(uint64_t(tokens) * top_k, f);
    SHRIKE_REQUIRE(workspace_bytes >= acts.total, "mx decode FFN: workspace of %zu bytes, %zu needed", workspace_bytes, acts.total);
    if (tokens == 0) return 0;
    MxArgs a = {};
    fill_mx_experts(a, moe, pool, pool_slot_stride, offsets);
    a.x = static_cast<const uint8_t *>(d_x_codes);
    a.x_scales = static_cast<const uint8_t *>(d_x_scales);
    a.rows = tokens; a.n = f; a.k = d; a.top_k = top_k;
    a.act = static_cast<uint8_t *>(d_workspace);
    a.act_scales = a.act + acts.scales;
    a.slots = d_resolved_slots;
    a.weights = static_cast<const uint16_t *>(d_routing_weights);
    a.residual = static_cast<const uint16_t *>(d_residual);
    a.y = static_cast<uint16_t *>(d_y);
    a.hidden = static_cast<uint16_t *>(d_hidden);
    hipStream_t s = as_stream(stream);
    hipLaunchKernelGGL((k_mx_few<SHRIKE_MX_E4M3, 1, 4, 4, MxWork::kGateUp>), dim3(f / 32u, tokens * top_k), dim3(256), 0, s, a);
    SHRIKE_HIP(hipGetLastError());
    a.x = a.act;
    a.x_scales = a.act_scales;
    a.n = d; a.k = f;
    hipLaunchKernelGGL((k_mx_few<SHRIKE_MX_E4M3, 1, 2, 4, MxWork::kDown>), dim3(d / 32u, tokens), dim3(256), 0, s, a);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
