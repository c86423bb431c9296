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

// where lanes past the end of a row load their codes and scales: zero codes under a scale that is no NaN
__device__ const uint32_t g_mx_zeros[4] = {0, 0, 0, 0};

// A row operand of a lane, for one step: two 16-byte pieces of E4M3 codes, one of E2M1.
template <int XF>
struct MxFragment {
    uint4 piece[XF == SHRIKE_MX_E4M3 ? 2 : 1];
};

template <int XF>
__device__ __forceinline__ f32x4 mx_multiply(uint4 w, const MxFragment<XF> &x, f32x4 c, uint32_t w_scale, uint32_t x_scale) {
    const i32x8 a = {int(w.x), int(w.y), int(w.z), int(w.w), 0, 0, 0, 0};
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
__device__ __forceinline__ f32x4 mx_bias4(const uint16_t *bias, uint32_t n, uint32_t rows) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (bias)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (n + i < rows) v[i] = bf16_to_f32(bias[n + i]);
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

// Steps [from, to) of a lane's row of each weight tile against its row of x, `blocks` blocks long.
template <int XF, int NT>
__device__ __forceinline__ void few_steps(f32x4 (&acc)[NT], const uint8_t *const (&w)[NT], const uint8_t *const (&ws)[NT], const uint8_t *x,
                                          const uint8_t *xs, uint32_t from, uint32_t to, uint32_t blocks) {
    const uint32_t q = (threadIdx.x & 63u) >> 4;
    constexpr uint32_t kStep = XF == SHRIKE_MX_E4M3 ? 128u : 64u;  // bytes of x
    struct Step {
        uint4 w[NT];
        uint32_t ws[NT], xs;
        MxFragment<XF> x;
    };
    auto load = [&](Step &t, uint32_t s) {
        const uint32_t b = 4u * s + q;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            t.w[i] = *reinterpret_cast<const uint4 *>(w[i] + 16u * b);
            t.ws[i] = ws[i][b];
        }
        t.x.piece[0] = *reinterpret_cast<const uint4 *>(x + kStep * s + 16u * q);
        if constexpr (XF == SHRIKE_MX_E4M3) t.x.piece[1] = *reinterpret_cast<const uint4 *>(x + kStep * s + 64u + 16u * q);
        t.xs = xs[b];
    };
    auto multiply = [&](const Step &t) {
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] = mx_multiply<XF>(t.w[i], t.x, acc[i], t.ws[i], t.xs);
    };
    const uint32_t whole = min(to, blocks / 4u);
    uint32_t s = from;
    constexpr uint32_t kAhead = 4;
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
    if (s < to) {  // the last step of a row that ends inside it: what lies past its blocks is zeros
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const uint32_t b = 4u * s + q;
        Step t;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            t.w[i] = zero;
            t.ws[i] = 0;
            if (b < blocks) {
                t.w[i] = *reinterpret_cast<const uint4 *>(w[i] + 16u * b);
                t.ws[i] = ws[i][b];
            }
        }
        t.xs = b < blocks ? xs[b] : 0u;
        if constexpr (XF == SHRIKE_MX_E4M3) {
            t.x.piece[0] = t.x.piece[1] = zero;
            if (4u * s + q / 2u < blocks) t.x.piece[0] = *reinterpret_cast<const uint4 *>(x + kStep * s + 16u * q);
            if (4u * s + 2u + q / 2u < blocks) t.x.piece[1] = *reinterpret_cast<const uint4 *>(x + kStep * s + 64u + 16u * q);
        } else {
            t.x.piece[0] = zero;
            if (b < blocks) t.x.piece[0] = *reinterpret_cast<const uint4 *>(x + kStep * s + 16u * q);
        }
        multiply(t);
    }
}

// A workgroup takes 16 rows of x against 16 NT weight rows (gate and up: NT / 2 tiles of each), its four waves a part of k each; the
// partial sums meet in LDS. Routed work takes one row, which every column of the instruction then holds.
template <int XF, int NT, MxWork WORK>
__global__ __launch_bounds__(256) void k_mx_few(MxArgs a) {
    __shared__ f32x4 s_part[4][NT][64];
    const uint32_t wave = wave_index(), lane = threadIdx.x & 63u, m = lane & 15u, q = lane >> 4;
    const uint32_t blocks = a.k / kMxBlock, steps = (blocks + 3u) / 4u;
    const uint32_t row_codes = a.k / 2u;
    f32x4 acc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint8_t *w[NT], *ws[NT], *base = nullptr;
    uint32_t n0 = blockIdx.x * 16u * NT;

    if constexpr (WORK == MxWork::kDense) {
        const uint32_t row = min(blockIdx.y * 16u + m, a.rows - 1u);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const size_t r = min(n0 + 16u * i + m, a.n - 1u);
            w[i] = a.w + r * row_codes;
            ws[i] = a.w_scales + r * blocks;
        }
        few_steps<XF, NT>(acc, w, ws, a.x + size_t(row) * mx_code_bytes<XF>(a.k), a.x_scales + size_t(row) * blocks, steps * wave / 4u,
                          steps * (wave + 1u) / 4u, blocks);
    } else if constexpr (WORK == MxWork::kGateUp) {
        n0 = blockIdx.x * 8u * NT;
        const uint32_t cell = a.slots[blockIdx.y];
        if (cell == kSentinel) return;
        base = cell_base_uniform(a.pool, cell, a.stride);
        const size_t row = blockIdx.y / a.top_k;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const bool up = i >= NT / 2;
            const size_t r = n0 + 16u * (i % (NT / 2)) + m;
            w[i] = base + (up ? a.off.up_w_off : a.off.gate_w_off) + r * row_codes;
            ws[i] = base + (up ? a.off.up_s_off : a.off.gate_s_off) + r * blocks;
        }
        few_steps<XF, NT>(acc, w, ws, a.x + row * a.k, a.x_scales + row * blocks, steps * wave / 4u, steps * (wave + 1u) / 4u, blocks);
    } else {
        // the positions' steps one behind the other, a quarter of them a wave; a position's sum is weighted when its steps end
        const uint32_t all = steps * a.top_k, to = all * (wave + 1u) / 4u;
        uint32_t at = all * wave / 4u;
        while (at < to) {
            const uint32_t position = at / steps, from = at - position * steps, until = min(steps, from + (to - at));
            at += until - from;
            const size_t pair = size_t(blockIdx.y) * a.top_k + position;
            const uint32_t cell = a.slots[pair];
            if (cell == kSentinel) continue;
            base = cell_base_uniform(a.pool, cell, a.stride);
            f32x4 sum[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const size_t r = min(n0 + 16u * i + m, a.n - 1u);
                w[i] = base + a.off.down_w_off + r * row_codes;
                ws[i] = base + a.off.down_s_off + r * blocks;
                sum[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            few_steps<XF, NT>(sum, w, ws, a.x + pair * a.k, a.x_scales + pair * blocks, from, until, blocks);
            const float weight = f16_to_f32(a.weights[pair]);
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[i] += weight * sum[i];
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) s_part[wave][i][lane] = acc[i];
    __syncthreads();
    auto total = [&](int i) { return (s_part[0][i][lane] + s_part[1][i][lane]) + (s_part[2][i][lane] + s_part[3][i][lane]); };

    if constexpr (WORK == MxWork::kGateUp) {
        constexpr int kBlocks = NT / 4;  // MX blocks of activations
        if (wave >= uint32_t(kBlocks)) return;
        const uint32_t f0 = n0 + 32u * wave;
        f32x4 gate[2], up[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            gate[i] = total(2 * wave + i);
            up[i] = total(NT / 2 + 2 * wave + i);
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
        return;
    } else {
        if (wave >= uint32_t(NT)) return;
        const uint32_t n = n0 + 16u * wave + 4u * q;
        f32x4 v = total(wave);
        if constexpr (WORK == MxWork::kDense) {
            const uint32_t row = blockIdx.y * 16u + m;
            v += mx_bias4(a.bias, n, a.n);
            if (row < a.rows) mx_store4(a.out + row * a.out_stride, n, a.n, v, a.out_dtype, a.out_whole);
        } else {
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
}

// ------------------------------------------------------------------ tiles of rows

// MT tiles of 16 rows against four waves of NT tiles of 16 weight rows. A chunk of 256 k at a time: the rows by asynchronous loads into
// one of two places in LDS, 16-byte pieces swapped about within a row so that 16 rows' same piece lies in 64 different banks; the
// weights straight into registers, as no other wave wants them; all of it asked for while the chunk before is multiplied.
template <int XF, int MT, int NT, MxWork WORK>
__global__ __launch_bounds__(256, 2) void k_mx_tile(MxArgs a) {
    constexpr uint32_t kRows = 16u * MT;
    constexpr uint32_t kRowBytes = XF == SHRIKE_MX_E4M3 ? 256u : 128u;  // of a chunk
    constexpr uint32_t kPieces = kRowBytes / 16u;
    constexpr uint32_t kLoads = kRows * kPieces / 256u;  // a thread
    static_assert(kRows * kPieces % 256u == 0 && kRows <= 256u);
    __shared__ __attribute__((aligned(16))) uint8_t s_x[2][kRows * kRowBytes];
    __shared__ uint2 s_scales[2][kRows];
    const uint32_t wave = wave_index(), lane = threadIdx.x & 63u, m = lane & 15u, q = lane >> 4;
    const uint32_t blocks = a.k / kMxBlock, chunks = (blocks + 7u) / 8u, whole_chunks = blocks / 8u;
    const uint32_t x_bytes = mx_code_bytes<XF>(a.k);

    uint32_t row0, rows, pair0 = 0, n0;
    const uint8_t *base = nullptr;
    if constexpr (WORK == MxWork::kDense) {
        row0 = blockIdx.y * kRows;
        rows = min(kRows, a.rows - row0);
        n0 = (blockIdx.x * 4u + wave) * 16u * NT;
    } else {
        if (blockIdx.y >= *a.tile_count) return;
        const shrike_row_tile tile = a.tiles[blockIdx.y];
        if (tile.cell == kSentinel) return;
        base = cell_base_uniform(a.pool, tile.cell, a.stride);
        row0 = blockIdx.y * kRowTile;  // of the activations
        rows = min(uint32_t(__builtin_amdgcn_readfirstlane(int(tile.rows))), kRows);
        if (rows == 0) return;
        pair0 = uint32_t(__builtin_amdgcn_readfirstlane(int(tile.pair_start)));
        n0 = (blockIdx.x * 4u + wave) * (WORK == MxWork::kGateUp ? 8u : 16u) * NT;
    }
    auto x_row = [&](uint32_t r) -> size_t {  // the row of x that is row r of the tile
        r = min(r, rows - 1u);
        if constexpr (WORK == MxWork::kGateUp) return a.pairs[pair0 + r].token;
        return row0 + r;
    };
    const uint8_t *x[kLoads];
    uint32_t x_piece[kLoads];
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
        const uint32_t at = (i * 4u + wave) * 64u + lane, r = at / kPieces;
        x_piece[i] = ((at % kPieces) ^ (XF == SHRIKE_MX_E4M3 ? r : r >> 1)) % kPieces;
        x[i] = a.x + x_row(r) * x_bytes + 16u * x_piece[i];
    }
    const uint8_t *xs = a.x_scales + x_row(threadIdx.x) * blocks;  // (threads past the rows load the last one's)
    const uint8_t *w[NT], *ws[NT];
    const size_t row_codes = a.k / 2u;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        if constexpr (WORK == MxWork::kDense) {
            const size_t r = min(n0 + 16u * i + m, a.n - 1u);
            w[i] = a.w + r * row_codes;
            ws[i] = a.w_scales + r * blocks;
        } else if constexpr (WORK == MxWork::kGateUp) {
            const bool up = i >= NT / 2;
            const size_t r = min(n0 + 16u * (i % (NT / 2)) + m, a.n - 1u);
            w[i] = base + (up ? a.off.up_w_off : a.off.gate_w_off) + r * row_codes;
            ws[i] = base + (up ? a.off.up_s_off : a.off.gate_s_off) + r * blocks;
        } else {
            const size_t r = min(n0 + 16u * i + m, a.n - 1u);
            w[i] = base + a.off.down_w_off + r * row_codes;
            ws[i] = base + a.off.down_s_off + r * blocks;
        }
        w[i] += 16u * q;
    }

    struct Chunk {
        uint4 w[2][NT];
        u32x2_by1 ws[NT];
    };
    // eight scale bytes of a chunk, those past the row's end zero
    auto scales8 = [&](const uint8_t *p, uint32_t c) -> u32x2_by1 {
        if (c < whole_chunks) return *reinterpret_cast<const u32x2_by1 *>(p + 8u * c);
        u32x2_by1 v = {0, 0};
        for (uint32_t i = 0; i < blocks - 8u * c; ++i) v[i / 4u] |= uint32_t(p[8u * c + i]) << 8u * (i % 4u);
        return v;
    };
    u32x2_by1 x_scales;
    auto load = [&](uint32_t c, Chunk &to) {
        const uint32_t lds = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)s_x[c & 1u]));
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const void *from = x[i] + c * kRowBytes;
            if (c >= whole_chunks && c * kRowBytes + 16u * x_piece[i] >= x_bytes) from = g_mx_zeros;
            lds_load16(uint32_t(__builtin_amdgcn_readfirstlane(int(lds + (i * 4u + wave) * 1024u))), from);
        }
        x_scales = scales8(xs, c);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            to.ws[i] = scales8(ws[i], c);
#pragma unroll
            for (uint32_t s = 0; s < 2; ++s) {
                const void *from = w[i] + c * 128u + 64u * s;
                if (c >= whole_chunks && 8u * c + 4u * s + q >= blocks) from = g_mx_zeros;
                to.w[s][i] = *reinterpret_cast<const uint4 *>(from);
            }
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[t][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto step = [&](uint32_t c, Chunk &now, Chunk &next) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0) in the compiler's own count: it need not wait for the next chunk's loads before it uses this one's
        if (threadIdx.x < kRows) s_scales[c & 1u][threadIdx.x] = make_uint2(x_scales[0], x_scales[1]);
        wait_loads_and_sync<0>();
        if (c + 1u < chunks) load(c + 1u, next);
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t *lds = s_x[c & 1u];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (16u * t >= rows) break;
            const uint2 sx = s_scales[c & 1u][16u * t + m];
#pragma unroll
            for (uint32_t s = 0; s < 2; ++s) {
                MxFragment<XF> f;
                const uint32_t r = 16u * t + m;
                if constexpr (XF == SHRIKE_MX_E4M3) {
                    f.piece[0] = *reinterpret_cast<const uint4 *>(lds + r * 256u + 16u * ((8u * s + q) ^ m));
                    f.piece[1] = *reinterpret_cast<const uint4 *>(lds + r * 256u + 16u * ((8u * s + 4u + q) ^ m));
                } else {
                    f.piece[0] = *reinterpret_cast<const uint4 *>(lds + r * 128u + 16u * ((4u * s + q) ^ (m >> 1)));
                }
                const uint32_t x_scale = (s ? sx.y : sx.x) >> 8u * q;
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[t][i] = mx_multiply<XF>(now.w[s][i], f, acc[t][i], now.ws[i][s] >> 8u * q, x_scale);
            }
        }
    };
    Chunk even, odd;
    load(0, even);
    for (uint32_t c = 0; c < chunks; c += 2u) {
        step(c, even, odd);
        if (c + 1u < chunks) step(c + 1u, odd, even);
    }

#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const uint32_t r = 16u * t + m;
        if constexpr (WORK == MxWork::kDense) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const uint32_t n = n0 + 16u * i + 4u * q;
                const f32x4 v = acc[t][i] + mx_bias4(a.bias, n, a.n);
                if (r < rows) mx_store4(a.out + (row0 + r) * a.out_stride, n, a.n, v, a.out_dtype, a.out_whole);
            }
        } else if constexpr (WORK == MxWork::kGateUp) {
#pragma unroll
            for (int b = 0; b < NT / 4; ++b) {
                const uint32_t f0 = n0 + 32u * b;
                f32x4 gate[2], up[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    gate[i] = acc[t][2 * b + i];
                    up[i] = acc[t][NT / 2 + 2 * b + i];
                    if (a.ebias) {
                        gate[i] += mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.gate_ab_off), f0 + 16u * i + 4u * q, a.n);
                        up[i] += mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.up_ab_off), f0 + 16u * i + 4u * q, a.n);
                    }
                }
                const MxActBlock q8 = mx_activate(gate, up, a.act_kind);
                if (r < rows && f0 < a.n) {
                    uint8_t *to = a.act + size_t(row0 + r) * a.n + f0 + 4u * q;
                    *reinterpret_cast<uint32_t *>(to) = q8.codes[0];
                    *reinterpret_cast<uint32_t *>(to + 16) = q8.codes[1];
                    if (q == 0) a.act_scales[size_t(row0 + r) * (a.n / kMxBlock) + f0 / kMxBlock] = uint8_t(q8.scale);
                }
            }
        } else {
            if (r >= rows) continue;
            const shrike_token_expert_pair p = a.pairs[pair0 + r];
            uint16_t *to = a.out + (size_t(p.token) * a.top_k + p.rank) * a.n;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const uint32_t n = n0 + 16u * i + 4u * q;
                f32x4 v = acc[t][i];
                if (a.ebias) v += mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.down_ab_off), n, a.n);
                mx_store4(to, n, a.n, v, SHRIKE_ELEM_F16, true);
            }
        }
    }
}

template <int XF>
static int launch_product(const MxArgs &a, hipStream_t s) {
    if (a.rows <= 16u) {
        hipLaunchKernelGGL((k_mx_few<XF, 2, MxWork::kDense>), dim3((a.n + 31u) / 32u, 1), dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL((k_mx_tile<XF, 4, 4, MxWork::kDense>), dim3((a.n + 255u) / 256u, (a.rows + 63u) / 64u), dim3(256), 0, s, a);
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
    hipLaunchKernelGGL((k_mx_tile<SHRIKE_MX_E4M3, 4, 4, MxWork::kGateUp>), dim3((f + 127u) / 128u, tiles), dim3(256), 0, s, a);
    SHRIKE_HIP(hipGetLastError());
    a.x = a.act;
    a.x_scales = a.act_scales;
    a.n = d; a.k = f;
    a.out = static_cast<uint16_t *>(d_route_partials);
    hipLaunchKernelGGL((k_mx_tile<SHRIKE_MX_E4M3, 4, 4, MxWork::kDown>), dim3((d + 255u) / 256u, tiles), dim3(256), 0, s, a);
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
    hipLaunchKernelGGL((k_mx_few<SHRIKE_MX_E4M3, 4, MxWork::kGateUp>), dim3(f / 32u, tokens * top_k), dim3(256), 0, s, a);
    SHRIKE_HIP(hipGetLastError());
    a.x = a.act;
    a.x_scales = a.act_scales;
    a.n = d; a.k = f;
    hipLaunchKernelGGL((k_mx_few<SHRIKE_MX_E4M3, 2, MxWork::kDown>), dim3(d / 32u, tokens), dim3(256), 0, s, a);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
