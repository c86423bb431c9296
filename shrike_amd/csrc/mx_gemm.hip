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
// Three kernels. k_mx_few: up to 64 rows a workgroup, weights read straight from memory into the operands' registers, k split over the waves.
// mx_tile: 256 rows against 256 weight rows through LDS, four waves, bound by the matrix cores and LDS. mx_thin: up to 64 rows of an
// expert against 128 weight rows, through LDS too, several workgroups a compute unit, bound by reading the weights.
#include "decode_launch.h"
#include "mx_common.h"
#include "prefill_common.h"

#include <cstddef>
#include <type_traits>

namespace shrike {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A row operand of a lane, for one step: two 16-byte pieces of E4M3 codes, one of E2M1.
template <int XF>
struct MxFragment {
    u32x4 piece[XF == SHRIKE_MX_E4M3 ? 2 : 1];
};

template <int XF>
__device__ __forceinline__ f32x4 mx_multiply(u32x4 w, const MxFragment<XF> &x, f32x4 c, uint32_t w_scale, uint32_t x_scale) {
    const i32x8 a = {int(w[0]), int(w[1]), int(w[2]), int(w[3]), 0, 0, 0, 0};
    const u32x4 p = x.piece[0];
    if constexpr (XF == SHRIKE_MX_E4M3) {
        const u32x4 p2 = x.piece[1];
        const i32x8 b = {int(p[0]), int(p[1]), int(p[2]), int(p[3]), int(p2[0]), int(p2[1]), int(p2[2]), int(p2[3])};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, int(w_scale), 0, int(x_scale));
    } else {
        const i32x8 b = {int(p[0]), int(p[1]), int(p[2]), int(p[3]), 0, 0, 0, 0};
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
// l ^ 48. The activation goes to eight bits from fp32, without a rounding to fp16 between. (The clamps drop a NaN: it is put back.)
struct MxActBlock {
    uint32_t codes[2];  // of the lane's four values in either tile
    uint32_t scale;
};
__device__ __forceinline__ MxActBlock mx_activate(const f32x4 (&gate)[2], const f32x4 (&up)[2], uint32_t act_kind) {
    float v[8];
    uint32_t top = 0;
    auto each = [&](auto kind) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float g = gate[i / 4][i % 4], u = up[i / 4][i % 4];
            v[i] = glu_rt_fast(g, u, decltype(kind)::value);
            if (decltype(kind)::value == SHRIKE_ACT_CLAMPED_SWIGLU) {
                asm volatile("" : "+v"(v[i]));  // (or the compiler branches round the exponential, lane by lane)
                v[i] = __builtin_isunordered(g, u) ? __uint_as_float(0x7fc00000u) : v[i];
            }
            top = max(top, magnitude_bits(v[i]));
        }
    };
    if (act_kind == SHRIKE_ACT_SILU) each(std::integral_constant<uint32_t, SHRIKE_ACT_SILU>{});
    else if (act_kind == SHRIKE_ACT_CLAMPED_SWIGLU) each(std::integral_constant<uint32_t, SHRIKE_ACT_CLAMPED_SWIGLU>{});
    else each(std::integral_constant<uint32_t, SHRIKE_ACT_GELU_TANH>{});
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

// the same where the four are there: experts' outputs are multiples of 64
__device__ __forceinline__ f32x4 mx_bias4(const uint16_t *bias, uint32_t n) {
    const u16x4_by2 b = *reinterpret_cast<const u16x4_by2 *>(bias + n);
    return f32x4{bf16_to_f32(b[0]), bf16_to_f32(b[1]), bf16_to_f32(b[2]), bf16_to_f32(b[3])};
}

// Four outputs to the nearest of 16 bits. (Both conversions are made, two values an instruction, and one is taken: fewer cycles than a branch.)
__device__ __forceinline__ uint2 mx_pack4(f32x4 v, uint32_t dtype) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t lo = {v[0], v[1]}, hi = {v[2], v[3]};
    const uint32_t f16[2] = {__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, f16x2_t)), __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, f16x2_t))};
    const uint32_t bf16[2] = {__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf16x2_t)), __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf16x2_t))};
    return dtype == SHRIKE_ELEM_F16 ? make_uint2(f16[0], f16[1]) : make_uint2(bf16[0], bf16[1]);
}
// four neighbouring outputs; `whole`: rows start at multiples of 16 bytes, so that four in a row are one store
__device__ __forceinline__ void mx_store4(uint16_t *row, uint32_t n, uint32_t outputs, f32x4 v, uint32_t dtype, bool whole) {
    const uint2 h = mx_pack4(v, dtype);
    if (whole && n + 4u <= outputs) {
        *reinterpret_cast<uint2 *>(row + n) = h;
    } else {
        const uint32_t words[2] = {h.x, h.y};
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (n + i < outputs) row[n + i] = uint16_t(words[i / 2u] >> 16u * (i % 2u));
    }
}

enum class MxWork { kDense, kGateUp, kDown };

struct MxRuns;

struct MxArgs {
    const MxRuns *runs;
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

// The scales of rows on their way through LDS, a row a lane: up to 32 blocks of a row from `start` on, in two slots of 16. A slot holds 16
// scales from its first block on, or the row's last 16 where it has fewer left; a row that has not 16 at all is read byte by byte.
struct MxFewScales {
    u32x4 slot[2];
};
__device__ __forceinline__ MxFewScales few_scales(buffer_t from, uint32_t at, uint32_t start, uint32_t blocks) {
    MxFewScales s;
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
        s.slot[j] = u32x4{0, 0, 0, 0};
        if (blocks >= 16u) {
            s.slot[j] = load16(from, at, min(start + 16u * j, blocks - 16u));
        } else if (j == 0) {
#pragma unroll
            for (uint32_t b = 0; b < 15; ++b)
                if (b < blocks) s.slot[0][b / 4u] |= uint32_t(__builtin_amdgcn_raw_buffer_load_b8(from, at + b, 0, 0)) << 8u * (b % 4u);
        }
    }
    return s;
}
// Block b's byte among a row's two slots.
__device__ __forceinline__ uint32_t few_scale_byte(uint32_t b, uint32_t start, uint32_t blocks) {
    const uint32_t ahead = (b - start) / 16u * 16u;
    return ahead + b - (blocks >= 16u ? min(start + ahead, blocks - 16u) : 0u);
}

// Steps [from, to) of a wave's NT tiles of 16 weight rows against its MT tiles of rows of x, `blocks` blocks long: AHEAD steps on their way.
// Codes come straight from memory into the operands' registers: 16 neighbouring lanes want a piece each of 16 rows, which takes the
// address unit a cycle a lane, so that a compute unit takes 16 bytes a cycle: enough for weights that are read once. The scales would
// cost as many cycles again, a byte each, and come through LDS. All the addresses are those of a lane's row. The rows of x take the same
// road, and more of it: a k of 16 weight rows is 8 bytes, of 16 rows of E4M3 16, of E2M1 8. With one tile of E4M3 rows a third of the
// bytes are weights', with four a ninth, and that bounds calls of many weights (201,088 x 2,880 by 1, 16, 17 and 64 E4M3 rows 98, 140, 232 and
// 339 us, 3.1 to 0.9 TB/s of weights). Down's row, which every column of the instruction holds, is asked for sixteen times.
struct MxFewRows {
    const uint8_t *codes, *scales;  // what the offsets count from
};
template <int XF, int MT, int NT, int AHEAD>
__device__ __forceinline__ void few_steps(f32x4 (&acc)[MT][NT], uint8_t *lds, MxFewRows w, const uint32_t (&w_at)[NT], uint32_t w_scale_at, MxFewRows x, const uint32_t (&x_at)[MT],
                                          uint32_t x_scale_at, uint32_t from, uint32_t to, uint32_t blocks) {
    const uint32_t lane = threadIdx.x & 63u, m = lane & 15u, q = lane >> 4;
    constexpr uint32_t kStep = XF == SHRIKE_MX_E4M3 ? 128u : 64u;  // bytes of x
    struct Step {
        u32x4 w[NT];
        MxFragment<XF> x[MT];
    };
    const buffer_t w_codes = buffer_of(w.codes), w_scales = buffer_of(w.scales), x_codes = buffer_of(x.codes), x_scales = buffer_of(x.scales);
    // In a last step that the rows end in, the lanes past their end take the last block's place, with zero codes of weights.
    auto load = [&](Step &t, uint32_t s) {
        uint32_t back = 0, at0 = 16u * q, at1 = 64u + 16u * q;
        if (4u * s + 4u > blocks) {
            const uint32_t last = blocks - 4u * s - 1u, b = min(q, last);
            back = 16u * (q - b);
            if constexpr (XF == SHRIKE_MX_E4M3) {
                at0 = min(at0, 32u * last + 16u);
                at1 = min(at1, 32u * last + 16u);
            } else {
                at0 = 16u * b;
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) t.w[i] = load16(w_codes, w_at[i] + 16u * q - back, 64u * s);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            t.x[j].piece[0] = load16(x_codes, x_at[j] + at0, kStep * s);
            if constexpr (XF == SHRIKE_MX_E4M3) t.x[j].piece[1] = load16(x_codes, x_at[j] + at1, kStep * s);
        }
    };
    uint8_t *const lds_w = lds, *const lds_x = lds + NT * 16u * 32u;
    auto multiply = [&](Step &t, uint32_t s, uint32_t start) {
        const uint32_t byte = few_scale_byte(min(4u * s + q, blocks - 1u), start, blocks);
        if (4u * s + 4u > blocks)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) t.w[i][e] = 4u * s + q < blocks ? t.w[i][e] : 0u;
        uint32_t ws[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) ws[i] = lds_w[(16u * i + m) * 32u + byte];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const uint32_t x_scale = lds_x[(16u * j + m) * 32u + byte];
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[j][i] = mx_multiply<XF>(t.w[i], t.x[j], acc[j][i], ws[i], x_scale);
        }
    };
    if (from >= to) return;
    constexpr uint32_t kSegment = AHEAD % 3 == 0 ? 6 : 8;  // steps: a multiple of AHEAD
    static_assert(kSegment % AHEAD == 0);
    Step t[AHEAD];
    const bool w_row = lane < 16u * NT, x_row = lane < 16u * MT;
    MxFewScales sw = few_scales(w_scales, w_scale_at, 4u * from, blocks), sx = few_scales(x_scales, x_scale_at, 4u * from, blocks);
#pragma unroll
    for (uint32_t i = 0; i < AHEAD; ++i)
        if (from + i < to) load(t[i], from + i);
    for (uint32_t first = from; first < to; first += kSegment) {
        // a segment's scales into the wave's own part of LDS (no other wave reads it), and the next segment's on their way
        if (w_row) {
            reinterpret_cast<u32x4 *>(lds_w + lane * 32u)[0] = sw.slot[0];
            reinterpret_cast<u32x4 *>(lds_w + lane * 32u)[1] = sw.slot[1];
        }
        if (x_row) {
            reinterpret_cast<u32x4 *>(lds_x + lane * 32u)[0] = sx.slot[0];
            reinterpret_cast<u32x4 *>(lds_x + lane * 32u)[1] = sx.slot[1];
        }
        __builtin_amdgcn_wave_barrier();
        if (first + kSegment < to) {
            sw = few_scales(w_scales, w_scale_at, 4u * (first + kSegment), blocks);
            sx = few_scales(x_scales, x_scale_at, 4u * (first + kSegment), blocks);
        }
        const uint32_t until = min(to, first + kSegment);
        for (uint32_t s = first; s < until; s += AHEAD)
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
                if (s + i < until) {
                    multiply(t[i], s + i, 4u * first);
                    if (s + i + AHEAD < to) load(t[i], s + i + AHEAD);
                }
        __builtin_amdgcn_wave_barrier();
    }
}

// The pairs from `pair` on that are at the same cell, up to 16: lane m of each 16 gets the m-th (past their end: `pair`). Returns their
// count, 0 where an earlier pair's workgroup takes this one along.
__device__ __forceinline__ uint32_t same_cell_pairs(const uint32_t *slots, uint32_t pairs, uint32_t pair, uint32_t cell, uint32_t &mine) {
    const uint32_t lane = threadIdx.x & 63u, m = lane & 15u;
    mine = pair;
    uint32_t before = 0, count = 0;
    for (uint32_t first = 0; first < pairs; first += 64u) {
        uint64_t same = __ballot(first + lane < pairs && slots[first + lane] == cell);
        if (pair > first) {
            const uint64_t earlier = pair - first >= 64u ? ~uint64_t(0) : (uint64_t(1) << (pair - first)) - 1u;
            before += uint32_t(__popcll(same & earlier));
            same &= ~earlier;
        }
        for (; same != 0 && count < 16u; ++count, same &= same - 1u)
            if (m == count) mine = first + uint32_t(__builtin_ctzll(same));
    }
    return before % 16u == 0 ? count : 0u;
}

// Waves take 16 MT rows of x against 16 NT weight rows (gate and up: NT / 2 tiles of each), a part of k each, and their sums meet in LDS: a row's 1,440 bytes are few for one wave, and a call of few rows is a launch and a few latencies (2,880 x 2,880 by one row 4.6 us,
// by 64 rows 7.9). Gate and up: the rows are those of up to 16 pairs of one expert, whose weights are then read once. Down: one token's, a
// position behind the other, a row that every column of the instruction holds.
template <int XF, int MT, int NT, int WAVES, int AHEAD, MxWork WORK, int LEAST = MT == 1 ? 4 : 2>
__global__ __launch_bounds__(64 * WAVES, LEAST) void k_mx_few(MxArgs a) {
    constexpr uint32_t kScales = 16u * (NT + MT) * 32u;  // of a wave
    __shared__ __attribute__((aligned(16))) uint8_t s_scales[WAVES * kScales];
    __shared__ f32x4 s_part[WAVES][MT * NT][64];
    const uint32_t wave = wave_index(), lane = threadIdx.x & 63u, m = lane & 15u, q = lane >> 4;
    const uint32_t blocks = a.k / kMxBlock, steps = (blocks + 3u) / 4u, row_codes = blocks * 16u;
    const uint32_t n0 = blockIdx.x * (WORK == MxWork::kGateUp ? 8u : 16u) * NT;
    uint8_t *const lds = s_scales + wave * kScales;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT * NT; ++i) {
        acc[i / NT][i % NT] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        asm volatile("" : "+v"(acc[i / NT][i % NT]));  // (a loop that starts from a zero that it can see, the compiler takes apart word by word)
    }
    const uint8_t *base = nullptr;
    uint32_t w_at[NT], w_scale_at, x_at[MT], x_scale_at;
    uint32_t pair = 0, columns = 0;  // gate and up: the lane's column's pair, and how many columns are pairs'
    // (rows past the last are the last again: nobody stores them)
    auto weight_row = [&](uint32_t r) { return min(n0 + r, a.n - 1u); };

    if constexpr (WORK == MxWork::kDense) {
        const uint32_t first = min(n0, a.n - 1u), row0 = blockIdx.y * 16u * MT;
        auto x_row = [&](uint32_t r) { return min(row0 + r, a.rows - 1u) - row0; };
#pragma unroll
        for (int i = 0; i < NT; ++i) w_at[i] = (weight_row(16u * i + m) - first) * row_codes;
        w_scale_at = (weight_row(lane % (16u * NT)) - first) * blocks;
#pragma unroll
        for (int j = 0; j < MT; ++j) x_at[j] = x_row(16u * j + m) * mx_code_bytes<XF>(a.k);
        x_scale_at = x_row(lane % (16u * MT)) * blocks;
        few_steps<XF, MT, NT, AHEAD>(acc, lds, {a.w + size_t(first) * row_codes, a.w_scales + size_t(first) * blocks}, w_at, w_scale_at,
                                     {a.x + size_t(row0) * mx_code_bytes<XF>(a.k), a.x_scales + size_t(row0) * blocks}, x_at, x_scale_at,
                                     steps * wave / WAVES, steps * (wave + 1u) / WAVES, blocks);
    } else if constexpr (WORK == MxWork::kGateUp) {
        const uint32_t cell = a.slots[blockIdx.y];
        if (cell == kSentinel) return;
        columns = same_cell_pairs(a.slots, a.rows * a.top_k, blockIdx.y, cell, pair);
        if (columns == 0) return;
        base = cell_base_uniform(a.pool, cell, a.stride);
#pragma unroll
        for (int i = 0; i < NT; ++i) w_at[i] = (i >= NT / 2 ? a.off.up_w_off : a.off.gate_w_off) + weight_row(16u * (i % (NT / 2)) + m) * row_codes;
        w_scale_at = (lane >= 8u * NT ? a.off.up_s_off : a.off.gate_s_off) + weight_row(lane % (8u * NT)) * blocks;
        x_at[0] = pair / a.top_k * a.k;
        x_scale_at = pair / a.top_k * blocks;
        few_steps<XF, MT, NT, AHEAD>(acc, lds, {base, base}, w_at, w_scale_at, {a.x, a.x_scales}, x_at, x_scale_at, steps * wave / WAVES, steps * (wave + 1u) / WAVES, blocks);
    } else {
        // the positions' steps one behind the other, an equal part of them a wave; a position's sum is weighted when its steps end
        const uint32_t all = steps * a.top_k, to = all * (wave + 1u) / WAVES;
        uint32_t at = all * wave / WAVES;
#pragma unroll
        for (int i = 0; i < NT; ++i) w_at[i] = a.off.down_w_off + weight_row(16u * i + m) * row_codes;
        w_scale_at = a.off.down_s_off + weight_row(lane % (16u * NT)) * blocks;
        x_at[0] = x_scale_at = 0;
        while (at < to) {
            const uint32_t position = at / steps, from = at - position * steps, until = min(steps, from + (to - at));
            at += until - from;
            const size_t row = size_t(blockIdx.y) * a.top_k + position;
            const uint32_t cell = a.slots[row];
            if (cell == kSentinel) continue;
            base = cell_base_uniform(a.pool, cell, a.stride);
            f32x4 sum[1][NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                sum[0][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                asm volatile("" : "+v"(sum[0][i]));
            }
            few_steps<XF, 1, NT, AHEAD>(sum, lds, {base, base}, w_at, w_scale_at, {a.x + row * a.k, a.x_scales + row * blocks}, x_at, x_scale_at, from, until, blocks);
            const float weight = f16_to_f32(a.weights[row]);
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[0][i] += weight * sum[0][i];
        }
    }
#pragma unroll
    for (int i = 0; i < MT * NT; ++i) s_part[wave][i][lane] = acc[i / NT][i % NT];
    __syncthreads();
    // the sum of tile i of the wave's rows over the parts of k
    auto total = [&](uint32_t i) {
        f32x4 v = s_part[0][i][lane];
#pragma unroll
        for (int p = 1; p < WAVES; ++p) v += s_part[p][i][lane];
        return v;
    };

    if constexpr (WORK == MxWork::kGateUp) {
        static_assert(NT == 4 && MT == 1, "a wave's gate and up rows are one MX block of activations");
        if (wave != 0) return;
        f32x4 gate[2], up[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            gate[i] = total(i);
            up[i] = total(2u + i);
            if (a.ebias) {
                gate[i] += mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.gate_ab_off), n0 + 16u * i + 4u * q);
                up[i] += mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.up_ab_off), n0 + 16u * i + 4u * q);
            }
        }
        const MxActBlock b = mx_activate(gate, up, a.act_kind);
        if (m < columns) {
            uint8_t *to = a.act + size_t(pair) * a.n + n0 + 4u * q;
            *reinterpret_cast<uint32_t *>(to) = b.codes[0];
            *reinterpret_cast<uint32_t *>(to + 16) = b.codes[1];
            if (q == 0) a.act_scales[size_t(pair) * (a.n / kMxBlock) + n0 / kMxBlock] = uint8_t(b.scale);
        }
    } else if constexpr (WORK == MxWork::kDense) {
        for (uint32_t i = wave; i < uint32_t(MT * NT); i += WAVES) {
            const uint32_t row = (blockIdx.y * MT + i / NT) * 16u + m, n = n0 + 16u * (i % NT) + 4u * q;
            const f32x4 v = total(i) + mx_bias4(a.bias, n, a.n);
            if (row < a.rows) mx_store4(a.out + row * a.out_stride, n, a.n, v, a.out_dtype, a.out_whole);
        }
    } else {
        static_assert(WAVES >= NT);
        if (wave >= uint32_t(NT)) return;
        const uint32_t n = n0 + 16u * wave + 4u * q;
        f32x4 v = total(wave);
        if (m != 0 || n >= a.n) return;  // (n and a.n are multiples of four)
        if (a.ebias)
            for (uint32_t p = 0; p < a.top_k; ++p) {
                const size_t row = size_t(blockIdx.y) * a.top_k + p;
                const uint32_t cell = a.slots[row];
                if (cell == kSentinel) continue;
                const uint8_t *at = cell_base(a.pool, cell, a.stride) + a.off.down_ab_off;
                v += f16_to_f32(a.weights[row]) * mx_bias4(reinterpret_cast<const uint16_t *>(at), n);
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

// A tile of up to 32 MT rows against 256 weight rows by four waves, 16 MT rows against 128 weight rows each (gate and up: 64 of either).
// Everything comes through LDS by asynchronous loads, of whole 128-byte lines: a load that takes half a line of each of 16 rows costs the
// cache what the whole lines do (14 against 33 TB/s of cache hits over the device), and straight from memory into the operands'
// registers, where 16 neighbouring lanes want a piece each of 16 rows, a line a lane. A part a wave as large as its registers hold, since
// every operand is read from LDS by two waves. A line is a unit of k, 256 of E2M1 codes, 128 of E4M3; two units of either operand have a
// place, and the next one is asked for while the last one is multiplied. The pieces of a line are swapped about so that 16 rows' same
// piece lies in 64 different banks.
// Measured: 4,096 x 4,096 x 2,880 of E4M3 rows 42.5 us (2,270 TFLOP/s), of which 17 are start, outputs and end; a step of 128 k 1.2 to 1.4 us
// where its products take 0.9, of E2M1 rows 0.85 and 0.6. Reading the next step's weights ahead of its barrier, or rows two tiles ahead, makes
// no step shorter; touching lines two steps ahead of their loads makes it a tenth longer.
template <int MT>
struct MxTileLds {
    static constexpr uint32_t kRows = 32u * MT, kWeights = 256u;
    static constexpr uint32_t kX = kRows * 128u, kW = kWeights * 128u;  // a unit
    // two places of either, and the scales of four steps, 16 bytes a row, twice
    static constexpr uint32_t kAtW = 2u * kX, kScales = kAtW + 2u * kW, kScalePlace = (kWeights + kRows) * 16u, kBytes = kScales + 2u * kScalePlace;
    static_assert(kBytes <= 160u * 1024u);
};

// Where a lane's parts of the weight rows start, from an address that the workgroup shares: the 16 bytes that its eight asynchronous loads take
// (of a line, `piece` bytes from the row's own start), and the scales of the row that the thread's number names.
struct MxTileWeights {
    const uint8_t *codes, *scales;
    uint32_t at[8], piece, scale_at;
};

// An address that is the same in every lane, in scalar registers.
__device__ __forceinline__ const uint8_t *uniform(const uint8_t *p) {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(at)))), hi = uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(at >> 32))));
    return reinterpret_cast<const uint8_t *>(uint64_t(hi) << 32 | lo);
}

// The piece of a line that a lane of an asynchronous load takes: a load is 8 rows of 8 pieces, and a row's pieces are swapped by half its
// number within 16 (`load`: the load's number, which tells the rows 0..7 of 16 from 8..15).
__device__ __forceinline__ uint32_t mx_piece(uint32_t load) {
    const uint32_t lane = threadIdx.x & 63u;
    return 16u * ((lane & 7u) ^ (lane >> 4) ^ (load % 2u * 4u));
}

template <int XF, int MT>
struct MxTile {
    using L = MxTileLds<MT>;
    static constexpr uint32_t kLoads = MT;  // of x, a wave and unit
    static constexpr uint32_t kSteps = XF == SHRIKE_MX_E4M3 ? 1u : 2u;  // of a unit of x
    f32x4 acc[MT][8];

    // x, xs: where the rows that `row(r)` numbers start
    template <typename Row>
    __device__ __forceinline__ void run(uint8_t *lds, const MxTileWeights &w, const uint8_t *x, const uint8_t *xs, uint32_t blocks, Row row) {
        const uint32_t wave = wave_index(), lane = threadIdx.x & 63u, m = lane & 15u, q = lane >> 4, wm = wave / 2u, wn = wave % 2u;
        const uint32_t steps = (blocks + 3u) / 4u;
        const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds));
        // Load i of a unit: rows (4 i + wave) * 8 + lane / 8. Offsets of the lane's piece of the first unit, and of the row's last piece: past its end
        // that is asked for again.
        const uint32_t piece = mx_piece(wave), x_bytes = blocks * (XF == SHRIKE_MX_E4M3 ? 32u : 16u);
        uint32_t x_at[kLoads], x_end[kLoads], w_end[8];
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t start = row((4u * i + wave) * 8u + lane / 8u) * x_bytes;
            x_at[i] = start + piece;
            x_end[i] = start + x_bytes - 16u;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) w_end[i] = w.at[i] - w.piece + blocks * 16u - 16u;
        const uint8_t *const x0 = uniform(x), *const w0 = uniform(w.codes);
        auto load_x = [&](uint32_t u, uint32_t i) { lds_load16(lds0 + (u & 1u) * L::kX + (4u * i + wave) * 1024u, x0, min(x_at[i] + u * 128u, x_end[i])); };
        auto load_w = [&](uint32_t u, uint32_t i) { lds_load16(lds0 + L::kAtW + (u & 1u) * L::kW + (4u * i + wave) * 1024u, w0, min(w.at[i] + u * 128u, w_end[i])); };
        // The scales of steps 4 g .. 4 g + 3: 16 bytes a row, a weight row a thread and a row of x too. Where the row has fewer left, its last 16; a row
        // that has not as many is read byte by byte.
        const uint32_t xs_at = row(threadIdx.x) * blocks;
        u32x4 sw, sx;
        auto load_scales = [&](uint32_t g) {
            typedef uint32_t u32x4_by1 __attribute__((ext_vector_type(4), aligned(1)));
            const uint32_t from = min(16u * g, blocks - 16u);
            sw = *reinterpret_cast<const u32x4_by1 *>(w.scales + (w.scale_at + from));
            sx = *reinterpret_cast<const u32x4_by1 *>(xs + (xs_at + from));
        };
        auto load_few_scales = [&] {
            sw = sx = u32x4{0, 0, 0, 0};
#pragma unroll
            for (uint32_t b = 0; b < 15; ++b)
                if (b < blocks) {
                    sw[b / 4u] |= uint32_t(w.scales[w.scale_at + b]) << 8u * (b % 4u);
                    sx[b / 4u] |= uint32_t(xs[xs_at + b]) << 8u * (b % 4u);
                }
        };
        // Into LDS so that a lane finds the four steps' bytes of its block in one word (read byte by byte, a step each: 43.0 us in place of 42.5 for 4,096 x
        // 4,096 x 2,880): word j takes bytes j, 4 + j, 8 + j, 12 + j. The last 16 of a row are moved up to where they belong, the last one behind them (the codes
        // there are zeros).
        auto by_steps = [&](u32x4 v, uint32_t g) {
            if (blocks >= 16u && 16u * g > blocks - 16u) {
                const uint32_t ahead = 16u * g - (blocks - 16u), last = (v[3] >> 24) * 0x01010101u;
                for (uint32_t i = 0; i < ahead / 4u; ++i) v = u32x4{v[1], v[2], v[3], last};
                const uint32_t by = ahead % 4u;
                v = u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], by), __builtin_amdgcn_alignbyte(v[2], v[1], by), __builtin_amdgcn_alignbyte(v[3], v[2], by),
                          __builtin_amdgcn_alignbyte(last, v[3], by)};
            }
            const uint32_t low01 = __builtin_amdgcn_perm(v[1], v[0], 0x05010400u), high01 = __builtin_amdgcn_perm(v[1], v[0], 0x07030602u);
            const uint32_t low23 = __builtin_amdgcn_perm(v[3], v[2], 0x05010400u), high23 = __builtin_amdgcn_perm(v[3], v[2], 0x07030602u);
            return u32x4{__builtin_amdgcn_perm(low23, low01, 0x05040100u), __builtin_amdgcn_perm(low23, low01, 0x07060302u),
                         __builtin_amdgcn_perm(high23, high01, 0x05040100u), __builtin_amdgcn_perm(high23, high01, 0x07060302u)};
        };
        auto store_scales = [&](uint32_t g) {
            uint8_t *to = lds + L::kScales + (g & 1u) * L::kScalePlace;
            reinterpret_cast<u32x4 *>(to)[threadIdx.x] = by_steps(sw, g);
            if (threadIdx.x < L::kRows) reinterpret_cast<u32x4 *>(to + L::kWeights * 16u)[threadIdx.x] = by_steps(sx, g);
        };
        // the wave's scales of four steps; the lowest byte is the next one's
        uint32_t w_scale[8], x_scale[MT];
        auto fetch_scales = [&](uint32_t g) {
            const uint8_t *from = lds + L::kScales + (g & 1u) * L::kScalePlace + m * 16u + q * 4u;
#pragma unroll
            for (int i = 0; i < 8; ++i) w_scale[i] = *reinterpret_cast<const uint32_t *>(from + (wn * 8u + i) * 256u);
#pragma unroll
            for (int t = 0; t < MT; ++t) x_scale[t] = *reinterpret_cast<const uint32_t *>(from + L::kWeights * 16u + (wm * MT + t) * 256u);
        };
        // A step: 16 rows of x against the wave's 128 weight rows at a time, and between them, one by one, the next units' loads. (All at once they
        // would hold up every wave for as long as the address unit takes.) LAST: the rows may end inside the step; the weights' codes past their end
        // are made zeros.
        auto multiply = [&](uint32_t s, auto next_x, auto next_w, auto last) {
            constexpr bool LAST = decltype(last)::value, NEXT_X = decltype(next_x)::value, NEXT_W = decltype(next_w)::value;
            const uint32_t half_w = 4u * (s & 1u), half_x = XF == SHRIKE_MX_E4M3 ? 0u : half_w;  // pieces from the unit's start
            const uint8_t *weights = lds + L::kAtW + (s / 2u & 1u) * L::kW + wn * 16384u + m * 128u;
            const uint8_t *rows = lds + (s / kSteps & 1u) * L::kX + wm * (MT * 2048u) + m * 128u;
            auto fetch = [&](MxFragment<XF> &f, int t, int part) {
                if (part == 0) f.piece[0] = *reinterpret_cast<const u32x4 *>(rows + t * 2048u + 16u * ((half_x + q) ^ (m >> 1)));
                if constexpr (XF == SHRIKE_MX_E4M3)
                    if (part == 1) f.piece[1] = *reinterpret_cast<const u32x4 *>(rows + t * 2048u + 16u * ((4u + q) ^ (m >> 1)));
            };
            MxFragment<XF> now, next;
#pragma unroll
            for (int part = 0; part < 2; ++part) fetch(now, 0, part);
            next = now;
            u32x4 wf[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                wf[i] = *reinterpret_cast<const u32x4 *>(weights + i * 2048u + 16u * ((half_w + q) ^ (m >> 1)));
                if (LAST)
#pragma unroll
                    for (int e = 0; e < 4; ++e) wf[i][e] = 4u * s + q < blocks ? wf[i][e] : 0u;
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                // between the products, one thing each: the next rows' operands, then loads
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    acc[t][i] = mx_multiply<XF>(wf[i], now, acc[t][i], w_scale[i], x_scale[t]);
                    __builtin_amdgcn_sched_barrier(0);
                    if (t + 1 < MT && i < 2) fetch(next, t + 1, i);
                    if (i >= 3) issue<NEXT_X, NEXT_W>(s, 5 * t + i - 3, load_x, load_w);
                    __builtin_amdgcn_sched_barrier(0);
                }
                // (the products stay ahead of what follows: they have no effect that would keep the compiler from moving them)
#pragma unroll
                for (int i = 0; i < 8; ++i) asm volatile("" : "+a"(acc[t][i]));
                x_scale[t] >>= 8;
                now = next;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) w_scale[i] >>= 8;
        };
#pragma unroll
        for (int i = 0; i < MT * 8; ++i) {
            acc[i / 8][i % 8] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            asm volatile("" : "+a"(acc[i / 8][i % 8]));  // (a loop that starts from a zero that it can see, the compiler takes apart word by word)
        }
        if (blocks >= 16u) load_scales(0);
        else load_few_scales();
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) load_x(0, i);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) load_w(0, i);
        // Two steps a turn. Ahead of the first, everything has landed. In its course the rows' next unit is asked for (E2M1 rows: and the weights'), in the
        // second one's the unit after it and the weights'.
        const std::true_type yes;
        const std::false_type no;
        const std::integral_constant<bool, kSteps == 1u> one;
        auto turn = [&](uint32_t s) {
            __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0) in the compiler's own count
            if (s % 4u == 0) store_scales(s / 4u);
            wait_loads_and_sync<0>();
            if (s % 4u == 0) {
                fetch_scales(s / 4u);
                if (s + 4u < steps) load_scales(s / 4u + 1u);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        auto middle = [&] {
            if constexpr (kSteps == 1u) wait_loads_and_sync<0>();
            __builtin_amdgcn_sched_barrier(0);
        };
        uint32_t s = 0;
        for (; s + 2u < steps; s += 2u) {
            turn(s);
            multiply(s, yes, yes, no);
            if constexpr (kSteps == 1u) wait_loads_and_sync<8>();  // (all but the weights')
            __builtin_amdgcn_sched_barrier(0);
            multiply(s + 1u, one, no, no);
        }
        turn(s);
        if (s + 1u < steps) {
            multiply(s, one, no, yes);
            middle();
            ++s;
        }
        multiply(s, no, no, yes);
    }

    // The load for place `at` of a step's 5 MT between products: the rows' first, one a place, then the weights', spread over what is left.
    template <bool NEXT_X, bool NEXT_W, typename LoadX, typename LoadW>
    static __device__ __forceinline__ void issue(uint32_t s, int at, LoadX load_x, LoadW load_w) {
        constexpr int kPlaces = 5 * MT - MT;
        if constexpr (NEXT_X)
            if (at < MT) load_x(s / kSteps + 1u, at);
        if constexpr (NEXT_W)
            if (at >= MT)
#pragma unroll
                for (int j = 8 * (at - MT) / kPlaces; j < 8 * (at - MT + 1) / kPlaces; ++j) load_w(s / 2u + 1u, j);
    }
};

template <int XF, int MT, MxWork WORK>
__device__ __forceinline__ void mx_tile(const MxArgs &a, uint8_t *lds, uint32_t number, uint32_t row0, uint32_t rows, uint32_t pair0, const uint8_t *base) {
    const uint32_t wave = wave_index(), lane = threadIdx.x & 63u, m = lane & 15u, q = lane >> 4, wm = wave / 2u, wn = wave % 2u;
    const uint32_t blocks = a.k / kMxBlock;
    const uint32_t first = number * (WORK == MxWork::kGateUp ? 128u : 256u);  // output of the workgroup
    // Weight row r of the workgroup's 256: 128 of a wave of each half, gate and up by turns of 64 of them. (Rows past the last are the last again:
    // nobody stores them.)
    auto weight_row = [&](uint32_t r) { return WORK == MxWork::kGateUp ? min(first + r / 128u * 64u + r % 64u, a.n - 1u) : min(first + r, a.n - 1u); };
    MxTileWeights w;
    w.piece = mx_piece(wave);
    uint32_t from = 0;
    if constexpr (WORK == MxWork::kDense) {
        w.codes = a.w + size_t(first) * blocks * 16u;
        w.scales = a.w_scales + size_t(first) * blocks;
        from = first;
    } else {
        w.codes = w.scales = base;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t r = (4u * i + wave) * 8u + lane / 8u;
        w.at[i] = (weight_row(r) - from) * blocks * 16u + w.piece;
        if constexpr (WORK == MxWork::kGateUp) w.at[i] += r % 128u >= 64u ? a.off.up_w_off : a.off.gate_w_off;
        if constexpr (WORK == MxWork::kDown) w.at[i] += a.off.down_w_off;
    }
    w.scale_at = (weight_row(threadIdx.x) - from) * blocks;
    if constexpr (WORK == MxWork::kGateUp) w.scale_at += threadIdx.x % 128u >= 64u ? a.off.up_s_off : a.off.gate_s_off;
    if constexpr (WORK == MxWork::kDown) w.scale_at += a.off.down_s_off;
    MxTile<XF, MT> tile;
    // the rows past the tile's are its last one again; gate and up take a pair's token's row of the chunk
    auto clamped = [&](uint32_t r) { return min(r, rows - 1u); };
    if constexpr (WORK == MxWork::kGateUp)
        tile.run(lds, w, a.x, a.x_scales, blocks, [&](uint32_t r) -> uint32_t { return a.pairs[pair0 + clamped(r)].token; });
    else
        tile.run(lds, w, a.x + size_t(row0) * mx_code_bytes<XF>(a.k), a.x_scales + size_t(row0) * blocks, blocks, clamped);

    const uint32_t r0 = wm * 16u * MT + m;
    if constexpr (WORK == MxWork::kGateUp) {
        // Through LDS, where a wave has room for its own rows of 64 codes, so that a store takes 64 neighbouring ones.
        constexpr uint32_t kRoom = MT * 16u * 64u;
        wait_loads_and_sync<0>();
        uint8_t *room = lds + wave * kRoom;
        if (first + wn * 64u >= a.n) return;  // (outputs are multiples of 64)
        uint32_t scale[MT];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t f0 = first + wn * 64u + 32u * b;
            f32x4 bias[4] = {};
            if (a.ebias)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    bias[i] = mx_bias4(reinterpret_cast<const uint16_t *>(base + (i < 2u ? a.off.gate_ab_off : a.off.up_ab_off)), f0 + 16u * (i % 2u) + 4u * q);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const uint32_t r = r0 + 16u * t;
                const f32x4 gate[2] = {tile.acc[t][2 * b] + bias[0], tile.acc[t][2 * b + 1] + bias[1]};
                const f32x4 up[2] = {tile.acc[t][4 + 2 * b] + bias[2], tile.acc[t][4 + 2 * b + 1] + bias[3]};
                const MxActBlock q8 = mx_activate(gate, up, a.act_kind);
                uint32_t *to = reinterpret_cast<uint32_t *>(room + (16u * t + m) * 64u) + q;
                to[4u * ((2u * b) ^ (m / 4u))] = q8.codes[0];
                to[4u * ((2u * b + 1u) ^ (m / 4u))] = q8.codes[1];
                scale[t] = b == 0 ? q8.scale : scale[t] | q8.scale << 8;
                if (b == 1 && q == 0 && r < rows) *reinterpret_cast<uint16_t *>(a.act_scales + size_t(row0 + r) * (a.n / kMxBlock) + f0 / kMxBlock - 1u) = uint16_t(scale[t]);
            }
        }
        const uint32_t f16 = first + wn * 64u + 16u * (lane % 4u);
#pragma unroll
        for (uint32_t t = 0; t < uint32_t(MT); ++t) {
            const uint32_t r = 16u * t + lane / 4u, at = wm * 16u * MT + r;
            const uint4 v = *reinterpret_cast<const uint4 *>(room + r * 64u + 16u * ((lane % 4u) ^ (r / 4u & 3u)));
            if (at < rows && f16 < a.n) *reinterpret_cast<uint4 *>(a.act + size_t(row0 + at) * a.n + f16) = v;
        }
    } else {
        const uint32_t n0 = first + wn * 128u + 4u * q;
        f32x4 bias[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (WORK == MxWork::kDense) bias[i] = mx_bias4(a.bias, n0 + 16u * i, a.n);
            else if (a.ebias) bias[i] = mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.down_ab_off), min(n0 + 16u * i, a.n - 4u));
            else bias[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        // Through LDS, where a wave has room for its own rows of 128 outputs: so that a store takes whole lines of four rows. (Straight from the
        // registers a line is four stores of a quarter of it each: 4,096 x 4,096 outputs 17 us in place of 7.) 16-byte pieces swapped as ever.
        constexpr uint32_t kRoom = MT * 16u * 256u;
        static_assert(4u * kRoom <= MxTileLds<MT>::kBytes);
        wait_loads_and_sync<0>();
        uint8_t *room = lds + wave * kRoom;
        // down: where a lane's rows go, the wave's rows lane and lane + 64
        uint32_t place[2] = {0, 0};
        if constexpr (WORK == MxWork::kDown)
#pragma unroll
            for (uint32_t i = 0; i < (MT > 4 ? 2u : 1u); ++i) {
                const shrike_token_expert_pair p = a.pairs[pair0 + min(wm * 16u * MT + 64u * i + lane, rows - 1u)];
                place[i] = p.token * a.top_k + p.rank;
            }
        const uint32_t n8 = first + wn * 128u + 8u * m;
#pragma unroll
        for (uint32_t t = 0; t < uint32_t(MT); ++t) {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint2 h = mx_pack4(tile.acc[t][i] + bias[i], WORK == MxWork::kDense ? a.out_dtype : uint32_t(SHRIKE_ELEM_F16));
                *reinterpret_cast<uint2 *>(room + (16u * t + m) * 256u + 16u * ((2u * i + q / 2u) ^ m) + q % 2u * 8u) = h;
            }
#pragma unroll
            for (uint32_t j = 4u * t; j < 4u * t + 4u; ++j) {
                const uint32_t r = 4u * j + q, at = wm * 16u * MT + r;
                const uint4 v = *reinterpret_cast<const uint4 *>(room + r * 256u + 16u * (m ^ (r & 15u)));
                const uint32_t slot = uint32_t(__shfl(int(place[MT > 4 ? j / 16u : 0u]), int(r % 64u)));
                if (at >= rows || n8 >= a.n) continue;
                uint16_t *to;
                bool whole = true;
                if constexpr (WORK == MxWork::kDense) {
                    to = a.out + (row0 + at) * a.out_stride;
                    whole = a.out_whole && n8 + 8u <= a.n;
                } else {
                    to = a.out + size_t(slot) * a.n;
                }
                if (whole) {
                    *reinterpret_cast<uint4 *>(to + n8) = v;
                } else {
                    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e)
                        if (n8 + e < a.n) to[n8 + e] = uint16_t(words[e / 2u] >> 16u * (e % 2u));
                }
            }
        }
    }
}

template <int XF, int MT>
__global__ __launch_bounds__(256, 1) void k_mx_product(MxArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    // Workgroups go to the eight dies by turns: each die takes neighbouring tiles, four tiles of rows by as many columns, whose rows and weights
    // meet in its cache.
    const uint32_t columns = (a.n + 255u) / 256u, heights = (a.rows + 32u * MT - 1u) / (32u * MT);
    const uint32_t number = blockIdx.x % 8u * (gridDim.x / 8u) + blockIdx.x / 8u;
    if (number >= columns * heights) return;
    const uint32_t group = number / (4u * columns), within = number % (4u * columns), high = min(4u, heights - 4u * group);
    const uint32_t row0 = (4u * group + within % high) * 32u * MT;
    mx_tile<XF, MT, MxWork::kDense>(a, lds, within / high, row0, min(32u * MT, a.rows - row0), 0, nullptr);
}

// Whether the table's record goes on where the one before it ends: the same expert's next rows.
__device__ __forceinline__ bool goes_on(const shrike_row_tile &before, const shrike_row_tile &tile) {
    return before.expert == tile.expert && before.cell == tile.cell && before.rows == kRowTile && before.pair_start + kRowTile == tile.pair_start;
}

// The table's records as the workgroups take them: up to four that go on to each other, 256 rows, from the first, fifth ... of such a run on. The ones of
// most rows come first: they are dealt out in this order, and one that starts last would be waited for. One workgroup.
struct MxRun {
    uint32_t record, rows;
};
struct MxRuns {
    uint32_t count, pad[3];
    MxRun run[1];
};
static constexpr size_t mx_runs_bytes(size_t records) { return (sizeof(MxRuns) + records * sizeof(MxRun) + 255u) & ~size_t(255); }
constexpr uint32_t kRunThreads = 256, kRunClasses = 16;  // by 16 rows

__global__ __launch_bounds__(kRunThreads) void k_mx_expert_runs(const shrike_row_tile *tiles, const uint32_t *tile_count, uint32_t records, MxRuns *runs) {
    __shared__ uint32_t starts[kRunThreads / 64u], counts[kRunClasses], at[kRunClasses];
    const uint32_t count = min(*tile_count, records), lane = threadIdx.x & 63u, wave = threadIdx.x / 64u;
    if (threadIdx.x < kRunClasses) counts[threadIdx.x] = 0;
    // rows of the run that starts with record i, or 0; every thread calls it, 256 neighbouring records at a time
    auto rows_of = [&](uint32_t i, uint32_t &carried) -> uint32_t {
        const bool there = i < count, start = there && (i == 0 || !goes_on(tiles[i - 1u], tiles[i]));
        const uint64_t in_wave = __ballot(start);
        __syncthreads();
        if (lane == 0) starts[wave] = in_wave ? (i | 63u) - uint32_t(__builtin_clzll(in_wave)) : ~0u;
        __syncthreads();
        const uint64_t mine = in_wave & (~0ull >> (63u - lane));
        uint32_t first = carried;
        for (uint32_t w = 0; w < kRunThreads / 64u; ++w) {
            if (w == wave && mine == 0) break;
            if (w == wave) { first = (i & ~63u) + 63u - uint32_t(__builtin_clzll(mine)); break; }
            if (starts[w] != ~0u) first = starts[w];
        }
        for (uint32_t w = 0; w < kRunThreads / 64u; ++w)
            if (starts[w] != ~0u) carried = starts[w];
        if (!there || (i - first) % 4u != 0) return 0;
        shrike_row_tile part[4];  // (all asked for at once)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) part[j] = tiles[min(i + j, count - 1u)];
        if (part[0].cell == kSentinel) return 0;
        uint32_t rows = min(part[0].rows, kRowTile);
        bool on = true;
#pragma unroll
        for (uint32_t j = 1; j < 4; ++j) {
            on = on && i + j < count && goes_on(part[j - 1u], part[j]);
            rows += on ? min(part[j].rows, kRowTile) : 0u;
        }
        return rows;
    };
    const uint32_t end = (count + kRunThreads - 1u) & ~(kRunThreads - 1u);
    uint32_t carried = 0, rows = 0;
    for (uint32_t i = threadIdx.x; i < end; i += kRunThreads)
        if ((rows = rows_of(i, carried)) != 0) atomicAdd(&counts[(256u - rows) / 16u], 1u);
    __syncthreads();
    if (threadIdx.x < kRunClasses) {
        uint32_t before = 0;
        for (uint32_t c = 0; c < threadIdx.x; ++c) before += counts[c];
        at[threadIdx.x] = before;
        if (threadIdx.x == kRunClasses - 1u) runs->count = before + counts[threadIdx.x];
    }
    __syncthreads();
    carried = 0;
    for (uint32_t i = threadIdx.x; i < end; i += kRunThreads) {
        if (end > kRunThreads) rows = rows_of(i, carried);
        if (rows != 0) runs->run[atomicAdd(&at[(256u - rows) / 16u], 1u)] = {i, rows};  // (their order within a class is nobody's concern)
    }
}

template <MxWork WORK>
__global__ __launch_bounds__(256, 1) void k_mx_expert_rows(MxArgs a) {
    constexpr int XF = SHRIKE_MX_E4M3;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const MxRun run = a.runs->run[blockIdx.y];  // (the grid is no higher than the list; one latency with the count's)
    if (blockIdx.y >= a.runs->count) return;
    const shrike_row_tile tile = a.tiles[run.record];
    const uint32_t pair0 = uint32_t(__builtin_amdgcn_readfirstlane(int(tile.pair_start))), row0 = run.record * kRowTile;
    const uint32_t rows = uint32_t(__builtin_amdgcn_readfirstlane(int(run.rows)));
    const uint8_t *base = cell_base_uniform(a.pool, tile.cell, a.stride);
    if (rows > 128u) mx_tile<XF, 8, WORK>(a, lds, blockIdx.x, row0, rows, pair0, base);
    else if (rows > 64u) mx_tile<XF, 4, WORK>(a, lds, blockIdx.x, row0, rows, pair0, base);
    else mx_tile<XF, 2, WORK>(a, lds, blockIdx.x, row0, rows, pair0, base);
}

// ------------------------------------------------------------------ experts of few rows

// Up to 64 rows of one expert's against 128 weight rows by two waves, 64 of them each: for experts of few rows, whose weights are read once
// and whose products the matrix cores have done long before. The same asynchronous loads as above, two chunks of 256 k at a time, and little
// enough LDS that a compute unit holds three workgroups: one's start and end are then the others' middle. 512 tokens over 256 experts of
// 2,048 x 512, 16 rows each and uneven: gate and up 67 us (4.3 TB/s of weights), down 38 (3.8; two chunks a workgroup); by the
// tiles above 116 and 79.
struct MxThinLds {
    static constexpr uint32_t kRows = 32u * 256u, kWeights = 128u * 128u;  // a chunk of each
    static constexpr uint32_t kScales = 2u * (kRows + kWeights), kBytes = kScales + (128u + 32u) * 24u;
    static_assert(2u * kRows + kWeights + (128u + 64u) * 24u <= kBytes);  // (64 rows and one chunk instead)
    static_assert(3u * ((kBytes + 1279u) / 1280u * 1280u) <= 160u * 1024u);  // (it is given out in pieces of 1,280 bytes)
};

// 16 MT rows. (64 take one chunk at a time.) The k of the loop are 256 a step; the scales lie in LDS for three steps, 24 a row.
template <int MT, MxWork WORK, typename Rows>
__device__ __forceinline__ void mx_thin(const MxArgs &a, uint8_t *lds, uint32_t rows, const Rows &which, const uint8_t *base) {
    using L = MxThinLds;
    constexpr uint32_t kPlaces = MT <= 2 ? 2u : 1u, kX = MT <= 2 ? L::kRows : 2u * L::kRows, kPlace = kX + L::kWeights, kScales = kPlaces * kPlace;
    auto place_of = [](uint32_t c) { return kPlaces == 2u ? (c & 1u) * kPlace : 0u; };
    const uint32_t wave = wave_index(), lane = threadIdx.x & 63u, m = lane & 15u, q = lane >> 4;
    const uint32_t blocks = a.k / kMxBlock, chunks = (blocks + 7u) / 8u;
    const uint32_t first = blockIdx.x * (WORK == MxWork::kGateUp ? 64u : 128u);  // output of the workgroup
    // The wave's weight row r of 64: gate and up 32 each. (Rows past the last are the last again, of either operand: nobody stores them.)
    auto weight_row = [&](uint32_t r) { return min(first + (WORK == MxWork::kGateUp ? wave * 32u + r % 32u : wave * 64u + r), a.n - 1u); };
    auto codes_of = [&](uint32_t r) { return WORK == MxWork::kDown ? a.off.down_w_off : r >= 32u ? a.off.up_w_off : a.off.gate_w_off; };
    auto scales_of = [&](uint32_t r) { return WORK == MxWork::kDown ? a.off.down_s_off : r >= 32u ? a.off.up_s_off : a.off.gate_s_off; };
    auto x_row = [&](uint32_t r) -> uint32_t { return which.x_row(min(r, rows - 1u)); };
    const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds));
    // Offsets of a lane's pieces of the first chunk, and of the last piece of the same row, which is asked for again past the row's end.
    uint32_t w_at[8], w_end[8], x_at[2 * MT], x_end[2 * MT];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t r = i * 8u + lane / 8u, start = codes_of(r) + weight_row(r) * blocks * 16u;
        w_at[i] = start + mx_piece(i);
        w_end[i] = start + blocks * 16u - 16u;
    }
#pragma unroll
    for (uint32_t i = 0; i < 2 * MT; ++i) {
        const uint32_t r = (wave * 2u * MT + i) * 4u + lane / 16u, start = x_row(r) * a.k;
        x_at[i] = start + 16u * (m ^ (r % 16u));
        x_end[i] = start + a.k - 16u;
    }
    const uint8_t *const w0 = uniform(base), *const x0 = uniform(a.x + size_t(which.x_row0()) * a.k);
    auto load = [&](uint32_t c) {
        const uint32_t place = lds0 + place_of(c);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) lds_load16(place + kX + wave * 8192u + i * 1024u, w0, min(w_at[i] + c * 128u, w_end[i]));
#pragma unroll
        for (uint32_t i = 0; i < 2 * MT; ++i) lds_load16(place + (wave * 2u * MT + i) * 1024u, x0, min(x_at[i] + c * 256u, x_end[i]));
    };
    // The scales of three chunks, 8 a chunk: a weight row a lane, a row of x by one wave's 32. Where the row has fewer left, its last 8; a row that has not
    // as many is read byte by byte.
    const uint8_t *const w_scales = base + scales_of(lane) + weight_row(lane) * blocks;
    const uint8_t *const x_scales = a.x_scales + size_t(which.x_row0() + x_row(MT <= 2 ? min(lane % 32u, 16u * MT - 1u) : lane)) * blocks;
    uint2 sw[3], sx[3];
    auto scales_from = [&](uint32_t c) { return blocks >= 8u ? min(8u * c, blocks - 8u) : 0u; };
    auto load_scales = [&](uint32_t c) {
        if (blocks >= 8u) {
#pragma unroll
            for (uint32_t i = 0; i < 3; ++i) {
                const u32x2_by1 w = *reinterpret_cast<const u32x2_by1 *>(w_scales + scales_from(c + i));
                const u32x2_by1 x = *reinterpret_cast<const u32x2_by1 *>(x_scales + scales_from(c + i));
                sw[i] = make_uint2(w[0], w[1]);
                sx[i] = make_uint2(x[0], x[1]);
            }
        } else {
            uint32_t w[2] = {0, 0}, x[2] = {0, 0};
#pragma unroll
            for (uint32_t b = 0; b < 7; ++b)
                if (b < blocks) {
                    w[b / 4u] |= uint32_t(w_scales[b]) << 8u * (b % 4u);
                    x[b / 4u] |= uint32_t(x_scales[b]) << 8u * (b % 4u);
                }
            sw[0] = sw[1] = sw[2] = make_uint2(w[0], w[1]);
            sx[0] = sx[1] = sx[2] = make_uint2(x[0], x[1]);
        }
    };
    uint8_t *const scales = lds + kScales;
    auto store_scales = [&] {
        uint2 *to = reinterpret_cast<uint2 *>(scales);
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i) {
            to[threadIdx.x * 3u + i] = sw[i];
            if (threadIdx.x < 16u * MT) to[(128u + threadIdx.x) * 3u + i] = sx[i];
        }
    };
    f32x4 acc[MT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[t][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            asm volatile("" : "+v"(acc[t][i]));  // (a loop that starts from a zero that it can see, the compiler takes apart word by word)
        }
    uint32_t third = 0;  // c % 3
    auto multiply = [&](uint32_t c, uint32_t s, auto last) {
        constexpr bool LAST = decltype(last)::value;
        const uint8_t *rows_at = lds + place_of(c) + m * 256u, *weights = lds + place_of(c) + kX + wave * 8192u + m * 128u;
        const uint32_t b = 8u * c + 4u * s + q, byte = 8u * third + (LAST ? min(b, blocks - 1u) : b) - scales_from(c);
        MxFragment<SHRIKE_MX_E4M3> f[MT];
        uint32_t x_scale[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            f[t].piece[0] = *reinterpret_cast<const u32x4 *>(rows_at + t * 4096u + 16u * ((8u * s + q) ^ m));
            f[t].piece[1] = *reinterpret_cast<const u32x4 *>(rows_at + t * 4096u + 16u * ((8u * s + 4u + q) ^ m));
            x_scale[t] = scales[(128u + 16u * t + m) * 24u + byte];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u32x4 wf = *reinterpret_cast<const u32x4 *>(weights + i * 2048u + 16u * ((4u * s + q) ^ (m >> 1)));
            const uint32_t w_scale = scales[(wave * 64u + 16u * i + m) * 24u + byte];
            if (LAST)
#pragma unroll
                for (int e = 0; e < 4; ++e) wf[e] = b < blocks ? wf[e] : 0u;
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t][i] = mx_multiply<SHRIKE_MX_E4M3>(wf, f[t], acc[t][i], w_scale, x_scale[t]);
        }
        // (the products stay ahead of what follows: they have no effect that would keep the compiler from moving them)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(acc[t][i]));
    };
    load_scales(0);
    load(0);
    if (kPlaces == 2u && chunks > 1u) load(1);
    uint32_t c = 0;
    for (; c + 1u < chunks; ++c) {
        if (third == 0) store_scales();
        wait_loads_and_sync<kPlaces == 2u ? 8 + 2 * MT : 0>();
        multiply(c, 0, std::false_type{});
        multiply(c, 1, std::false_type{});
        __syncthreads();
        if (third == 0 && c + 3u < chunks) load_scales(c + 3u);
        if (c + kPlaces < chunks) load(c + kPlaces);
        third = third == 2u ? 0u : third + 1u;
    }
    if (third == 0) store_scales();
    wait_loads_and_sync<0>();
    multiply(c, 0, std::true_type{});
    if (8u * c + 4u < blocks) multiply(c, 1, std::true_type{});

#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const uint32_t row = 16u * t + m;
        if constexpr (WORK == MxWork::kGateUp) {
            const uint32_t f0 = first + wave * 32u;
            if (f0 >= a.n) return;
            f32x4 gate[2] = {acc[t][0], acc[t][1]}, up[2] = {acc[t][2], acc[t][3]};
            if (a.ebias)
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    gate[i] += mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.gate_ab_off), f0 + 16u * i + 4u * q);
                    up[i] += mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.up_ab_off), f0 + 16u * i + 4u * q);
                }
            const MxActBlock q8 = mx_activate(gate, up, a.act_kind);
            const size_t to_row = which.out_row(row);
            if (row < rows) {
                uint8_t *to = a.act + to_row * a.n + f0 + 4u * q;
                *reinterpret_cast<uint32_t *>(to) = q8.codes[0];
                *reinterpret_cast<uint32_t *>(to + 16) = q8.codes[1];
                if (q == 0) a.act_scales[to_row * (a.n / kMxBlock) + f0 / kMxBlock] = uint8_t(q8.scale);
            }
        } else {
            if (first + wave * 64u >= a.n) return;
            // Through LDS, the rows' halves of 128 bytes, so that whole lines leave; a wave's own half of its weights, which it has read.
            uint8_t *stage = lds + place_of(c + kPlaces - 1u) + kX + wave * 8192u;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                f32x4 v = acc[t][i];
                if (a.ebias) v += mx_bias4(reinterpret_cast<const uint16_t *>(base + a.off.down_ab_off), first + wave * 64u + 16u * i + 4u * q);
                *reinterpret_cast<uint2 *>(stage + row * 128u + 8u * ((4u * i + q) ^ (2u * (m & 7u)))) = mx_pack4(v, SHRIKE_ELEM_F16);
            }
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                const uint32_t r = 16u * t + 8u * i + lane / 8u, n = first + wave * 64u + 8u * (lane % 8u);
                const size_t to_row = which.out_row(r);
                if (r >= rows || n >= a.n) continue;
                *reinterpret_cast<u32x4 *>(a.out + to_row * a.n + n) = *reinterpret_cast<const u32x4 *>(stage + r * 128u + 16u * ((lane % 8u) ^ (r & 7u)));
            }
        }
    }
}

// Rows of a chunk: gate and up take a pair's token's, and leave them in the table's order; down leaves them with the pair's token.
template <MxWork WORK>
struct MxChunkRows {
    uint32_t row0, there;  // `there`: of row `lane`, gate and up its token, down where it goes
    __device__ __forceinline__ uint32_t of(uint32_t r) const { return uint32_t(__shfl(int(there), int(r))); }
    __device__ __forceinline__ uint32_t x_row0() const { return WORK == MxWork::kGateUp ? 0u : row0; }  // (the activations may pass 4 GiB)
    __device__ __forceinline__ uint32_t x_row(uint32_t r) const { return WORK == MxWork::kGateUp ? of(r) : r; }
    __device__ __forceinline__ size_t out_row(uint32_t r) const { return WORK == MxWork::kGateUp ? row0 + r : of(r); }
};
template <MxWork WORK>
__global__ __launch_bounds__(128, 2) void k_mx_expert_thin(MxArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const uint32_t number = blockIdx.y;
    const shrike_row_tile tile = a.tiles[number];  // (the grid is as high as the table; one latency with the count's)
    if (number >= *a.tile_count) return;
    if (tile.cell == kSentinel || tile.rows == 0) return;
    const uint8_t *base = cell_base_uniform(a.pool, tile.cell, a.stride);
    const uint32_t rows = min(uint32_t(__builtin_amdgcn_readfirstlane(int(tile.rows))), kRowTile), pair0 = uint32_t(__builtin_amdgcn_readfirstlane(int(tile.pair_start)));
    const shrike_token_expert_pair p = a.pairs[pair0 + min(threadIdx.x & 63u, rows - 1u)];
    const MxChunkRows<WORK> which = {number * kRowTile, WORK == MxWork::kGateUp ? p.token : p.token * a.top_k + p.rank};
    if (rows > 32u) mx_thin<4, WORK>(a, lds, rows, which, base);
    else if (rows > 16u) mx_thin<2, WORK>(a, lds, rows, which, base);
    else mx_thin<1, WORK>(a, lds, rows, which, base);
}

// Gate and up of single tokens' pairs, up to 16 at the same cell.
struct MxPairRows {
    uint32_t pair, top_k;  // lane m of each 16: row m's
    __device__ __forceinline__ uint32_t of(uint32_t r) const { return uint32_t(__shfl(int(pair), int(r & 15u))); }
    __device__ __forceinline__ uint32_t x_row0() const { return 0; }
    __device__ __forceinline__ uint32_t x_row(uint32_t r) const { return of(r) / top_k; }
    __device__ __forceinline__ size_t out_row(uint32_t r) const { return of(r); }
};
__global__ __launch_bounds__(128, 2) void k_mx_decode_thin(MxArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const uint32_t cell = a.slots[blockIdx.y];
    if (cell == kSentinel) return;
    MxPairRows which = {0, a.top_k};
    const uint32_t rows = same_cell_pairs(a.slots, a.rows * a.top_k, blockIdx.y, cell, which.pair);
    if (rows != 0) mx_thin<1, MxWork::kGateUp>(a, lds, rows, which, cell_base_uniform(a.pool, cell, a.stride));
}

constexpr uint32_t kMxExpertLds = MxTileLds<8>::kBytes;  // the widest instance's

template <int XF, int MT>
static void launch_tiles(const MxArgs &a, hipStream_t s) {
    const uint32_t tiles = (a.n + 255u) / 256u * ((a.rows + 32u * MT - 1u) / (32u * MT));
    hipLaunchKernelGGL((k_mx_product<XF, MT>), dim3((tiles + 7u) / 8u * 8u), dim3(256), MxTileLds<MT>::kBytes, s, a);
}

// By rows and by how many workgroups a shape would have. Measured, us, E4M3 | E2M1 rows:
//                                  64 x 16 outputs, k over 8 waves   64 x 256    128 x 256   256 x 256
//    65 rows of 2,880 x 2,880              11.4 |  7.7              15.7 | 13.7 22.5 | 18.1 35.8 | 25.8
//   128                                    13.6 |  9.0              15.6 | 13.9 22.5 | 18.4 36.6 | 26.8
//   128 rows of 4,096 x 2,304              14.4 |  8.5              13.1 | 11.6 19.1 | 15.7 30.9 | 23.2
//   256 rows of 2,880 x 2,880              19.9 | 12.4              15.7 | 13.9 22.7 | 18.7 36.8 | 27.1
//   256 rows of 4,096 x 2,304              26.8 | 14.9              13.4 | 12.0 19.3 | 16.2 30.9 | 23.6
// 1,024 rows of 2,880 x 2,880              70.5 | 40.0              18.4 | 15.8 24.2 | 20.0 38.2 | 28.5
// 1,536 (288 workgroups of 64 x 256)      101   | 54.8              36.7 | 33.6 25.1 | 21.0 38.7 | 29.2
// 2,048                                   134   | 72.3              36.9 | 34.2 26.2 | 22.1 39.0 | 29.9
// Few workgroups read the rows once each: 384 of them from E4M3's bytes, 768 from E2M1's, are where that costs as much as the tiles' start.
// Up to 64 rows that kernel is taken however many workgroups it has, and of many outputs it loses by that. The same two, calls back to back over
// three sets of weights:
//    17 | 64 rows of  2,880 x 2,880   E4M3  6.6,  7.7 (tiles 14.1, 14.9)   E2M1  5.6,  6.3 (12.4, 13.1)
//                     8,192 x 2,880        10.4, 13.8       (17.7, 18.5)         7.3, 10.4 (16.7, 17.8)
//                    32,768 x 2,304        33.1, 51.4       (15.7, 16.5)        19.3, 27.3 (14.3, 15.0)
//                   201,088 x 2,880         232,  339       ( 148,  158)         134,  243 ( 123,  131)
//     1 | 16 rows of 32,768 x 2,304        13.7, 18.4       (15.3, 15.7)        12.4, 14.5 (14.1, 14.2)
//                   201,088 x 2,880          98,  140       ( 147,  149)          94,  119 ( 121,  123)
// Of the tiles the lowest that are dealt out in one go: a compute unit takes one at a time.
template <int XF>
static int launch_product(const MxArgs &a, hipStream_t s) {
    const uint64_t columns = (a.n + 255u) / 256u, few = uint64_t((a.n + 15u) / 16u) * ((a.rows + 63u) / 64u);
    if (a.rows <= 16u)
        hipLaunchKernelGGL((k_mx_few<XF, 1, 1, 8, 4, MxWork::kDense>), dim3((a.n + 15u) / 16u, 1), dim3(512), 0, s, a);
    else if (a.rows <= 64u || few <= (XF == SHRIKE_MX_E4M3 ? 384u : 768u))
        hipLaunchKernelGGL((k_mx_few<XF, 4, 1, 8, 2, MxWork::kDense>), dim3((a.n + 15u) / 16u, (a.rows + 63u) / 64u), dim3(512), 0, s, a);
    else if (columns * ((a.rows + 63u) / 64u) <= 256u)
        launch_tiles<XF, 2>(a, s);
    else if (columns * ((a.rows + 127u) / 128u) <= 256u)
        launch_tiles<XF, 4>(a, s);
    else
        launch_tiles<XF, 8>(a, s);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}

static bool mx_aligned(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16u == 0; }

// An expert's blob in a cell: what the codes' 16-byte loads and the cell's size allow.
static int check_mx_offsets(const shrike_expert_offsets *o, uint64_t stride, uint32_t d, uint32_t f, bool biases) {
    const uint64_t codes = uint64_t(d) * f / 2u, scales = uint64_t(d) * f / kMxBlock;
    // The kernels' offsets from a cell's start are 32 bits, and those of codes reach up to a line past a row's end ahead of the clamp to it.
    stride = std::min<uint64_t>(stride, 0xffffffffull);
    const uint64_t codes_end = std::min<uint64_t>(stride, 0xffffffffull - 128u);
    SHRIKE_REQUIRE(o->gate_w_off % 16u == 0 && o->up_w_off % 16u == 0 && o->down_w_off % 16u == 0, "mx experts: code offsets must be multiples of 16");
    SHRIKE_REQUIRE(o->gate_w_off + codes <= codes_end && o->up_w_off + codes <= codes_end && o->down_w_off + codes <= codes_end
                       && o->gate_s_off + scales <= stride && o->up_s_off + scales <= stride && o->down_s_off + scales <= stride,
                   "mx experts: a projection of %u x %u does not fit a cell of %llu bytes", d, f, (unsigned long long)stride);
    if (biases) {
        SHRIKE_REQUIRE(o->gate_ab_off % 2u == 0 && o->up_ab_off % 2u == 0 && o->down_ab_off % 2u == 0, "mx experts: bias offsets must be even");
        SHRIKE_REQUIRE(o->gate_ab_off + 2ull * f <= stride && o->up_ab_off + 2ull * f <= stride && o->down_ab_off + 2ull * d <= stride,
                       "mx experts: the biases do not fit a cell of %llu bytes", (unsigned long long)stride);
    }
    return 0;
}

// (of a handle, these calls read the description alone, and first of all: a bare one at its head is refused as a handle's would be)
static_assert(offsetof(shrike_hip_moe, desc) == 0);
static int check_mx_experts(const shrike_hip_moe *moe, const shrike_pool_bases *pool, uint64_t stride, const shrike_expert_offsets *offsets, uint32_t d,
                            uint32_t f, uint32_t top_k) {
    SHRIKE_REQUIRE(moe && pool && offsets, "mx experts: NULL argument");
    SHRIKE_REQUIRE(d == moe->desc.d && f == moe->desc.f, "mx experts: shape %ux%u differs from the handle's %ux%u", d, f, moe->desc.d, moe->desc.f);
    // (a tile's 256 rows of activations are reached by 32 bits)
    SHRIKE_REQUIRE(f <= SHRIKE_MX_MAX_K, "mx experts: f=%u is more than %u", f, SHRIKE_MX_MAX_K);
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
    a.out_whole = mx_aligned(d_out) && (rows == 1u || out_stride_elements % 8u == 0);
    return x_format == SHRIKE_MX_E4M3 ? launch_product<SHRIKE_MX_E4M3>(a, as_stream(stream)) : launch_product<SHRIKE_MX_E2M1>(a, as_stream(stream));
}

size_t shrike_hip_mx_ffn_workspace_bytes(uint32_t max_row_tiles, uint32_t f) {
    return mx_acts(uint64_t(max_row_tiles) * kRowTile, f).total + mx_runs_bytes(max_row_tiles);
}

int shrike_hip_mx_grouped_ffn(shrike_hip_moe *moe, void *stream, const shrike_pool_bases *pool, uint64_t pool_slot_stride,
                              const shrike_expert_offsets *offsets, const shrike_hip_grouped_routes *routes, uint32_t max_row_tiles,
                              const void *d_x_codes, const void *d_x_scales, void *d_route_partials, void *d_workspace, size_t workspace_bytes,
                              uint32_t query_count, uint32_t d, uint32_t f, uint32_t top_k) {
    if (int rc = check_mx_experts(moe, pool, pool_slot_stride, offsets, d, f, top_k)) return rc;
    SHRIKE_REQUIRE(routes && routes->sorted_pairs && routes->row_tiles && routes->row_tile_count, "mx grouped FFN: routes are not bound");
    SHRIKE_REQUIRE(d_x_codes && d_x_scales && d_route_partials && d_workspace, "mx grouped FFN: NULL buffer");
    SHRIKE_REQUIRE(mx_aligned(d_x_codes) && mx_aligned(d_route_partials), "mx grouped FFN: codes and partials must be 16-byte aligned");
    SHRIKE_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 256u == 0, "mx grouped FFN: workspace must be 256-byte aligned");
    // (the rows' codes are reached by 32 bits, and past a row's end ahead of the clamp)
    SHRIKE_REQUIRE(uint64_t(query_count) * d <= 0xffffffffull - 1024u, "mx grouped FFN: %u rows of %u are more than 4 GiB of codes", query_count, d);
    if (query_count == 0 || max_row_tiles == 0) return 0;
    // (an expert's last tile may be partly filled: more tiles than this there cannot be)
    const uint32_t tiles = readable_records(max_row_tiles, uint64_t(query_count) * top_k, moe->desc.num_experts);
    SHRIKE_REQUIRE(tiles <= 65535u, "mx grouped FFN: %u row tiles are too many", tiles);
    const MxActs acts = mx_acts(uint64_t(max_row_tiles) * kRowTile, f);
    const size_t needed = shrike_hip_mx_ffn_workspace_bytes(max_row_tiles, f);
    SHRIKE_REQUIRE(workspace_bytes >= needed, "mx grouped FFN: workspace of %zu bytes, %zu needed", workspace_bytes, needed);
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
    // Experts of few rows are bound by their weights, and by what a workgroup's start and end cost where k is short: measured both ways, the two
    // meet at 50 rows an expert of f 2,880, 130 of 1,024 and 230 of 512. (All three kernels of a chunk, us, workgroups of 64 rows | of
    // 256: f 2,880, d 2,880, 32 experts: 32 rows each 140 | 165, 64: 197 | 183; f 1,024, d 2,304, 256 experts: 64: 302 | 372, 128: 485 |
    // 505, 192: 686 | 590; f 512, d 2,048, 256 experts: 64: 159 | 206, 128: 260 | 294, 256: 471 | 457.)
    const bool thin = uint64_t(query_count) * top_k * f < uint64_t(moe->desc.num_experts) << 17;
    if (!thin) {
        MxRuns *runs = reinterpret_cast<MxRuns *>(a.act + acts.total);
        a.runs = runs;
        hipLaunchKernelGGL(k_mx_expert_runs, dim3(1), dim3(kRunThreads), 0, s, a.tiles, a.tile_count, tiles, runs);
        SHRIKE_HIP(hipGetLastError());
    }
    if (thin) hipLaunchKernelGGL(k_mx_expert_thin<MxWork::kGateUp>, dim3((f + 63u) / 64u, tiles), dim3(128), MxThinLds::kBytes, s, a);
    else hipLaunchKernelGGL(k_mx_expert_rows<MxWork::kGateUp>, dim3((f + 127u) / 128u, tiles), dim3(256), kMxExpertLds, s, a);
    SHRIKE_HIP(hipGetLastError());
    a.x = a.act;
    a.x_scales = a.act_scales;
    a.n = d; a.k = f;
    a.out = static_cast<uint16_t *>(d_route_partials);
    if (thin) hipLaunchKernelGGL(k_mx_expert_thin<MxWork::kDown>, dim3((d + 127u) / 128u, tiles), dim3(128), MxThinLds::kBytes, s, a);
    else hipLaunchKernelGGL(k_mx_expert_rows<MxWork::kDown>, dim3((d + 255u) / 256u, tiles), dim3(256), kMxExpertLds, s, a);
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
    SHRIKE_REQUIRE(tokens <= SHRIKE_MX_MAX_DECODE_TOKENS, "mx decode FFN: %u tokens are too many, %u at most", tokens, SHRIKE_MX_MAX_DECODE_TOKENS);
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
    // Gate and up, a cell's weights through LDS by workgroups that go through all of k, or, where those were fewer than one a compute unit, by four
    // waves with a part of k each: 64 workgroups (8 pairs, f 512) 9.8 us and 8.1, 128 (f 1,024) 10.8 and 9.9, 256 (16 pairs) 12.5 and 14.2,
    // 2,048 (128 pairs) 50 and 60. (2 of gpt-oss's tokens, 360, are the other way about: 25.8 and 23.4.)
    const uint32_t pairs = tokens * top_k, workgroups = (f + 63u) / 64u * pairs;
    if (workgroups >= 256u) hipLaunchKernelGGL(k_mx_decode_thin, dim3((f + 63u) / 64u, pairs), dim3(128), MxThinLds::kBytes, s, a);
    else hipLaunchKernelGGL((k_mx_few<SHRIKE_MX_E4M3, 1, 4, 4, 3, MxWork::kGateUp, 3>), dim3(f / 32u, pairs), dim3(256), 0, s, a);
    SHRIKE_HIP(hipGetLastError());
    a.x = a.act;
    a.x_scales = a.act_scales;
    a.n = d; a.k = f;
    // Down, a token's 32 outputs by eight waves, or 16 by sixteen where those were no more than one a compute unit: 144 workgroups (d 2,304) 8.0 us and
    // 10.5 with half as many, 180 (d 2,880) 10.9 and 13.5, 256 (2 tokens of 2,048) 6.5 and 7.2, 288 13.6 and 10.4, 2,304 (16 tokens) 58 and 38.
    // Every pair reads its expert, however many share it: with few experts that is what bounds a batch (gpt-oss's down, 16 tokens 67 us and 64 tokens 205,
    // where the experts that they use are 25 and 29 us of bytes; 16 tokens over 8 experts of 2,048 x 1,024, all of them each, 27, 2 of bytes).
    if (d / 16u * tokens <= 256u) hipLaunchKernelGGL((k_mx_few<SHRIKE_MX_E4M3, 1, 1, 16, 3, MxWork::kDown>), dim3(d / 16u, tokens), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((k_mx_few<SHRIKE_MX_E4M3, 1, 2, 8, 3, MxWork::kDown>), dim3((d + 31u) / 32u, tokens), dim3(512), 0, s, a);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
