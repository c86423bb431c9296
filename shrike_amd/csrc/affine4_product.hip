// Products with 4-bit weights and a scale (and a bias) a group:
//
//   out[r, i] = sum_g scale[i, g] (sum_{k in g} x[r, k] code[i, k]) + sum_g bias[i, g] (sum_{k in g} x[r, k]) + bias[i]
//
// The weights never become 16-bit weights. A code enters the matrix instruction as it is: the byte 0x0c, c a code, is c * 2^-9 in E4M3 whatever
// the code, and one instruction widens two of them to c in fp16 or bf16. (The fp16 subnormals 0x000c would take two instructions fewer of nine a
// word, and multiply exactly too; but the instruction lines their products up as if they were normal and drops what lies below, 8.5e-6 of
// the result of 2,880 k where this leaves 1e-7.) A group's products are summed by a chain of instructions in fp32 and scaled on the vector unit. The bias term is one more
// short product, of the rows' group sums with the groups' biases, in bf16: an fp32 sum is three bf16 terms, an fp16 bias two, and what
// is left out is below 2^-24 of a product.
#include "prefill_common.h"

#include <type_traits>

namespace shrike {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct Affine4Args {
    const uint16_t *x;
    uint64_t x_stride;  // elements
    const uint8_t *codes;
    const uint16_t *scales, *biases, *bias;
    void *out;
    uint64_t out_stride;  // elements
    uint32_t rows, n, k, group, meta, out_type;
    uint32_t parts;  // k_affine4_few: waves that share an output's k
};

union Affine4Frag {
    half8 h;
    bf8_t b;
    uint32_t u[4];
    uint4 v;
};

// The eight codes of a word in order, as the operand's elements
template <int XT>
__device__ __forceinline__ Affine4Frag affine4_codes(uint32_t w) {
    const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
    const uint32_t bytes[2] = {__builtin_amdgcn_perm(odd, even, 0x05010400u), __builtin_amdgcn_perm(odd, even, 0x07030602u)};
    Affine4Frag f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (XT == SHRIKE_ELEM_F16) {
            f.u[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes[i], 512.0f, false));
            f.u[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes[i], 512.0f, true));
        } else {
            f.u[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes[i], 512.0f, false));
            f.u[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes[i], 512.0f, true));
        }
    }
    return f;
}
template <int XT>
__device__ __forceinline__ f32x16 affine4_multiply(const Affine4Frag &x, const Affine4Frag &w, f32x16 c) {
    if constexpr (XT == SHRIKE_ELEM_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, w.h, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.b, w.b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 affine4_zero() { return f32x16{0}; }

// The sum of the eight values of a piece, on top of c
template <int XT>
__device__ __forceinline__ float affine4_add(const uint4 &v, float c) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (XT == SHRIKE_ELEM_F16) {
            const h2_t one = {_Float16(1.0f), _Float16(1.0f)};
            c = __builtin_amdgcn_fdot2(as_h2(w[i]), one, c, false);
        } else {
            c = __fadd_rn(c, __uint_as_float(w[i] << 16));
            c = __fadd_rn(c, __uint_as_float(w[i] & 0xffff0000u));
        }
    }
    return c;
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{lo, hi}), bf2_t));
}
// A value as three bf16 terms, here two values at a time
__device__ __forceinline__ void bf16_terms(float a, float b, uint32_t (&t)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        t[i] = bf16_pair(a, b);
        a = __fsub_rn(a, __uint_as_float(t[i] << 16));
        b = __fsub_rn(b, __uint_as_float(t[i] & 0xffff0000u));
    }
}

__device__ __forceinline__ void affine4_store(const Affine4Args &a, uint32_t r, uint32_t i, float v) {
    const uint64_t at = uint64_t(r) * a.out_stride + i;
    if (a.out_type == SHRIKE_ELEM_F32) static_cast<float *>(a.out)[at] = v;
    else if (a.out_type == SHRIKE_ELEM_F16) static_cast<uint16_t *>(a.out)[at] = f32_to_f16(v);
    else static_cast<uint16_t *>(a.out)[at] = uint16_t(bf16_pair(v, 0.0f));
}

// Loads from where `at` bytes of a tensor of `bytes` lie, up to its end.
typedef __amdgpu_buffer_rsrc_t buffer_t;
__device__ __forceinline__ buffer_t affine4_buffer(const void *tensor, uint64_t at, uint64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(static_cast<const uint8_t *>(tensor)) + at, 0,
                                             uint32_t(bytes - at < 0xffffffffull ? bytes - at : 0xffffffffull), 0x00020000);
}
__device__ __forceinline__ uint4 affine4_load16(buffer_t b, uint32_t at, uint32_t moving) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b128(b, at, moving, 0);
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// ------------------------------------------------------------------ few rows
//
// Up to 8 R8 rows a workgroup of eight waves; `parts` of them share an output block's k, the others have blocks of their own. A wave's
// block is 32 outputs, a lane's column of it one output. Codes and rows come through LDS, a unit of 256 k (four steps, a line of a row of codes)
// ahead, the codes a wave's own, the rows a part's. While a unit is multiplied, the group sums of its rows are formed beside it, and the bias term of the unit before is added.
//
// In a step lane half h has k = 32 h + 0..31 of both operands (groups of 32: 16 h + 0..15 of either group).

constexpr uint32_t kFewWaves = 8, kFewUnit = 256;  // k a unit
template <int R8>
struct FewLds {
    static constexpr uint32_t kX = 8u * R8 * kFewUnit * 2u;  // a part's rows of a unit
    static constexpr uint32_t kSums = 8u * R8 * 48u;         // their sums: three terms of up to eight groups
    static constexpr uint32_t kPart = 2u * (kX + kSums);     // two places
    static constexpr uint32_t kCodes = 32u * kFewUnit / 2u;  // a wave's codes of a unit
    static constexpr uint32_t bytes(uint32_t parts) { return parts * kPart + kFewWaves * 2u * kCodes; }
};

template <int XT, int GROUP, int R8>
__global__ __launch_bounds__(64 * kFewWaves, R8 == 4 ? 2 : 4) void k_affine4_few(Affine4Args a) {
    typedef FewLds<R8> L;
    constexpr bool SUB32 = GROUP == 32;
    constexpr int kRegs = 4 * R8;  // of a 32 x 32 block, those of the rows there are
    constexpr uint32_t kChains = SUB32 ? 8u : 4u;                      // of a unit
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const uint32_t lane = threadIdx.x & 63u, col = lane & 31u, half = lane >> 5;
    const uint32_t wave = wave_index(), part = wave % a.parts, block = blockIdx.x * (kFewWaves / a.parts) + wave / a.parts;
    const uint32_t row0 = blockIdx.y * 8u * R8, rows = min(a.rows - row0, 8u * R8);
    const uint32_t n0 = block * 32u;
    const uint32_t units = (a.k + kFewUnit - 1u) / kFewUnit, rounds = (units + a.parts - 1u) / a.parts;
    const uint32_t groups = a.k / a.group, pieces = a.k / 8u;
    const bool active = n0 < a.n;

    // a part's units lie one behind the other; the last part may have fewer, or none
    const uint32_t first = part * rounds, mine = first < units ? min(rounds, units - first) : 0u;

    // (outputs past the last are the last again: nobody stores them)
    const uint32_t n_first = min(n0, a.n - 1u);
    const uint8_t *const codes = a.codes + uint64_t(n_first) * (a.k / 2u);
    const buffer_t scales = affine4_buffer(a.scales, uint64_t(n_first) * groups * 2u, uint64_t(a.n) * groups * 2u);
    const buffer_t biases = a.biases ? affine4_buffer(a.biases, uint64_t(n_first) * groups * 2u, uint64_t(a.n) * groups * 2u) : scales;
    const uint32_t my_n = min(n0 + col, a.n - 1u) - n_first, meta_from = my_n * groups * 2u;
    const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds));
    auto x_place = [&](uint32_t p, uint32_t u) { return p * L::kPart + (u & 1u) * L::kX; };
    auto sums_place = [&](uint32_t p, uint32_t u) { return p * L::kPart + 2u * L::kX + (u & 1u) * L::kSums; };

    // The rows of every part's unit u into their places, a step of 64 k (128 bytes a row) behind the other: eight rows a load, eight lanes
    // each, a piece (eight values) a lane. Pieces are xor-ed with half their row's number, so that 16 rows read at one piece touch each bank
    // once; past k stands the row's last piece.
    constexpr uint32_t kStepX = 8u * R8 * 128u;
    auto load_x = [&](uint32_t u) {
        const uint32_t eights = (rows + 7u) / 8u, swizzled = lane & 7u, r8 = lane >> 3;
        for (uint32_t i = wave; i < a.parts * 4u * eights; i += kFewWaves) {
            const uint32_t s = i & 3u, p = (i >> 2) / eights, r = 8u * ((i >> 2) - p * eights) + r8;
            const uint32_t piece = (p * rounds + u) * (kFewUnit / 8u) + 8u * s;
            if (piece >= pieces) continue;
            lds_load16(lds0 + x_place(p, u) + s * kStepX + (r - r8) * 128u,
                       a.x + uint64_t(row0 + min(r, rows - 1u)) * a.x_stride + min(piece + (swizzled ^ ((r >> 1) & 7u)), pieces - 1u) * 8u);
        }
    };
    auto read_x = [&](uint32_t place, uint32_t s, uint32_t r, uint32_t piece) {
        return *reinterpret_cast<const uint4 *>(lds + place + s * kStepX + r * 128u + ((piece ^ ((r >> 1) & 7u)) * 16u));
    };

    // The wave's codes of unit u into its place: a line (128 bytes) of eight rows a load, eight lanes a row, xor-ed as the rows of x are; past
    // the row's end stands its last piece.
    const uint32_t lds_codes = a.parts * L::kPart + wave * 2u * L::kCodes;
    const uint32_t code_pieces = a.k / 32u, line_piece = (lane & 7u) ^ (lane >> 4);  // (xor-ed with 4 in every second load)
    uint32_t line_at[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) line_at[j] = (min(n0 + 8u * j + (lane >> 3), a.n - 1u) - n_first) * (a.k / 2u);
    struct Unit {
        uint32_t s[kChains / 2], b[kChains / 2];
    };
    auto load_unit = [&](Unit &t, uint32_t u) {
        const uint32_t unit = first + u, to = lds0 + lds_codes + (u & 1u) * L::kCodes;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            lds_load16(to + j * 1024u, codes, line_at[j] + min(unit * 8u + (line_piece ^ (4u * (j & 1u))), code_pieces - 1u) * 16u);
        // a unit's groups: four, or two of 128 to be taken twice, or eight of 32; one by one where the row has fewer left
        constexpr uint32_t per = kFewUnit / GROUP; const uint32_t g = unit * per;
        auto metas = [&](buffer_t from, uint32_t (&to)[kChains / 2]) {
            if (g + per > groups) {
#pragma unroll
                for (uint32_t j = 0; j < kChains; ++j) {
                    const uint32_t at = min(GROUP == 128 ? g + j / 2u : g + j, groups - 1u);
                    const uint32_t v = __builtin_amdgcn_raw_buffer_load_b16(from, meta_from, at * 2u, 0);
                    to[j / 2u] = j % 2u ? to[j / 2u] | v << 16 : v;
                }
            } else if constexpr (SUB32) {
                const uint4 v = affine4_load16(from, meta_from, g * 2u);
                to[0] = v.x;
                to[1] = v.y;
                to[2] = v.z;
                to[3] = v.w;
            } else if constexpr (GROUP == 64) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(from, meta_from, g * 2u, 0);
                to[0] = v[0];
                to[1] = v[1];
            } else {
                const uint32_t v = __builtin_amdgcn_raw_buffer_load_b32(from, meta_from, g * 2u, 0);
                to[0] = (v & 0xffffu) * 0x10001u;
                to[1] = (v >> 16) * 0x10001u;
            }
        };
        metas(scales, t.s);
        metas(biases, t.b);
    };
    auto meta_at = [&](const uint32_t (&m)[kChains / 2], uint32_t c) { return meta_f32(uint16_t(m[c / 2u] >> 16u * (c % 2u)), a.meta); };

    float acc[kRegs];
#pragma unroll
    for (int r = 0; r < kRegs; ++r) acc[r] = 0.0f;

    const uint32_t my_row = min(col, rows - 1u);  // the row of LDS that a lane's row of the operand is (rows past the last: the last)

    auto multiply = [&](const Unit &t, uint32_t u, auto whole) {
        const uint32_t left = decltype(whole)::value ? kFewUnit : a.k - (first + u) * kFewUnit;  // of the row, from this unit on
        const uint8_t *const my_codes = lds + lds_codes + (u & 1u) * L::kCodes + col * 128u;
#pragma unroll
        for (uint32_t s = 0; s < 4; ++s) {
            if (64u * s >= left) break;
            const uint4 v = *reinterpret_cast<const uint4 *>(my_codes + (((2u * s + half) ^ ((col >> 1) & 7u)) * 16u));
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            if constexpr (SUB32) {
                // lane half h has group h of the step: its halves to both (past the row's end there is no second group)
                if (64u * s + 32u >= left)
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = half ? 0u : w[j];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const auto r = __builtin_amdgcn_permlane32_swap(w[j], w[j + 2], false, false);
                    w[j] = r[0];
                    w[j + 2] = r[1];
                }
            }
            Affine4Frag f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = affine4_codes<XT>(w[j]);
            constexpr int kPer = SUB32 ? 2 : 4;
#pragma unroll
            for (int c = 0; c < 4 / kPer; ++c) {
                f32x16 p = affine4_zero();
#pragma unroll
                for (uint32_t j = c * kPer; j < c * kPer + kPer; ++j) {
                    Affine4Frag x;
                    x.v = read_x(x_place(part, u), s, my_row, SUB32 ? 4u * c + 2u * half + j % 2u : 4u * half + j);
                    p = affine4_multiply<XT>(x, f[j], p);
                }
                const float scale = meta_at(t.s, SUB32 ? 2u * s + c : s);
#pragma unroll
                for (int r = 0; r < kRegs; ++r) acc[r] = fmaf(scale, p[r], acc[r]);
            }
        }
    };
    // The group sums of every part's unit u, as three bf16 terms of each: a lane a piece, eight lanes (four) a group.
    auto form_sums = [&](uint32_t u) {
        for (uint32_t i = threadIdx.x; i < a.parts * rows * 32u; i += 64u * kFewWaves) {
            const uint32_t piece = i % 32u, r = i / 32u % rows, p = i / 32u / rows, at = (p * rounds + u) * kFewUnit + 8u * piece;
            float sum = affine4_add<XT>(read_x(x_place(p, u), piece / 8u, r, piece % 8u), 0.0f);
            sum = at < a.k ? sum : 0.0f;
            sum = __fadd_rn(sum, dpp_f32<0xB1>(sum));
            sum = __fadd_rn(sum, dpp_f32<0x4E>(sum));
            if constexpr (!SUB32) sum = __fadd_rn(sum, dpp_f32<0x141>(sum));  // row_half_mirror
            uint32_t terms[3];
            bf16_terms(sum, 0.0f, terms);
            constexpr uint32_t kLanes = 32u / kChains;
            uint16_t *to = reinterpret_cast<uint16_t *>(lds + sums_place(p, u) + r * 48u) + piece / kLanes;
            if (piece % kLanes == 0)
#pragma unroll
                for (int j = 0; j < 3; ++j) to[8 * j] = uint16_t(terms[j]);
            if (!SUB32 && piece % kLanes == 1)
#pragma unroll
                for (int j = 0; j < 3; ++j) to[8 * j + 4] = 0;
        }
    };
    // The bias term of unit u: its sums' terms against the biases, an fp16 bias as two bf16 terms.
    auto add_bias = [&](const uint32_t (&b)[kChains / 2], uint32_t u) {
        Affine4Frag high, low, high0;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) high.u[j] = low.u[j] = 0;
        const bool as_they_are = a.meta == SHRIKE_META_BF16 && a.biases;
#pragma unroll
        for (uint32_t j = 0; j < kChains / 2u; ++j) {
            if (as_they_are) {
                high.u[j] = b[j];
                continue;
            }
            const float factor = a.biases ? 1.0f : -8.0f;
            uint32_t terms[3];
            bf16_terms(meta_at(b, 2u * j) * factor, meta_at(b, 2u * j + 1u) * factor, terms);
            high.u[j] = terms[0];
            low.u[j] = terms[1];
        }
        // half 0 of the lanes adds the sums' high terms, half 1 the middle ones, then half 0 the low ones, each against the high bias
#pragma unroll
        for (int j = 0; j < 4; ++j) high0.u[j] = half ? 0u : high.u[j];
        const uint8_t *sums = lds + sums_place(part, u) + my_row * 48u;
        Affine4Frag both, rest;
        both.v = *reinterpret_cast<const uint4 *>(sums + 16u * half);
        rest.v = *reinterpret_cast<const uint4 *>(sums + 32u);
        f32x16 p = __builtin_amdgcn_mfma_f32_32x32x16_bf16(both.b, high.b, affine4_zero(), 0, 0, 0);
        p = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rest.b, high0.b, p, 0, 0, 0);
        if (a.meta == SHRIKE_META_F16) p = __builtin_amdgcn_mfma_f32_32x32x16_bf16(both.b, low.b, p, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < kRegs; ++r) acc[r] = __fadd_rn(acc[r], p[r]);
    };

    Unit t[2];
    uint32_t kept[kChains / 2];  // the biases of the unit before
    load_x(0);
    if (active && mine) load_unit(t[0], 0);
    auto phase = [&](Unit &now, Unit &next, uint32_t u) {
        // all that the unit needs has landed, for every wave; and nobody reads the places of the one before any more
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), in the compiler's own count too
        wait_loads_and_sync<0>();
        if (u + 1u < rounds) load_x(u + 1u);
        if (active && u + 1u < mine) load_unit(next, u + 1u);
        form_sums(u);
        if (active && u && u - 1u < mine) add_bias(kept, u - 1u);
        if (active && u < mine) {
            if ((first + u + 1u) * kFewUnit <= a.k) multiply(now, u, std::true_type{});
            else multiply(now, u, std::false_type{});
#pragma unroll
            for (uint32_t j = 0; j < kChains / 2u; ++j) kept[j] = now.b[j];
        }
    };
    for (uint32_t u = 0; u < rounds; u += 2u) {
        phase(t[0], t[1], u);
        if (u + 1u < rounds) phase(t[1], t[0], u + 1u);
    }
    __syncthreads();
    if (active && mine == rounds) add_bias(kept, rounds - 1u);

    auto store = [&](uint32_t r, float v) {
        const uint32_t row = 8u * (r / 4u) + 4u * half + r % 4u, n = n0 + col;
        if (row < rows && n < a.n) affine4_store(a, row0 + row, n, a.bias ? __fadd_rn(v, meta_f32(a.bias[n], a.meta)) : v);
    };
    if (a.parts == 1u) {
        if (!active) return;
#pragma unroll
        for (uint32_t r = 0; r < kRegs; ++r) store(r, acc[r]);
        return;
    }
    // the parts' sums meet in LDS; every part adds up some of the registers
    float *meet = reinterpret_cast<float *>(lds);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRegs; ++r) meet[(wave * kRegs + r) * 64u + lane] = acc[r];
    __syncthreads();
    if (!active) return;
    for (uint32_t r = part; r < uint32_t(kRegs); r += a.parts) {
        float v = 0.0f;
        for (uint32_t p = 0; p < a.parts; ++p) v = __fadd_rn(v, meet[((wave - part + p) * kRegs + r) * 64u + lane]);
        store(r, v);
    }
}

template <int XT, int GROUP, int R8>
static int launch_few(const Affine4Args &args, hipStream_t s) {
    typedef FewLds<R8> L;
    Affine4Args a = args;
    const uint32_t blocks = (a.n + 31u) / 32u, tiles = (a.rows + 8u * R8 - 1u) / (8u * R8), units = (a.k + kFewUnit - 1u) / kFewUnit;
    a.parts = 1;
    while (a.parts < 8u && L::bytes(2u * a.parts) <= 160u * 1024u && a.parts * 2u <= units && uint64_t(blocks) * tiles * a.parts < 8u * 256u) a.parts *= 2u;
    const uint32_t bytes = L::bytes(a.parts);
    static_assert(kFewWaves * 4u * R8 * 256u <= L::bytes(1), "the parts' sums fit");
    const uint32_t per = kFewWaves / a.parts;
    hipLaunchKernelGGL((k_affine4_few<XT, GROUP, R8>), dim3((blocks + per - 1u) / per, tiles), dim3(64u * kFewWaves), bytes, s, a);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}
template <int XT, int GROUP>
static int launch_affine4(const Affine4Args &a, hipStream_t s) {
    if (a.rows <= 8u) return launch_few<XT, GROUP, 1>(a, s);
    const uint64_t blocks = (a.n + 31u) / 32u;
    if (a.rows <= 16u || blocks * ((a.rows + 31u) / 32u) < 512u) return launch_few<XT, GROUP, 2>(a, s);
    return launch_few<XT, GROUP, 4>(a, s);
}
template <int XT>
static int launch_affine4(const Affine4Args &a, hipStream_t s) {
    if (a.group == 32u) return launch_affine4<XT, 32>(a, s);
    return a.group == 64u ? launch_affine4<XT, 64>(a, s) : launch_affine4<XT, 128>(a, s);
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
    a.meta = meta_dtype;
    a.out_type = out_dtype;
    constexpr uint32_t kMost = 16u * 65535u;  // rows of a launch: a grid's second dimension ends at 65,535
    for (uint32_t first = 0; first < rows; first += kMost) {
        Affine4Args part = a;
        part.x += uint64_t(first) * a.x_stride;
        part.out = static_cast<uint8_t *>(a.out) + uint64_t(first) * a.out_stride * (out_dtype == SHRIKE_ELEM_F32 ? 4u : 2u);
        part.rows = std::min(rows - first, kMost);
        const hipStream_t s = as_stream(stream);
        const int rc = x_dtype == SHRIKE_ELEM_F16 ? launch_affine4<SHRIKE_ELEM_F16>(part, s) : launch_affine4<SHRIKE_ELEM_BF16>(part, s);
        if (rc) return rc;
    }
    return 0;
}
