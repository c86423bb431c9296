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
#include <utility>

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
            const bf2_t one = {__bf16(1.0f), __bf16(1.0f)};
            c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2_t, w[i]), one, c, false);
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

// ------------------------------------------------------------------ one row
//
// A matrix-vector product is the reading of its weights. Lanes side by side read a row's 16-byte chunks (32 codes) side by side: 2^shift lanes a
// row, NCH chunks each, so that rows of any length leave few lanes idle (90 chunks of 2,880 k are three steps of 32 lanes, 94 %). A wave holds its
// slices of x in registers and takes a batch of rows a turn, turn after turn. (A row of x too long for that is read piece by piece with every turn.)
// The memory bounds it: 201,088 x 2,880 takes 65 us, 5.0 TB/s of all its bytes; 65,536 x 8,192 63 us, 4.7 TB/s. (A lane a row with x in LDS took 123 us of
// the first.) A small one is its launch: 2,048 x 2,048 3.8 us on the GPU.
constexpr int kGemvChunks = 6;
template <int NCH>
constexpr int kGemvBatch = NCH <= 2 ? 4 : 2;  // rows a lane and turn: four to twelve loads of codes on their way

struct GemvSlice {
    uint32_t p[16];  // 32 values as pairs, in the order that the codes come in
    float sum;
};
// fp16: pairs (0, 4) (1, 5) (2, 6) (3, 7) of eight; bf16: in order
template <int XT>
__device__ __forceinline__ void gemv_slice(GemvSlice &x, const uint4 (&v)[4]) {
    x.sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (XT == SHRIKE_ELEM_F16) {
            h2_t p[4];
            pairs_from_x8(v[j], p);
#pragma unroll
            for (int i = 0; i < 4; ++i) x.p[4 * j + i] = as_u32(p[i]);
        } else {
            x.p[4 * j] = v[j].x;
            x.p[4 * j + 1] = v[j].y;
            x.p[4 * j + 2] = v[j].z;
            x.p[4 * j + 3] = v[j].w;
        }
        x.sum = affine4_add<XT>(v[j], x.sum);
    }
}
template <int XT>
__device__ __forceinline__ float gemv_dot(const uint4 &w, const GemvSlice &x) {
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    if constexpr (XT == SHRIKE_ELEM_F16) {
        // a code in the low bits of 1024, or four bits further up in 64, is that number and the code; less the number it is the code, as a normal
        // fp16 (of the subnormals that need no subtraction this instruction, too, drops what lies low: 4e-6 of the result of 2,880 k for 1e-7)
        const h2_t k1024 = {_Float16(1024.0f), _Float16(1024.0f)}, k64 = {_Float16(64.0f), _Float16(64.0f)};
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t lo = words[j], hi = words[j] >> 8;
            sum = __builtin_amdgcn_fdot2(as_h2((lo & 0x000f000fu) | 0x64006400u) - k1024, as_h2(x.p[4 * j]), sum, false);
            sum = __builtin_amdgcn_fdot2(as_h2((lo & 0x00f000f0u) | 0x54005400u) - k64, as_h2(x.p[4 * j + 1]), sum, false);
            sum = __builtin_amdgcn_fdot2(as_h2((hi & 0x000f000fu) | 0x64006400u) - k1024, as_h2(x.p[4 * j + 2]), sum, false);
            sum = __builtin_amdgcn_fdot2(as_h2((hi & 0x00f000f0u) | 0x54005400u) - k64, as_h2(x.p[4 * j + 3]), sum, false);
        }
        return sum;
    } else {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const Affine4Frag f = affine4_codes<XT>(words[j]);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2_t, f.u[i]), __builtin_bit_cast(bf2_t, x.p[4 * j + i]), sum, false);
        }
        return sum;
    }
}

template <int XT, int NCH>
__global__ __launch_bounds__(256) void k_affine4_gemv(Affine4Args a, uint32_t shift, uint32_t turns) {
    const uint32_t lane = threadIdx.x & 63u, wave = blockIdx.x * 4u + wave_index(), waves = gridDim.x * 4u;
    const uint32_t cpr = a.k / 32u, per_row = a.k / 2u, groups = a.k / a.group, lanes = 1u << shift, rows = 64u >> shift;
    const uint32_t sub = lane >> shift, col = lane & (lanes - 1u), group_shift = a.group == 32u ? 0u : a.group == 64u ? 1u : 2u;
    const uint32_t segments = (cpr + NCH * lanes - 1u) / (NCH * lanes);
    GemvSlice x[NCH];
    auto load_x = [&](uint32_t segment) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const uint32_t c = (segment * NCH + i) * lanes + col;
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = reinterpret_cast<const uint4 *>(a.x)[min(c, cpr - 1u) * 4u + j];
                if (c >= cpr) v[j] = zero4();  // past the row's end the lane counts for nothing
            }
            gemv_slice<XT>(x[i], v);
        }
    };
    if (segments == 1u) load_x(0);
    for (uint32_t turn = 0; turn < turns; ++turn) {
        const uint32_t first = (turn * waves + wave) * kGemvBatch<NCH> * rows;
        if (first >= a.n) return;
        uint32_t n[kGemvBatch<NCH>];
        float acc[kGemvBatch<NCH>];
#pragma unroll
        for (int r = 0; r < kGemvBatch<NCH>; ++r) {
            n[r] = first + r * rows + sub;
            acc[r] = 0.0f;
        }
        for (uint32_t segment = 0; segment < segments; ++segment) {
            uint4 w[kGemvBatch<NCH>][NCH];
            uint16_t s[kGemvBatch<NCH>][NCH], b[kGemvBatch<NCH>][NCH];
#pragma unroll
            for (int r = 0; r < kGemvBatch<NCH>; ++r) {
                const uint32_t row = min(n[r], a.n - 1u);
                const uint8_t *codes = a.codes + uint64_t(row) * per_row;
                const uint16_t *scales = a.scales + uint64_t(row) * groups, *biases = (a.biases ? a.biases : a.scales) + uint64_t(row) * groups;
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const uint32_t c = min((segment * NCH + i) * lanes + col, cpr - 1u), g = c >> group_shift;
                    const u32x4_t *from = reinterpret_cast<const u32x4_t *>(codes) + c;
                    const u32x4_t v = __builtin_nontemporal_load(from);  // (201,088 x 2,880: 67.5 us without the hint, 66.3 with it; weights that a cache holds: as fast)
                    w[r][i] = make_uint4(v.x, v.y, v.z, v.w);
                    s[r][i] = scales[g];
                    b[r][i] = biases[g];
                }
            }
            if (segments > 1u) load_x(segment);
#pragma unroll
            for (int r = 0; r < kGemvBatch<NCH>; ++r)
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const float scale = meta_f32(s[r][i], a.meta), bias = a.biases ? meta_f32(b[r][i], a.meta) : -8.0f * scale;
                    acc[r] = fmaf(bias, x[i].sum, fmaf(scale, gemv_dot<XT>(w[r][i], x[i]), acc[r]));
                }
        }
#pragma unroll
        for (int r = 0; r < kGemvBatch<NCH>; ++r) acc[r] = seg_sum(acc[r], lanes);
#pragma unroll
        for (int r = 0; r < kGemvBatch<NCH>; ++r)
            if (col == lanes - 1u && n[r] < a.n) affine4_store(a, 0, n[r], a.bias ? __fadd_rn(acc[r], meta_f32(a.bias[n[r]], a.meta)) : acc[r]);
    }
}

template <int XT, int NCH>
static int launch_gemv(const Affine4Args &a, uint32_t shift, hipStream_t s) {
    // as many workgroups as the device holds at once; where there are more rows, each takes several turns, all of them as many
    const uint64_t batches = (a.n + kGemvBatch<NCH> * (64u >> shift) - 1u) / (kGemvBatch<NCH> * (64u >> shift)), groups_of_waves = (batches + 3u) / 4u;
    const uint32_t most = 256u * (NCH == 1 ? 5u : NCH <= 4 ? 3u : 2u), turns = uint32_t((groups_of_waves + most - 1u) / most);
    const uint32_t workgroups = uint32_t((groups_of_waves + turns - 1u) / turns);
    hipLaunchKernelGGL((k_affine4_gemv<XT, NCH>), dim3(workgroups), dim3(256), 0, s, a, shift, turns);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}
template <int XT>
static int launch_gemv(const Affine4Args &a, hipStream_t s) {
    // the lanes a row: of those whose share fits, the one that leaves the fewest idle, and of equals the most
    const uint32_t cpr = a.k / 32u;
    uint32_t best = 6, steps = kGemvChunks, idle = ~0u;
    for (uint32_t shift = 6; shift >= 2u; --shift) {
        const uint32_t n = ((cpr - 1u) >> shift) + 1u;
        if (n > uint32_t(kGemvChunks)) break;
        const uint32_t left = ((n << shift) - cpr) * 256u / (n << shift);
        if (left + 8u < idle) {  // (a gain of 3 % is worth its registers)
            idle = left;
            best = shift;
            steps = n;
        }
    }
    switch (steps) {
    case 1: return launch_gemv<XT, 1>(a, best, s);
    case 2: return launch_gemv<XT, 2>(a, best, s);
    case 3: return launch_gemv<XT, 3>(a, best, s);
    case 4: return launch_gemv<XT, 4>(a, best, s);
    case 5: return launch_gemv<XT, 5>(a, best, s);
    default: return launch_gemv<XT, 6>(a, best, s);
    }
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
// ahead, the rows a part's in two places, the codes a wave's own in one: they go on into registers before the next are asked for. While a unit is
// multiplied, the group sums of its rows are formed beside it, and the bias term of the unit before is added. What bounds it is waiting: a unit's loads have
// only the unit before to hide behind, and the waves meet at every unit. Of their time they wait 40 to 58 % (300 rows of 4,096 x 2,048 40, 64 of 16,384 x
// 2,304 53, 8 of 5,120 x 2,880 58); the vector unit is busy 51, 40 and 32 %, the matrix unit 16, 9 and 8. Of some 300 instructions a unit and wave 144 take
// the codes apart and 16 multiply. (Two sets of sums, so that one chain is scaled while the
// next is multiplied, took the registers of two waves and 3 us more of 22; two copies of the loop for the scales of two units no less time.)
// 8 rows of 5,120 x 2,880: 8.7 us; 37 of 2,049 x 2,304: 10.4; 64 of 16,384 x 2,304: 23.2 (0.86 TB/s of weights, 208 TFLOP/s).
//
// In a step lane half h has k = 32 h + 0..31 of both operands (groups of 32: 16 h + 0..15 of either group).

constexpr uint32_t kFewWaves = 8, kFewUnit = 256;  // k a unit
template <int R8>
struct FewLds {
    static constexpr uint32_t kX = 8u * R8 * kFewUnit * 2u;  // a part's rows of a unit
    static constexpr uint32_t kSums = 8u * R8 * 48u;         // their sums: three terms of up to eight groups
    static constexpr uint32_t kPart = 2u * (kX + kSums);     // two places
    static constexpr uint32_t kCodes = 32u * kFewUnit / 2u;  // a wave's codes of a unit
    static constexpr uint32_t bytes(uint32_t parts) { return parts * kPart + kFewWaves * kCodes; }
};

template <int XT, int GROUP, int R8>
__global__ __launch_bounds__(64 * kFewWaves, 2) void k_affine4_few(Affine4Args a) {
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
        const uint32_t swizzled = lane & 7u, r8 = lane >> 3;
        for (uint32_t i = wave; i < a.parts * 4u * R8; i += kFewWaves) {
            const uint32_t s = i & 3u, p = (i >> 2) / R8, eight = (i >> 2) % R8, r = 8u * eight + r8;
            const uint32_t piece = (p * rounds + u) * (kFewUnit / 8u) + 8u * s;
            if (8u * eight >= rows || piece >= pieces) continue;
            lds_load16(lds0 + x_place(p, u) + s * kStepX + (r - r8) * 128u,
                       a.x + uint64_t(row0 + min(r, rows - 1u)) * a.x_stride + min(piece + (swizzled ^ ((r >> 1) & 7u)), pieces - 1u) * 8u);
        }
    };
    auto read_x = [&](uint32_t place, uint32_t s, uint32_t r, uint32_t piece) {
        return *reinterpret_cast<const uint4 *>(lds + place + s * kStepX + r * 128u + ((piece ^ ((r >> 1) & 7u)) * 16u));
    };

    // The wave's codes of unit u into its place: a line (128 bytes) of eight rows a load, eight lanes a row, xor-ed as the rows of x are; past
    // the row's end stands its last piece.
    const uint32_t lds_codes = a.parts * L::kPart + wave * L::kCodes;
    const uint32_t code_pieces = a.k / 32u, line_piece = (lane & 7u) ^ (lane >> 4);  // (xor-ed with 4 in every second load)
    uint32_t line_at[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) line_at[j] = (min(n0 + 8u * j + (lane >> 3), a.n - 1u) - n_first) * (a.k / 2u);
    struct Unit {
        uint32_t s[kChains / 2], b[kChains / 2];
    };
    auto load_unit = [&](Unit &t, uint32_t u) {
        const uint32_t unit = first + u, to = lds0 + lds_codes;
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

    auto multiply = [&](const Unit &t, const uint4 (&codes)[4], uint32_t u, auto whole) {
        const uint32_t left = decltype(whole)::value ? kFewUnit : a.k - (first + u) * kFewUnit;  // of the row, from this unit on
#pragma unroll
        for (uint32_t s = 0; s < 4; ++s) {
            if (64u * s >= left) break;
            uint32_t w[4] = {codes[s].x, codes[s].y, codes[s].z, codes[s].w};
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
        for (uint32_t i = threadIdx.x; i < a.parts * 256u * R8; i += 64u * kFewWaves) {
            const uint32_t piece = i % 32u, r = i / 32u % (8u * R8), p = i / (256u * R8), at = (p * rounds + u) * kFewUnit + 8u * piece;
            if (r >= rows) continue;
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

    Unit next;
    uint32_t kept[kChains / 2];  // the biases of the unit before
    load_x(0);
    if (active && mine) load_unit(next, 0);
    for (uint32_t u = 0; u < rounds; ++u) {
        // all that the unit needs has landed, for every wave; and nobody reads the places of the one before any more
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), in the compiler's own count too
        wait_loads_and_sync<0>();
        const Unit now = next;
        // the unit's codes into registers, and the next ones into their place
        uint4 raw[4];
#pragma unroll
        for (uint32_t s = 0; s < 4; ++s) raw[s] = *reinterpret_cast<const uint4 *>(lds + lds_codes + col * 128u + (((2u * s + half) ^ ((col >> 1) & 7u)) * 16u));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (u + 1u < rounds) load_x(u + 1u);
        if (active && u + 1u < mine) load_unit(next, u + 1u);
        form_sums(u);
        if (active && u && u - 1u < mine) add_bias(kept, u - 1u);
        if (active && u < mine) {
            if ((first + u + 1u) * kFewUnit <= a.k) multiply(now, raw, u, std::true_type{});
            else multiply(now, raw, u, std::false_type{});
#pragma unroll
            for (uint32_t j = 0; j < kChains / 2u; ++j) kept[j] = now.b[j];
        }
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

// The parts that share k: twice as many as long as every CU has at most one workgroup and every part a unit. A second one costs what the halved k gives:
// 64 rows of 5,120 x 2,880 take 20 us in two parts (160 workgroups), 26 in four (320).
template <int R8>
static uint64_t few_workgroups(const Affine4Args &a, uint32_t parts) {
    const uint32_t blocks = (a.n + 31u) / 32u, per = kFewWaves / parts;
    return uint64_t((blocks + per - 1u) / per) * ((a.rows + 8u * R8 - 1u) / (8u * R8));
}
template <int R8>
static uint32_t few_parts(const Affine4Args &a) {
    const uint32_t units = (a.k + kFewUnit - 1u) / kFewUnit;
    uint32_t parts = 1;
    while (parts < kFewWaves && FewLds<R8>::bytes(2u * parts) <= 160u * 1024u && parts * 2u <= units && few_workgroups<R8>(a, 2u * parts) <= 256u) parts *= 2u;
    return parts;
}
template <int XT, int GROUP, int R8>
static int launch_few(const Affine4Args &args, hipStream_t s) {
    typedef FewLds<R8> L;
    Affine4Args a = args;
    a.parts = few_parts<R8>(a);
    const uint32_t blocks = (a.n + 31u) / 32u, tiles = (a.rows + 8u * R8 - 1u) / (8u * R8), bytes = L::bytes(a.parts);
    static_assert(kFewWaves * 4u * R8 * 256u <= L::bytes(1), "the parts' sums fit");
    const uint32_t per = kFewWaves / a.parts;
    hipLaunchKernelGGL((k_affine4_few<XT, GROUP, R8>), dim3((blocks + per - 1u) / per, tiles), dim3(64u * kFewWaves), bytes, s, a);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}
// ------------------------------------------------------------------ many rows
//
// 32 MT WM rows against 32 NT WN outputs a workgroup of KS parts of WM x WN waves, 32 MT x 32 NT a wave; the parts have a share of k each and their sums meet
// in LDS. Rows and codes come through LDS, a step of 64 k of the rows two steps ahead in three places, two steps of the codes (64 bytes a row) in two. A
// chunk is eight chains (a chain is a group's products, or half a group's of 128): its scales and biases come through LDS too, a chunk ahead, and the
// bias term is added a chunk behind from the sums of the rows' groups, which the waves form from the operands that they hold, WN waves a share of the
// tile's rows each. A wave takes a code apart for MT blocks of rows, and scales a chain while the next is multiplied.
//
// What bounds it is the issue of instructions beside the matrix ones: a step of a wave of 128 x 64 has 32 of these, 1,024 cycles, and some 390 of the vector
// unit, half of them the scaling; the vector unit is busy 54 % of the time and the matrix unit 39. 4,096 rows of 8,192 x 4,096:
// 322 to 338 us by the card, 815 to 855 TFLOP/s (a large fp16 product of the library, whose weights are not taken apart, 227); 512 of 8,192 x 2,048: 34 us. Without the loads the large one takes 12 % less, without the group sums 10 to 15. In two parts of k a CU
// with one small tile has two waves a SIMD: 512 of 8,192 x 2,048 39 us against 44.

// Four bytes a lane into LDS, as lds_load16
__device__ __forceinline__ void lds_load4(uint32_t lds, const void *base, uint32_t offset) {
    const void *moved;
    asm volatile("s_mov_b64 %0, %3\n\tglobal_load_lds_dword %2, %0" : "=&s"(moved) : "{m0}"(lds), "v"(offset), "s"(base) : "memory");
}

template <class Call, int... I>
__device__ __forceinline__ void each_of(Call &&call, std::integer_sequence<int, I...>) {
    (call(std::integral_constant<int, I>{}), ...);
}

// The lane's number, new at every call
__device__ __forceinline__ uint32_t lane_number() {
    uint32_t l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
    return l;
}

template <int MT, int NT, int WM, int WN, int P, int KS>
struct TileLds {
    static constexpr uint32_t kRows = 32u * MT * WM, kOuts = 32u * NT * WN, kWaves = WM * WN;
    static constexpr uint32_t kX = kRows * 128u;    // a step's rows
    static constexpr uint32_t kB = kOuts * 64u;     // two steps' codes
    static constexpr uint32_t kSums = kRows * 48u;  // a chunk's sums, three bf16 terms each
    static constexpr uint32_t kUnits = (P + 2u) / 2u;  // places of the codes: what is asked for beside a step is needed after its rows
    static constexpr uint32_t kCodes = P * kX, kSum = kCodes + kUnits * kB, kScales = kSum + kSums;
    // a chunk's scales (or biases) of a wave's outputs, a word of each at a time: up to eight, that may start in the middle of a word
    static constexpr uint32_t kMeta = 5u * 128u * NT, kBiases = kScales + 2u * WN * kMeta, kBytes = (kBiases + WN * kMeta + 127u) & ~127u;
    static constexpr int kLoadsX = int(kX / 1024u / kWaves), kLoadsB = int(kB / 1024u / kWaves);  // of a wave, a step (two steps)
    static_assert(kLoadsX * 1024u * kWaves == kX && kLoadsB * 1024u * kWaves == kB && KS * kBytes <= 160u * 1024u);
    static_assert(kWaves * 32u * (32u * NT * 4u + 16u) <= kBytes && (KS == 1 || kWaves * MT * NT * 4096u <= kBytes), "the outputs on their way out fit, and a part's sums");
};

template <int XT, int GROUP, int MT, int NT, int WM, int WN, int P, int KS>
__global__ __launch_bounds__(64 * WM * WN * KS, 2) void k_affine4_tile(Affine4Args a) {
    typedef TileLds<MT, NT, WM, WN, P, KS> L;
    constexpr bool SUB32 = GROUP == 32;
    constexpr uint32_t kSteps = SUB32 ? 4u : 8u;               // of a chunk
    constexpr uint32_t kMetas = GROUP == 128 ? 4u : 8u;        // a chunk's scales
    const uint32_t lane = threadIdx.x & 63u, col = lane & 31u, half = lane >> 5;
    // the workgroup's waves are KS parts of k, whole chunks each, with their own places in LDS
    const uint32_t part = wave_index() / L::kWaves, wave = wave_index() % L::kWaves, wm = wave / WN, wn = wave % WN;
    const uint32_t steps_in_all = (a.k + 63u) / 64u, chunks = ((steps_in_all + kSteps - 1u) / kSteps + KS - 1u) / KS;  // of a part, the first ones
    const uint32_t first_step = min(part * chunks * kSteps, steps_in_all), steps = min(chunks * kSteps, steps_in_all - first_step);
    const uint32_t my_k = steps ? a.k - first_step * 64u : 0u;  // what is left of a row where the part begins
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_of_parts[];  // (of a size that the compiler does not know: else it takes sums to the accumulation registers and back)
    uint8_t *const lds = lds_of_parts + part * L::kBytes;
    const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds_of_parts)) + part * L::kBytes;
    const uint32_t groups = a.k / uint32_t(GROUP), my_groups = my_k / uint32_t(GROUP);
    const uint32_t row0 = blockIdx.y * L::kRows, n0 = blockIdx.x * L::kOuts, rows = min(a.rows - row0, L::kRows);

    // ---- what the wave asks for: eight rows of x a load (eight lanes a row, pieces xor-ed with half the row's number), sixteen of codes
    // (four lanes a row, xor-ed with a quarter of it). Rows and outputs past the last are the last again; past k stands a row's last piece.
    const uint32_t pieces = my_k / 8u, code_pieces = my_k / 32u;
    const uint8_t *const x = reinterpret_cast<const uint8_t *>(a.x + uint64_t(row0) * a.x_stride) + first_step * 128u;
    const uint8_t *const codes = a.codes + uint64_t(n0) * (a.k / 2u) + first_step * 32u;
    // (The offsets are formed again from the lane's number at every use: held in registers, they are spilled.)
    const uint32_t stride = uint32_t(a.x_stride) * 2u, row_bytes = a.k / 2u;
    auto load_x = [&](uint32_t place, uint32_t g) {
        const uint32_t l = lane_number(), first = 8u * wave * L::kLoadsX, piece = (l & 7u) ^ (4u * (wave * L::kLoadsX & 1u) + (l >> 4));
        const uint32_t to = lds0 + place * L::kX + wave * L::kLoadsX * 1024u;
        const uint8_t *const from = x + size_t(g) * 128u;
        if (rows == L::kRows && (!SUB32 || 8u * g + 8u <= pieces)) {
            const uint32_t row = (first + (l >> 3)) * stride, even = row + piece * 16u, odd = row + (piece ^ 4u) * 16u;
#pragma unroll
            for (uint32_t j = 0; j < L::kLoadsX; ++j) lds_load16(to + j * 1024u, from + size_t(8u * j) * stride, j % 2u ? odd : even);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < L::kLoadsX; ++j)
                lds_load16(to + j * 1024u, from, min(first + 8u * j + (l >> 3), rows - 1u) * stride + min(j % 2u ? piece ^ 4u : piece, pieces - 1u - 8u * g) * 16u);
        }
    };
    auto load_b = [&](uint32_t place, uint32_t two) {
        const uint32_t l = lane_number(), first = 16u * wave * L::kLoadsB, piece = (l & 3u) ^ (l >> 4);
        const uint32_t to = lds0 + L::kCodes + place * L::kB + wave * L::kLoadsB * 1024u;
        const uint8_t *const from = codes + size_t(two) * 64u;
        if (n0 + L::kOuts <= a.n && 4u * two + 4u <= code_pieces) {
            const uint32_t at = (first + (l >> 2)) * row_bytes + piece * 16u;
#pragma unroll
            for (uint32_t j = 0; j < L::kLoadsB; ++j) lds_load16(to + j * 1024u, from + size_t(16u * j) * row_bytes, at);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < L::kLoadsB; ++j)
                lds_load16(to + j * 1024u, from, min(first + 16u * j + (l >> 2), a.n - 1u - n0) * row_bytes + min(piece, code_pieces - 1u - 4u * two) * 16u);
        }
    };

    // ---- a chunk's scales, a chunk ahead, and its biases, of the wave's outputs, a lane each: a run of 16-bit values that starts at any of them,
    // so the words that it lies in, none past the tensor's last one. Waves of the same outputs share them out (one asks for scales, one for biases).
    const uint32_t n_first = n0 + wn * 32u * NT;
    const bool active = n_first < a.n;
    const uint32_t n_base = min(n_first, a.n - 1u);
    constexpr uint32_t kWords = kMetas / 2u + 1u;
    constexpr int kMetaLoads = int(kWords) * (WM == 1 ? 2 : 1);  // of a wave, a chunk
    struct Run {
        const uint8_t *from;  // the word that the wave's first output's values start in
        uint32_t skew, last;  // where in it, and how far the tensor's last word lies from it, in bytes
    };
    auto run_of = [&](const uint16_t *tensor) {
        const uint8_t *const first = reinterpret_cast<const uint8_t *>(tensor + uint64_t(n_base) * groups + (steps ? part * chunks * kMetas : 0u));
        Run r;
        r.skew = uint32_t(reinterpret_cast<uintptr_t>(first) & 2u);
        r.from = first - r.skew;
        const uint64_t left = (uint64_t(a.n - n_base) * groups - (steps ? part * chunks * kMetas : 0u)) * 2u + r.skew - 2u;
        r.last = uint32_t(left < 0x7ffffffcull ? left : 0x7ffffffcull) & ~3u;
        return r;
    };
    const Run scales = run_of(a.scales), biases = run_of(a.biases ? a.biases : a.scales);
    // where the values of the lane's l-th output start, in bytes from `from` (a chunk's start is a whole number of words further on)
    auto meta_start = [&](const Run &r, uint32_t l) { return r.skew + (min(n_first + l, a.n - 1u) - n_base) * groups * 2u; };
    auto load_metas = [&](const Run &r, uint32_t to, uint32_t chunk) {
        const uint32_t l = lane_number(), at = (meta_start(r, l) & ~3u) + chunk * kMetas * 2u;
        if (NT == 2 || l < 32u)
#pragma unroll
        for (uint32_t j = 0; j < kWords; ++j) lds_load4(lds0 + to + j * (128u * NT), r.from, min(at + 4u * j, r.last));
    };
    auto load_both = [&](uint32_t chunk) {  // the next chunk's scales, this one's biases
        if (WM == 1 || wm == 0) load_metas(scales, L::kScales + (((chunk + 1u) & 1u) * WN + wn) * L::kMeta, chunk + 1u);
        if (WM == 1 || wm == 1) load_metas(biases, L::kBiases + wn * L::kMeta, chunk);
    };
    // a lane's scale of its i-th output and the chunk's chain c, an even or odd one of the chunk's scales
    uint32_t scale_from[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const uint32_t l = 32u * i + col;
        scale_from[i] = L::kScales + wn * L::kMeta + 4u * l + (meta_start(scales, l) & 2u);
    }
    auto scale_at = [&](uint32_t chunk, int i, uint32_t c) {
        const uint32_t e = GROUP == 128 ? c / 2u : c, into = scale_from[i] & 2u;
        const uint32_t odd = e % 2u ? (into ? 128u * NT - 2u : 2u) : 0u;
        return *reinterpret_cast<const uint16_t *>(lds + (chunk & 1u) * (WN * L::kMeta) + scale_from[i] + odd + e / 2u * (128u * NT));
    };

    f32x16 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            acc[m][i] = affine4_zero();
            asm volatile("" : "+v"(acc[m][i]));
        }
    constexpr int kPer = SUB32 ? 2 : 4, kSubs = 4 / kPer;  // instructions a chain, chains a block and step
    uint8_t *const sums = lds + L::kSum;
    const uint32_t my_rows = wm * 32u * MT;  // the wave's first row of the tile
    const uint8_t *const my_x = lds + (my_rows + col) * 128u;
    auto read_x = [&](uint32_t place, uint32_t m, uint32_t j) {
        const uint32_t piece = SUB32 ? 4u * (j / 2u) + 2u * half + j % 2u : 4u * half + j;
        return *reinterpret_cast<const uint4 *>(my_x + place * L::kX + m * 4096u + ((piece ^ ((col >> 1) & 7u)) * 16u));
    };
    auto read_codes = [&](uint32_t from, uint32_t g, uint4 (&to)[NT]) {
        const uint32_t l = lane_number(), c = l & 31u;  // (32 rows further on a quarter of the row's number is the same but for bits that are not looked at)
        const uint8_t *const at = lds + L::kCodes + from * L::kB + (wn * 32u * NT + c) * 64u + (((2u * (g & 1u) + (l >> 5)) ^ ((c >> 2) & 3u)) * 16u);
#pragma unroll
        for (int i = 0; i < NT; ++i) to[i] = *reinterpret_cast<const uint4 *>(at + i * 2048u);
    };
    // of groups of 32 lane half h has group h of the step: its halves to both (past the row's end there is no second group)
    auto deal = [&](uint4 &v, uint32_t g) {
        if constexpr (SUB32) {
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            if (64u * g + 32u >= my_k)
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = half ? 0u : w[j];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const auto q = __builtin_amdgcn_permlane32_swap(w[j], w[j + 2], false, false);
                w[j] = q[0];
                w[j + 2] = q[1];
            }
            v = make_uint4(w[0], w[1], w[2], w[3]);
        }
    };
    auto word = [](const uint4 &v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; };
    // The sums of a step's groups of the rows that are this wave's share: its pieces are read, added and written a few instructions a slot.
    static_assert(MT <= WN && MT * NT >= 2, "a wave has a share of 32 rows at most, and the reads stand ahead of the meeting");
    const uint32_t share = min(wn, uint32_t(MT - 1));
    uint4 sum_piece[2];
    float sum_of[kSubs];
    auto form_sums = [&](auto slot_, uint32_t g, uint32_t place, uint32_t s) {
        constexpr int slot = decltype(slot_)::value;
        if constexpr (slot >= 2 && slot < 6) {
            constexpr int j = slot - 2, c = j / kPer;
            sum_of[c] = affine4_add<XT>(sum_piece[j % 2], j % kPer ? sum_of[c] : 0.0f);
        }
        if constexpr (slot < 4) {
            sum_piece[slot % 2] = read_x(place, share, slot);
        }
        if constexpr (slot == 6) {
            const uint32_t l = lane_number(), col = l & 31u, half = l >> 5;
#pragma unroll
            for (int c = 0; c < kSubs; ++c) {
                float v = add_xor32(sum_of[c]);
                if (SUB32 && c == 1 && 64u * g + 32u >= my_k) v = 0.0f;
                uint32_t terms[3];
                bf16_terms(v, 0.0f, terms);
                uint16_t *to = reinterpret_cast<uint16_t *>(sums + (my_rows + 32u * share + col) * 48u) + (SUB32 ? 2u * s + c : s);
                if (half == 0 && wn < uint32_t(MT))
#pragma unroll
                    for (int j = 0; j < 3; ++j) to[8 * j] = uint16_t(terms[j]);
            }
        }
    };
    // Where the next step's rows and codes have landed for every wave and the places of this step's are free again: of what was asked for after
    // them, the rows of P - 2 steps, codes at every odd one of these and a chunk's scales and biases at its first, all may still be on their way.
    auto meet = [&](uint32_t g, uint32_t place, uint32_t unit, uint32_t s, auto odd_, uint32_t chunk) {
        constexpr uint32_t S = decltype(odd_)::value, kBetween = P - 2u, kOdd = kBetween / 2u + (kBetween % 2u && S == 0 ? 1u : 0u);
        if (g + 2u * L::kUnits >= steps) wait_loads_and_sync<0>();
        else if (s >= 1u && s <= kBetween) wait_loads_and_sync<int(kBetween) * L::kLoadsX + int(kOdd) * L::kLoadsB + kMetaLoads>();
        else wait_loads_and_sync<int(kBetween) * L::kLoadsX + int(kOdd) * L::kLoadsB>();
        if (s == 0) load_both(chunk);
        if (S && g + 2u * L::kUnits - 1u < steps) load_b(unit, (g >> 1) + L::kUnits);
        if (g + P < steps) load_x(place, g + P);
    };
    // Step g, the s-th of its chunk: a chain of kPer instructions a block (and group of 32). Between a chain's instructions stand the scaling of the
    // chain before, the reads of the rows that come next into registers whose last use was the instruction ahead, and with the last
    // rows' chains the unpacking of the next step's codes.
    Affine4Frag f[NT][4], xf[4];
    uint4 raw[NT];
    constexpr bool kBehind = NT == 1 || !SUB32;  // (else the second sum is spilled)
    f32x16 p[kBehind ? 2 : 1];
    float before = 0.0f;  // the scale of the step before's last chain
    uint16_t next_scales[kSubs][NT];  // the next step's, as they are
    float factors[kSubs][NT] = {};
    auto read_scales = [&](uint32_t chunk, uint32_t s) {
#pragma unroll
        for (int c = 0; c < kSubs; ++c)
#pragma unroll
            for (int i = 0; i < NT; ++i) next_scales[c][i] = scale_at(chunk, i, SUB32 ? 2u * s + c : s);
    };
    auto step = [&](uint32_t g, uint32_t place, uint32_t next_place, uint32_t unit, uint32_t next_unit, uint32_t s, auto odd_, uint32_t chunk) {
        before = factors[kSubs - 1][NT - 1];
#pragma unroll
        for (int c = 0; c < kSubs; ++c)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                // (past the row's end there is no second group, but the next output's first scale, which may be anything)
                factors[c][i] = SUB32 && c == 1 && 64u * g + 32u >= my_k ? 0.0f : meta_f32(next_scales[c][i], a.meta);
            }
        auto slots = [&](auto slot_) {  // an instruction and what stands behind it
            constexpr int slot = decltype(slot_)::value, j = slot % kPer, chain = slot / kPer, i = chain % NT, c = chain / NT % kSubs, m = chain / NT / kSubs;
            constexpr int chains = MT * kSubs * NT, last = (chain + chains - 1) % chains, at = c * kPer + j;
            f32x16 &now = p[kBehind ? chain & 1 : 0], &old = p[kBehind ? (chain & 1) ^ 1 : 0];
            f32x16 &into = acc[last / NT / kSubs][last % NT];
            if constexpr (j == 0) {
                if constexpr (m == MT - 1 && c == 0 && i == 0) {
                    meet(g, place, unit, s, odd_, chunk);
                    read_codes(next_unit, g + 1u, raw);  // (behind the last step: something)
#pragma unroll
                    for (int n = 0; n < NT; ++n) asm volatile("" : "+v"(raw[n].x), "+v"(raw[n].y), "+v"(raw[n].z), "+v"(raw[n].w));
                }
                if constexpr (m == MT - 1 && c == 0) deal(raw[i], g + 1u);
            }
            now = affine4_multiply<XT>(xf[at], f[i][at], j == 0 ? affine4_zero() : now);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (slot == 1) read_scales(s + 1u == kSteps ? chunk + 1u : chunk, s + 1u == kSteps ? 0u : s + 1u);
            if constexpr (i == NT - 1) xf[at].v = m + 1 < MT ? read_x(place, m + 1u, at) : read_x(next_place, 0u, at);
            if constexpr (m == MT - 1) {
                f[i][at] = affine4_codes<XT>(word(raw[i], at));
                asm volatile("" : "+v"(f[i][at].v.x), "+v"(f[i][at].v.y), "+v"(f[i][at].v.z), "+v"(f[i][at].v.w));  // (here: else it sinks behind the branches)
            }
            form_sums(slot_, g, place, s);
            if constexpr (kBehind) {
                constexpr int kEach = 16 / kPer;
#pragma unroll
                for (int r = j * kEach; r < (j + 1) * kEach; ++r) into[r] = fmaf(chain ? factors[last / NT % kSubs][last % NT] : before, old[r], into[r]);
                asm volatile("" : "+v"(into));
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!kBehind && j == kPer - 1) {
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[m][i][r] = fmaf(factors[c][i], now[r], acc[m][i][r]);
                asm volatile("" : "+v"(acc[m][i]));
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        each_of(slots, std::make_integer_sequence<int, MT * NT * 4>{});
    };
    static_assert(MT * kSubs * NT % 2 == 0, "the chains alternate between two sums across steps");
    // what no chain of a last chunk has written
    auto clear_sums = [&](uint32_t chains) {
        for (uint32_t m = wn; m < uint32_t(MT); m += WN)
            for (uint32_t c = chains; c < 8u && half == 0; ++c)
#pragma unroll
                for (int j = 0; j < 3; ++j) reinterpret_cast<uint16_t *>(sums + (my_rows + 32u * m + col) * 48u)[8 * j + c] = 0;
    };
    // The bias term of a chunk of `chains` chains: the lanes of half 0 add the sums' high terms, those of half 1 the middle ones, then half 0 the
    // low ones, each against the (high) bias; an fp16 bias is two bf16 terms.
    auto add_bias = [&](uint32_t chains) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const float factor = a.biases ? 1.0f : -8.0f;
            const uint32_t l = lane_number(), col = l & 31u, half = l >> 5;
            // the run's words, brought to where it starts; of groups of 128 each value twice
            const uint8_t *const run = lds + L::kBiases + wn * L::kMeta + 4u * (32u * i + col);
            const uint32_t skew = 8u * (meta_start(biases, 32u * i + col) & 2u);
            uint32_t words[kWords], pairs[4];
#pragma unroll
            for (uint32_t j = 0; j < kWords; ++j) words[j] = *reinterpret_cast<const uint32_t *>(run + j * (128u * NT));
#pragma unroll
            for (uint32_t j = 0; j + 1u < kWords; ++j) words[j] = __builtin_amdgcn_alignbit(words[j + 1u], words[j], skew);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) pairs[j] = GROUP == 128 ? (words[j / 2u] >> 16u * (j % 2u) & 0xffffu) * 0x10001u : words[j];
            Affine4Frag high, low;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                uint32_t terms[3];
                auto value = [&](uint32_t c) { return c < chains ? meta_f32(uint16_t(pairs[c / 2u] >> 16u * (c % 2u)), a.meta) * factor : 0.0f; };
                bf16_terms(value(2u * j), value(2u * j + 1u), terms);
                high.u[j] = terms[0];
                low.u[j] = terms[1];
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const uint8_t *at = sums + (my_rows + 32u * m + col) * 48u;
                Affine4Frag both, rest;
                both.v = *reinterpret_cast<const uint4 *>(at + 16u * half);
                rest.v = *reinterpret_cast<const uint4 *>(at + 32u);
#pragma unroll
                for (int j = 0; j < 4; ++j) rest.u[j] = half ? 0u : rest.u[j];
                f32x16 q = NT == 1 ? affine4_zero() : acc[m][i];
                q = __builtin_amdgcn_mfma_f32_32x32x16_bf16(both.b, high.b, q, 0, 0, 0);
                q = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rest.b, high.b, q, 0, 0, 0);
                if (a.meta == SHRIKE_META_F16) q = __builtin_amdgcn_mfma_f32_32x32x16_bf16(both.b, low.b, q, 0, 0, 0);
                if (NT == 1)
#pragma unroll
                    for (int r = 0; r < 16; ++r) q[r] = __fadd_rn(acc[m][i][r], q[r]);
                acc[m][i] = q;
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    if (WM == 1 || wm == 0) load_metas(scales, L::kScales + wn * L::kMeta, 0);
    // as if steps -P ... -1 had asked for them
    if (steps) load_b(0, 0);
#pragma unroll
    for (int v = 0; v < P; ++v) {
        constexpr int kAhead = P % 2;  // v - P is odd where v is of the other parity than P
        const uint32_t u = uint32_t((v - P - 1) / 2 + int(L::kUnits));
        if (v % 2 != kAhead && u != 0u && 2u * u < steps) load_b(u, u);
        if (uint32_t(v) < steps) load_x(v, v);
    }
    wait_loads_and_sync<0>();
#pragma unroll
    for (int r = 0; kBehind && r < 16; ++r) p[kBehind][r] = 0.0f;
    auto begin = [&](uint32_t place, uint32_t unit, uint32_t g) {
        read_codes(unit, g, raw);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            deal(raw[i], g);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[i][j] = affine4_codes<XT>(word(raw[i], j));
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) xf[j].v = read_x(place, 0, j);
    };
    begin(0, 0, 0);
    read_scales(0, 0);
    uint32_t place = 0, unit = 0;
    const uint32_t most_steps = min(chunks * kSteps, steps_in_all);
    for (uint32_t chunk = 0; chunk < chunks; ++chunk) {
        auto one = [&](uint32_t s, auto odd_) {
            const uint32_t g = chunk * kSteps + s, next_place = place == P - 1u ? 0u : place + 1u;
            const uint32_t next_unit = !decltype(odd_)::value ? unit : unit == L::kUnits - 1u ? 0u : unit + 1u;
            step(g, place, next_place, unit, next_unit, s, odd_, chunk);
            place = next_place;
            unit = next_unit;
        };
#pragma unroll 1
        for (uint32_t s = 0; s < kSteps; s += 2u) {
            const uint32_t g = chunk * kSteps + s;
            if (KS == 1 && g >= steps) break;
            // (a part that ends earlier meets the others all the same, as far as the first part, the longest, goes)
            if (g < steps) one(s, std::integral_constant<uint32_t, 0>{});
            else if (g < most_steps) wait_loads_and_sync<0>();
            if (g + 1u < steps) one(s + 1u, std::integral_constant<uint32_t, 1>{});
            else if (g + 1u < most_steps) wait_loads_and_sync<0>();
        }
        // the chunk's bias term, once every wave has formed its sums
        const uint32_t done = min(chunk * kSteps, steps), chains = min(8u, SUB32 ? my_groups - min(chunk * 8u, my_groups) : steps - done);
        if (chains < 8u) clear_sums(chains);
        if (done + kSteps >= steps) wait_loads<0>();  // (in the last one its biases may still be on their way)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (chains) add_bias(chains);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        begin(place, unit, (chunk + 1u) * kSteps);  // (held across the bias term, the operands are spilled)
    }
#pragma unroll
    for (int r = 0; kBehind && r < 16; ++r) acc[MT - 1][NT - 1][r] = fmaf(factors[kSubs - 1][NT - 1], p[kBehind][r], acc[MT - 1][NT - 1][r]);
    __syncthreads();
    if constexpr (KS > 1) {  // the second part's sums by way of LDS; the first has the rest
        static_assert(KS == 2);
        float *const meet_at = reinterpret_cast<float *>(lds_of_parts) + wave * (MT * NT * 1024u) + lane;
        if (part == 1u)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) meet_at[((m * NT + i) * 16 + r) * 64] = acc[m][i][r];
        __syncthreads();
        if (part == 0)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[m][i][r] = __fadd_rn(acc[m][i][r], meet_at[((m * NT + i) * 16 + r) * 64]);
        __syncthreads();
        if (part == 1u) return;
    }
    if (!active) return;

    // ---- out: a block of 32 rows at a time through the wave's own part of LDS, so that a row's outputs leave 16 bytes a lane
    const uint32_t size = a.out_type == SHRIKE_ELEM_F32 ? 4u : 2u, pitch = 32u * NT * size + 16u, outs = min(32u * NT, a.n - n_first);
    uint8_t *const stage = lds + wave * 32u * (32u * NT * 4u + 16u);
    const bool whole = (reinterpret_cast<uintptr_t>(a.out) | (a.out_stride * size)) % 16u == 0;
    float extra[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) extra[i] = a.bias ? meta_f32(a.bias[min(n_first + 32u * i + col, a.n - 1u)], a.meta) : 0.0f;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (my_rows + 32u * m >= rows) break;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (uint32_t r = 0; r < 16; ++r) {
                const float v = __fadd_rn(acc[m][i][r], extra[i]);
                uint8_t *to = stage + (8u * (r / 4u) + 4u * half + r % 4u) * pitch + (32u * i + col) * size;
                if (size == 4u) *reinterpret_cast<float *>(to) = v;
                else *reinterpret_cast<uint16_t *>(to) = a.out_type == SHRIKE_ELEM_F16 ? f32_to_f16(v) : uint16_t(bf16_pair(v, 0.0f));
            }
        __builtin_amdgcn_wave_barrier();
        const uint32_t per = 32u * NT * size / 16u;  // lanes a row
        for (uint32_t at = lane; at < 32u * per; at += 64u) {
            const uint32_t r = at / per, first = (at % per) * (16u / size), row = my_rows + 32u * m + r;
            if (row >= rows || first >= outs) continue;
            const uint8_t *from = stage + r * pitch + first * size;
            uint8_t *to = static_cast<uint8_t *>(a.out) + (uint64_t(row0 + row) * a.out_stride + n_first + first) * size;
            if (whole && first + 16u / size <= outs) {
                *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(from);
            } else {
                for (uint32_t j = 0; j < 16u / size && first + j < outs; ++j) {
                    if (size == 4u) reinterpret_cast<uint32_t *>(to)[j] = reinterpret_cast<const uint32_t *>(from)[j];
                    else reinterpret_cast<uint16_t *>(to)[j] = reinterpret_cast<const uint16_t *>(from)[j];
                }
            }
        }
    }
}

template <int XT, int GROUP, int MT, int NT, int WM, int WN, int P, int KS>
static int launch_tile(const Affine4Args &a, hipStream_t s) {
    typedef TileLds<MT, NT, WM, WN, P, KS> L;
    hipLaunchKernelGGL((k_affine4_tile<XT, GROUP, MT, NT, WM, WN, P, KS>), dim3((a.n + L::kOuts - 1u) / L::kOuts, (a.rows + L::kRows - 1u) / L::kRows),
                       dim3(64u * L::kWaves * KS), KS * L::kBytes, s, a);
    SHRIKE_HIP(hipGetLastError());
    return 0;
}

// Which shape: the one that takes the least, in tenths of a microsecond, by its rounds (of 256 workgroups), the units of 256 k a round, and what a unit,
// a round and the call take. Measured, in us:
//   rows x n x k              8 rows   16 rows   32 rows   128 x 128   256 x 256
//   16 x 4,096 x 4,096           9.7      15.8      27.0        53.5       141.9
//   64 x 8,192 x 2,048          18.7      14.3      18.8        30.7        75.7
//   64 x 16,384 x 2,304         30.5      22.7      22.1        38.3        85.3
//   128 x 4,096 x 4,096         31.5      22.9      31.1        55.6       148.1
//   300 x 4,096 x 2,048         37.3      28.1      24.9        33.3        79.5
//   512 x 8,192 x 2,048         94.0      77.6      49.3        35.2        80.4
//   2,048 x 4,096 x 4,096      370.2     284.9     176.6       116.5       148.8
//   2,048 x 6,144 x 4,096      547.5     410.9     261.3       172.0       153.7
//   4,096 x 5,120 x 2,048      449.4     372.6     228.0       162.9       166.0
//   513 x 26,428 x 320          86.9      53.6      39.3        80.5        54.6
//   1,724 x 2,822 x 1,216       88.2      56.0      40.1        65.0        68.4
//   3,108 x 14,040 x 64        139.7      91.3      63.4       111.4        53.8
template <int R8>
static uint64_t few_cost(const Affine4Args &a) {
    const uint32_t parts = few_parts<R8>(a), units = (a.k + kFewUnit - 1u) / kFewUnit, each = (units + parts - 1u) / parts;
    const uint64_t rounds = (few_workgroups<R8>(a, parts) + 255u) / 256u;
    return R8 == 1 ? rounds * each * 15u + 60u : R8 == 2 ? rounds * each * 20u + 60u : rounds * (each * 26u + 8u) + 50u;
}
static uint64_t tile_cost(const Affine4Args &a, uint32_t side, uint32_t unit, uint32_t call) {
    const uint64_t tiles = uint64_t((a.rows + side - 1u) / side) * ((a.n + side - 1u) / side);
    return (tiles + 255u) / 256u * ((a.k + kFewUnit - 1u) / kFewUnit * unit + 70u) + call;
}
template <int XT, int GROUP>
static int launch_affine4(const Affine4Args &a, hipStream_t s) {
    if (a.rows <= 8u) return launch_few<XT, GROUP, 1>(a, s);  // (8 rows of 16,384 x 4,096: 15.9 us, by 16 a workgroup 17.4; of 5,120 x 2,880 9.5 and 12.4)
    const uint64_t few[3] = {few_cost<1>(a), few_cost<2>(a), few_cost<4>(a)}, least = std::min(few[0], std::min(few[1], few[2]));
    if (a.x_stride * 512u < uint64_t(1) << 32) {  // (a tile's rows are reached by 32 bits)
        const uint64_t tile = tile_cost(a, 128, 29, 50), large = tile_cost(a, 256, 90, 100);
        if (std::min(tile, large) < least) return tile <= large ? launch_tile<XT, GROUP, 4, 1, 1, 4, 3, 2>(a, s) : launch_tile<XT, GROUP, 4, 2, 2, 4, 3, 1>(a, s);
    }
    if (few[1] == least) return launch_few<XT, GROUP, 2>(a, s);
    return few[2] == least ? launch_few<XT, GROUP, 4>(a, s) : launch_few<XT, GROUP, 1>(a, s);
}
template <int XT>
static int launch_affine4(const Affine4Args &a, hipStream_t s) {
    if (a.rows == 1u) return launch_gemv<XT>(a, s);
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
    constexpr uint32_t kMost = 8u * 65535u;  // rows of a launch: a grid's second dimension ends at 65,535, and the lowest workgroup has 8 rows
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
