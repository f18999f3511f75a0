// Products whose operands are rows of bytes along K: 8-bit integers with a scale for each token and channel, and fp16 or bf16 values.
//
// One instruction takes 64 bytes of K of either kind (v_mfma_i32_16x16x64_i8, v_mfma_f32_16x16x32_f16 and _bf16): a lane holds 16 bytes of one row, lane l those of row l % 16
// at byte 16 (l / 16), and of a result four neighbouring rows of the first operand and one of the second.  So one kernel moves the bytes of all three, in steps of 128.
//
// Weights are laid out once: a tile is 16 channels x 128 bytes of K, 2048 bytes as [piece 0..7][channel][16 bytes]; the tiles of the same K lie behind one another.
// A wave's load of an operand is whole kilobytes, with nothing to unpack.  Channels are padded to 64, four tiles, and K to 256 bytes, two steps, with zeros.  What a channel has (scale, sum, bias) lies by tiles too.
// SwiGLU: tiles of gate channels and of their up channels take turns, so a lane has both of a pair.
//
// Rows of 8-bit integers: x = (q - z) s with an fp32 scale s, and a zero point z or none, for each row; behind K, up to a multiple of 256, the code of 0 (z, or 0 without zero points), which meets the
// weights' zeros.  Dense rows lie by tiles of 16 rows x 128, [piece][row][16], the tiles of the same rows along K behind one another; rows of experts, which a product takes from anywhere, an odd
// multiple of 128 bytes apart (at a multiple of 4 KiB they meet in few channels of the L2).  Channel c has an fp32 scale t and S = sum of its weights w:
//   y = (sum_k q w - z S) t s + bias, the bracket exact in 32 bits up to K = 65536 (255 * 128 * 65536 < 2^31), then one rounding for each operation and one for the output.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "mx_device.h"

namespace orx {
namespace bytes {

using mx::v4f;
using mx::v4i;
using mx::v4u;

constexpr int kStep = 128;        // bytes of K to a step, of which there are pairs
constexpr int kTileBytes = 2048;  // 16 channels of a step
constexpr int kMostIntegerK = 65536;
constexpr int steps_of_bytes(int64_t bytes) { return (int)((bytes + 2 * kStep - 1) / (2 * kStep) * 2); }

enum Kind { I8 = 0, F16 = 1, BF16 = 2 };  // of the operands

template <int KIND>
struct Operands {
    using Sum = v4f;
    static constexpr int value_bytes = 2;
};
template <>
struct Operands<I8> {
    using Sum = v4i;
    static constexpr int value_bytes = 1;
};

template <int KIND>
__device__ __forceinline__ typename Operands<KIND>::Sum multiply(v4i weight, v4i row, typename Operands<KIND>::Sum sum) {
    typedef _Float16 half8 __attribute__((ext_vector_type(8)));
    typedef __bf16 brain8 __attribute__((ext_vector_type(8)));
    if constexpr (KIND == I8) return __builtin_amdgcn_mfma_i32_16x16x64_i8(weight, row, sum, 0, 0, 0);
    else if constexpr (KIND == F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, weight), __builtin_bit_cast(half8, row), sum, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(brain8, weight), __builtin_bit_cast(brain8, row), sum, 0, 0, 0);
}

// The same in one register, in and out: left to itself the compiler moves the sums about between unrolled steps, which takes the registers of half a set more.  What it would have inserted is on
// the caller: two instructions between the last write of an operand by an instruction (not a load) and the multiply, and a pause (settle) in front of the first reading of a sum.
template <int KIND>
__device__ __forceinline__ void multiply_in_place(typename Operands<KIND>::Sum& sum, const v4i& weight, const v4i& row) {
    if constexpr (KIND == I8) asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+v"(sum) : "v"(weight), "v"(row));
    else if constexpr (KIND == F16) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+v"(sum) : "v"(weight), "v"(row));
    else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(sum) : "v"(weight), "v"(row));
}
__device__ __forceinline__ void settle() { asm volatile("s_nop 15"); }

// What a product reads and writes.
struct Product {
    const uint8_t* a;      // dense rows of 8-bit integers by tiles, others `pitch` bytes apart
    const float* scale;    // of the rows (8-bit integers)
    const int* zero;       // zero points of the rows, or null
    const uint8_t* w;      // tiles
    const float* w_scale;  // of the channels, by tiles
    const int* w_sum;      // sums of the channels' weights, by tiles (with zero points)
    const float* bias;     // by tiles, or null
    void* out;
    int64_t pitch;
    int m, cols, steps;  // rows, output columns, steps of K
    int row_bytes;       // of K, of a row
    int tiles;           // 16-channel tiles of the weights (of one expert)
    int type;            // of the output (mx::Type)
    // experts: unit = expert, first slot, slots (TileUnits); a slot's row is its token's or its own
    const int4* units;
    const int* unit_count;
    int most_units;  // that the list holds
    int runs;  // of neighbouring tiles that an XCD has, where weights go straight to registers
    const int* slot_token;
};

// A row's scale and zero point.
struct RowScale {
    float scale;
    int zero;
};

// What four channels have: their scales, and with zero points and biases those sums and biases (zeros where there are none).
struct Channels {
    v4f scale;
    v4i sum;
    v4f bias;
};
// Four channels of one row.  EXTRAS: zero points and biases there may be.
template <int KIND, bool EXTRAS>
__device__ __forceinline__ v4f scaled(typename Operands<KIND>::Sum sum, const Channels& channel, const RowScale& row) {
    v4f y;
    if constexpr (KIND == I8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (EXTRAS) sum[j] -= row.zero * channel.sum[j];
            y[j] = ((float)sum[j] * channel.scale[j]) * row.scale;
            if constexpr (EXTRAS) y[j] += channel.bias[j];
        }
    } else {
        y = sum;
    }
    return y;
}

// ---- rows to 8-bit integers ---------------------------------------------------------------------------------------------------------------------
// s = max(largest / 127, 2^-100), q = x / s; with zero points s = max((high - low) / 255, 2^-100) over low = min(x, 0) and high = max(x, 0), z = round(-low / s) - 128, q = round(x / s) + z
// within [-128, 127].  Quotients round to the nearest whole number, ties to even.  (2^-100: the residuals below keep all of their bits.)  A row with an infinity or NaN, or whose range leaves
// fp32, has the scale NaN and codes 0, so its products are NaN.
constexpr float kSmallestScale = 7.888609052210118e-31f;  // 2^-100

// What a row's values leave, bits as the type orders its magnitudes: `high` of the largest magnitude; with zero points of the largest value that is not negative, and `low` of the lowest value,
// with its sign (without it where none is negative).  As whole numbers the values from 0 on order as they are and lie above the negative ones, and without a sign the negative ones lie
// above the others, the lowest on top: one maximum each.
struct RowRange {
    uint32_t high, low;
};
template <int TYPE, bool ZERO, int WORDS>
__device__ __forceinline__ void widen(RowRange& range, const uint32_t (&words)[WORDS]) {
    typedef short signed_pair __attribute__((ext_vector_type(2)));
    typedef unsigned short pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < WORDS; ++j) {
        if constexpr (!ZERO) range.high = TYPE == mx::F32 ? max(range.high, words[j] & 0x7FFFFFFFu) : mx::pair_max(range.high, words[j]);  // (16 bits: both halves apart)
        else if constexpr (TYPE == mx::F32) range.high = (uint32_t)max((int)range.high, (int)words[j]), range.low = max(range.low, words[j]);
        else {
            range.high = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(signed_pair, range.high), __builtin_bit_cast(signed_pair, words[j])));
            range.low = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pair, range.low), __builtin_bit_cast(pair, words[j])));
        }
    }
}
// over the wave, known to all of it
template <int TYPE, bool ZERO>
__device__ __forceinline__ RowRange over_wave(RowRange range) {
    auto both = [](uint32_t bits) { return wave_max_u32(TYPE == mx::F32 ? bits : max(bits & 0xFFFFu, bits >> 16)); };
    return {both(range.high), ZERO ? both(range.low) : 0u};
}
__device__ __forceinline__ RowRange wider(const RowRange& a, const RowRange& b) { return {max(a.high, b.high), max(a.low, b.low)}; }
struct RowCode {
    float scale, inverse;
    int zero;
    bool bad;
};
// the largest of the negatives' magnitudes
template <int TYPE>
__device__ __forceinline__ uint32_t low_bits(const RowRange& range) {
    constexpr uint32_t sign = TYPE == mx::F32 ? 0x80000000u : 0x8000u;
    return range.low & sign ? range.low & (sign - 1) : 0u;
}
template <int TYPE, bool ZERO>
__device__ __forceinline__ RowCode row_code(const RowRange& range) {
    RowCode code;
    const uint32_t low = ZERO ? low_bits<TYPE>(range) : 0u;
    const float span = mx::Bits<TYPE>::value(range.high) + (ZERO ? mx::Bits<TYPE>::value(low) : 0.f);
    code.bad = max(range.high, low) >= mx::Bits<TYPE>::infinity || span == __builtin_inff();
    code.scale = fmaxf(__fdiv_rn(code.bad ? 0.f : span, ZERO ? 255.f : 127.f), kSmallestScale);
    code.inverse = __fdiv_rn(1.f, code.scale);
    code.zero = 0;
    return code;
}
// The nearest whole number to value / scale, ties to even: the product with the inverse decides, which is within 256 * 2^-23 of the quotient, except within 2^-14 of a tie k + 1/2, where the
// residual value - (k + 1/2) scale does: one fused multiply-add, whose sign is exact.
__device__ __forceinline__ float whole_near_tie(float value, const RowCode& code) {
    const float below = rintf(__builtin_fmaf(value, code.inverse, -0.5f)), tie = below + 0.5f;
    const float rest = __builtin_fmaf(-tie, code.scale, value);
    return rest > 0.f ? below + 1.f : rest < 0.f ? below : rintf(tie);
}
__device__ __forceinline__ float whole_of(float value, const RowCode& code) {
    const float product = value * code.inverse, r = rintf(product);
    return fabsf(fabsf(product - r) - 0.5f) < 6.103515625e-05f ? whole_near_tie(value, code) : r;
}
// Four codes in a word; one test for the four: the multiply-add rounds the exact product to a whole number (1.5 * 2^23 more, whose low byte it then is).
template <bool ZERO>
__device__ __forceinline__ uint32_t four_codes(const float (&value)[4], const RowCode& code) {
    constexpr float kWhole = 12582912.0f;
    float r[4], farthest = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        r[j] = __builtin_fmaf(value[j], code.inverse, kWhole);
        farthest = fmaxf(farthest, fabsf(__builtin_fmaf(value[j], code.inverse, kWhole - r[j])));
    }
    if (__builtin_expect(farthest > 0.49993896484375f, 0)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = whole_of(value[j], code) + kWhole;
    }
    uint32_t word[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (ZERO) r[j] = __builtin_amdgcn_fmed3f(r[j] + (float)code.zero, kWhole - 128.f, kWhole + 127.f);
        else r[j] = __builtin_amdgcn_fmed3f(r[j], kWhole - 127.f, kWhole + 127.f);  // (a scale's rounding can bring a quotient a little above 127, never to 127.5)
        word[j] = __float_as_uint(r[j]);
    }
    const uint32_t low = __builtin_amdgcn_perm(word[1], word[0], 0x0C0C0400u), high = __builtin_amdgcn_perm(word[3], word[2], 0x0C0C0400u);
    return code.bad ? 0u : low | high << 16;
}
// zero point of a row whose lowest value is -low
__device__ __forceinline__ int zero_point(float low, const RowCode& code) { return (int)whole_of(low, code) - 128; }

// eight values from the words that hold them
template <int TYPE, int WORDS>
__device__ __forceinline__ void eight_values(float (&value)[8], const uint32_t (&words)[WORDS]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (TYPE == mx::F32) value[j] = __uint_as_float(words[j]);
        else value[j] = mx::Bits<TYPE>::value((j & 1) ? words[j / 2] >> 16 : words[j / 2] & 0xFFFFu);
    }
}
template <int TYPE, bool ZERO, int WORDS>
__device__ __forceinline__ uint2 eight_codes(const uint32_t (&words)[WORDS], const RowCode& code) {
    float value[8];
    eight_values<TYPE>(value, words);
    const float low[4] = {value[0], value[1], value[2], value[3]}, high[4] = {value[4], value[5], value[6], value[7]};
    return make_uint2(four_codes<ZERO>(low, code), four_codes<ZERO>(high, code));
}
// What a row's range makes of it.
template <int TYPE, bool ZERO>
__device__ __forceinline__ RowCode code_of(const RowRange& range) {
    RowCode code = row_code<TYPE, ZERO>(range);
    if constexpr (ZERO) code.zero = code.bad ? 0 : zero_point(mx::Bits<TYPE>::value(low_bits<TYPE>(range)), code);
    return code;
}
__device__ __forceinline__ float stored_scale(const RowCode& code) { return code.bad ? __uint_as_float(0x7FC00000u) : code.scale; }

}  // namespace bytes
}  // namespace orx
