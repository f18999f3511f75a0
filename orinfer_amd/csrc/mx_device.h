// Microscaled 4-bit floating point (MXFP4) on gfx950: the format, its quantiser and the layout that the products read.
//
// A row is cut into blocks of 32 along K.  A block has one power of two, kept as a byte e for 2^(e - 127) (255: the block is NaN), and 32 codes of a sign, two
// exponent and one mantissa bits, 0 0.5 1 1.5 2 3 4 6, two to a byte with the even element in the low half.
//
// Rows (activations): codes (rows, KP / 2), bytes (rows, KP / 32), KP = K rounded up to whole blocks, or for the products
// to an odd multiple of 256; what is behind K is zero.  (Odd: rows that lie a multiple of 4 KiB apart meet in few channels of the L2.)
// Tiles (weights, laid out once): 16 channels x 256 K are 2048 bytes of codes, [block 0..7][channel][16 bytes], and 128 bytes of powers,
// [channel][block & 1][block >> 1]; tiles of one 16 channels lie along K behind one another.  One 16-byte piece is what a lane holds of an operand of v_mfma_scale_f32_*_f8f6f4
// with 4-bit codes: 32 elements of one row, whose one power comes from a byte of the lane's scale register.  So a wave's load of an operand is whole kilobytes,
// with nothing to unpack, and no lane needs another's power.  The order of the blocks within a product is free as long as both operands agree.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "a8_device.h"

namespace orx {
namespace mx {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));

constexpr int kBlock = 32;        // elements to a power
constexpr int kStepK = 256;       // K of a tile
constexpr int kTileBytes = 2048;  // codes of 16 channels x 256 K
constexpr int kTilePowers = 128;

enum Type { F16 = 0, BF16 = 1, F32 = 2 };

// Bits of a magnitude as they order (infinity and NaN behind all others), and where those begin.
template <int TYPE>
struct Bits;
template <>
struct Bits<F16> {
    static constexpr uint32_t infinity = 0x7C00;
    static __device__ __forceinline__ float value(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (unsigned short)bits); }
};
template <>
struct Bits<BF16> {
    static constexpr uint32_t infinity = 0x7F80;
    static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits << 16); }
};
template <>
struct Bits<F32> {
    static constexpr uint32_t infinity = 0x7F800000;
    static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits); }
};

// The power's byte of a block whose largest magnitude has these bits: the largest's own power of two less the two that the code 4..6 has.  What is above 6 of
// those units then saturates; `ceil` takes the next power for such a block.  The smallest byte is 0, also that of a block of zeros.
template <int TYPE>
__device__ __forceinline__ uint32_t power_byte(uint32_t largest, bool ceil) {
    if (largest >= Bits<TYPE>::infinity) return 255u;
    const uint32_t bits = __float_as_uint(Bits<TYPE>::value(largest));  // (16-bit subnormals are normal numbers here)
    const int exponent = (int)(bits >> 23) - 2 + (ceil && (bits & 0x7FFFFFu) > 0x400000u ? 1 : 0);
    return (uint32_t)max(exponent, 0);
}

// Largest magnitude bits of two 16-bit values in a word and so far.
__device__ __forceinline__ uint32_t pair_max(uint32_t so_far, uint32_t word) {
    typedef unsigned short pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pair, so_far), __builtin_bit_cast(pair, word & 0x7FFF7FFFu)));
}

// largest over the four lanes of a quad
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
}

// Eight codes of one block, rounded to nearest, ties to the even code, saturating: the conversion instruction divides by the power of the scale's exponent
// field, also by 2^-127 where that is zero (it agrees with the rule for every fp16 and bf16 value, fp32 values of every exponent, and every power that power_byte gives).
template <int TYPE>
__device__ __forceinline__ uint32_t eight_codes(const uint32_t* words, uint32_t byte) {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
    const float power = __uint_as_float(byte << 23);
    uint32_t codes = 0;
    if constexpr (TYPE == F16) {
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(half2v, words[0]), power, 0);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(half2v, words[1]), power, 1);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(half2v, words[2]), power, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(half2v, words[3]), power, 3);
    } else if constexpr (TYPE == BF16) {
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf2v, words[0]), power, 0);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf2v, words[1]), power, 1);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf2v, words[2]), power, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf2v, words[3]), power, 3);
    } else {
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(words[0]), __uint_as_float(words[1]), power, 0);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(words[2]), __uint_as_float(words[3]), power, 1);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(words[4]), __uint_as_float(words[5]), power, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(words[6]), __uint_as_float(words[7]), power, 3);
    }
    return byte == 255u ? 0u : codes;
}

template <int BYTE_A, int BYTE_B>
__device__ __forceinline__ v4f multiply_16(v4i a, v4i b, v4f sum, int powers_a, int powers_b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(v8i{a[0], a[1], a[2], a[3], 0, 0, 0, 0}, v8i{b[0], b[1], b[2], b[3], 0, 0, 0, 0}, sum, 4, 4,
                                                            BYTE_A, powers_a, BYTE_B, powers_b);
}
template <int BYTE_A, int BYTE_B>
__device__ __forceinline__ v16f multiply_32(v4i a, v4i b, v16f sum, int powers_a, int powers_b) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v8i{a[0], a[1], a[2], a[3], 0, 0, 0, 0}, v8i{b[0], b[1], b[2], b[3], 0, 0, 0, 0}, sum, 4, 4,
                                                           BYTE_A, powers_a, BYTE_B, powers_b);
}

// silu(gate) * up in fp32, rounded once with the output (with the library exponential and quotient 32 thousand expert rows of 512 pairs took 87 us in tiles of 256, 78 now)
__device__ __forceinline__ float swiglu(float gate, float up) { return gate * sigmoid_value(gate) * up; }

__device__ __forceinline__ uint32_t two_values(float a, float b, int type) {
    if (type == F16) {
        typedef _Float16 half2v __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, half2v{(_Float16)a, (_Float16)b});
    }
    typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf2v{(__bf16)a, (__bf16)b});
}

// Neighbouring results of a row from column `col` on, of `cols` columns: a store for all of them at any address of the type's own alignment (this target's memory
// instructions take it), those of a last, short piece one after another.
typedef unsigned int words2 __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned int words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef float floats4 __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void store_eight_halves(void* out, int64_t row_start, int col, int cols, v4u v) {
    unsigned short* to = reinterpret_cast<unsigned short*>(out) + row_start + col;
    if (col + 8 <= cols) {
        *reinterpret_cast<words4*>(to) = v;
    } else {
#pragma unroll 1
        for (; col < cols; ++col) {
            *to++ = (unsigned short)v[0];
            v = v4u{__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16), __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] >> 16};
        }
    }
}
__device__ __forceinline__ void store_four(void* out, int type, int64_t row_start, int col, int cols, v4f v) {
    if (type == F32) {
        float* to = reinterpret_cast<float*>(out) + row_start + col;
        if (col + 4 <= cols) {
            *reinterpret_cast<floats4*>(to) = v;
        } else {
#pragma unroll 1
            for (; col < cols; ++col) *to++ = v[0], v = v4f{v[1], v[2], v[3], 0.f};
        }
        return;
    }
    unsigned short* to = reinterpret_cast<unsigned short*>(out) + row_start + col;
    uint32_t low = two_values(v[0], v[1], type), high = two_values(v[2], v[3], type);
    if (col + 4 <= cols) {
        *reinterpret_cast<words2*>(to) = words2{low, high};
    } else {
#pragma unroll 1
        for (; col < cols; ++col) *to++ = (unsigned short)low, low = __builtin_amdgcn_alignbit(high, low, 16), high >>= 16;
    }
}

// What a product reads and writes.
struct Product {
    const uint8_t* a;   // codes of the rows (rows, pitch)
    const uint8_t* as;  // their powers (rows, pitch / 16)
    const uint8_t* w;   // tiles
    const uint8_t* ws;
    void* out;
    int m, cols, k, steps;  // rows, output columns, K, K / 256
    int pitch;             // bytes of a row's codes
    int tiles;             // 16-channel tiles of the weights (of one expert)
    int type;              // of the output
    // experts: unit = expert, first slot, slots (TileUnits), row of a slot's token or of the slot itself
    const int4* units;
    const int* unit_count;
    int most_units;  // that the list holds
    const int* slot_token;
};

}  // namespace mx
}  // namespace orx
