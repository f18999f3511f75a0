// Rows of 16-bit or 32-bit values to MXFP4 and back (the format: mx_device.h).
//
//   a = max |x| of a block, e = max(exponent(a) - 2, 0), code = E2M1(x / 2^(e - 127)), nearest, ties to even, saturating.
// Bound by memory: 2 bytes in and 17/32 out an element.  A lane takes eight values (16 bytes of 16-bit ones), four lanes a block: the largest magnitude is two
// exchanges within a quad, a lane's eight codes are one word, so both sides are whole lines, and nothing is kept across lanes otherwise.
#include <algorithm>

#include "mx_device.h"
#include "orx_internal.h"

namespace orx {
namespace {

constexpr int kThreads = 256, kPieces = 4;  // eight-value pieces to a thread

struct QuantParams {
    const void* x;
    uint8_t *q, *s;
    int64_t pieces_total;
    uint32_t pieces;  // of a row
    int k, ceil;
};

// bits of the largest magnitude of a lane's eight values
template <int TYPE, int WORDS>
__device__ __forceinline__ uint32_t largest_of(const uint32_t (&words)[WORDS]) {
    uint32_t found = 0;
#pragma unroll
    for (int j = 0; j < WORDS; ++j) found = TYPE == mx::F32 ? max(found, words[j] & 0x7FFFFFFFu) : mx::pair_max(found, words[j]);
    return TYPE == mx::F32 ? found : max(found & 0xFFFFu, found >> 16);
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void mx_quantise_kernel(QuantParams p) {
    constexpr int WORDS = TYPE == mx::F32 ? 8 : 4;
    const int64_t base = (int64_t)blockIdx.x * (kThreads * kPieces);
    const int64_t first_row = base / p.pieces;  // uniform: once a workgroup
    const uint32_t first_piece = (uint32_t)(base - first_row * p.pieces);
    uint32_t words[kPieces][WORDS];
    int64_t row[kPieces];
    uint32_t piece[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const uint32_t at = first_piece + i * kThreads + threadIdx.x;
        const uint32_t down = at / p.pieces;
        row[i] = first_row + down, piece[i] = at - down * p.pieces;
        const bool live = base + i * kThreads + threadIdx.x < p.pieces_total;
        const int first = (int)piece[i] * 8, count = live ? p.k - first : 0;
#pragma unroll
        for (int j = 0; j < WORDS; ++j) words[i][j] = 0;
        const int64_t offset = row[i] * p.k + first;
        if (count >= 8) {
            const mx::words4* const from = reinterpret_cast<const mx::words4*>(reinterpret_cast<const uint8_t*>(p.x) + offset * (TYPE == mx::F32 ? 4 : 2));
#pragma unroll
            for (int j = 0; j < WORDS / 4; ++j) {
                const mx::v4u four = from[j];
                words[i][4 * j] = four[0], words[i][4 * j + 1] = four[1], words[i][4 * j + 2] = four[2], words[i][4 * j + 3] = four[3];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < count) {
                    if constexpr (TYPE == mx::F32)
                        words[i][j] = reinterpret_cast<const uint32_t*>(p.x)[offset + j];
                    else
                        words[i][j / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(p.x)[offset + j] << (16 * (j & 1));
                }
        }
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        // (a row is whole blocks, so the lanes of a quad are pieces of one block, or all behind the end)
        const uint32_t byte = mx::power_byte<TYPE>(mx::quad_max(largest_of<TYPE>(words[i])), p.ceil != 0);
        if (base + i * kThreads + threadIdx.x >= p.pieces_total) continue;
        const int64_t at = row[i] * p.pieces + piece[i];
        reinterpret_cast<uint32_t*>(p.q)[at] = mx::eight_codes<TYPE>(words[i], byte);
        if ((threadIdx.x & 3) == 0) p.s[at >> 2] = (uint8_t)byte;
    }
}

// The same by tiles of 16 rows x 256 (the layout of the products): a wave takes 16 rows x 128, four rows of 256 bytes to a load, and its stores are runs of 64 bytes.  Rows
// of the last tile that are not there become 0.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void mx_quantise_tiles_kernel(QuantParams p, int rows, int steps, int groups) {
    constexpr int WORDS = TYPE == mx::F32 ? 8 : 4;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int tile = blockIdx.x / groups, window = (int)(blockIdx.x % groups) * (kThreads / 64) + wave;  // of 128 columns
    if (window >= 2 * steps) return;
    const int column = window * 128 + (lane & 15) * 8;
    uint32_t words[4][WORDS];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = (int64_t)tile * 16 + 4 * i + (lane >> 4);
        const int count = row < rows ? p.k - column : 0;
        const int64_t offset = row * p.k + column;
#pragma unroll
        for (int j = 0; j < WORDS; ++j) words[i][j] = 0;
        if (count >= 8) {
            const mx::words4* const from = reinterpret_cast<const mx::words4*>(reinterpret_cast<const uint8_t*>(p.x) + offset * (TYPE == mx::F32 ? 4 : 2));
#pragma unroll
            for (int j = 0; j < WORDS / 4; ++j) {
                const mx::v4u four = from[j];
                words[i][4 * j] = four[0], words[i][4 * j + 1] = four[1], words[i][4 * j + 2] = four[2], words[i][4 * j + 3] = four[3];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < count) {
                    if constexpr (TYPE == mx::F32)
                        words[i][j] = reinterpret_cast<const uint32_t*>(p.x)[offset + j];
                    else
                        words[i][j / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(p.x)[offset + j] << (16 * (j & 1));
                }
        }
    }
    const int64_t at = (int64_t)tile * steps + (window >> 1);
    const int block = (window & 1) * 4 + ((lane & 15) >> 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * i + (lane >> 4);
        const uint32_t byte = mx::power_byte<TYPE>(mx::quad_max(largest_of<TYPE>(words[i])), p.ceil != 0);
        *reinterpret_cast<uint32_t*>(p.q + at * mx::kTileBytes + block * 256 + r * 16 + (lane & 3) * 4) = mx::eight_codes<TYPE>(words[i], byte);
        if ((lane & 3) == 0) p.s[at * mx::kTilePowers + r * 8 + (block & 1) * 4 + (block >> 1)] = (uint8_t)byte;
    }
}

struct DequantParams {
    const uint8_t *q, *s;
    void* y;
    int64_t pieces_total;
    uint32_t pieces;
    int k, type;
};

__global__ __launch_bounds__(kThreads) void mx_dequantise_kernel(DequantParams p) {
    const int64_t base = (int64_t)blockIdx.x * (kThreads * kPieces);
    const int64_t first_row = base / p.pieces;
    const uint32_t first_piece = (uint32_t)(base - first_row * p.pieces);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        if (base + i * kThreads + threadIdx.x >= p.pieces_total) return;
        const uint32_t at = first_piece + i * kThreads + threadIdx.x;
        const uint32_t down = at / p.pieces, piece = at - down * p.pieces;
        const int64_t row = first_row + down, from = row * p.pieces + piece;
        const int first = (int)piece * 8;
        if (first >= p.k) continue;
        const uint32_t codes = reinterpret_cast<const uint32_t*>(p.q)[from];
        const uint32_t byte = p.s[from >> 2];
        const float power = __uint_as_float(byte << 23);
        auto two = [&](auto pair, float& a, float& b) { a = byte == 255u ? __uint_as_float(0x7FC00000u) : pair[0], b = byte == 255u ? __uint_as_float(0x7FC00000u) : pair[1]; };
        float v[8];
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, power, 0), v[0], v[1]);
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, power, 1), v[2], v[3]);
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, power, 2), v[4], v[5]);
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, power, 3), v[6], v[7]);
        const mx::v4f low = {v[0], v[1], v[2], v[3]}, high = {v[4], v[5], v[6], v[7]};
        if (p.type != mx::F32) {
            mx::store_eight_halves(p.y, row * p.k, first, p.k, mx::v4u{mx::two_values(v[0], v[1], p.type), mx::two_values(v[2], v[3], p.type),
                                                                      mx::two_values(v[4], v[5], p.type), mx::two_values(v[6], v[7], p.type)});
            continue;
        }
        mx::store_four(p.y, p.type, row * p.k, first, p.k, low);
        mx::store_four(p.y, p.type, row * p.k, first + 4, p.k, high);
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------------
// slots used: K, stride (K as stored), algorithm (type), flags (ceil), flags2 (tiles)
int geometry(const orx_function& f, int rows, Geometry* g) {
    if (f.flags2) {
        g->grid[0] = ceil_div(rows, 16) * ceil_div(2 * (f.stride / mx::kStepK), kThreads / 64);
        g->block[0] = kThreads;
        return ORX_OK;
    }
    g->grid[0] = (uint32_t)(((int64_t)rows * (f.stride / 8) + kThreads * kPieces - 1) / (kThreads * kPieces));
    g->block[0] = kThreads;
    return ORX_OK;
}
// Q, S, X, rows
int quantise_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    QuantParams p;
    p.q = pointer_arg<uint8_t>(args, 0), p.s = pointer_arg<uint8_t>(args, 1), p.x = pointer_arg<const void>(args, 2);
    p.pieces = (uint32_t)f.stride / 8, p.pieces_total = (int64_t)rows * p.pieces;
    p.k = f.K, p.ceil = f.flags;
    const dim3 grid(g.grid[0]), block(kThreads);
    if (f.flags2) {  // tiles
        const int steps = f.stride / mx::kStepK, groups = (2 * steps + kThreads / 64 - 1) / (kThreads / 64);
        if (f.algorithm == mx::F16) ORX_LAUNCH(mx_quantise_tiles_kernel<mx::F16>, grid, block, 0, s, p, rows, steps, groups);
        else if (f.algorithm == mx::BF16) ORX_LAUNCH(mx_quantise_tiles_kernel<mx::BF16>, grid, block, 0, s, p, rows, steps, groups);
        else ORX_LAUNCH(mx_quantise_tiles_kernel<mx::F32>, grid, block, 0, s, p, rows, steps, groups);
        return hip_check(hipGetLastError(), "launch mxfp4_quantization");
    }
    if (f.algorithm == mx::F16) ORX_LAUNCH(mx_quantise_kernel<mx::F16>, grid, block, 0, s, p);
    else if (f.algorithm == mx::BF16) ORX_LAUNCH(mx_quantise_kernel<mx::BF16>, grid, block, 0, s, p);
    else ORX_LAUNCH(mx_quantise_kernel<mx::F32>, grid, block, 0, s, p);
    return hip_check(hipGetLastError(), "launch mxfp4_quantization");
}
// Q, S, Y, rows
int dequantise_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    DequantParams p;
    p.q = pointer_arg<const uint8_t>(args, 0), p.s = pointer_arg<const uint8_t>(args, 1), p.y = pointer_arg<void>(args, 2);
    p.pieces = (uint32_t)f.stride / 8, p.pieces_total = (int64_t)rows * p.pieces;
    p.k = f.K, p.type = f.algorithm;
    ORX_LAUNCH(mx_dequantise_kernel, dim3(g.grid[0]), dim3(kThreads), 0, s, p);
    return hip_check(hipGetLastError(), "launch mxfp4_dequantization");
}

constexpr int kMaxK = 1 << 24;

int shape(const Variant& v, orx_function* f, const char* type_key) {
    bool bad = false;
    f->K = (int)v.integer("K", 0, &bad);
    const int pad = (int)v.integer("pad", mx::kBlock, &bad);
    f->algorithm = mx_type(v, type_key, "float16", &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    if (f->K <= 0 || f->K > kMaxK || (pad != mx::kBlock && pad != mx::kStepK)) {
        set_error("%s: need 0 < K <= %d and pad 32 or 256", f->symbol.c_str(), kMaxK);
        return ORX_ERR_BAD_VARIANT;
    }
    f->stride = pad == mx::kBlock ? (f->K + 31) / 32 * 32 : ((f->K + 255) / 256 | 1) * 256;  // (for the products an odd multiple)
    f->dynamic_rows = true;
    // (a launch's threads are counted in 32 bits)
    const int most = (int)std::min<int64_t>(1 << 24, ((1ll << 32) / kThreads - 1) * (kThreads * kPieces) / (f->stride / 8 + 64)) - 16;  // (or the tiles that these rows touch)
    f->capacity = (int)v.integer("M", most, &bad);
    if (bad || f->capacity < 1 || f->capacity > most) {
        if (!bad) set_error("%s: M must be 1 to %d for this K", f->symbol.c_str(), most);
        return ORX_ERR_BAD_VARIANT;
    }
    f->geometry = geometry;
    return ORX_OK;
}
int make_quantise(const Variant& v, orx_function* f) {
    const int code = shape(v, f, "input_dtype");
    if (code != ORX_OK) return code;
    bool bad = false;
    const std::string scale = v.string("scale", "floor", &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    const std::string layout = v.string("layout", "rows", &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    if (layout != "rows" && (layout != "tiles" || v.has("pad"))) {
        set_error("mxfp4_quantization: layout must be rows or tiles, and pad goes with rows");
        return ORX_ERR_BAD_VARIANT;
    }
    if (layout == "tiles") f->flags2 = 1, f->stride = (f->K + mx::kStepK - 1) / mx::kStepK * mx::kStepK;
    if (scale != "floor" && scale != "ceil") {
        set_error("mxfp4_quantization: scale must be floor or ceil");
        return ORX_ERR_BAD_VARIANT;
    }
    f->flags = scale == "ceil";
    f->args = {{"Q", ArgPointer, 4}, {"S", ArgPointer, 1}, {"X", ArgPointer, f->algorithm == mx::F32 ? 4u : 2u}, {"rows", ArgI32, 4}};
    f->launch = quantise_launch;
    f->device_function = f->flags2 ? (f->algorithm == mx::F16    ? reinterpret_cast<const void*>(&mx_quantise_tiles_kernel<mx::F16>)
                                      : f->algorithm == mx::BF16 ? reinterpret_cast<const void*>(&mx_quantise_tiles_kernel<mx::BF16>)
                                                                 : reinterpret_cast<const void*>(&mx_quantise_tiles_kernel<mx::F32>))
                         : f->algorithm == mx::F16    ? reinterpret_cast<const void*>(&mx_quantise_kernel<mx::F16>)
                         : f->algorithm == mx::BF16 ? reinterpret_cast<const void*>(&mx_quantise_kernel<mx::BF16>)
                                                    : reinterpret_cast<const void*>(&mx_quantise_kernel<mx::F32>);
    return ORX_OK;
}
int make_dequantise(const Variant& v, orx_function* f) {
    const int code = shape(v, f, "output_dtype");
    if (code != ORX_OK) return code;
    f->args = {{"Q", ArgPointer, 4}, {"S", ArgPointer, 1}, {"Y", ArgPointer, f->algorithm == mx::F32 ? 4u : 2u}, {"rows", ArgI32, 4}};
    f->launch = dequantise_launch;
    f->device_function = reinterpret_cast<const void*>(&mx_dequantise_kernel);
    return ORX_OK;
}

}  // namespace

int mx_type(const Variant& v, const char* key, const char* fallback, bool* bad) {
    const std::string name = v.string(key, fallback, bad);
    if (name == "float16") return mx::F16;
    if (name == "bfloat16") return mx::BF16;
    if (name == "float32") return mx::F32;
    if (!*bad) set_error("%s must be float16, bfloat16 or float32", key);
    *bad = true;
    return mx::F16;
}

int make_mx_projection(const Variant& v, orx_function* f);
int make_mx_grouped(const Variant& v, orx_function* f);

const Registration* mx_registrations(int* count) {
    static const Registration rows[] = {
        {"mxfp4_quantization", make_quantise, "K, input_dtype=float16|bfloat16|float32, scale=floor|ceil, layout=rows|tiles, pad=32|256, M=capacity", "Q,S,X,rows"},
        {"mxfp4_dequantization", make_dequantise, "K, output_dtype=float16|bfloat16|float32, pad=32|256, M=capacity", "Q,S,Y,rows"},
        {"mxfp4_projection", make_mx_projection, "M, N, K, dynamic_rows=false, input_dtype=mxfp4|float16|bfloat16 (up to 16 rows), epilogue=none|swiglu, output_dtype=float16|bfloat16|float32",
         "A[,AS],Out,W,WS[,m]"},
        {"mxfp4_grouped", make_mx_grouped,
         "rows, E, N, K, tiles, block_m=16|32|64|128|256, gather=false, input_dtype=mxfp4|float16 (block_m=16), epilogue=none|swiglu, "
         "output_dtype=float16|bfloat16|float32",
         "A[,AS],Out[,SlotToken],TileCount,TileUnits,W,WS"},
    };
    *count = (int)(sizeof(rows) / sizeof(rows[0]));
    return rows;
}

}  // namespace orx
