// Rows of 16-bit or 32-bit values to MXFP4 and back (the format: mx_device.h).
//
//   a = max |x| of a block, e = max(exponent(a) - 2, 0), code = E2M1(x / 2^(e - 127)), nearest, ties to even, saturating.
// Bound by memory: 2 bytes in and 17/32 out an element.  A lane takes eight values (16 bytes of 16-bit ones), four lanes a block: the largest magnitude is two
// exchanges within a quad, a lane's eight codes are one word, so both sides are whole lines, and nothing is kept across lanes otherwise.  Read past the caches: 8192 x 5120 bf16
// 25.0 -> 17.4 us (6.1 TB/s), by tiles 8192 x 4096 fp16 22.8 -> 17.5; two or eight pieces to a thread instead of four 24.0, 18.5.
#include <algorithm>

#include "mx_device.h"
#include "orx_internal.h"

namespace orx {
namespace {

constexpr int kThreads = 256;
// Eight-value pieces to a thread, all of whose loads are on their way together: four, one where there are few (us with four / one: 3 rows of 2048 3.1 / 2.4, 2048 of 512 5.0 / 3.0,
// 4096 of 2048 6.8 / 6.5, 32768 of 512 level, 8192 of 5120 19.9 / 21.9).
constexpr int kPieces = 4;
constexpr int64_t kFewPieces = 1 << 21;

// Rows of `pieces` eight-value pieces, one behind the other in one sequence of fewer than 2^32.
struct Rows {
    uint32_t total, pieces, inverse;  // inverse = floor(2^32 / pieces)
    uint32_t pitch;                   // pieces from one stored row to the next
    int k;
    // Row and piece of number `at`: the quotient by the inverse is at most one too small.
    __device__ __forceinline__ void split(uint32_t at, uint32_t& row, uint32_t& piece) const {
        row = __umulhi(at, inverse), piece = at - row * pieces;
        if (piece >= pieces) ++row, piece -= pieces;
    }
};
Rows rows_of(int rows, int pieces, int pitch, int k) {
    return {(uint32_t)rows * (uint32_t)pieces, (uint32_t)pieces, (uint32_t)std::min<uint64_t>((1ull << 32) / pieces, 0xFFFFFFFFull), (uint32_t)pitch, k};
}

struct QuantParams {
    const void* x;
    uint8_t *q, *s;
    Rows rows;
    int ceil;
};

// bits of the largest magnitude of a lane's eight values
template <int TYPE, int WORDS>
__device__ __forceinline__ uint32_t largest_of(const uint32_t (&words)[WORDS]) {
    uint32_t found = 0;
#pragma unroll
    for (int j = 0; j < WORDS; ++j) found = TYPE == mx::F32 ? max(found, words[j] & 0x7FFFFFFFu) : mx::pair_max(found, words[j]);
    return TYPE == mx::F32 ? found : max(found & 0xFFFFu, found >> 16);
}

// `count` of eight values from an address of their own alignment; what is not there is 0
template <int TYPE, int WORDS>
__device__ __forceinline__ void read_eight(uint32_t (&words)[WORDS], const void* x, int64_t offset, int count) {
#pragma unroll
    for (int j = 0; j < WORDS; ++j) words[j] = 0;
    if (count >= 8) {
        const mx::words4* const from = reinterpret_cast<const mx::words4*>(reinterpret_cast<const uint8_t*>(x) + offset * (TYPE == mx::F32 ? 4 : 2));
#pragma unroll
        for (int j = 0; j < WORDS / 4; ++j) {
            const mx::v4u four = __builtin_nontemporal_load(from + j);
            words[4 * j] = four[0], words[4 * j + 1] = four[1], words[4 * j + 2] = four[2], words[4 * j + 3] = four[3];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) {
                if constexpr (TYPE == mx::F32)
                    words[j] = reinterpret_cast<const uint32_t*>(x)[offset + j];
                else
                    words[j / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(x)[offset + j] << (16 * (j & 1));
            }
    }
}

// WHOLE: rows of whole blocks without a gap on either side, so that a piece's number is its place and no row is looked for.
template <int TYPE, bool WHOLE, int PIECES>
__global__ __launch_bounds__(kThreads) void mx_quantise_kernel(QuantParams p) {
    constexpr int WORDS = TYPE == mx::F32 ? 8 : 4;
    const uint32_t base = blockIdx.x * (kThreads * PIECES) + threadIdx.x;
    uint32_t words[PIECES][WORDS], to[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const uint32_t at = base + i * kThreads;
        const bool live = at < p.rows.total;
        int count = live ? 8 : 0;
        int64_t offset = (int64_t)at * 8;
        to[i] = at;
        if constexpr (!WHOLE) {
            uint32_t row, piece;
            p.rows.split(at, row, piece);
            count = live ? p.rows.k - (int)piece * 8 : 0;
            offset = (int64_t)row * p.rows.k + piece * 8;
            to[i] = row * p.rows.pitch + piece;
        }
        read_eight<TYPE>(words[i], p.x, offset, count);
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        // (a row is whole blocks, so the lanes of a quad are pieces of one block, or all behind the end)
        const uint32_t byte = mx::power_byte<TYPE>(mx::quad_max(largest_of<TYPE>(words[i])), p.ceil != 0);
        if (base + i * kThreads >= p.rows.total) continue;
        reinterpret_cast<uint32_t*>(p.q)[to[i]] = mx::eight_codes<TYPE>(words[i], byte);
        if ((threadIdx.x & 3) == 0) p.s[to[i] >> 2] = (uint8_t)byte;
    }
}

// The same by tiles of 16 rows x 256 (the layout of the products): a wave takes 4 LOADS rows x 128, four rows of 256 bytes to a load, and its stores are runs of 64 bytes.  Rows
// of the last tile that are not there become 0.
template <int TYPE, int LOADS>
__global__ __launch_bounds__(kThreads) void mx_quantise_tiles_kernel(QuantParams p, int rows, int steps, int groups) {
    constexpr int PARTS = 4 / LOADS;  // of a tile
    constexpr int WORDS = TYPE == mx::F32 ? 8 : 4;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int at_tile = blockIdx.x / groups, tile = at_tile / PARTS, first = at_tile % PARTS * (4 * LOADS), window = (int)(blockIdx.x % groups) * (kThreads / 64) + wave;  // of 128 columns
    if (window >= 2 * steps) return;
    const int column = window * 128 + (lane & 15) * 8;
    uint32_t words[LOADS][WORDS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int64_t row = (int64_t)tile * 16 + first + 4 * i + (lane >> 4);
        read_eight<TYPE>(words[i], p.x, row * p.rows.k + column, row < rows ? p.rows.k - column : 0);
    }
    const int64_t at = (int64_t)tile * steps + (window >> 1);
    const int block = (window & 1) * 4 + ((lane & 15) >> 2);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r = first + 4 * i + (lane >> 4);
        const uint32_t byte = mx::power_byte<TYPE>(mx::quad_max(largest_of<TYPE>(words[i])), p.ceil != 0);
        *reinterpret_cast<uint32_t*>(p.q + at * mx::kTileBytes + block * 256 + r * 16 + (lane & 3) * 4) = mx::eight_codes<TYPE>(words[i], byte);
        if ((lane & 3) == 0) p.s[at * mx::kTilePowers + r * 8 + (block & 1) * 4 + (block >> 1)] = (uint8_t)byte;
    }
}

struct DequantParams {
    const uint8_t *q, *s;
    void* y;
    Rows rows;
    int type;
};

template <bool WHOLE, int PIECES>
__global__ __launch_bounds__(kThreads) void mx_dequantise_kernel(DequantParams p) {
    const uint32_t base = blockIdx.x * (kThreads * PIECES) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const uint32_t at = base + i * kThreads;
        if (at >= p.rows.total) return;
        uint32_t from = at;
        int64_t row_start = 0;
        int first = 0, k = 8;
        if constexpr (WHOLE) {
            row_start = (int64_t)at * 8;
        } else {
            uint32_t row, piece;
            p.rows.split(at, row, piece);
            from = row * p.rows.pitch + piece, row_start = (int64_t)row * p.rows.k, first = (int)piece * 8, k = p.rows.k;
            if (first >= k) continue;
        }
        const uint32_t codes = reinterpret_cast<const uint32_t*>(p.q)[from];
        const uint32_t byte = p.s[from >> 2];
        const float power = __uint_as_float(byte << 23);
        float v[8];
        auto two = [&](auto pair, float& a, float& b) { a = byte == 255u ? __uint_as_float(0x7FC00000u) : pair[0], b = byte == 255u ? __uint_as_float(0x7FC00000u) : pair[1]; };
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, power, 0), v[0], v[1]);
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, power, 1), v[2], v[3]);
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, power, 2), v[4], v[5]);
        two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, power, 3), v[6], v[7]);
        if (p.type != mx::F32) {
            mx::store_eight_halves(p.y, row_start, first, k, mx::v4u{mx::two_values(v[0], v[1], p.type), mx::two_values(v[2], v[3], p.type), mx::two_values(v[4], v[5], p.type),
                                                                     mx::two_values(v[6], v[7], p.type)});
            continue;
        }
        mx::store_four(p.y, p.type, row_start, first, k, mx::v4f{v[0], v[1], v[2], v[3]});
        mx::store_four(p.y, p.type, row_start, first + 4, k, mx::v4f{v[4], v[5], v[6], v[7]});
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------------
// slots used: K, group (K in whole blocks, or in steps of 256 for the products), stride (from one stored row to the next), algorithm (type), flags (ceil), flags2 (tiles)
bool few_pieces(const orx_function& f, int rows) { return (int64_t)rows * (f.group / 8) <= kFewPieces; }
int geometry(const orx_function& f, int rows, Geometry* g) {
    const bool few = few_pieces(f, rows);
    const int64_t pieces = (int64_t)rows * (f.group / 8), to_a_block = kThreads * (few ? 1 : kPieces);
    g->grid[0] = f.flags2 ? ceil_div(rows, 16) * (few ? 4 : 1) * ceil_div(f.group / 128, kThreads / 64) : (uint32_t)((pieces + to_a_block - 1) / to_a_block);
    g->block[0] = kThreads;
    return ORX_OK;
}
template <int TYPE, int PIECES>
void quantise(const orx_function& f, int rows, const Geometry& g, hipStream_t s, const QuantParams& p) {
    const dim3 grid(g.grid[0]), block(kThreads);
    if (f.flags2) ORX_LAUNCH((mx_quantise_tiles_kernel<TYPE, PIECES>), grid, block, 0, s, p, rows, f.group / mx::kStepK, (int)ceil_div(f.group / 128, kThreads / 64));
    else if (f.K == f.stride) ORX_LAUNCH((mx_quantise_kernel<TYPE, true, PIECES>), grid, block, 0, s, p);
    else ORX_LAUNCH((mx_quantise_kernel<TYPE, false, PIECES>), grid, block, 0, s, p);
}
template <int TYPE>
void quantise(const orx_function& f, int rows, const Geometry& g, hipStream_t s, const QuantParams& p) {
    if (few_pieces(f, rows)) quantise<TYPE, 1>(f, rows, g, s, p);
    else quantise<TYPE, kPieces>(f, rows, g, s, p);
}
template <int PIECES>
void dequantise(const orx_function& f, const Geometry& g, hipStream_t s, const DequantParams& p) {
    if (f.K == f.stride) ORX_LAUNCH((mx_dequantise_kernel<true, PIECES>), dim3(g.grid[0]), dim3(kThreads), 0, s, p);
    else ORX_LAUNCH((mx_dequantise_kernel<false, PIECES>), dim3(g.grid[0]), dim3(kThreads), 0, s, p);
}
// Q, S, X, rows
int quantise_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    QuantParams p;
    p.q = pointer_arg<uint8_t>(args, 0), p.s = pointer_arg<uint8_t>(args, 1), p.x = pointer_arg<const void>(args, 2);
    p.rows = rows_of(rows, f.group / 8, f.stride / 8, f.K), p.ceil = f.flags;
    if (f.algorithm == mx::F16) quantise<mx::F16>(f, rows, g, s, p);
    else if (f.algorithm == mx::BF16) quantise<mx::BF16>(f, rows, g, s, p);
    else quantise<mx::F32>(f, rows, g, s, p);
    return hip_check(hipGetLastError(), "launch mxfp4_quantization");
}
// Q, S, Y, rows
int dequantise_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    DequantParams p;
    p.q = pointer_arg<const uint8_t>(args, 0), p.s = pointer_arg<const uint8_t>(args, 1), p.y = pointer_arg<void>(args, 2);
    p.rows = rows_of(rows, f.group / 8, f.stride / 8, f.K), p.type = f.algorithm;
    if (few_pieces(f, rows)) dequantise<1>(f, g, s, p);
    else dequantise<kPieces>(f, g, s, p);
    return hip_check(hipGetLastError(), "launch mxfp4_dequantization");
}

constexpr int kMaxK = 1 << 24;

int shape(const Variant& v, orx_function* f, const char* type_key, bool tiles) {
    bool bad = false;
    f->K = (int)v.integer("K", 0, &bad);
    const int pad = tiles ? mx::kStepK : (int)v.integer("pad", mx::kBlock, &bad);
    f->algorithm = mx_type(v, type_key, "float16", &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    if (f->K <= 0 || f->K > kMaxK || (pad != mx::kBlock && pad != mx::kStepK)) {
        set_error("%s: need 0 < K <= %d and pad 32 or 256", f->symbol.c_str(), kMaxK);
        return ORX_ERR_BAD_VARIANT;
    }
    f->flags2 = tiles;
    f->group = pad == mx::kBlock ? (f->K + 31) / 32 * 32 : (f->K + 255) / 256 * 256;
    f->stride = pad == mx::kBlock || tiles ? f->group : (f->group / 256 | 1) * 256;  // (for the products an odd multiple; what is behind `group` is not written)
    f->dynamic_rows = true;
    // Rows: pieces are counted in 32 bits (a launch's threads are a quarter of them).  Tiles: addresses are 64 bits wide, a launch's threads are fewer than 2^32.
    const int64_t counted = tiles ? 16 * (0xFFFFFFFFll / kThreads / ceil_div(f->group / 128, kThreads / 64)) : ((1ll << 32) - 65536) / (f->stride / 8);
    const int most = (int)std::min<int64_t>(1 << 24, counted);
    f->capacity = (int)v.integer("M", most, &bad);
    if (bad || f->capacity < 1 || f->capacity > most) {
        if (!bad) set_error("%s: M must be 1 to %d for this K", f->symbol.c_str(), most);
        return ORX_ERR_BAD_VARIANT;
    }
    f->geometry = geometry;
    return ORX_OK;
}
int make_quantise(const Variant& v, orx_function* f) {
    bool bad = false;
    const std::string scale = v.string("scale", "floor", &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    const std::string layout = v.string("layout", "rows", &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    if (layout != "rows" && (layout != "tiles" || v.has("pad"))) {
        set_error("mxfp4_quantization: layout must be rows or tiles, and pad goes with rows");
        return ORX_ERR_BAD_VARIANT;
    }
    if (scale != "floor" && scale != "ceil") {
        set_error("mxfp4_quantization: scale must be floor or ceil");
        return ORX_ERR_BAD_VARIANT;
    }
    const int code = shape(v, f, "input_dtype", layout == "tiles");
    if (code != ORX_OK) return code;
    f->flags = scale == "ceil";
    f->args = {{"Q", ArgPointer, 4}, {"S", ArgPointer, 1}, {"X", ArgPointer, f->algorithm == mx::F32 ? 4u : 2u}, {"rows", ArgI32, 4}};
    f->launch = quantise_launch;
    const bool whole = f->K == f->stride;
#define ORX_QUANTISE(TYPE)                                                                            \
    (f->flags2 ? reinterpret_cast<const void*>(&mx_quantise_tiles_kernel<TYPE, kPieces>)                       \
     : whole   ? reinterpret_cast<const void*>(&mx_quantise_kernel<TYPE, true, kPieces>)                       \
               : reinterpret_cast<const void*>(&mx_quantise_kernel<TYPE, false, kPieces>))
    f->device_function = f->algorithm == mx::F16 ? ORX_QUANTISE(mx::F16) : f->algorithm == mx::BF16 ? ORX_QUANTISE(mx::BF16) : ORX_QUANTISE(mx::F32);
#undef ORX_QUANTISE
    return ORX_OK;
}
int make_dequantise(const Variant& v, orx_function* f) {
    const int code = shape(v, f, "output_dtype", false);
    if (code != ORX_OK) return code;
    f->args = {{"Q", ArgPointer, 4}, {"S", ArgPointer, 1}, {"Y", ArgPointer, f->algorithm == mx::F32 ? 4u : 2u}, {"rows", ArgI32, 4}};
    f->launch = dequantise_launch;
    f->device_function = f->K == f->stride ? reinterpret_cast<const void*>(&mx_dequantise_kernel<true, kPieces>) : reinterpret_cast<const void*>(&mx_dequantise_kernel<false, kPieces>);
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
         "rows, E, N, K, tiles, block_m=16|64|128|256, gather=false, input_dtype=mxfp4|float16 (block_m=16), epilogue=none|swiglu, "
         "output_dtype=float16|bfloat16|float32",
         "A[,AS],Out[,SlotToken],TileCount,TileUnits,W,WS"},
    };
    *count = (int)(sizeof(rows) / sizeof(rows[0]));
    return rows;
}

}  // namespace orx
