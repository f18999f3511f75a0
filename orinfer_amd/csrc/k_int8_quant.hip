// Rows of 16-bit or 32-bit values to 8-bit integers with an fp32 scale and, if wanted, a zero point for each row (the rules: byte_device.h).
//
// Bound by memory: 2 bytes in and 1 out an element.  A row's values stay in registers between its largest magnitude and its codes, 8 values (16 bytes of 16-bit ones) to a piece, HELD pieces to a
// thread; what a longer row has beyond them is read again.
#include <algorithm>

#include "byte_device.h"
#include "orx_internal.h"

namespace orx {
namespace {

using namespace bytes;

constexpr int kHeld = 4;

struct QuantParams {
    const void* x;
    uint8_t* q;
    float* s;
    int* z;
    int rows, k, pieces;  // pieces of eight codes that a row has, zeros behind K among them
    int64_t pitch;
};

// `count` of eight values from an address of their own alignment; what is not there is 0
template <int TYPE, int WORDS>
__device__ __forceinline__ void read_eight(uint32_t (&words)[WORDS], const uint8_t* from, int count) {
#pragma unroll
    for (int j = 0; j < WORDS; ++j) words[j] = 0;
    if (count >= 8) {
#pragma unroll
        for (int j = 0; j < WORDS / 4; ++j) {
            const v4u four = __builtin_nontemporal_load(reinterpret_cast<const mx::words4*>(from) + j);
            words[4 * j] = four[0], words[4 * j + 1] = four[1], words[4 * j + 2] = four[2], words[4 * j + 3] = four[3];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) {
                if constexpr (TYPE == mx::F32) words[j] = reinterpret_cast<const uint32_t*>(from)[j];
                else words[j / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(from)[j] << (16 * (j & 1));
            }
    }
}

// WAVES waves to a row, at least four waves to a workgroup
template <int TYPE, int WAVES, bool ZERO>
__global__ __launch_bounds__(WAVES < 4 ? 256 : 64 * WAVES) void int8_quantise_kernel(QuantParams p) {
    constexpr int WORDS = TYPE == mx::F32 ? 8 : 4, BYTES = TYPE == mx::F32 ? 4 : 2, THREADS = 64 * WAVES, ROWS = WAVES < 4 ? 4 / WAVES : 1;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int at = (int)threadIdx.x % THREADS;
    __shared__ RowRange found[2][WAVES];
    int round = 0;
#pragma unroll 1
    for (int row = (int)blockIdx.x * ROWS + wave / WAVES; row < p.rows; row += (int)gridDim.x * ROWS) {
        const uint8_t* const x = reinterpret_cast<const uint8_t*>(p.x) + (int64_t)row * p.k * BYTES;
        RowRange range = {0, 0.f, 0.f};
        uint32_t words[kHeld][WORDS];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) read_eight<TYPE>(words[i], x + (int64_t)(at + i * THREADS) * (8 * BYTES), p.k - (at + i * THREADS) * 8);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) widen<TYPE, ZERO>(range, words[i]);
        for (int piece = at + kHeld * THREADS; piece < p.pieces; piece += THREADS) {
            uint32_t more[WORDS];
            read_eight<TYPE>(more, x + (int64_t)piece * (8 * BYTES), p.k - piece * 8);
            widen<TYPE, ZERO>(range, more);
        }
        range = over_wave<TYPE, ZERO>(range);
        if constexpr (WAVES > 1) {  // (all waves of a workgroup are at the same row; the other half is for the next one)
            RowRange(&mine)[WAVES] = found[round ^= 1];
            if ((threadIdx.x & 63) == 0) mine[wave] = range;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WAVES; ++i) range.bits = max(range.bits, mine[i].bits), range.high = fmaxf(range.high, mine[i].high), range.low = fmaxf(range.low, mine[i].low);
        }
        const RowCode code = code_of<TYPE, ZERO>(range);
        uint8_t* const q = p.q + row * p.pitch;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int piece = at + i * THREADS;
            if (piece < p.pieces) *reinterpret_cast<uint2*>(q + (int64_t)piece * 8) = eight_codes<TYPE, ZERO>(words[i], code);
        }
        for (int piece = at + kHeld * THREADS; piece < p.pieces; piece += THREADS) {
            uint32_t more[WORDS];
            read_eight<TYPE>(more, x + (int64_t)piece * (8 * BYTES), p.k - piece * 8);
            *reinterpret_cast<uint2*>(q + (int64_t)piece * 8) = eight_codes<TYPE, ZERO>(more, code);
        }
        if (at == 0) {
            p.s[row] = stored_scale(code);
            if constexpr (ZERO) p.z[row] = code.zero;
        }
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------------
// slots used: K, group (K in whole steps of 128), stride (from one stored row to the next), algorithm (type), flags (zero points)
constexpr int kMaxK = 1 << 24;
constexpr uint32_t kMostGroups = 1 << 21;  // (a launch's threads are fewer than 2^32)

// Waves to a row: those that hold it, up to sixteen.
int waves_to_a_row(const orx_function& f, int rows) {
    const int held = 64 * 8 * kHeld;
    return f.group <= held ? 1 : f.group <= 4 * held ? 4 : 16;
}
int geometry(const orx_function& f, int rows, Geometry* g) {
    const int waves = waves_to_a_row(f, rows);
    g->grid[0] = std::min<uint32_t>(waves < 4 ? ceil_div(rows, 4 / waves) : rows, kMostGroups);
    g->block[0] = waves < 4 ? 256 : 64 * waves;
    return ORX_OK;
}
template <int TYPE, bool ZERO>
void quantise(const orx_function& f, int rows, const Geometry& g, hipStream_t s, const QuantParams& p) {
    const int waves = waves_to_a_row(f, rows);
    const dim3 grid(g.grid[0]), block(g.block[0]);
    if (waves == 1) ORX_LAUNCH((int8_quantise_kernel<TYPE, 1, ZERO>), grid, block, 0, s, p);
    else if (waves == 4) ORX_LAUNCH((int8_quantise_kernel<TYPE, 4, ZERO>), grid, block, 0, s, p);
    else ORX_LAUNCH((int8_quantise_kernel<TYPE, 16, ZERO>), grid, block, 0, s, p);
}
template <int TYPE>
void quantise(const orx_function& f, int rows, const Geometry& g, hipStream_t s, const QuantParams& p) {
    if (f.flags) quantise<TYPE, true>(f, rows, g, s, p);
    else quantise<TYPE, false>(f, rows, g, s, p);
}
// Q, S, X[, Z], rows
int quantise_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    QuantParams p = {};
    p.q = pointer_arg<uint8_t>(args, 0), p.s = pointer_arg<float>(args, 1), p.x = pointer_arg<const void>(args, 2);
    p.z = f.flags ? pointer_arg<int>(args, 3) : nullptr;
    p.rows = rows, p.k = f.K, p.pieces = f.group / 8, p.pitch = f.stride;
    if (f.algorithm == mx::F16) quantise<mx::F16>(f, rows, g, s, p);
    else if (f.algorithm == mx::BF16) quantise<mx::BF16>(f, rows, g, s, p);
    else quantise<mx::F32>(f, rows, g, s, p);
    return hip_check(hipGetLastError(), "launch int8_token_quantization");
}
int make_quantise(const Variant& v, orx_function* f) {
    bool bad = false;
    f->K = (int)v.integer("K", 0, &bad);
    f->algorithm = mx_type(v, "input_dtype", "float16", &bad);
    f->flags = v.boolean("zero_points", false, &bad);
    f->capacity = (int)v.integer("M", 1 << 24, &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    if (f->K <= 0 || f->K > kMaxK || f->capacity < 1 || f->capacity > 1 << 24) {
        set_error("int8_token_quantization: need 0 < K <= %d and M from 1 to %d", kMaxK, 1 << 24);
        return ORX_ERR_BAD_VARIANT;
    }
    f->group = (f->K + kStep - 1) / kStep * kStep;
    f->stride = (f->group / kStep | 1) * kStep;
    f->dynamic_rows = true;
    f->geometry = geometry;
    f->args = {{"Q", ArgPointer, 8}, {"S", ArgPointer, 4}, {"X", ArgPointer, f->algorithm == mx::F32 ? 4u : 2u}};
    if (f->flags) f->args.push_back({"Z", ArgPointer, 4});
    f->args.push_back({"rows", ArgI32, 4});
    f->launch = quantise_launch;
    return ORX_OK;
}

}  // namespace

int make_int8_projection(const Variant& v, orx_function* f);
int make_int8_grouped(const Variant& v, orx_function* f);
int make_half_grouped(const Variant& v, orx_function* f);

const Registration* byte_registrations(int* count) {
    static const Registration rows[] = {
        {"int8_token_quantization", make_quantise, "K, input_dtype=float16|bfloat16|float32, zero_points=false, M=capacity", "Q,S,X[,Z],rows"},
        {"int8_token_projection", make_int8_projection,
         "M, N, K, dynamic_rows=false, input_dtype=int8|float16|bfloat16 (few rows), zero_points=false, bias=false, epilogue=none|swiglu, output_dtype=float16|bfloat16|float32",
         "A[,AS][,AZ][,Bias],Out,W,WS[,WSum][,m]"},
        {"int8_token_grouped", make_int8_grouped,
         "rows, E, N, K, tiles, block_m=16|64|128|256, gather=false, input_dtype=int8|float16|bfloat16 (block_m=16), epilogue=none|swiglu, output_dtype=float16|bfloat16|float32",
         "A[,AS],Out[,SlotToken],TileCount,TileUnits,W,WS"},
        {"half_grouped", make_half_grouped,
         "rows, E, N, K, tiles, block_m=16|64|128|256, gather=false, dtype=float16|bfloat16, epilogue=none|swiglu, output_dtype=float16|bfloat16|float32",
         "A,Out[,SlotToken],TileCount,TileUnits,W"},
    };
    *count = (int)(sizeof(rows) / sizeof(rows[0]));
    return rows;
}

}  // namespace orx
