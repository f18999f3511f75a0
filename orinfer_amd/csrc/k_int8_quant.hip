// Rows of 16-bit or 32-bit values to 8-bit integers with an fp32 scale and, if wanted, a zero point for each row (the rules: byte_device.h).
//
// Bound by memory: 2 bytes in and 1 out an element.  A row's values stay in registers between its largest magnitude and its codes, 8 values (16 bytes of 16-bit ones) to a piece, HELD pieces to a
// thread; what a longer row has beyond them is read again.  Many rows: a wave or two to each, eight rows to a workgroup, because a line of a tile has pieces of eight rows (and lines that
// several XCDs write in part reach the memory in parts); few rows: a workgroup to each.
#include <algorithm>

#include "byte_device.h"
#include "orx_internal.h"

namespace orx {
namespace {

using namespace bytes;

struct QuantParams {
    const void* x;
    uint8_t* q;
    float* s;
    int* z;
    int rows, k, pieces;  // pieces of eight codes that a row has, those behind K among them
    int64_t pitch;  // by rows
    int steps;      // by tiles of 16 rows
};

// `count` of eight values from an address of their own alignment; what is not there is 0.  WHOLE: all eight or none.
template <int TYPE, bool WHOLE, int WORDS>
__device__ __forceinline__ void read_eight(uint32_t (&words)[WORDS], const uint8_t* from, int count) {
#pragma unroll
    for (int j = 0; j < WORDS; ++j) words[j] = 0;
    if (count >= 8) {
#pragma unroll
        for (int j = 0; j < WORDS / 4; ++j) {
            const v4u four = __builtin_nontemporal_load(reinterpret_cast<const mx::words4*>(from) + j);
            words[4 * j] = four[0], words[4 * j + 1] = four[1], words[4 * j + 2] = four[2], words[4 * j + 3] = four[3];
        }
    } else if constexpr (!WHOLE) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) {
                if constexpr (TYPE == mx::F32) words[j] = reinterpret_cast<const uint32_t*>(from)[j];
                else words[j / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(from)[j] << (16 * (j & 1));
            }
    }
}

// Where a row's eight codes number `piece` go: rows lie `pitch` apart, or by tiles of 16 rows x 128, [piece of 16 codes][row][16] (tiles of the same rows along K behind one another).
template <bool TILES>
__device__ __forceinline__ uint8_t* place_of(const QuantParams& p, int row, int piece) {
    if constexpr (TILES) return p.q + ((int64_t)(row >> 4) * p.steps + (piece >> 4)) * kTileBytes + ((piece >> 1) & 7) * 256 + (row & 15) * 16 + (piece & 1) * 8;
    return p.q + row * p.pitch + (int64_t)piece * 8;
}

// How rows are dealt: EACH rows to a wave at a time, ROWS x EACH to a workgroup, WAVES waves to a row, HELD pieces to a thread.
template <int EACH_, int ROWS_, int WAVES_, int HELD_>
struct Deal {
    static constexpr int EACH = EACH_, ROWS = ROWS_, WAVES = WAVES_, HELD = HELD_;
    static_assert(EACH == 1 || WAVES == 1, "rows of several waves meet one by one");
};

template <int TYPE, typename DEAL, bool WHOLE, bool ZERO, bool TILES>
__global__ __launch_bounds__(64 * DEAL::ROWS * DEAL::WAVES, 4) void int8_quantise_kernel(QuantParams p) {
    constexpr int EACH = DEAL::EACH, ROWS = DEAL::ROWS, WAVES = DEAL::WAVES, HELD = DEAL::HELD;
    constexpr int WORDS = TYPE == mx::F32 ? 8 : 4, BYTES = TYPE == mx::F32 ? 4 : 2, THREADS = 64 * WAVES;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int at = (int)threadIdx.x % THREADS;
    __shared__ RowRange found[2][ROWS * WAVES];
    // Eight rows' codes by tiles meet in LDS and leave as whole lines: 16-byte pieces of eight rows, and 16 bytes more so that pieces behind one another lie in other banks.
    constexpr bool MEET = TILES && ROWS == 8;
    extern __shared__ __align__(16) uint8_t lds[];
    int round = 0;
#pragma unroll 1
    for (int64_t base = (int64_t)blockIdx.x * (ROWS * EACH); base < p.rows; base += (int64_t)gridDim.x * (ROWS * EACH)) {
        uint32_t words[EACH][HELD][WORDS];
        int row[EACH];
        const uint8_t* x[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            row[e] = (int)base + wave / WAVES + ROWS * e;
            x[e] = reinterpret_cast<const uint8_t*>(p.x) + (int64_t)row[e] * p.k * BYTES;
            const int k = row[e] < p.rows ? p.k : 0;
#pragma unroll
            for (int i = 0; i < HELD; ++i) read_eight<TYPE, WHOLE>(words[e][i], x[e] + (int64_t)(at + i * THREADS) * (8 * BYTES), k - (at + i * THREADS) * 8);
        }
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const bool live = row[e] < p.rows;
            RowRange range = {0, 0};
#pragma unroll
            for (int i = 0; i < HELD; ++i) widen<TYPE, ZERO>(range, words[e][i]);
            for (int piece = at + HELD * THREADS; live && piece < p.pieces; piece += THREADS) {
                uint32_t more[WORDS];
                read_eight<TYPE, WHOLE>(more, x[e] + (int64_t)piece * (8 * BYTES), p.k - piece * 8);
                widen<TYPE, ZERO>(range, more);
            }
            range = over_wave<TYPE, ZERO>(range);
            if constexpr (WAVES > 1) {  // (all waves of a workgroup are at the same rows; the other half is for the next ones)
                RowRange(&mine)[ROWS * WAVES] = found[round ^= 1];
                if ((threadIdx.x & 63) == 0) mine[wave] = range;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < WAVES; ++i) range = wider(range, mine[wave / WAVES * WAVES + i]);
            }
            const RowCode code = code_of<TYPE, ZERO>(range);
            auto place = [&](int piece) -> uint8_t* {
                if constexpr (MEET) return lds + ((piece >> 1) + e * (p.pieces >> 1)) * 144 + wave / WAVES * 16 + (piece & 1) * 8;
                else return place_of<TILES>(p, row[e], piece);
            };
            if (live) {
#pragma unroll
                for (int i = 0; i < HELD; ++i) {
                    const int piece = at + i * THREADS;
                    if (piece < p.pieces) *reinterpret_cast<uint2*>(place(piece)) = eight_codes<TYPE, ZERO>(words[e][i], code);
                    __builtin_amdgcn_sched_barrier(0);  // (all pieces' values at once take twice the registers)
                }
                for (int piece = at + HELD * THREADS; piece < p.pieces; piece += THREADS) {
                    uint32_t more[WORDS];
                    read_eight<TYPE, WHOLE>(more, x[e] + (int64_t)piece * (8 * BYTES), p.k - piece * 8);
                    *reinterpret_cast<uint2*>(place(piece)) = eight_codes<TYPE, ZERO>(more, code);
                }
                if (at == 0) {
                    p.s[row[e]] = stored_scale(code);
                    if constexpr (ZERO) p.z[row[e]] = code.zero;
                }
            }
        }
        if constexpr (MEET) {
            __syncthreads();
            const int pieces = p.pieces >> 1;  // of 16 codes
            for (int i = threadIdx.x; i < EACH * pieces * 8; i += 64 * ROWS * WAVES) {
                const int r = i & 7, in = i >> 3, e = in / pieces, piece = in - e * pieces;
                const int to = (int)base + r + ROWS * e;
                if (to < p.rows) *reinterpret_cast<v4u*>(place_of<true>(p, to, 2 * piece)) = *reinterpret_cast<const v4u*>(lds + in * 144 + r * 16);
            }
            __syncthreads();
        }
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------------
// slots used: K, group (K in whole pairs of steps), stride (from one stored row to the next), algorithm (type), flags (zero points), flags2 (by tiles)
constexpr int kMaxK = 1 << 24;
constexpr uint32_t kMostGroups = 1 << 21;  // (a launch's threads are fewer than 2^32)

// The deal for `rows` rows of K values; and whether they are whole pieces of eight, which the others only have few of.  us of bf16 rows, with zero points up to a tenth more, the deal taken first
// (rows x K):
//   four rows to a wave or one: 32768 x 512 15.0 and 16.6, 8192 x 512 7.3 and 6.6;
//   by rows: eight rows to a workgroup or one: 8192 x 2048 12.3 and 14.6, 2048 x 2048 7.6 and 6.5, 8192 x 4096 22.7 and 19.6, 8192 x 8192 48.8 and 34.6; four waves to a row or sixteen:
//     8192 x 5120 23.3 and 46.0, 2048 x 17408 29.5 and 24.0, 64 x 17408 11.2 and 5.7;
//   by tiles: eight rows or one: 2048 x 2048 6.6 and 9.4, 2048 x 4096 10.2 and 13.9, 1024 x 4096 8.6 and 7.4; of eight rows two waves to a row or one: 8192 x 4096 23.7 and 25.8, 8192 x 8192
//     52.1 and 64.6, 4096 x 2048 8.9 and 10.0, 8192 x 2048 14.7 and 13.3.
template <typename BODY>
void with_deal(const orx_function& f, int rows, BODY body) {
    const int k = f.K;
    const bool tiles = f.flags2;
    if (k % 8) {
        if (k <= 1024 || (tiles && k <= 8192 && rows >= 2048)) body(Deal<1, 8, 1, 4>{}, std::false_type{});
        else body(Deal<1, 1, 4, 4>{}, std::false_type{});
    } else if (k <= 512 && rows >= 16384) body(Deal<4, 8, 1, 1>{}, std::true_type{});
    else if (k <= 1024 || (k <= 2048 && rows >= 8192)) body(Deal<1, 8, 1, 4>{}, std::true_type{});
    else if (k > 8192) body(Deal<1, 1, 16, 4>{}, std::true_type{});
    else if (!tiles || rows < (k <= 2048 ? 1024 : 1536)) body(Deal<1, 1, 4, 4>{}, std::true_type{});
    else body(Deal<1, 8, 2, 4>{}, std::true_type{});
}
int geometry(const orx_function& f, int rows, Geometry* g) {
    with_deal(f, rows, [&](auto deal, auto) {
        using DEAL = decltype(deal);
        g->grid[0] = std::min<uint32_t>(ceil_div(rows, DEAL::ROWS * DEAL::EACH), kMostGroups);
        g->block[0] = 64 * DEAL::ROWS * DEAL::WAVES;
        g->shared = f.flags2 && DEAL::ROWS == 8 ? DEAL::EACH * (f.group / 16) * 144 : 0;
    });
    return ORX_OK;
}
constexpr uint32_t kMostLds = 8192 / 16 * 144;  // (of the eight rows that a workgroup has)
template <int TYPE, typename DEAL, bool WHOLE, bool ZERO, bool TILES>
int launch_one(const Geometry& g, hipStream_t s, const QuantParams& p) {
    constexpr auto kernel = &int8_quantise_kernel<TYPE, DEAL, WHOLE, ZERO, TILES>;
    if constexpr (TILES && DEAL::ROWS == 8) {
        static DeviceOnce ready;
        const int code = ready.run([] { return hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds), "hipFuncSetAttribute"); });
        if (code != ORX_OK) return code;
    }
    ORX_LAUNCH(kernel, dim3(g.grid[0]), dim3(g.block[0]), g.shared, s, p);
    return hip_check(hipGetLastError(), "launch int8_token_quantization");
}
template <int TYPE, bool ZERO>
int quantise(const orx_function& f, int rows, const Geometry& g, hipStream_t s, const QuantParams& p) {
    int code = ORX_OK;
    with_deal(f, rows, [&](auto deal, auto whole) {
        using DEAL = decltype(deal);
        constexpr bool WHOLE = decltype(whole)::value;
        code = f.flags2 ? launch_one<TYPE, DEAL, WHOLE, ZERO, true>(g, s, p) : launch_one<TYPE, DEAL, WHOLE, ZERO, false>(g, s, p);
    });
    return code;
}
template <int TYPE>
int quantise(const orx_function& f, int rows, const Geometry& g, hipStream_t s, const QuantParams& p) {
    return f.flags ? quantise<TYPE, true>(f, rows, g, s, p) : quantise<TYPE, false>(f, rows, g, s, p);
}
// Q, S, X[, Z], rows
int quantise_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    QuantParams p = {};
    p.q = pointer_arg<uint8_t>(args, 0), p.s = pointer_arg<float>(args, 1), p.x = pointer_arg<const void>(args, 2);
    p.z = f.flags ? pointer_arg<int>(args, 3) : nullptr;
    p.rows = rows, p.k = f.K, p.pieces = f.group / 8, p.pitch = f.stride, p.steps = f.group / kStep;
    if (f.algorithm == mx::F16) return quantise<mx::F16>(f, rows, g, s, p);
    return f.algorithm == mx::BF16 ? quantise<mx::BF16>(f, rows, g, s, p) : quantise<mx::F32>(f, rows, g, s, p);
}
int make_quantise(const Variant& v, orx_function* f) {
    bool bad = false;
    f->K = (int)v.integer("K", 0, &bad);
    f->algorithm = mx_type(v, "input_dtype", "float16", &bad);
    f->flags = v.boolean("zero_points", false, &bad);
    f->capacity = (int)v.integer("M", 1 << 24, &bad);
    const std::string layout = v.string("layout", "rows", &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    if (layout != "rows" && layout != "tiles") {
        set_error("int8_token_quantization: layout must be rows or tiles");
        return ORX_ERR_BAD_VARIANT;
    }
    f->flags2 = layout == "tiles";
    if (f->K <= 0 || f->K > kMaxK || f->capacity < 1 || f->capacity > 1 << 24) {
        set_error("int8_token_quantization: need 0 < K <= %d and M from 1 to %d", kMaxK, 1 << 24);
        return ORX_ERR_BAD_VARIANT;
    }
    f->group = steps_of_bytes(f->K) * kStep;
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
        {"int8_token_quantization", make_quantise, "K, input_dtype=float16|bfloat16|float32, zero_points=false, layout=rows|tiles, M=capacity", "Q,S,X[,Z],rows"},
        {"int8_token_projection", make_int8_projection,
         "M, N, K, dynamic_rows=false, input_dtype=int8|float16|bfloat16 (few rows), zero_points=false, bias=false, epilogue=none|swiglu, output_dtype=float16|bfloat16|float32",
         "A[,AS][,AZ][,Bias],Out,W,WS[,WSum][,m]"},
        {"int8_token_grouped", make_int8_grouped,
         "rows, E, N, K, tiles, block_m=16|64|128, gather=false, input_dtype=int8|float16|bfloat16 (block_m=16), epilogue=none|swiglu, output_dtype=float16|bfloat16|float32",
         "A[,AS],Out[,SlotToken],TileCount,TileUnits,W,WS"},
        {"half_grouped", make_half_grouped,
         "rows, E, N, K, tiles, block_m=16|64|128, gather=false, dtype=float16|bfloat16, epilogue=none|swiglu, output_dtype=float16|bfloat16|float32",
         "A,Out[,SlotToken],TileCount,TileUnits,W"},
    };
    *count = (int)(sizeof(rows) / sizeof(rows[0]));
    return rows;
}

}  // namespace orx
