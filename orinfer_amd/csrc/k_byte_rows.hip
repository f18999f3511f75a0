// Products of few rows with weights by byte tiles (dense and routed experts), and the symbols of both.
//
// Bound by the weights' bytes: a wave streams whole tiles (2 KiB a step and 16 channels) into registers, AHEAD steps on their way; the steps are dealt to the waves of a workgroup, whose sums
// meet in LDS.  The weights are the first operand, so a lane ends with four neighbouring channels of one row.
// 16-bit rows of a product in 8-bit integers (QUANTISE): a workgroup makes their codes itself, into LDS, while its first weights are on their way.
#include <algorithm>

#include "byte_device.h"
#include "byte_tiles.h"
#include "orx_internal.h"

namespace orx {
namespace {

using namespace bytes;

// 16 bytes of a lane from a buffer of `bytes`; what lies behind its end reads as 0 and is not fetched.
struct Buffer {
    __amdgpu_buffer_rsrc_t from;
    __device__ __forceinline__ Buffer(const uint8_t* base, int bytes) : from(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, bytes, 0x00027000)) {}
    __device__ __forceinline__ v4i load_16(int offset) const { return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(from, offset, 0, 0)); }
};

constexpr int kPieces = 8;  // of eight values, of a thread, that a row of a workgroup of eight waves may take (QUANTISE)

// ROWS blocks of 16 rows, two tiles of 16 channels (SwiGLU: gate and up) to a workgroup of WAVES waves.  SOURCE: mx::F16 or mx::BF16 rows to quantise, -1 rows as the product takes them.
template <int KIND, int ROWS, int WAVES, int AHEAD, int SOURCE, bool ZERO, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(WAVES * 64) void byte_rows_kernel(Product p) {
    using Sum = typename Operands<KIND>::Sum;
    constexpr int TILES = 2;
    constexpr bool QUANTISE = SOURCE >= 0;
    extern __shared__ __align__(16) uint8_t lds[];  // sums, or the rows' codes before them
    Sum(*const sums)[ROWS * TILES][64] = reinterpret_cast<Sum(*)[ROWS * TILES][64]>(lds);
    __shared__ RowRange ranges[WAVES];
    __shared__ RowScale row_scales[16 * ROWS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int groups = (p.tiles + TILES - 1) / TILES;
    const int unit = blockIdx.x / groups, group = blockIdx.x % groups;
    int first_row = unit * (16 * ROWS), rows = min(p.m - first_row, 16 * ROWS);
    const uint8_t* w = p.w;
    int64_t channels = 0;  // of the experts in front of this one
    if (GROUPED) {
        if (unit >= *p.unit_count) return;
        const int4 u = p.units[unit];
        first_row = __builtin_amdgcn_readfirstlane(u.y), rows = __builtin_amdgcn_readfirstlane(u.z);
        const int64_t tile = (int64_t)__builtin_amdgcn_readfirstlane(u.x) * p.tiles;
        w += tile * p.steps * kTileBytes, channels = tile * 16;
    }
    auto row_at = [&](int local) {
        int64_t row = max(first_row + min(local, rows - 1), 0);  // (rows that are not there repeat the last: their sums go nowhere)
        if (GROUPED && p.slot_token != nullptr) row = p.slot_token[row];
        return row;
    };
    const int r = lane & 15, piece = lane >> 4;  // lane's channel or row; its pieces of a step, and 4 behind

    // ---- rows to quantise: what a thread holds of its row ----
    constexpr int TYPE = QUANTISE ? SOURCE : mx::F16;
    const int row_waves = rows == 1 ? WAVES : rows == 2 ? WAVES / 2 : rows <= 4 ? WAVES / 4 : 1;  // to a row
    const int row_pieces = p.steps * 16, my_row = wave / row_waves, in_row = wave % row_waves * 64 + lane;
    uint32_t words[QUANTISE ? kPieces : 1][4];
    auto read_row = [&](int row) {
        const uint16_t* const x = reinterpret_cast<const uint16_t*>(p.a) + row_at(row) * (p.row_bytes);  // (row_bytes of codes, as many values)
#pragma unroll
        for (int i = 0; i < (QUANTISE ? kPieces : 0); ++i) {
            const int first = (in_row + i * row_waves * 64) * 8, count = p.row_bytes - first;
            v4u four = {0, 0, 0, 0};
            if (i * row_waves * 64 < row_pieces) {
                if (count >= 8) {
                    four = *reinterpret_cast<const mx::words4*>(x + first);
                } else {
                    for (int j = 0; j < count; ++j) four[j / 2] |= (uint32_t)x[first + j] << (16 * (j & 1));
                }
            }
            words[i][0] = four[0], words[i][1] = four[1], words[i][2] = four[2], words[i][3] = four[3];
        }
    };
    if constexpr (QUANTISE) read_row(min(my_row, rows - 1));

    // ---- weights on their way ----
    struct Step {
        v4i w[TILES][2], a[ROWS][2];
    };
    const uint8_t* a[ROWS];
    if constexpr (!QUANTISE) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) a[i] = p.a + row_at(16 * i + r) * p.pitch;
    }
    auto load = [&](Step& s, int step) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int64_t tile = (int64_t)step * p.tiles + min(group * TILES + t, p.tiles - 1);
            const Buffer codes(w + tile * kTileBytes, step < p.steps ? kTileBytes : 0);
            s.w[t][0] = codes.load_16(lane * 16);
            s.w[t][1] = codes.load_16(lane * 16 + 1024);
        }
        if constexpr (!QUANTISE) {
            // (16-bit rows end where they end: pieces behind that are 0, and read the row's first one)
            const int at = min(step, p.steps - 1) * kStep + piece * 16;
            const bool there[2] = {KIND == I8 || at < p.row_bytes, KIND == I8 || at + 64 < p.row_bytes};
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const v4i value = *reinterpret_cast<const v4i*>(a[i] + (there[half] ? at + 64 * half : 0));
                    s.a[i][half] = there[half] ? value : v4i{0, 0, 0, 0};
                }
        }
    };
    Step held[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(held[i], wave + i * WAVES);

    // ---- the rows' codes ----
    const int live = min(rows, 16);
    if constexpr (QUANTISE) {
        for (int first = 0; first < rows; first += WAVES / row_waves) {
            const int row = first + my_row;
            if (first > 0) read_row(min(row, rows - 1));
            RowRange range = {0, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kPieces; ++i) widen<TYPE, ZERO>(range, words[i]);
            range = over_wave<TYPE, ZERO>(range);
            if (row_waves > 1) {  // (then one round takes all rows)
                if (lane == 0) ranges[wave] = range;
                __syncthreads();
                for (int i = 0; i < row_waves; ++i) {
                    const RowRange other = ranges[my_row * row_waves + i];
                    range.bits = max(range.bits, other.bits), range.high = fmaxf(range.high, other.high), range.low = fmaxf(range.low, other.low);
                }
            }
            const RowCode code = code_of<TYPE, ZERO>(range);
            if (row < rows) {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const int at = in_row + i * row_waves * 64;
                    if (at < row_pieces) *reinterpret_cast<uint2*>(lds + ((int64_t)(at >> 1) * live + row) * 16 + (at & 1) * 8) = eight_codes<TYPE, ZERO>(words[i], code);
                }
                if (wave % row_waves == 0 && lane == 0) row_scales[row] = {stored_scale(code), code.zero};
            }
        }
        __syncthreads();
    } else if constexpr (KIND == I8) {
        for (int i = threadIdx.x; i < 16 * ROWS; i += WAVES * 64) {
            const int64_t row = row_at(i);
            row_scales[i] = {p.scale[row], ZERO ? p.zero[row] : 0};
        }
    }

    Sum sum[ROWS][TILES];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int t = 0; t < TILES; ++t) sum[i][t] = Sum{};
    auto multiply_step = [&](Step& s, int step) {
        if constexpr (QUANTISE) {
            const int there = min(step, p.steps - 1), row = min(r, live - 1);
            const uint8_t* const from = lds + ((there * 8 + piece) * live + row) * 16;
            s.a[0][0] = *reinterpret_cast<const v4i*>(from);
            s.a[0][1] = *reinterpret_cast<const v4i*>(from + 4 * live * 16);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
#pragma unroll
                for (int t = 0; t < TILES; ++t) sum[i][t] = multiply<KIND>(s.w[t][half], s.a[i][half], sum[i][t]);
    };
#pragma unroll 1
    for (int step = wave; step < p.steps; step += AHEAD * WAVES) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (step + i * WAVES < p.steps) multiply_step(held[i], step + i * WAVES);
            if (step + (i + AHEAD) * WAVES < p.steps) load(held[i], step + (i + AHEAD) * WAVES);
        }
    }
    if constexpr (QUANTISE) __syncthreads();  // (the sums take the codes' place)
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int t = 0; t < TILES; ++t) sums[wave][i * TILES + t][lane] = sum[i][t];
    __syncthreads();
    constexpr int KINDS = SWIGLU ? 2 : 1;
    for (int q = threadIdx.x; q < ROWS * TILES / KINDS * 64; q += WAVES * 64) {
        const int l = q & 63, i = (q >> 6) / (TILES / KINDS), t = (q >> 6) % (TILES / KINDS);
        const int row = 16 * i + (l & 15);
        v4f total[KINDS];
#pragma unroll
        for (int kind = 0; kind < KINDS; ++kind) {
            Sum all = sums[0][i * TILES + t * KINDS + kind][l];
#pragma unroll
            for (int other = 1; other < WAVES; ++other) all += sums[other][i * TILES + t * KINDS + kind][l];
            const int64_t at = channels + min(group * TILES + t * KINDS + kind, p.tiles - 1) * 16 + 4 * (l >> 4);
            Channels channel = {};
            if constexpr (KIND == I8) {
                channel.scale = *reinterpret_cast<const v4f*>(p.w_scale + at);
                if (ZERO) channel.sum = *reinterpret_cast<const v4i*>(p.w_sum + at);
                if (!GROUPED && p.bias != nullptr) channel.bias = *reinterpret_cast<const v4f*>(p.bias + at);
            }
            total[kind] = scaled<KIND, !GROUPED>(all, channel, KIND == I8 ? row_scales[min(row, rows - 1)] : RowScale{});
        }
        if constexpr (SWIGLU) {
#pragma unroll
            for (int j = 0; j < 4; ++j) total[0][j] = mx::swiglu(total[0][j], total[KINDS - 1][j]);
        }
        if (row < rows)
            mx::store_four(p.out, p.type, (int64_t)(first_row + row) * p.cols, ((group * TILES) / KINDS + t) * 16 + 4 * (l >> 4), p.cols, total[0]);
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------------
// slots used: M (rows; experts: slots), N, K, E, tiles (units), block_m, flags, flags2 (kind), algorithm (output type), H (output columns), slots (16-channel tiles), packed_k (source of the rows, plus 1)
enum { kSwiglu = 1, kGather = 2, kZero = 4, kBias = 8 };
constexpr int kMostLds = 80 * 1024;

int steps_of(const orx_function& f) { return (f.K * (f.flags2 == I8 ? 1 : 2) + kStep - 1) / kStep; }

// What a launch of `rows` rows runs: a unit's rows, and the form of the tiles from LDS (-1: the kernel above, 32 channels to a workgroup), or its waves
struct Plan {
    int rows, form, waves;
};
Plan few_rows(int unit_rows) { return {unit_rows, -1, unit_rows == 64 ? 4 : 8}; }
Plan plan(const orx_function& f, int rows) {
    if (f.E > 0) return f.block_m == 16 ? few_rows(16) : Plan{f.block_m, f.block_m == 64 ? kTiles64 : f.block_m == 256 ? kTiles256 : kTiles128x256, 0};
    if (rows <= 64) return few_rows(rows <= 16 ? 16 : rows <= 32 ? 32 : 64);
    return rows >= 1024 ? Plan{256, kTiles256, 0} : Plan{128, kTiles128, 0};
}
uint32_t few_rows_lds(const orx_function& f, int rows, const Plan& plan) {
    const uint32_t sums = (uint32_t)plan.waves * (plan.rows / 16) * 2 * 1024;
    const uint32_t codes = f.packed_k == 0 ? 0 : (uint32_t)steps_of(f) * kStep * std::min(f.E > 0 ? 16 : rows, 16);
    return std::max(sums, codes);
}

int geometry(const orx_function& f, int rows, Geometry* g) {
    const Plan plan = orx::plan(f, rows);
    const TilesShape shape = plan.form < 0 ? TilesShape{plan.rows, 32} : byte_tiles_shape(f.flags2, plan.form, f.E > 0);
    const int64_t units = f.E > 0 ? (int64_t)f.tiles : ceil_div(rows, plan.rows);
    int64_t blocks = units * ceil_div(f.slots, shape.channels / 16);
    if (blocks >= (1ll << 32) / 512) {
        set_error("%s: %d rows of %d channels are more than one launch takes", f.symbol.c_str(), rows, f.N);
        return ORX_ERR_ROWS;
    }
    if (plan.form >= 0) {
        blocks = std::min<int64_t>(blocks, (int64_t)device_compute_units() * shape.to_a_cu);
        g->block[0] = shape.threads;
        g->shared = shape.lds;
    } else {
        g->block[0] = 64 * plan.waves;
        g->shared = few_rows_lds(f, rows, plan);
    }
    g->grid[0] = (uint32_t)blocks;
    return ORX_OK;
}

template <int KIND, int ROWS, int WAVES, int AHEAD, int SOURCE, bool ZERO, bool GROUPED, bool SWIGLU>
int launch_one(const Product& p, const Geometry& g, hipStream_t s) {
    constexpr auto kernel = &byte_rows_kernel<KIND, ROWS, WAVES, AHEAD, SOURCE, ZERO, GROUPED, SWIGLU>;
    static DeviceOnce ready;
    const int code = ready.run([] { return hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds), "hipFuncSetAttribute"); });
    if (code != ORX_OK) return code;
    ORX_LAUNCH(kernel, dim3(g.grid[0]), dim3(64 * WAVES), g.shared, s, p);
    return hip_check(hipGetLastError(), "launch byte product");
}
template <int KIND, int ROWS, int WAVES, int AHEAD, int SOURCE, bool ZERO, bool GROUPED>
int launch_of(const orx_function& f, const Product& p, const Geometry& g, hipStream_t s) {
    return f.flags & kSwiglu ? launch_one<KIND, ROWS, WAVES, AHEAD, SOURCE, ZERO, GROUPED, true>(p, g, s) : launch_one<KIND, ROWS, WAVES, AHEAD, SOURCE, ZERO, GROUPED, false>(p, g, s);
}
template <int ROWS, int WAVES, int AHEAD, int SOURCE>
int launch_dense(const orx_function& f, const Product& p, const Geometry& g, hipStream_t s) {
    return f.flags & kZero ? launch_of<I8, ROWS, WAVES, AHEAD, SOURCE, true, false>(f, p, g, s) : launch_of<I8, ROWS, WAVES, AHEAD, SOURCE, false, false>(f, p, g, s);
}
int launch_product(const orx_function& f, int rows, const Geometry& g, hipStream_t s, const Product& p) {
    const Plan plan = orx::plan(f, rows);
    if (plan.form >= 0) return launch_byte_tiles(p, f.flags2, plan.form, f.E > 0, f.flags & kSwiglu, g.grid[0], s);
    if (f.E > 0) {
        if (f.flags2 == F16) return launch_of<F16, 1, 8, 2, -1, false, true>(f, p, g, s);
        if (f.flags2 == BF16) return launch_of<BF16, 1, 8, 2, -1, false, true>(f, p, g, s);
        if (f.packed_k == 0) return launch_of<I8, 1, 8, 2, -1, false, true>(f, p, g, s);
        return f.packed_k - 1 == mx::F16 ? launch_of<I8, 1, 8, 2, mx::F16, false, true>(f, p, g, s) : launch_of<I8, 1, 8, 2, mx::BF16, false, true>(f, p, g, s);
    }
    if (f.packed_k != 0) return f.packed_k - 1 == mx::F16 ? launch_dense<1, 8, 2, mx::F16>(f, p, g, s) : launch_dense<1, 8, 2, mx::BF16>(f, p, g, s);
    if (plan.rows == 16) return launch_dense<1, 8, 2, -1>(f, p, g, s);
    return plan.rows == 32 ? launch_dense<2, 8, 2, -1>(f, p, g, s) : launch_dense<4, 4, 1, -1>(f, p, g, s);
}

Product product_of(const orx_function& f, int rows) {
    Product p = {};
    p.m = rows, p.cols = f.H, p.steps = steps_of(f), p.tiles = f.slots, p.type = f.algorithm;
    p.row_bytes = f.K * (f.flags2 == I8 ? 1 : 2);
    p.pitch = f.flags2 == I8 ? (int64_t)(p.steps | 1) * kStep : p.row_bytes;
    return p;
}

// A[, AS][, AZ][, Bias], Out, W, WS[, WSum][, m]
int projection_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    Product p = product_of(f, rows);
    int at = 0;
    p.a = pointer_arg<const uint8_t>(args, at++);
    if (f.packed_k == 0) p.scale = pointer_arg<const float>(args, at++);
    if (f.packed_k == 0 && f.flags & kZero) p.zero = pointer_arg<const int>(args, at++);
    if (f.flags & kBias) p.bias = pointer_arg<const float>(args, at++);
    p.out = pointer_arg<void>(args, at++), p.w = pointer_arg<const uint8_t>(args, at++), p.w_scale = pointer_arg<const float>(args, at++);
    if (f.flags & kZero) p.w_sum = pointer_arg<const int>(args, at++);
    return launch_product(f, rows, g, s, p);
}
// A[, AS], Out[, SlotToken], TileCount, TileUnits, W[, WS]
int grouped_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    Product p = product_of(f, rows);
    int at = 0;
    p.a = pointer_arg<const uint8_t>(args, at++);
    if (f.flags2 == I8 && f.packed_k == 0) p.scale = pointer_arg<const float>(args, at++);
    p.out = pointer_arg<void>(args, at++);
    if (f.flags & kGather) p.slot_token = pointer_arg<const int>(args, at++);
    p.unit_count = pointer_arg<const int>(args, at++), p.units = pointer_arg<const int4>(args, at++), p.most_units = f.tiles;
    p.w = pointer_arg<const uint8_t>(args, at++);
    if (f.flags2 == I8) p.w_scale = pointer_arg<const float>(args, at++);
    return launch_product(f, rows, g, s, p);
}

// Rows that a product quantises itself: their codes fit LDS, and a thread holds its part of a row.
bool quantises(const orx_function& f, int rows) {
    const int row_waves = rows == 1 ? 8 : rows == 2 ? 4 : rows <= 4 ? 2 : 1;
    return rows <= 16 && few_rows_lds(f, rows, few_rows(16)) <= (uint32_t)kMostLds && steps_of(f) * 16 <= row_waves * 64 * kPieces;
}

// What all three have: N, K, epilogue, types.
int shape(const Variant& v, orx_function* f) {
    bool bad = false;
    const bool halves = f->symbol == "half_grouped";
    f->N = (int)v.integer("N", 0, &bad), f->K = (int)v.integer("K", 0, &bad);
    const std::string epilogue = v.string("epilogue", "none", &bad);
    f->algorithm = mx_type(v, "output_dtype", "float16", &bad);
    const std::string input = v.string(halves ? "dtype" : "input_dtype", halves ? "float16" : "int8", &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    if ((input != "int8" || halves) && input != "float16" && input != "bfloat16") {
        set_error("%s: %s must be %sfloat16 or bfloat16", f->symbol.c_str(), halves ? "dtype" : "input_dtype", halves ? "" : "int8, ");
        return ORX_ERR_BAD_VARIANT;
    }
    f->flags2 = !halves ? I8 : input == "float16" ? F16 : BF16;
    f->packed_k = halves || input == "int8" ? 0 : 1 + (input == "float16" ? mx::F16 : mx::BF16);
    if (epilogue != "none" && epilogue != "swiglu") {
        set_error("%s: epilogue must be none or swiglu", f->symbol.c_str());
        return ORX_ERR_BAD_VARIANT;
    }
    const bool swiglu = epilogue == "swiglu";
    f->flags |= swiglu ? kSwiglu : 0;
    const int most = halves ? 1 << 20 : kMostIntegerK, unit = halves ? 8 : 1;
    if (f->N <= 0 || f->N > 1 << 24 || (swiglu && f->N % 2) || f->K <= 0 || f->K % unit || f->K > most) {
        set_error("%s: need 0 < N <= %d (even for swiglu) and K a multiple of %d up to %d", f->symbol.c_str(), 1 << 24, unit, most);
        return ORX_ERR_BAD_VARIANT;
    }
    f->H = swiglu ? f->N / 2 : f->N;
    f->slots = (f->H + 15) / 16 * (swiglu ? 2 : 1);
    f->geometry = geometry;
    return ORX_OK;
}

int make_grouped(const Variant& v, orx_function* f) {
    bool bad = false;
    f->M = (int)v.integer("rows", 0, &bad), f->E = (int)v.integer("E", 0, &bad), f->tiles = (int)v.integer("tiles", 0, &bad);
    f->block_m = (int)v.integer("block_m", 16, &bad);
    f->flags = v.boolean("gather", false, &bad) ? kGather : 0;
    if (bad) return ORX_ERR_BAD_VARIANT;
    const int code = shape(v, f);
    if (code != ORX_OK) return code;
    if (f->M <= 0 || f->M > 1 << 24 || f->E <= 0 || f->tiles <= 0 || f->tiles > 1 << 24 || (f->block_m != 16 && f->block_m != 64 && f->block_m != 128 && f->block_m != 256)) {
        set_error("%s: need rows, E and tiles above 0 and block_m 16, 64, 128 or 256", f->symbol.c_str());
        return ORX_ERR_BAD_VARIANT;
    }
    f->capacity = f->M;
    if (f->packed_k != 0 && (f->block_m != 16 || !quantises(*f, 16))) {
        set_error("%s: 16-bit rows go with block_m 16 and K up to %d", f->symbol.c_str(), 64 * 8 * kPieces);
        return ORX_ERR_BAD_VARIANT;
    }
    f->args = {{"A", ArgPointer, f->packed_k != 0 ? 2u : 16u}};
    if (f->flags2 == I8 && f->packed_k == 0) f->args.push_back({"AS", ArgPointer, 4});
    f->args.push_back({"Out", ArgPointer, f->algorithm == mx::F32 ? 4u : 2u});
    if (f->flags & kGather) f->args.push_back({"SlotToken", ArgPointer, 4});
    for (const ArgSpec& a : std::initializer_list<ArgSpec>{{"TileCount", ArgPointer, 4}, {"TileUnits", ArgPointer, 16}, {"W", ArgPointer, 16}}) f->args.push_back(a);
    if (f->flags2 == I8) f->args.push_back({"WS", ArgPointer, 16});
    f->launch = grouped_launch;
    Geometry g;
    return geometry(*f, f->M, &g);
}

}  // namespace

int make_int8_projection(const Variant& v, orx_function* f) {
    bool bad = false;
    f->M = (int)v.integer("M", 0, &bad);
    f->dynamic_rows = v.boolean("dynamic_rows", false, &bad);
    f->flags = (v.boolean("zero_points", false, &bad) ? kZero : 0) | (v.boolean("bias", false, &bad) ? kBias : 0);
    if (bad) return ORX_ERR_BAD_VARIANT;
    const int code = shape(v, f);
    if (code != ORX_OK) return code;
    if (f->M <= 0 || f->M > 1 << 24) {
        set_error("int8_token_projection: need 0 < M <= %d", 1 << 24);
        return ORX_ERR_BAD_VARIANT;
    }
    f->capacity = f->M;
    if (f->packed_k != 0 && !quantises(*f, f->M)) {
        set_error("int8_token_projection: 16-bit rows go with M up to 16 and short K: codes of all rows up to %d bytes, rows of %d values (M 1: 8 times that, 2: 4, 4: 2)", kMostLds, 64 * 8 * kPieces);
        return ORX_ERR_BAD_VARIANT;
    }
    f->args = {{"A", ArgPointer, f->packed_k != 0 ? 2u : 16u}};
    if (f->packed_k == 0) f->args.push_back({"AS", ArgPointer, 4});
    if (f->packed_k == 0 && f->flags & kZero) f->args.push_back({"AZ", ArgPointer, 4});
    if (f->flags & kBias) f->args.push_back({"Bias", ArgPointer, 16});
    f->args.push_back({"Out", ArgPointer, f->algorithm == mx::F32 ? 4u : 2u});
    f->args.push_back({"W", ArgPointer, 16}), f->args.push_back({"WS", ArgPointer, 16});
    if (f->flags & kZero) f->args.push_back({"WSum", ArgPointer, 16});
    if (f->dynamic_rows) f->args.push_back({"m", ArgI32, 4});
    f->launch = projection_launch;
    return ORX_OK;
}
int make_int8_grouped(const Variant& v, orx_function* f) { return make_grouped(v, f); }
int make_half_grouped(const Variant& v, orx_function* f) { return make_grouped(v, f); }

}  // namespace orx
