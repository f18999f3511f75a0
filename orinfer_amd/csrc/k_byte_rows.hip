// Products of few rows with weights by byte tiles (dense and routed experts), and the symbols of both.
//
// Bound by the weights' bytes: a wave streams whole tiles (2 KiB a step and 16 channels) into registers, AHEAD steps on their way; the steps are dealt to the waves of a workgroup, whose sums
// meet in LDS.  The weights are the first operand, so a lane ends with four neighbouring channels of one row.
// 16-bit rows of a product in 8-bit integers (QUANTISE): a workgroup makes their codes itself, into LDS, while its first weights are on their way.
// us: a bf16 row by 9728 x 2560 int8 7.6 (25 MB, 3.3 TB/s: half of it start, row and first weights), 16 rows of codes by 17408 x 5120 20.6 (4.3 TB/s), by 4096 x 4096 7.2; three tokens' routes to
// 128 experts of 1024 x 2048 9.6 int8 (50 MB, 5.2 TB/s), one token's in bf16 8.1 (34 MB, 4.1 TB/s).
#include <algorithm>

#include "byte_device.h"
#include "byte_tiles.h"
#include "orx_internal.h"

namespace orx {
namespace {

using namespace bytes;

// Waves that share a row which is quantised here, of all that a workgroup has.
__host__ __device__ constexpr int rows_waves(int rows, int waves) { return rows == 1 ? waves : rows == 2 ? waves / 2 : rows <= waves / 2 ? waves / (rows <= 4 ? 4 : 8) : 1; }

// 16 bytes of a lane from a buffer of `bytes`; what lies behind its end reads as 0 and is not fetched.
struct Buffer {
    __amdgpu_buffer_rsrc_t from;
    __device__ __forceinline__ Buffer(const uint8_t* base, int bytes) : from(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, bytes, 0x00027000)) {}
    __device__ __forceinline__ v4i load_16(int offset) const { return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(from, offset, 0, 0)); }
};

// ROWS blocks of 16 rows to a workgroup of WAVES waves, and two tiles of 16 channels (SwiGLU: gate and up), one where the rows are quantised here and a tile has its results for itself.
// SOURCE: mx::F16 or mx::BF16 rows to quantise, up to PIECES pieces of eight values to a thread; -1 rows as the product takes them.
constexpr int tiles_of(int source, bool swiglu) { return source >= 0 && !swiglu ? 1 : 2; }

// (Two workgroups to a CU, of long rows too where gate and up are, us of one and two: 8 rows of 9728 x 2560 13.7 and 10.9, with zero points 16.6 and 12.9, of 14336 x 4096 28.0 and 19.6, 25.9 and
// 18.6, 4 rows of 17408 x 5120 29.6 and 26.0, 32.9 and 28.2; without gate and up 8 rows took 16.2 and 19.6.  Long rows of bf16 leave 12 to 20 bytes to scratch in front of the first multiply, nothing behind.)
template <int KIND, int ROWS, int WAVES, int AHEAD, int SOURCE, int PIECES, bool ZERO, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(WAVES * 64, ROWS == 1 && (PIECES <= 4 || SWIGLU) ? 4 : 2) void byte_rows_kernel(Product p) {
    using Sum = typename Operands<KIND>::Sum;
    constexpr int TILES = tiles_of(SOURCE, SWIGLU);
    constexpr bool QUANTISE = SOURCE >= 0, DEALT = QUANTISE && !GROUPED;
    constexpr bool TILED = KIND == I8 && !GROUPED && !QUANTISE;  // the rows' layout
    extern __shared__ __align__(16) uint8_t lds[];  // the rows' codes, and behind them the waves' sums (where several items are dealt, two items' in turn)
    __shared__ RowRange ranges[WAVES];
    __shared__ RowScale row_scales[16 * ROWS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int groups = (p.tiles + TILES - 1) / TILES;

    // ---- items: the rows of a unit by TILES tiles of channels; where dense rows are quantised here several to a workgroup (once then for all), whose weights follow one another without a pause ----
    struct Item {
        int first_row, rows, group;
        int64_t tile;  // of its expert, the first
    };
    const int items = !DEALT ? 0 : groups * ((p.m + 16 * ROWS - 1) / (16 * ROWS));
    auto item_of = [&](int id) __attribute__((always_inline)) {
        Item item;
        const int unit = id / groups;
        item.group = id % groups, item.first_row = unit * (16 * ROWS), item.rows = min(p.m - item.first_row, 16 * ROWS), item.tile = 0;
        if (GROUPED) {
            const int4 u = p.units[unit];
            item.first_row = __builtin_amdgcn_readfirstlane(u.y), item.rows = __builtin_amdgcn_readfirstlane(u.z);
            item.tile = (int64_t)__builtin_amdgcn_readfirstlane(u.x) * p.steps * p.tiles;
        }
        return item;
    };
    Item item = item_of(blockIdx.x);  // (a list holds as many units as there are workgroups for: read beside their number)
    if (GROUPED && (int)(blockIdx.x / groups) >= __builtin_amdgcn_readfirstlane(*p.unit_count)) return;
    auto row_at = [&](const Item& item, int local) __attribute__((always_inline)) {
        int64_t row = max(item.first_row + min(local, item.rows - 1), 0);  // (rows that are not there repeat the last: their sums go nowhere)
        if (GROUPED && p.slot_token != nullptr) row = p.slot_token[row];
        return row;
    };
    const int r = lane & 15, piece = lane >> 4;  // lane's channel or row; its pieces of a step, and 4 behind

    // ---- rows to quantise: what a thread holds of its row ----
    constexpr int TYPE = QUANTISE ? SOURCE : mx::F16;
    const int rows = item.rows, row_waves = rows_waves(rows, WAVES);  // to a row
    const int row_pieces = p.steps * 16, my_row = wave / row_waves, in_row = wave % row_waves * 64 + lane;
    uint32_t words[QUANTISE ? PIECES : 1][4];
    auto read_row = [&](int row) __attribute__((always_inline)) {
        const uint16_t* const x = reinterpret_cast<const uint16_t*>(p.a) + row_at(item, row) * p.row_bytes;  // (row_bytes of codes, as many values)
#pragma unroll
        for (int i = 0; i < (QUANTISE ? PIECES : 0); ++i) {
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
    auto aim = [&](const Item& item) __attribute__((always_inline)) {
        if constexpr (!QUANTISE) {
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
                a[i] = TILED ? p.a + (int64_t)min(item.first_row / 16 + i, (p.m - 1) / 16) * p.steps * kTileBytes : p.a + row_at(item, 16 * i + r) * p.pitch;
        }
    };
    auto load = [&](Step& s, const Item& item, int step) __attribute__((always_inline)) {  // (what lies behind the last step reads as 0)
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int64_t tile = item.tile + (int64_t)step * p.tiles + min(item.group * TILES + t, p.tiles - 1);
            const Buffer codes(p.w + tile * kTileBytes, step < p.steps ? kTileBytes : 0);
            s.w[t][0] = codes.load_16(lane * 16);
            s.w[t][1] = codes.load_16(lane * 16 + 1024);
        }
        if constexpr (TILED) {
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                if constexpr (ROWS == 1) {  // (beside the weights' loads; with 64 rows plain loads are faster)
                    const Buffer codes(a[i] + (int64_t)step * kTileBytes, step < p.steps ? kTileBytes : 0);
                    s.a[i][0] = codes.load_16(lane * 16), s.a[i][1] = codes.load_16(lane * 16 + 1024);
                } else {
                    const uint8_t* const from = a[i] + (int64_t)min(step, p.steps - 1) * kTileBytes + lane * 16;
                    s.a[i][0] = *reinterpret_cast<const v4i*>(from), s.a[i][1] = *reinterpret_cast<const v4i*>(from + 1024);
                }
            }
        } else if constexpr (!QUANTISE) {
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
    aim(item);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(held[i], item, wave + i * WAVES);

    // ---- the rows' codes ----
    const int live = min(rows, 16);
    const uint32_t codes_bytes = QUANTISE ? (uint32_t)p.steps * kStep * live : 0;
    if constexpr (QUANTISE) {
        for (int first = 0; first < rows; first += WAVES / row_waves) {
            const int row = first + my_row;
            if (first > 0) read_row(min(row, rows - 1));
            RowRange range = {0, 0};
#pragma unroll
            for (int i = 0; i < PIECES; ++i) widen<TYPE, ZERO>(range, words[i]);
            range = over_wave<TYPE, ZERO>(range);
            if (row_waves > 1) {  // (then one round takes all rows)
                if (lane == 0) ranges[wave] = range;
                __syncthreads();
                for (int i = 0; i < row_waves; ++i) range = wider(range, ranges[my_row * row_waves + i]);
            }
            const RowCode code = code_of<TYPE, ZERO>(range);
            if (row < rows) {
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const int at = in_row + i * row_waves * 64;
                    if (at < row_pieces) *reinterpret_cast<uint2*>(lds + ((int64_t)(at >> 1) * live + row) * 16 + (at & 1) * 8) = eight_codes<TYPE, ZERO>(words[i], code);
                }
                if (wave % row_waves == 0 && lane == 0) row_scales[row] = {stored_scale(code), code.zero};
            }
        }
        __syncthreads();
    }

    const int chunks = (p.steps + AHEAD * WAVES - 1) / (AHEAD * WAVES);  // of AHEAD steps to a wave
    constexpr int KINDS = SWIGLU ? 2 : 1;
    int turn = 0;
#pragma unroll 1
    for (int id = blockIdx.x;;) {
        const int next_id = id + (int)gridDim.x;
        const bool more = DEALT && next_id < items;
        const Item next = more ? item_of(next_id) : item;
        if constexpr (KIND == I8 && !QUANTISE) {
            for (int i = threadIdx.x; i < 16 * ROWS; i += WAVES * 64) {
                const int64_t row = row_at(item, i);
                row_scales[i] = {p.scale[row], ZERO ? p.zero[row] : 0};
            }
        }
        Sum sum[ROWS][TILES];
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int t = 0; t < TILES; ++t) sum[i][t] = Sum{};
        auto multiply_step = [&](Step& s, int step) __attribute__((always_inline)) {
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
        int step = wave;
#pragma unroll 1
        for (int chunk = 0; chunk < chunks; ++chunk) {
            // (the next chunk's weights, or the next item's first ones, or none)
            const bool last = chunk == chunks - 1;
            if (last && more) aim(next);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                // (dealt items load zeros behind the last step, others nothing)
                if (DEALT || step + i * WAVES < p.steps) multiply_step(held[i], step + i * WAVES);
                const int then = last ? (more ? wave + i * WAVES : p.steps) : step + (i + AHEAD) * WAVES;
                if (DEALT || then < p.steps) load(held[i], last ? next : item, then);
            }
            step += AHEAD * WAVES;
        }
        Sum(*const sums)[ROWS * TILES][64] = reinterpret_cast<Sum(*)[ROWS * TILES][64]>(lds + codes_bytes) + turn * WAVES;
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int t = 0; t < TILES; ++t) sums[wave][i * TILES + t][lane] = sum[i][t];
        __syncthreads();
        for (int q = threadIdx.x; q < ROWS * TILES / KINDS * 64; q += WAVES * 64) {
            const int l = q & 63, i = (q >> 6) / (TILES / KINDS), t = (q >> 6) % (TILES / KINDS);
            const int row = 16 * i + (l & 15);
            v4f total[KINDS];
#pragma unroll
            for (int kind = 0; kind < KINDS; ++kind) {
                Sum all = sums[0][i * TILES + t * KINDS + kind][l];
#pragma unroll
                for (int other = 1; other < WAVES; ++other) all += sums[other][i * TILES + t * KINDS + kind][l];
                const int64_t at = item.tile / p.steps * 16 + min(item.group * TILES + t * KINDS + kind, p.tiles - 1) * 16 + 4 * (l >> 4);
                Channels channel = {};
                if constexpr (KIND == I8) {
                    channel.scale = *reinterpret_cast<const v4f*>(p.w_scale + at);
                    if (ZERO) channel.sum = *reinterpret_cast<const v4i*>(p.w_sum + at);
                    if (!GROUPED && p.bias != nullptr) channel.bias = *reinterpret_cast<const v4f*>(p.bias + at);
                }
                total[kind] = scaled<KIND, !GROUPED>(all, channel, KIND == I8 ? row_scales[min(row, item.rows - 1)] : RowScale{});
                // (One kind's sums after the other's: both at once, beside the next item's weights on their way, left 44 bytes to scratch with zero points, and every reload waited for those weights:
                // 8 rows of 9728 x 2560 14.2 -> 12.9 us, one of 17408 x 5120 28.7 -> 23.5.)
                if constexpr (QUANTISE && SWIGLU) asm volatile("" : "+v"(total[kind])::"memory");
            }
            if constexpr (SWIGLU) {
#pragma unroll
                for (int j = 0; j < 4; ++j) total[0][j] = mx::swiglu(total[0][j], total[KINDS - 1][j]);
            }
            if (row < item.rows)
                mx::store_four(p.out, p.type, (int64_t)(item.first_row + row) * p.cols, ((item.group * TILES) / KINDS + t) * 16 + 4 * (l >> 4), p.cols, total[0]);
        }
        if (!more) return;
        item = next, id = next_id;
        turn ^= 1;
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------------
// slots used: M (rows; experts: slots), N, K, E, tiles (units), block_m, flags, flags2 (kind), algorithm (output type), H (output columns), slots (16-channel tiles), packed_k (source of the rows, plus 1)
enum { kSwiglu = 1, kGather = 2, kZero = 4, kBias = 8 };
constexpr int kMostLds = 128 * 1024;

int steps_of(const orx_function& f) { return steps_of_bytes((int64_t)f.K * (f.flags2 == I8 ? 1 : 2)); }

// What a launch of `rows` rows runs: a unit's rows, and the form of the tiles from LDS (-1: the kernel above), or its waves
struct Plan {
    int rows, form, waves;
};
// Of few steps fewer waves have one.
Plan few_rows(const orx_function& f, int unit_rows) { return {unit_rows, -1, unit_rows == 64 || (unit_rows == 16 && steps_of(f) <= 8) ? 4 : 8}; }
// Of dense launches the form whose estimate is least: fixed + step * steps * rounds over the CUs, in units of 10 ns.  Fitted to times of 1 to 8192 rows by seven sizes of weights (2048 x 1024
// to 17408 x 5120 and 5120 x 17408); the estimates are within a fifth, except below the time that the weights take from memory, and the form that is picked within a tenth of the fastest, within a fifth
// at 96 and 128 rows of 5120 x 17408 (40 by tiles of 64 x 64, 32 to 35 by the kernel above with 64 rows).  us at
// 7168 x 5120 of the kernel above with 16 and with 64 rows, and of tiles of 64 x 64, 64 x 128, 96 x 128, 128 x 128, 128 x 256 and 256 x 256:
//     16 rows: 9.1, 11.3, 14.7, 18.7, -, 23, 33, -;  64: -, 12.5, 15.3, 22, 23, 24, 35, -;  128: -, 18, 15.5, 21, 22, 27, 39, -;  256: -, 27, 25, 21, 24, 27, 39, 61;
//     333: -, 35, 33, 35, 23, 26, 37, 57;  512: -, 45, 43, 38, 41, 27, 39, 59;  1024: -, -, 71, 67, -, 51, 40, 59;  4096: 256 x 256 128 and 128 x 256 132;  8192: 247 and 242
struct Form {
    int form, rows, channels, fixed, step;
};
constexpr Form kForms[] = {{-1, 16, 32, 500, 10}, {-1, 64, 32, 600, 15}, {kTiles64x64, 64, 64, 300, 27}, {kTiles64, 64, 128, 300, 46}, {kTiles96, 96, 128, 400, 47}, {kTiles128, 128, 128, 400, 53},
                           {kWide128, 128, 256, 600, 72}, {kTiles256, 256, 256, 800, 125}};
Plan plan(const orx_function& f, int rows) {
    if (f.E > 0) return f.block_m == 16 ? few_rows(f, 16) : Plan{f.block_m, f.block_m == 64 ? kWide64 : kWide128, 0};
    if (f.packed_k != 0) return few_rows(f, 16);
    const int64_t units = device_compute_units();
    const Form* best = nullptr;
    int64_t least = 0;
    for (const Form& form : kForms) {
        if (form.form == kWide128 && (int64_t)f.slots * steps_of(f) * kTileBytes >= 1ll << 32) continue;  // (its loads of weights count 32 bits)
        const int64_t tiles = (int64_t)ceil_div(rows, form.rows) * ceil_div(f.slots, form.channels / 16);
        const int64_t estimate = form.fixed + (tiles + units - 1) / units * form.step * steps_of(f);
        if (best == nullptr || estimate < least) least = estimate, best = &form;
    }
    return best->form < 0 ? few_rows(f, best->rows) : Plan{best->rows, best->form, 0};
}
int tiles_of(const orx_function& f) { return tiles_of(f.packed_k - 1, f.flags & kSwiglu); }
uint32_t few_rows_lds(const orx_function& f, int rows, const Plan& plan) {
    const uint32_t sums = (uint32_t)plan.waves * (plan.rows / 16) * tiles_of(f) * 1024;
    const uint32_t codes = f.packed_k == 0 ? 0 : (uint32_t)steps_of(f) * kStep * std::min(f.E > 0 ? 16 : rows, 16);
    return codes + (f.E == 0 && f.packed_k != 0 ? 2 : 1) * sums;
}

int geometry(const orx_function& f, int rows, Geometry* g) {
    const Plan plan = orx::plan(f, rows);
    const TilesShape shape = plan.form < 0 ? TilesShape{plan.rows, 16 * tiles_of(f)} : byte_tiles_shape(f.flags2, plan.form, f.E > 0);
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
        // Of rows that are quantised here as many workgroups as the CUs hold at once, sixteen waves to a CU, all with as many items.  (Others take one item: 9.1 us either way at 7168 x 5120, and 20.6
        // instead of 24.8 at 17408 x 5120, where workgroups that end early make room for the next.)
        if (f.E == 0 && f.packed_k != 0) {
            const int64_t most = (int64_t)device_compute_units() * std::min(16 / plan.waves, (int)(160 * 1024 / (g->shared + 1024)));
            blocks = ceil_div(blocks, ceil_div(blocks, most));
        }
    }
    g->grid[0] = (uint32_t)blocks;
    return ORX_OK;
}

// Pieces to a thread where the rows are quantised by the product: a row of the most that there may be at once (of an expert 16).
int pieces_of(const orx_function& f, int rows, int waves) { return (steps_of(f) * 16 + 64 * rows_waves(f.E > 0 ? 16 : rows, waves) - 1) / (64 * rows_waves(f.E > 0 ? 16 : rows, waves)); }

template <int KIND, int ROWS, int WAVES, int AHEAD, int SOURCE, int PIECES, bool ZERO, bool GROUPED, bool SWIGLU>
int launch_one(const Product& p, const Geometry& g, hipStream_t s) {
    constexpr auto kernel = &byte_rows_kernel<KIND, ROWS, WAVES, AHEAD, SOURCE, PIECES, ZERO, GROUPED, SWIGLU>;
    static DeviceOnce ready;
    const int code = ready.run([] { return hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds), "hipFuncSetAttribute"); });
    if (code != ORX_OK) return code;
    ORX_LAUNCH(kernel, dim3(g.grid[0]), dim3(64 * WAVES), g.shared, s, p);
    return hip_check(hipGetLastError(), "launch byte product");
}
template <int KIND, int ROWS, int WAVES, int AHEAD, int SOURCE, int PIECES, bool GROUPED, bool SWIGLU>
int launch_with(const orx_function& f, const Product& p, const Geometry& g, hipStream_t s) {
    if constexpr (KIND == I8 && !GROUPED)
        if (f.flags & kZero) return launch_one<KIND, ROWS, WAVES, AHEAD, SOURCE, PIECES, true, GROUPED, SWIGLU>(p, g, s);
    return launch_one<KIND, ROWS, WAVES, AHEAD, SOURCE, PIECES, false, GROUPED, SWIGLU>(p, g, s);
}
template <int KIND, int ROWS, int WAVES, int AHEAD, int SOURCE, int PIECES, bool GROUPED>
int launch_of(const orx_function& f, const Product& p, const Geometry& g, hipStream_t s) {
    return f.flags & kSwiglu ? launch_with<KIND, ROWS, WAVES, AHEAD, SOURCE, PIECES, GROUPED, true>(f, p, g, s) : launch_with<KIND, ROWS, WAVES, AHEAD, SOURCE, PIECES, GROUPED, false>(f, p, g, s);
}
// 16 rows as the product takes them: two steps on their way, of an expert's that has many four (dense, which follow one another, they do not fit the registers).
template <int KIND, bool GROUPED>
int launch_16(const orx_function& f, int waves, const Product& p, const Geometry& g, hipStream_t s) {
    if (waves == 4) return launch_of<KIND, 1, 4, 2, -1, 1, GROUPED>(f, p, g, s);
    if constexpr (GROUPED)
        if (steps_of(f) > 16) return launch_of<KIND, 1, 8, 4, -1, 1, GROUPED>(f, p, g, s);
    return launch_of<KIND, 1, 8, 2, -1, 1, GROUPED>(f, p, g, s);
}
template <int SOURCE, bool GROUPED>
int launch_quantising(const orx_function& f, int rows, int waves, const Product& p, const Geometry& g, hipStream_t s) {
    if (waves == 4) return launch_of<I8, 1, 4, 2, SOURCE, 4, GROUPED>(f, p, g, s);
    if (pieces_of(f, rows, waves) > 4) return launch_of<I8, 1, 8, 2, SOURCE, 8, GROUPED>(f, p, g, s);
    if constexpr (GROUPED) return launch_of<I8, 1, 8, 4, SOURCE, 4, true>(f, p, g, s);
    // (gate and up, dealt: four steps of both do not fit the registers)
    return f.flags & kSwiglu ? launch_with<I8, 1, 8, 2, SOURCE, 4, GROUPED, true>(f, p, g, s) : launch_with<I8, 1, 8, 4, SOURCE, 4, GROUPED, false>(f, p, g, s);
}
int launch_product(const orx_function& f, int rows, const Geometry& g, hipStream_t s, const Product& p) {
    const Plan plan = orx::plan(f, rows);
    if (plan.form >= 0) return launch_byte_tiles(p, f.flags2, plan.form, f.E > 0, f.flags & kSwiglu, g.grid[0], s);
    if (f.packed_k != 0) {
        const bool brains = f.packed_k - 1 == mx::BF16;
        if (f.E > 0) return brains ? launch_quantising<mx::BF16, true>(f, rows, plan.waves, p, g, s) : launch_quantising<mx::F16, true>(f, rows, plan.waves, p, g, s);
        return brains ? launch_quantising<mx::BF16, false>(f, rows, plan.waves, p, g, s) : launch_quantising<mx::F16, false>(f, rows, plan.waves, p, g, s);
    }
    if (f.E > 0) {
        if (f.flags2 == F16) return launch_16<F16, true>(f, plan.waves, p, g, s);
        return f.flags2 == BF16 ? launch_16<BF16, true>(f, plan.waves, p, g, s) : launch_16<I8, true>(f, plan.waves, p, g, s);
    }
    if (plan.rows == 16) return launch_16<I8, false>(f, plan.waves, p, g, s);
    return launch_of<I8, 4, 4, 1, -1, 1, false>(f, p, g, s);
}

Product product_of(const orx_function& f, int rows) {
    Product p = {};
    p.m = rows, p.cols = f.H, p.steps = steps_of(f), p.tiles = f.slots, p.type = f.algorithm;
    p.runs = 1;
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
    // Units come largest first, those that multiply half last: with one run to an XCD the last XCDs have little to do, with short runs XCDs share units and experts.  (us of both products with 1, 2, 4
    // and 8 runs; fp16, 128 experts of 2048 and 512: 256 tokens, units of 64 110, 107, 104, 105, 1024, of 128 187, 170, 172, 169, 4096 345, 348, 336, 341; 16 experts of 4096 and 1536: 2048 tokens,
    // 48 units 226, 225, 241, 249, 4096, 80 units 379, 380, 387, 408.  Seven banks, int8 and bf16, 16 to 512 routes to an expert of skewed and of even
    // popularity: within 5 % of the best of the four, but 10 to 25 % slower than 8 runs at 128 even routes to each of 16 or 60 experts.)
    p.runs = f.tiles >= 128 ? 4 : f.tiles >= 32 ? 2 : 1;
    p.w = pointer_arg<const uint8_t>(args, at++);
    if (f.flags2 == I8) p.w_scale = pointer_arg<const float>(args, at++);
    return launch_product(f, rows, g, s, p);
}

// Rows that a product quantises itself: their codes fit LDS, and a thread holds its part of a row.
constexpr int kMostPieces = 8;
bool quantises(const orx_function& f, int rows) {
    const Plan plan = few_rows(f, 16);
    return rows <= 16 && few_rows_lds(f, rows, plan) <= (uint32_t)kMostLds && pieces_of(f, rows, plan.waves) <= (plan.waves == 4 ? 4 : kMostPieces);
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
    f->slots = swiglu ? (f->H + 31) / 32 * 4 : (f->H + 63) / 64 * 4;
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
    if (f->M <= 0 || f->M > 1 << 24 || f->E <= 0 || f->tiles <= 0 || f->tiles > 1 << 24 || (f->block_m != 16 && f->block_m != 64 && f->block_m != 128)) {
        set_error("%s: need rows, E and tiles above 0 and block_m 16, 64 or 128", f->symbol.c_str());
        return ORX_ERR_BAD_VARIANT;
    }
    f->capacity = f->M;
    if (f->block_m > 16 && (int64_t)f->slots * steps_of(*f) * kTileBytes >= 1ll << 32) {  // (weights' loads count 32 bits from an expert's first one)
        set_error("%s: an expert's weights of 4 GiB and more go with block_m 16", f->symbol.c_str());
        return ORX_ERR_BAD_VARIANT;
    }
    if (f->packed_k != 0 && (f->block_m != 16 || !quantises(*f, 16))) {
        set_error("%s: 16-bit rows go with block_m 16 and K up to %d", f->symbol.c_str(), 64 * 8 * kMostPieces);
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
        set_error("int8_token_projection: 16-bit rows go with M up to 16 and short K: codes of all rows up to %d bytes, rows of %d values (M 1: 8 times that, 2: 4, 4: 2)", kMostLds, 64 * 8 * kMostPieces);
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
