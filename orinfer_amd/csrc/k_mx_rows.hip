// Products of few rows with MXFP4 weights (dense and routed experts), and the symbols of both.
//
//   out[m, n] = sum_k A[m, k] W[n, k], fp32 sums of exact products, rounded once; SwiGLU: columns are pairs of a gate and an up channel.
// Bound by the weights' bytes, 17/32 each: a wave streams whole tiles (2 KiB of codes, 128 bytes of powers) into registers; the K steps are dealt to the waves of a workgroup,
// whose sums meet in LDS.  The weights are the first operand, so a lane ends with four neighbouring channels of one row.  Dense rows come as tiles too: as rows of 128 bytes a step they
// took as long as the weights (weights out of cache, 17408 x 5120: 32 rows 16.7 us, as tiles 12.6, 64 rows 25.0 / 16.6).
// Rows of 16-bit values (QUANTISE, up to 16): a workgroup makes their codes itself, into LDS, while its first weights are on their way.
#include <algorithm>
#include <cmath>

#include "mx_device.h"
#include "mx_tiles.h"
#include "orx_internal.h"

namespace orx {
namespace {

using namespace mx;

// 16 or 4 bytes of a lane from a buffer of `bytes`; what lies behind its end reads as 0 and is not fetched.
struct Buffer {
    __amdgpu_buffer_rsrc_t from;
    __device__ __forceinline__ Buffer(const uint8_t* base, int bytes) : from(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, bytes, 0x00027000)) {}
    __device__ __forceinline__ v4i load_16(int offset) const { return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(from, offset, 0, 0)); }
    __device__ __forceinline__ int load_4(int offset) const { return (int)__builtin_amdgcn_raw_buffer_load_b32(from, offset, 0, 0); }
};

enum Source { Codes = 0, Halves = 1, Brains = 2 };  // of the rows: codes, fp16, bf16

// ROWS blocks of 16 rows, two tiles of 16 channels (SwiGLU: gate and up) to a workgroup of WAVES waves
template <int ROWS, int WAVES, int SOURCE, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(WAVES * 64) void mx_rows_kernel(Product p) {
    constexpr int TILES = 2;
    extern __shared__ __align__(16) uint8_t lds[];  // sums; in front of them the rows' codes and powers where they are made here
    v4f(*const sums)[ROWS * TILES][64] = reinterpret_cast<v4f(*)[ROWS * TILES][64]>(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int groups = (p.tiles + TILES - 1) / TILES;
    const int unit = blockIdx.x / groups, group = blockIdx.x % groups;
    int first_row = unit * (16 * ROWS), rows = p.m - first_row;
    const uint8_t *w = p.w, *ws = p.ws;
    if (GROUPED) {
        if (unit >= *p.unit_count) return;
        const int4 u = p.units[unit];
        first_row = __builtin_amdgcn_readfirstlane(u.y), rows = __builtin_amdgcn_readfirstlane(u.z);
        const int64_t tile = (int64_t)__builtin_amdgcn_readfirstlane(u.x) * p.tiles * p.steps;
        w += tile * kTileBytes, ws += tile * kTilePowers;
    }
    auto row_at = [&](int local) {
        int64_t row = first_row + min(local, rows - 1);  // (rows that are not there repeat the last: their sums go nowhere)
        if (GROUPED && p.slot_token != nullptr) row = p.slot_token[row];
        return row;
    };
    const int r = lane & 15, block = lane >> 4;  // lane's channel or row; its blocks of a step, and 4 behind

    // ---- weights on their way ----
    const int w_lane = lane * 16, ws_lane = r * 8 + (block & 1) * 4, ws_shift = (block >> 1) * 8;
    const uint32_t in_row = 0x0400u + 0x0101u * block;  // a row's eight powers: this lane's two, for v_perm
    struct Step {
        v4i w[TILES][2], a[ROWS][2];
        int wp[TILES];
        uint2 ap[ROWS];
    };
    const uint8_t *a[ROWS], *as[ROWS];
    if constexpr (SOURCE == Codes) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if constexpr (GROUPED) {
                const int64_t row = row_at(16 * i + r);
                a[i] = p.a + row * p.pitch + block * 16;
                as[i] = p.as + row * (p.pitch / 16);
            } else {
                const int64_t tile = min(first_row / 16 + i, (p.m - 1) / 16);
                a[i] = p.a + tile * p.steps * kTileBytes;
                as[i] = p.as + tile * p.steps * kTilePowers;
            }
        }
    }
    auto load = [&](Step& s, int step) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int64_t tile = min(group * TILES + t, p.tiles - 1);
            const Buffer codes(w + tile * p.steps * kTileBytes, p.steps * kTileBytes), powers(ws + tile * p.steps * kTilePowers, p.steps * kTilePowers);
            s.w[t][0] = codes.load_16(w_lane + step * kTileBytes);
            s.w[t][1] = codes.load_16(w_lane + step * kTileBytes + 1024);
            s.wp[t] = powers.load_4(ws_lane + step * kTilePowers);
        }
        if constexpr (SOURCE == Codes && GROUPED) {
            const int there = min(step, p.steps - 1);  // (a wave without a step)
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                s.a[i][0] = *reinterpret_cast<const v4i*>(a[i] + there * 128);
                s.a[i][1] = *reinterpret_cast<const v4i*>(a[i] + there * 128 + 64);
                s.ap[i] = *reinterpret_cast<const uint2*>(as[i] + there * 8);
            }
        } else if constexpr (SOURCE == Codes) {
            // The compiler makes one plain load of the first step's and the next one's, behind the wait for the weights.  Loads from buffers stay with the weights', and up to 32 rows that is
            // faster (us with buffers / without, 32 rows: 17408 x 5120 14.9 / 15.5, 9728 x 2560 6.6 / 6.7, 1056 x 2080 3.6 / 4.0), with 64 it is not (200 rows of 5120 x 17408 44.4 / 38.9).
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                if constexpr (ROWS <= 2) {
                    const Buffer codes(a[i], p.steps * kTileBytes), powers(as[i], p.steps * kTilePowers);
                    s.a[i][0] = codes.load_16(w_lane + step * kTileBytes);
                    s.a[i][1] = codes.load_16(w_lane + step * kTileBytes + 1024);
                    s.ap[i].x = (uint32_t)powers.load_4(ws_lane + step * kTilePowers);
                } else {
                    const int there = min(step, p.steps - 1);
                    s.a[i][0] = *reinterpret_cast<const v4i*>(a[i] + w_lane + there * kTileBytes);
                    s.a[i][1] = *reinterpret_cast<const v4i*>(a[i] + w_lane + there * kTileBytes + 1024);
                    s.ap[i].x = *reinterpret_cast<const uint32_t*>(as[i] + ws_lane + there * kTilePowers);
                }
            }
        }
    };
    Step held;
    load(held, wave);

    // ---- the rows' codes ----
    const int live = min(rows, 16);
    uint8_t* const codes = lds;
    uint8_t* const powers = lds + p.steps * 128 * live;
    if constexpr (SOURCE != Codes) {
        constexpr int TYPE = SOURCE == Halves ? F16 : BF16;
        const int pieces = p.steps * 32;  // of eight values, of a row
        for (int at = threadIdx.x; at < live * pieces; at += WAVES * 64) {
            const int row = at / pieces, piece = at - row * pieces;
            v4u words = {0, 0, 0, 0};
            if (piece * 8 < p.k) words = *reinterpret_cast<const words4*>(reinterpret_cast<const uint16_t*>(p.a) + row_at(row) * p.k + piece * 8);
            uint32_t two = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) two = pair_max(two, words[j]);
            const uint32_t byte = power_byte<TYPE>(quad_max(max(two & 0xFFFFu, two >> 16)), false);
            const uint32_t four[4] = {words[0], words[1], words[2], words[3]};
            *reinterpret_cast<uint32_t*>(codes + ((piece >> 2) * live + row) * 16 + (piece & 3) * 4) = eight_codes<TYPE>(four, byte);
            if ((piece & 3) == 0) powers[((piece >> 5) * live + row) * 8 + ((piece >> 2) & 7)] = (uint8_t)byte;
        }
        __syncthreads();
    }

    v4f sum[ROWS][TILES];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int t = 0; t < TILES; ++t) sum[i][t] = v4f{0, 0, 0, 0};
    auto multiply = [&](Step& s, int step) {
        if constexpr (SOURCE != Codes) {
            const int there = min(step, p.steps - 1), row = min(r, live - 1);
            const uint8_t* const from = codes + ((there * 8 + block) * live + row) * 16;
            s.a[0][0] = *reinterpret_cast<const v4i*>(from);
            s.a[0][1] = *reinterpret_cast<const v4i*>(from + 4 * live * 16);
            s.ap[0] = *reinterpret_cast<const uint2*>(powers + (there * live + row) * 8);
        }
        int wp[TILES];  // bytes 0 and 2, or 0 and 1, are this lane's
#pragma unroll
        for (int t = 0; t < TILES; ++t) wp[t] = (int)((uint32_t)s.wp[t] >> ws_shift);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            constexpr bool TILED = SOURCE == Codes && !GROUPED;
            const int ap = TILED ? (int)(s.ap[i].x >> ws_shift) : (int)__builtin_amdgcn_perm(s.ap[i].y, s.ap[i].x, in_row);
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                sum[i][t] = multiply_16<0, 0>(s.w[t][0], s.a[i][0], sum[i][t], wp[t], ap);
                sum[i][t] = multiply_16<2, TILED ? 2 : 1>(s.w[t][1], s.a[i][1], sum[i][t], wp[t], ap);
            }
        }
    };
#pragma unroll 1
    for (int step = wave; step < p.steps; step += WAVES) {
        multiply(held, step);
        if (step + WAVES < p.steps) load(held, step + WAVES);  // (what lies behind the end would still be waited for: 7168 x 5120, 32 rows 7.5 us, else 9.2)
    }
    if constexpr (SOURCE != Codes) __syncthreads();  // (the sums take the codes' place)
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int t = 0; t < TILES; ++t) sums[wave][i * TILES + t][lane] = sum[i][t];
    __syncthreads();
    constexpr int KINDS = SWIGLU ? 2 : 1;
    for (int q = threadIdx.x; q < ROWS * TILES / KINDS * 64; q += WAVES * 64) {
        const int l = q & 63, i = (q >> 6) / (TILES / KINDS), t = (q >> 6) % (TILES / KINDS);
        v4f total[KINDS];
#pragma unroll
        for (int kind = 0; kind < KINDS; ++kind) {
            total[kind] = sums[0][i * TILES + t * KINDS + kind][l];
#pragma unroll
            for (int other = 1; other < WAVES; ++other) total[kind] += sums[other][i * TILES + t * KINDS + kind][l];
        }
        if constexpr (SWIGLU) {
#pragma unroll
            for (int j = 0; j < 4; ++j) total[0][j] = swiglu(total[0][j], total[1][j]);
        }
        const int row = 16 * i + (l & 15);
        if (row < rows)
            store_four(p.out, p.type, (int64_t)(first_row + row) * p.cols, ((group * TILES) / KINDS + t) * 16 + 4 * (l >> 4), p.cols, total[0]);
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------------
// slots used: M (rows; experts: slots), N, K, E, tiles (units), block_m, flags (kSwiglu, kGather), algorithm (output type), H (output columns), slots (16-channel tiles)
// packed_k (source of the rows)
constexpr int kMostLds = 80 * 1024;  // of the few-rows kernel
enum { kSwiglu = 1, kGather = 2 };

// What a launch of `rows` rows runs: a unit's rows, and channels to a workgroup of the tiles from LDS, whose waves may take K in two halves (0: the kernel above, 32 channels), or its waves
struct Plan {
    int rows, channels, waves, halves = 1;
};
// Eight waves share K, four with 64 rows (us with four / eight, weights out of cache: 16 rows, 7168 x 5120 7.1 / 6.4, 17408 x 5120 13.4 / 13.0, 9728 x 2560 level; 32 rows, 7168 x 5120 7.9 / 7.5,
// 17408 x 5120 16.0 / 15.4, 2048 x 1024 3.4 / 3.1; 64 rows to a unit, 160 of 7168 x 5120 14.3 / 16.5, 333 of 4096 x 4096 11.4 / 13.7, 64 of 1024 x 4096 level).
Plan few_rows(int unit_rows) { return {unit_rows, 0, unit_rows == 64 ? 4 : 8}; }
// Us that a launch takes, weights out of cache, 256 CUs (within a fifth of what was measured at 32-700 rows of 7168 x 5120, 4096 x 4096, 1024 x 4096, 17408 x 5120, 5120 x 17408, 2048 x 1024,
// 1056 x 2080, 9728 x 2560).  The kernel above: a chain of steps for each wave, or what all workgroups read through the L2s.  Tiles: a chain of steps, longer where a CU has several
// workgroups side by side or one after another.  So few rows of few channels go to the former (128 rows of 4096 x 4096: 6.8, tiles 12.1 and 14.0), 32 to a unit first (64 rows: 5.3, as one
// unit 6.7), tiles where there are enough for all CUs, in halves of K where there are not (333 rows of 7168 x 5120: 20.1, else 23.1; 333 rows of 5120 x 17408 45, else 57).  64 rows x 64
// channels to a workgroup of the former were within a tenth of the better of the others.
double few_rows_us(const orx_function& f, int rows, const Plan& plan) {
    const double steps = (f.K + kStepK - 1) / kStepK, workgroups = (double)ceil_div(rows, plan.rows) * ((f.slots + 1) / 2);
    const double chain = std::ceil(steps / plan.waves) * (plan.rows == 64 ? 1.2 : 1.1);
    return 2.5 + std::max(chain, workgroups * (plan.rows + 32) * steps * 136 / 15.2e6 * (256.0 / device_compute_units()));
}
double tiles_us(const orx_function& f, int rows, const Plan& tile) {
    const int64_t cus = device_compute_units(), tiles = (int64_t)ceil_div(rows, tile.rows) * ceil_div(f.slots, tile.channels / 16);
    const double steps = (f.K + kStepK - 1) / kStepK, to_a_cu = (double)((tiles + cus - 1) / cus);
    if (tile.halves == 2) return tiles > cus || steps < 2 ? 1e30 : 2.5 + std::ceil(steps / 2) * (tile.rows == 64 ? 1.35 : 1.65);
    if (tile.rows == 64) return 2.5 + steps * std::max(0.85, 0.45 * to_a_cu);
    return 2.5 + steps * (tile.rows == 256 ? 1.8 * to_a_cu : to_a_cu == 1 ? 1.0 : 1.27 * std::ceil(to_a_cu / 2));
}
Plan plan(const orx_function& f, int rows) {
    if (f.E > 0) {
        // (of few steps: 128 experts x 8, 16 tokens, 512 deep, us with four / eight waves 10.4 / 13.5, 2048 deep 12.5 / 12.9)
        if (f.block_m == 16) return {16, 0, f.packed_k == Codes ? 4 : 8};
        return {f.block_m, f.block_m == 256 ? 256 : 128, 0};
    }
    if (rows <= 32) return few_rows(rows <= 16 ? 16 : 32);
    Plan best = few_rows(32);
    double best_us = few_rows_us(f, rows, best);
    auto weigh = [&](const Plan& other, double us) {
        if (us < best_us) best = other, best_us = us;
    };
    weigh(few_rows(64), few_rows_us(f, rows, few_rows(64)));
    if (rows > 64)
        for (const Plan& tile : {Plan{64, 128, 0, 1}, Plan{64, 128, 0, 2}, Plan{128, 128, 0, 1}, Plan{128, 128, 0, 2}, Plan{256, 256, 0, 1}}) weigh(tile, tiles_us(f, rows, tile));
    return best;
}
uint32_t few_rows_lds(const orx_function& f, int rows, const Plan& plan) {
    const uint32_t sums = (uint32_t)plan.waves * (plan.rows / 16) * 2 * 1024;
    const uint32_t codes = f.packed_k == Codes ? 0 : (uint32_t)((f.K + kStepK - 1) / kStepK) * 136 * std::min(f.E > 0 ? 16 : rows, 16);
    return std::max(sums, codes);
}

int geometry(const orx_function& f, int rows, Geometry* g) {
    const Plan plan = orx::plan(f, rows);
    const int64_t units = f.E > 0 ? f.tiles : ceil_div(rows, plan.rows);
    int64_t blocks = units * ceil_div(f.slots, plan.channels ? plan.channels / 16 : 2);
    if (blocks >= (1ll << 32) / 512) {
        set_error("%s: %d rows of %d channels are more than one launch takes", f.symbol.c_str(), rows, f.N);
        return ORX_ERR_ROWS;
    }
    if (plan.channels) {
        if (plan.halves == 1) blocks = std::min<int64_t>(blocks, (int64_t)device_compute_units() * mx_tiles_to_a_cu(plan.rows));
        g->block[0] = mx_tiles_threads(plan.rows, plan.halves);
        g->shared = mx_tiles_lds(plan.rows, plan.channels, plan.halves);
    } else {
        g->block[0] = 64 * plan.waves;
        g->shared = few_rows_lds(f, rows, plan);
    }
    g->grid[0] = (uint32_t)blocks;
    return ORX_OK;
}

template <int ROWS, int WAVES, int SOURCE, bool GROUPED, bool SWIGLU>
int launch_one(const Product& p, const Geometry& g, hipStream_t s) {
    constexpr auto kernel = &mx_rows_kernel<ROWS, WAVES, SOURCE, GROUPED, SWIGLU>;
    static DeviceOnce ready;
    const int code = ready.run([] { return hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds), "hipFuncSetAttribute"); });
    if (code != ORX_OK) return code;
    ORX_LAUNCH(kernel, dim3(g.grid[0]), dim3(64 * WAVES), g.shared, s, p);
    return hip_check(hipGetLastError(), "launch mxfp4 product");
}
template <int ROWS, int WAVES, int SOURCE>
int launch_of(const orx_function& f, const Product& p, const Geometry& g, hipStream_t s) {
    const bool swiglu = f.flags & kSwiglu;
    if constexpr (SOURCE == Halves)
        if (f.E > 0) return swiglu ? launch_one<ROWS, WAVES, SOURCE, true, true>(p, g, s) : launch_one<ROWS, WAVES, SOURCE, true, false>(p, g, s);
    return swiglu ? launch_one<ROWS, WAVES, SOURCE, false, true>(p, g, s) : launch_one<ROWS, WAVES, SOURCE, false, false>(p, g, s);
}
int launch_product(const orx_function& f, int rows, const Geometry& g, hipStream_t s, const Product& p) {
    const Plan plan = orx::plan(f, rows);
    if (plan.channels) return launch_mx_tiles(p, plan.rows, plan.channels, plan.halves, f.E > 0, f.flags & kSwiglu, g.grid[0], s);
    if (f.packed_k == Halves) return launch_of<1, 8, Halves>(f, p, g, s);
    if (f.packed_k == Brains) return launch_of<1, 8, Brains>(f, p, g, s);
    if (f.E > 0) return f.flags & kSwiglu ? launch_one<1, 4, Codes, true, true>(p, g, s) : launch_one<1, 4, Codes, true, false>(p, g, s);
    if (plan.rows == 16) return launch_of<1, 8, Codes>(f, p, g, s);
    return plan.rows == 32 ? launch_of<2, 8, Codes>(f, p, g, s) : launch_of<4, 4, Codes>(f, p, g, s);
}

Product product_of(const orx_function& f, int rows) {
    Product p = {};
    p.m = rows, p.cols = f.H, p.k = f.K, p.steps = (f.K + kStepK - 1) / kStepK, p.pitch = (p.steps | 1) * (kStepK / 2), p.tiles = f.slots, p.type = f.algorithm;
    return p;
}

// A[, AS], Out, W, WS[, m]
int projection_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    Product p = product_of(f, rows);
    const int codes = f.packed_k == Codes ? 1 : 0;
    p.a = pointer_arg<const uint8_t>(args, 0), p.as = codes ? pointer_arg<const uint8_t>(args, 1) : nullptr, p.out = pointer_arg<void>(args, 1 + codes);
    p.w = pointer_arg<const uint8_t>(args, 2 + codes), p.ws = pointer_arg<const uint8_t>(args, 3 + codes);
    return launch_product(f, rows, g, s, p);
}
// A[, AS], Out[, SlotToken], TileCount, TileUnits, W, WS
int grouped_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    Product p = product_of(f, rows);
    const int codes = f.packed_k == Codes ? 1 : 0, gather = f.flags & kGather ? 1 : 0;
    p.a = pointer_arg<const uint8_t>(args, 0), p.as = codes ? pointer_arg<const uint8_t>(args, 1) : nullptr, p.out = pointer_arg<void>(args, 1 + codes);
    p.slot_token = gather ? pointer_arg<const int>(args, 2 + codes) : nullptr;
    const int at = 2 + codes + gather;
    p.unit_count = pointer_arg<const int>(args, at), p.units = pointer_arg<const int4>(args, at + 1), p.most_units = f.tiles;
    p.w = pointer_arg<const uint8_t>(args, at + 2), p.ws = pointer_arg<const uint8_t>(args, at + 3);
    return launch_product(f, rows, g, s, p);
}
void row_arguments(orx_function* f) {
    f->args = {{"A", ArgPointer, f->packed_k == Codes ? 16u : 2u}};
    if (f->packed_k == Codes) f->args.push_back({"AS", ArgPointer, 8});
    f->args.push_back({"Out", ArgPointer, f->algorithm == F32 ? 4u : 2u});
}

int shape(const Variant& v, orx_function* f) {
    bool bad = false;
    f->N = (int)v.integer("N", 0, &bad), f->K = (int)v.integer("K", 0, &bad);
    const std::string epilogue = v.string("epilogue", "none", &bad);
    f->algorithm = mx_type(v, "output_dtype", "float16", &bad);
    // 16-bit rows are quantised on their way (few rows)
    const std::string input = v.string("input_dtype", "mxfp4", &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    if (input != "mxfp4" && input != "float16" && (input != "bfloat16" || f->E > 0)) {
        set_error("%s: input_dtype must be mxfp4 or float16%s", f->symbol.c_str(), f->E > 0 ? "" : " or bfloat16");
        return ORX_ERR_BAD_VARIANT;
    }
    f->packed_k = input == "mxfp4" ? Codes : input == "float16" ? Halves : Brains;
    if (epilogue != "none" && epilogue != "swiglu") {
        set_error("%s: epilogue must be none or swiglu", f->symbol.c_str());
        return ORX_ERR_BAD_VARIANT;
    }
    const bool swiglu = epilogue == "swiglu";
    f->flags = swiglu ? kSwiglu : 0;
    if (f->N <= 0 || f->N > 1 << 24 || (swiglu && f->N % 2) || f->K <= 0 || f->K % kBlock || f->K > 1 << 20) {
        set_error("%s: need 0 < N <= %d (even for swiglu) and K a multiple of %d up to %d", f->symbol.c_str(), 1 << 24, kBlock, 1 << 20);
        return ORX_ERR_BAD_VARIANT;
    }
    f->H = swiglu ? f->N / 2 : f->N;
    f->slots = (f->H + 15) / 16 * (swiglu ? 2 : 1);
    f->geometry = geometry;
    return ORX_OK;
}

}  // namespace

int make_mx_projection(const Variant& v, orx_function* f) {
    bool bad = false;
    f->M = (int)v.integer("M", 0, &bad);
    f->dynamic_rows = v.boolean("dynamic_rows", false, &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    const int code = shape(v, f);
    if (code != ORX_OK) return code;
    if (f->M <= 0 || f->M > 1 << 24) {
        set_error("mxfp4_projection: need 0 < M <= %d", 1 << 24);
        return ORX_ERR_BAD_VARIANT;
    }
    f->capacity = f->M;
    if (f->packed_k != Codes && (f->M > 16 || few_rows_lds(*f, f->M, {16, 0, 8}) > (uint32_t)kMostLds)) {
        set_error("mxfp4_projection: 16-bit rows go with M up to 16 and codes of all rows up to %d bytes", kMostLds);
        return ORX_ERR_BAD_VARIANT;
    }
    row_arguments(f);
    f->args.push_back({"W", ArgPointer, 16}), f->args.push_back({"WS", ArgPointer, 8});
    if (f->dynamic_rows) f->args.push_back({"m", ArgI32, 4});
    f->launch = projection_launch;
    return ORX_OK;
}

int make_mx_grouped(const Variant& v, orx_function* f) {
    bool bad = false;
    f->M = (int)v.integer("rows", 0, &bad), f->E = (int)v.integer("E", 0, &bad), f->tiles = (int)v.integer("tiles", 0, &bad);
    f->block_m = (int)v.integer("block_m", 16, &bad);
    const bool gather = v.boolean("gather", false, &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    const int code = shape(v, f);
    if (code != ORX_OK) return code;
    if (f->M <= 0 || f->M > 1 << 24 || f->E <= 0 || f->tiles <= 0 || f->tiles > 1 << 24 || (f->block_m != 16 && f->block_m != 64 && f->block_m != 128 && f->block_m != 256)) {
        set_error("mxfp4_grouped: need rows, E and tiles above 0 and block_m 16, 64, 128 or 256");
        return ORX_ERR_BAD_VARIANT;
    }
    f->flags |= gather ? kGather : 0;
    f->capacity = f->M;
    if (f->packed_k != Codes && (f->block_m != 16 || few_rows_lds(*f, f->M, {16, 0, 8}) > (uint32_t)kMostLds)) {
        set_error("mxfp4_grouped: 16-bit rows go with block_m 16 and codes of 16 rows up to %d bytes", kMostLds);
        return ORX_ERR_BAD_VARIANT;
    }
    row_arguments(f);
    if (gather) f->args.push_back({"SlotToken", ArgPointer, 4});
    for (const ArgSpec& a : std::initializer_list<ArgSpec>{{"TileCount", ArgPointer, 4}, {"TileUnits", ArgPointer, 16}, {"W", ArgPointer, 16}, {"WS", ArgPointer, 8}}) f->args.push_back(a);
    f->launch = grouped_launch;
    Geometry g;
    return geometry(*f, f->M, &g);
}

}  // namespace orx
