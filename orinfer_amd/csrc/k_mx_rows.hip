// Products of few rows with MXFP4 weights (dense and routed experts), and the symbols of both.
//
//   out[m, n] = sum_k A[m, k] W[n, k], fp32 sums of exact products, rounded once; SwiGLU: columns are pairs of a gate and an up channel.
// Bound by the weights' bytes, 17/32 each: a wave streams whole tiles (2 KiB of codes, 128 bytes of powers, no LDS in front of the multiplier) and the K steps are dealt to
// the waves of a workgroup, whose sums meet in LDS.  The weights are the first operand, so a lane ends with four neighbouring channels of one row.
#include <algorithm>

#include "mx_device.h"
#include "mx_tiles.h"
#include "orx_internal.h"

namespace orx {
namespace {

using namespace mx;

// ROWS blocks of 16 rows, TILES tiles of 16 channels (SwiGLU: gate and up in turn) to a workgroup of WAVES waves
template <int ROWS, int TILES, int WAVES, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(WAVES * 64) void mx_rows_kernel(Product p) {
    static_assert(!SWIGLU || TILES % 2 == 0, "pairs");
    __shared__ v4f sums[WAVES][ROWS * TILES][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int groups = (p.tiles + TILES - 1) / TILES;
    const int unit = blockIdx.x / groups, group = blockIdx.x % groups;
    int first_row = unit * (16 * ROWS), rows = p.m - first_row;
    const uint8_t *w = p.w, *ws = p.ws;
    if (GROUPED) {
        if (unit >= *p.unit_count) return;
        const int4 u = p.units[unit];
        first_row = u.y, rows = u.z;
        w += (int64_t)u.x * p.tiles * p.steps * kTileBytes, ws += (int64_t)u.x * p.tiles * p.steps * kTilePowers;
    }
    const int r = lane & 15, low = (lane >> 4) & 1, half = lane >> 5;  // lane's channel or row; its blocks 4 half + low and + 2 of every step
    const uint8_t *a[ROWS], *as[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        int64_t row = first_row + min(16 * i + r, rows - 1);  // (rows that are not there repeat the last: their sums go nowhere)
        if (GROUPED && p.slot_token != nullptr) row = p.slot_token[row];
        a[i] = p.a + row * p.pitch + (4 * half + low) * 16;
        as[i] = p.as + row * (p.pitch / 16) + 4 * half;
    }
    const uint8_t *wt[TILES], *wst[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int64_t tile = min(group * TILES + t, p.tiles - 1);
        wt[t] = w + tile * p.steps * kTileBytes + (4 * half + low) * 256 + r * 16;
        wst[t] = ws + tile * p.steps * kTilePowers + r * 8 + low * 4 + half * 2;
    }
    v4f sum[ROWS][TILES];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int t = 0; t < TILES; ++t) sum[i][t] = v4f{0, 0, 0, 0};
    for (int step = wave; step < p.steps; step += WAVES) {
        v4i wc[TILES][2], ac[ROWS][2];
        int wp[TILES], ap[ROWS];
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const uint8_t* const from = wt[t] + (int64_t)step * kTileBytes;
            wc[t][0] = *reinterpret_cast<const v4i*>(from);
            wc[t][1] = *reinterpret_cast<const v4i*>(from + 512);
            wp[t] = *reinterpret_cast<const unsigned short*>(wst[t] + (int64_t)step * kTilePowers);
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            ac[i][0] = *reinterpret_cast<const v4i*>(a[i] + step * 128);
            ac[i][1] = *reinterpret_cast<const v4i*>(a[i] + step * 128 + 32);
            ap[i] = *reinterpret_cast<const int*>(as[i] + step * 8) >> (8 * low);
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                sum[i][t] = multiply_16<0, 0>(wc[t][0], ac[i][0], sum[i][t], wp[t], ap[i]);
                sum[i][t] = multiply_16<1, 2>(wc[t][1], ac[i][1], sum[i][t], wp[t], ap[i]);
            }
    }
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
enum { kSwiglu = 1, kGather = 2 };
constexpr int kWaves = 4;

// What a launch of `rows` rows runs: a unit's rows, and channels to a workgroup of the tiles from LDS (0: the kernel above, 32 of them)
struct Plan {
    int rows, channels;
};
// us that tiles of one kind take: a start, then what the busiest CU has to do, step by step, or all of them at the rate that they sustain (the clock falls with the power that
// the multipliers draw).  Measured alone, 256 CUs, M x N x K, us with 64 x 128 / 128 x 128 / 256 x 256: 512 x 4096 x 4096 10.1 / 12.1 / 25.6; 2048 x 4096 x 4096 29.2 / 26.8 / 32.2;
// 8192 x 4096 x 4096 105 / 91 / 76; 333 x 7168 x 5120 16.3 / 15.6 / 31.9; 1500 x 7168 x 5120 49.4 / 44.7 / 38.1; 512 x 17408 x 5120 40.0 / 43.4 / 35.8; 1024 x 17408 x 5120 74 / 69 / 76.
double tiles_us(int64_t tiles, int steps, int rows, int channels, double step_us, double petaflops) {
    const int cus = device_compute_units();
    const double busiest = (double)((tiles + cus - 1) / cus) * steps * step_us;
    const double all = (double)tiles * steps * (2e-9 * kStepK * rows * channels) / petaflops * (256.0 / cus);
    return 2.5 + std::max(busiest, all);
}
Plan plan(const orx_function& f, int rows) {
#ifdef MX_SWEEP
    const char* force = getenv("MX_FORCE");
    if (force && rows >= 100) { int r, c; sscanf(force, "%d,%d", &r, &c); if (f.E == 0 || f.block_m == r) return {r, c}; }
#endif
    if (f.E > 0) return {f.block_m, f.block_m >= 64 ? (f.block_m == 256 ? 256 : 128) : 0};
    if (rows <= 64) return {rows <= 16 ? 16 : rows <= 32 ? 32 : 64, 0};
    const int steps = (f.K + kStepK - 1) / kStepK;
    const int64_t across = ceil_div(f.slots, 8);
    const double small = tiles_us(ceil_div(rows, 64) * across, steps, 64, 128, 0.40, 2.6), medium = tiles_us(ceil_div(rows, 128) * across, steps, 128, 128, 0.62, 3.05);
    const double large = tiles_us((int64_t)ceil_div(rows, 256) * ceil_div(f.slots, 16), steps, 256, 256, 1.75, 3.65);
    if (large <= medium && large <= small) return {256, 256};
    return medium <= small ? Plan{128, 128} : Plan{64, 128};
}

int geometry(const orx_function& f, int rows, Geometry* g) {
    const Plan plan = orx::plan(f, rows);
    const int64_t units = f.E > 0 ? f.tiles : ceil_div(rows, plan.rows);
    int64_t blocks = units * ceil_div(f.slots, plan.channels ? plan.channels / 16 : 2);
    if (blocks >= (1ll << 32) / 256) {
        set_error("%s: %d rows of %d channels are more than one launch takes", f.symbol.c_str(), rows, f.N);
        return ORX_ERR_ROWS;
    }
    if (plan.channels) {
        blocks = std::min<int64_t>(blocks, (int64_t)device_compute_units() * mx_tiles_to_a_cu(plan.rows));
        g->block[0] = mx_tiles_threads(plan.rows);
        g->shared = mx_tiles_lds(plan.rows, plan.channels);
    } else {
        g->block[0] = 64 * kWaves;
    }
    g->grid[0] = (uint32_t)blocks;
    return ORX_OK;
}

int launch_product(const orx_function& f, int rows, const Geometry& g, hipStream_t s, const Product& p) {
    const Plan plan = orx::plan(f, rows);
    if (plan.channels) return launch_mx_tiles(p, plan.rows, plan.channels, f.E > 0, f.flags & kSwiglu, g.grid[0], s);
    const dim3 grid(g.grid[0]), block(64 * kWaves);
#define ORX_MX(ROWS)                                                                                                          \
    do {                                                                                                                      \
        if (f.E > 0) {                                                                                                        \
            if (f.flags & kSwiglu) ORX_LAUNCH((mx_rows_kernel<ROWS, 2, kWaves, true, true>), grid, block, 0, s, p);            \
            else ORX_LAUNCH((mx_rows_kernel<ROWS, 2, kWaves, true, false>), grid, block, 0, s, p);                             \
        } else {                                                                                                              \
            if (f.flags & kSwiglu) ORX_LAUNCH((mx_rows_kernel<ROWS, 2, kWaves, false, true>), grid, block, 0, s, p);           \
            else ORX_LAUNCH((mx_rows_kernel<ROWS, 2, kWaves, false, false>), grid, block, 0, s, p);                            \
        }                                                                                                                     \
    } while (0)
    if (plan.rows == 16) ORX_MX(1);
    else if (plan.rows == 32) ORX_MX(2);
    else ORX_MX(4);
#undef ORX_MX
    return hip_check(hipGetLastError(), "launch mxfp4 product");
}

Product product_of(const orx_function& f, int rows) {
    Product p = {};
    p.m = rows, p.cols = f.H, p.steps = (f.K + kStepK - 1) / kStepK, p.pitch = (p.steps | 1) * (kStepK / 2), p.tiles = f.slots, p.type = f.algorithm;
    return p;
}

// A, AS, Out, W, WS[, m]
int projection_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    Product p = product_of(f, rows);
    p.a = pointer_arg<const uint8_t>(args, 0), p.as = pointer_arg<const uint8_t>(args, 1), p.out = pointer_arg<void>(args, 2);
    p.w = pointer_arg<const uint8_t>(args, 3), p.ws = pointer_arg<const uint8_t>(args, 4);
    return launch_product(f, rows, g, s, p);
}
// A, AS, Out[, SlotToken], TileCount, TileUnits, W, WS
int grouped_launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    Product p = product_of(f, rows);
    const int gather = f.flags & kGather ? 1 : 0;
    p.a = pointer_arg<const uint8_t>(args, 0), p.as = pointer_arg<const uint8_t>(args, 1), p.out = pointer_arg<void>(args, 2);
    p.slot_token = gather ? pointer_arg<const int>(args, 3) : nullptr;
    p.unit_count = pointer_arg<const int>(args, 3 + gather), p.units = pointer_arg<const int4>(args, 4 + gather);
    p.w = pointer_arg<const uint8_t>(args, 5 + gather), p.ws = pointer_arg<const uint8_t>(args, 6 + gather);
    return launch_product(f, rows, g, s, p);
}

int shape(const Variant& v, orx_function* f) {
    bool bad = false;
    f->N = (int)v.integer("N", 0, &bad), f->K = (int)v.integer("K", 0, &bad);
    const std::string epilogue = v.string("epilogue", "none", &bad);
    f->algorithm = mx_type(v, "output_dtype", "float16", &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
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
    f->args = {{"A", ArgPointer, 16}, {"AS", ArgPointer, 8}, {"Out", ArgPointer, f->algorithm == F32 ? 4u : 2u}, {"W", ArgPointer, 16}, {"WS", ArgPointer, 8}};
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
    if (f->M <= 0 || f->M > 1 << 24 || f->E <= 0 || f->tiles <= 0 || f->tiles > 1 << 24 || (f->block_m != 16 && f->block_m != 32 && f->block_m != 64 && f->block_m != 128 && f->block_m != 256)) {
        set_error("mxfp4_grouped: need rows, E and tiles above 0 and block_m 16, 32, 64, 128 or 256");
        return ORX_ERR_BAD_VARIANT;
    }
    f->flags |= gather ? kGather : 0;
    f->capacity = f->M;
    f->args = {{"A", ArgPointer, 16}, {"AS", ArgPointer, 8}, {"Out", ArgPointer, f->algorithm == F32 ? 4u : 2u}};
    if (gather) f->args.push_back({"SlotToken", ArgPointer, 4});
    for (const ArgSpec& a : std::initializer_list<ArgSpec>{{"TileCount", ArgPointer, 4}, {"TileUnits", ArgPointer, 16}, {"W", ArgPointer, 16}, {"WS", ArgPointer, 8}}) f->args.push_back(a);
    f->launch = grouped_launch;
    Geometry g;
    return geometry(*f, f->M, &g);
}

}  // namespace orx
