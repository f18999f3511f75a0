// Dense products of many rows of 8-bit integers with weights by byte tiles: tiles of the output from LDS.
//
// DOWN x ACROSS waves share a tile, each ROWS x CHANNELS blocks of 16 x 16 of it; K goes in steps of 128 bytes.  Rows and weights come from memory to LDS without passing a register, a kilobyte to a
// request as they are laid out.  A workgroup goes through its tiles as one sequence of steps: the next tile's first steps are on their way while the last ones are multiplied, and results drain
// under the next multiplies.
// 256 x 256 results, two stages: bound by the multiplier where tiles fill the CUs (1.25 us a step, 1.7 times the multiplies' own time at 2.4 GHz: at 8192 rows of 4096 x 4096 the pipe is busy in 0.64 of
// the cycles, and these take 1.8 GHz, where launches that multiply less run at 2.0 to 2.5).
// 128 x 128, 96 x 128, 64 x 128 and 64 x 64, for launches of fewer tiles than CUs: a CU took in 50-60 GB/s of operands in every form.  No unit is full then (333 rows of 7168 x 5120: pipe 0.26 of the
// cycles, LDS 0.16, 21 bytes a cycle from the L2, 2.3 TB/s from memory; waves wait in 0.38): it is what latency and one workgroup to a CU leave.  Four, five and six stages are under way (128 x 128:
// 0.54 us a step of 32 KB, with two stages 0.8, with two stages and half of K to either half of a workgroup 0.65; by eight waves 29.0 us at 128 rows of 17408 x 5120, by four 30.9; 96 x 128: 0.47; 64 x 128: 0.46, with
// two stages 0.75, with halves of K 0.55).  Of 64 x 64 four stages leave room for two workgroups to a CU (0.27 each).
// (A wave more that brought later steps' lines to the L2 made all of them 30-50 % slower: the lines that are asked for are what counts.)
#include "byte_wide_kernel.h"
#include "lds_asm.h"
#include "orx_internal.h"
#include "tile_requests.h"

namespace orx {
namespace {

using namespace bytes;
using namespace tile_requests;
using lds_asm::Each;

template <int ROWS, int CHANNELS, int DOWN, int ACROSS, int STAGES>
struct Form {
    static constexpr int rows = ROWS, channels = CHANNELS, across = ACROSS, stages = STAGES;
    static constexpr int bm = 16 * ROWS * DOWN, row_places = (bm + 63) / 64 * 64, bn = 16 * CHANNELS * ACROSS, waves = DOWN * ACROSS, stage = (bm + bn) * kStep;
    // what a tile's rows and channels have, for the results: scales, zero points, sums and biases; of the tile that is multiplied and of as many as there are stages
    static constexpr int scale_bytes = 4 * (2 * row_places + 3 * bn), lds = STAGES * stage + (STAGES + 1) * scale_bytes;
    static_assert(lds <= 160 * 1024, "a CU's LDS");
};

template <typename FORM, bool WIDE, bool SWIGLU>
__global__ __launch_bounds__(64 * FORM::waves, FORM::waves / 4 * (160 * 1024 / FORM::lds)) void byte_tiles_kernel(Product p) {
    using Sum = Operands<I8>::Sum;
    constexpr int ROWS = FORM::rows, CHANNELS = FORM::channels, ACROSS = FORM::across, WAVES = FORM::waves, STAGES = FORM::stages, BM = FORM::bm, BN = FORM::bn;
    constexpr bool HALF = BM / 16 % WAVES != 0;  // rows are requested by halves of tiles
    constexpr int A_REQUESTS = BM / (HALF ? 8 : 16) / WAVES, W_REQUESTS = BN / 16 / WAVES;  // of a wave and step
    constexpr int kAll = A_REQUESTS + W_REQUESTS, kLoads = (HALF ? 1 : 2) * A_REQUESTS + 2 * W_REQUESTS;
    static_assert(A_REQUESTS * WAVES == BM / (HALF ? 8 : 16) && W_REQUESTS * WAVES == BN / 16, "all of a stage");
    constexpr int kW = BM * kStep, kStage = FORM::stage, kScales = STAGES * kStage, kScaleBytes = FORM::scale_bytes;
    constexpr int kZeros = 4 * FORM::row_places, kChannels = 8 * FORM::row_places;  // of a tile's scales
    extern __shared__ __align__(128) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wave_m = wave / ACROSS, wave_n = wave % ACROSS;

    // ---- which results: tiles blockIdx.x, blockIdx.x + gridDim.x, .. of an order in which every XCD has one run ----
    const int groups = (p.tiles + BN / 16 - 1) / (BN / 16);
    const int row_tiles = (p.m + BM - 1) / BM;
    const int total = row_tiles * groups;
    const int my_tiles = __builtin_amdgcn_readfirstlane((total - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x);
    if (my_tiles <= 0) return;
    struct Tile {
        int first_row, rows, group;
    };
    auto tile_of = [&](int number) __attribute__((always_inline)) {
        const int at = (int)blockIdx.x + number * (int)gridDim.x, xcd = at & 7;
        const int id = xcd * (total >> 3) + min(xcd, total & 7) + (at >> 3);
        // eight tiles of rows for each tile of channels, so that an L2 holds what neighbours share
        const int band = id / (8 * groups), in_band = min(8, row_tiles - 8 * band), within = id % (8 * groups);
        Tile t;
        t.first_row = (8 * band + within % in_band) * BM, t.group = within / in_band, t.rows = min(BM, p.m - t.first_row);
        return t;
    };
    const uint32_t lds_base = lds_asm::lds_address_of(lds);

    // ---- requests ----
    const uint8_t *a_from[A_REQUESTS], *w_from[W_REQUESTS];  // tiles
    const int64_t step_bytes = (int64_t)p.tiles * kTileBytes;  // of the weights
    int load_tile = 0, load_step = 0, load_scales = 0, scales = 0;  // the tile and step whose requests come next, and where its scales and those of the tile that is multiplied lie
    auto turn = [&](int& at) __attribute__((always_inline)) { at = at == STAGES * kScaleBytes ? 0 : at + kScaleBytes; };
    Tile load_at;
    auto aim = [&]() __attribute__((always_inline)) {
        load_at = tile_of(load_tile);
#pragma unroll
        for (int b = 0; b < A_REQUESTS; ++b) {
            const int at = wave * A_REQUESTS + b;
            a_from[b] = uniform_pointer(p.a + (int64_t)min(load_at.first_row / 16 + (HALF ? at / 2 : at), (p.m - 1) / 16) * p.steps * kTileBytes + (HALF ? at % 2 * 1024 : 0));
        }
#pragma unroll
        for (int b = 0; b < W_REQUESTS; ++b) w_from[b] = uniform_pointer(p.w + (int64_t)min(load_at.group * (BN / 16) + wave * W_REQUESTS + b, p.tiles - 1) * kTileBytes);
    };
    auto request_scales = [&]() __attribute__((always_inline)) {  // in front of a tile's first step
        constexpr int R = FORM::row_places / 64, C = BN / 64, CHUNKS = 2 * R + 3 * C;
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds_base + kScales + load_scales);
#pragma unroll
        for (int c = 0; c < (CHUNKS + WAVES - 1) / WAVES; ++c) {
            const int chunk = wave + c * WAVES;  // (uniform)
            const bool of_rows = chunk < 2 * R;
            // Rows that are not there repeat the last: their sums go nowhere.
            const int64_t row = load_at.first_row + min(chunk % R * 64 + lane, load_at.rows - 1);
            const int64_t channel = min((load_at.group * C + (chunk - 2 * R) % C) * 64 + lane, p.tiles * 16 - 1);
            const int kind = of_rows ? chunk / R : 2 + (chunk - 2 * R) / C;
            const uint8_t* const base = reinterpret_cast<const uint8_t*>(kind == 0 ? (const void*)p.scale : kind == 1 ? (const void*)p.zero : kind == 2 ? (const void*)p.w_scale : kind == 3 ? (const void*)p.w_sum : (const void*)p.bias);
            request_4_from(base + (of_rows ? row : channel) * 4, to + chunk * 256, __builtin_amdgcn_readfirstlane(base == nullptr ? 0 : CHUNKS - chunk));
        }
        turn(load_scales);
    };
    auto advance = [&]() __attribute__((always_inline)) {
        if (++load_step < p.steps) return;
        load_step = 0;
        if (++load_tile < my_tiles) aim();
    };
    auto request = [&](auto id, uint32_t stage, int wanted) __attribute__((always_inline)) {  // the next step's; in order
        constexpr int ID = decltype(id)::value;
        // (uniform, which the compiler does not see in every form)
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds_base + stage);
        const int take = __builtin_amdgcn_readfirstlane(wanted);
        if constexpr (ID < A_REQUESTS) {
            if constexpr (HALF) request_half_tile(lane * 16, a_from[ID], to + (wave * A_REQUESTS + ID) * (kTileBytes / 2), take);
            else request_tile(lane * 16, a_from[ID], to + (wave * A_REQUESTS + ID) * kTileBytes, take);
            a_from[ID] += kTileBytes;
        } else {
            constexpr int B = ID - A_REQUESTS;
            request_tile(lane * 16, w_from[B], to + kW + (wave * W_REQUESTS + B) * kTileBytes, take);
            w_from[B] += step_bytes;
        }
    };

    // ---- operands: halves of a step, 64 bytes of K ----
    const uint32_t a_at = wave_m * ROWS * kTileBytes + lane * 16, w_at = kW + wave_n * CHANNELS * kTileBytes + lane * 16;
    // A half's operands are read while the half before is multiplied.  Rows, where there are many, into the registers whose last multiply has just been issued.
    constexpr int kHeldRows = ROWS > 4 ? 1 : 2;
    v4i fa[kHeldRows][ROWS], fw[2][CHANNELS];
    auto read_row = [&](auto half, auto i, uint32_t stage) __attribute__((always_inline)) {
        constexpr int H = decltype(half)::value, I = decltype(i)::value;
        fa[H % kHeldRows][I] = *reinterpret_cast<const v4i*>(lds + (a_at + stage) + (I * kTileBytes + H * 1024));
    };
    auto read_weight = [&](auto half, auto j, uint32_t stage) __attribute__((always_inline)) {
        constexpr int H = decltype(half)::value, J = decltype(j)::value;
        fw[H][J] = *reinterpret_cast<const v4i*>(lds + (w_at + stage) + (J * kTileBytes + H * 1024));
    };
    Sum sum[ROWS][CHANNELS];
    using Fresh = std::true_type;
    using Added = std::false_type;
    using H0 = std::integral_constant<int, 0>;
    using H1 = std::integral_constant<int, 1>;
    uint32_t stage = 0;
    int left = my_tiles * p.steps;  // steps, with this one
    auto next_stage_is_there = [&]() __attribute__((always_inline)) {
        if constexpr (STAGES == 2) everybody_arrived();
        else everybody_arrived_but<(STAGES - 2) * kLoads>(left - STAGES + 1);
        if (load_step == 0 && left > STAGES) request_scales();
    };
    // Half H of a step; behind every multiply stands at most a read or a request.  In the second half, once the first row's multiplies are on their way, the next stage is whole and nobody reads
    // this one any more.  FRESH: the first of a tile, whose sums are 0.
    auto half_step = [&](auto half, auto fresh, uint32_t next) __attribute__((always_inline)) {
        constexpr int H = decltype(half)::value;
        using Other = std::integral_constant<int, 1 - H>;
        Each<ROWS>::run([&](auto i) {
            constexpr int I = decltype(i)::value;
            Each<CHANNELS>::run([&](auto jj) {
                constexpr int JJ = decltype(jj)::value, J = I & 1 ? CHANNELS - 1 - JJ : JJ;  // one operand changes between neighbours
                sum[I][J] = multiply<I8>(fw[H][J], fa[H % kHeldRows][I], decltype(fresh)::value ? Sum{} : sum[I][J]);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (H == 1 && I == 0 && JJ == CHANNELS - 1) {
                    next_stage_is_there();
                    __builtin_amdgcn_sched_barrier(0);
                }
                // reads of weights and requests spread over the rows' multiplies
                constexpr int SKIPPED = H == 1 ? CHANNELS - 1 : 0, AT = I * CHANNELS + JJ - SKIPPED, COUNT = ROWS * CHANNELS - SKIPPED;
                if constexpr (AT >= 0) {
                    Each<CHANNELS>::run([&](auto w) {
                        if constexpr (decltype(w)::value * COUNT / (ROWS * CHANNELS) == AT) read_weight(Other{}, w, H == 0 ? stage : next);
                    });
                    if constexpr (H == 1)
                        Each<kAll>::run([&](auto q) {
                            if constexpr ((2 * decltype(q)::value + 1) * COUNT / (2 * kAll) == AT) request(q, stage, left - STAGES);
                        });
                }
                if constexpr (JJ == CHANNELS - 1) read_row(Other{}, i, H == 0 ? stage : next);
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        if constexpr (H == 1) advance();
    };

    // ---- results: block (i, j) has channels 4 piece .. of row r; pairs of blocks change rows of lanes, and a lane has eight neighbours ----
    constexpr int KINDS = SWIGLU ? 2 : 1, BLOCKS = CHANNELS / KINDS;  // of results
    const int r = lane & 15, piece = lane >> 4;
    auto store = [&](const Tile& t) __attribute__((always_inline)) {
        const int first_col = (t.group * (BN / 16) + wave_n * CHANNELS) / KINDS * 16;
        const uint8_t* const values = lds + kScales + scales;
        auto channel_of = [&](int block) {  // block of the weights
            Channels c = {};
            const uint8_t* const at = values + kChannels + ((wave_n * CHANNELS + block) * 16 + 4 * piece) * 4;
            c.scale = *reinterpret_cast<const v4f*>(at);
            if (p.w_sum != nullptr) c.sum = *reinterpret_cast<const v4i*>(at + 4 * BN);
            if (p.bias != nullptr) c.bias = *reinterpret_cast<const v4f*>(at + 8 * BN);
            return c;
        };
        const bool whole = first_col + BLOCKS * 16 <= p.cols;
        Each<BLOCKS / 2>::run([&](auto pair) {
            constexpr int J0 = 2 * decltype(pair)::value, J1 = J0 + 1;
            Channels channel[2 * KINDS];
#pragma unroll
            for (int b = 0; b < 2 * KINDS; ++b) channel[b] = channel_of(J0 * KINDS + b);
            Each<ROWS>::run([&](auto i) {
                constexpr int I = decltype(i)::value;
                const int local = (wave_m * ROWS + I) * 16 + r;
                const int64_t row_start = (int64_t)(t.first_row + local) * p.cols;
                RowScale row = {*reinterpret_cast<const float*>(values + 4 * local), 0};
                if (p.zero != nullptr) row.zero = *reinterpret_cast<const int*>(values + kZeros + 4 * local);
                v4f y[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    y[b] = scaled<I8, true>(sum[I][(J0 + b) * KINDS], channel[b * KINDS], row);
                    if constexpr (SWIGLU) {
                        const v4f up = scaled<I8, true>(sum[I][(J0 + b) * KINDS + KINDS - 1], channel[b * KINDS + KINDS - 1], row);
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[b][e] = mx::swiglu(y[b][e], up[e]);
                    }
                }
                if (WIDE || !whole) {
                    if (local < t.rows) {
                        mx::store_four(p.out, WIDE ? mx::F32 : p.type, row_start, first_col + J0 * 16 + 4 * piece, p.cols, y[0]);
                        mx::store_four(p.out, WIDE ? mx::F32 : p.type, row_start, first_col + J1 * 16 + 4 * piece, p.cols, y[1]);
                    }
                } else {
                    uint32_t a[2], b[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (p.type == mx::F16) a[e] = mx::two_values(y[0][2 * e], y[0][2 * e + 1], mx::F16), b[e] = mx::two_values(y[1][2 * e], y[1][2 * e + 1], mx::F16);
                        else a[e] = mx::two_values(y[0][2 * e], y[0][2 * e + 1], mx::BF16), b[e] = mx::two_values(y[1][2 * e], y[1][2 * e + 1], mx::BF16);
                    }
                    // lanes of an even `piece` get eight channels of the first block, of an odd one of the second
                    auto low = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
                    auto high = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
                    const int col = first_col + (J0 + (piece & 1)) * 16 + (piece >> 1) * 8;
                    if (local < t.rows) *reinterpret_cast<mx::words4*>(reinterpret_cast<unsigned short*>(p.out) + row_start + col) = v4u{low[0], high[0], low[1], high[1]};
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        });
    };

    aim();
#pragma unroll 1
    for (int s = 0; s < STAGES; ++s) {
        if (load_step == 0 && left > s) request_scales();
        Each<kAll>::run([&](auto q) { request(q, s * kStage, left - s); });
        advance();
    }
    if constexpr (STAGES == 2) everybody_arrived_but<kLoads>(left - 1);
    else everybody_arrived_but<(STAGES - 1) * kLoads>(left - STAGES + 1);
    Each<ROWS>::run([&](auto i) { read_row(H0{}, i, 0); });
    Each<CHANNELS>::run([&](auto j) { read_weight(H0{}, j, 0); });
    // One sequence of steps over all tiles: the next tile's first steps are on their way while this one's last are multiplied.  (The last step of all reads a stage that nobody filled.)
    auto one_step = [&](auto fresh) __attribute__((always_inline)) {
        const uint32_t next = stage == (STAGES - 1) * kStage ? 0 : stage + kStage;
        half_step(H0{}, fresh, next);
        half_step(H1{}, Added{}, next);
        stage = next;
        --left;
    };
#pragma unroll 1
    for (int tile = 0; tile < my_tiles; ++tile) {
        one_step(Fresh{});
#pragma unroll 1
        for (int step = 1; step < p.steps; ++step) one_step(Added{});
        store(tile_of(tile));
        turn(scales);
    }
}

template <typename FORM, bool WIDE, bool SWIGLU>
int launch_one(const Product& p, uint32_t blocks, hipStream_t s) {
    constexpr auto kernel = &byte_tiles_kernel<FORM, WIDE, SWIGLU>;
    static DeviceOnce ready;
    const int code = ready.run([] { return hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, FORM::lds), "hipFuncSetAttribute"); });
    if (code != ORX_OK) return code;
    ORX_LAUNCH(kernel, dim3(blocks), dim3(64 * FORM::waves), FORM::lds, s, p);
    return hip_check(hipGetLastError(), "launch byte tiles");
}
template <typename BODY>
auto with_form(int form, BODY body) {
    switch (form) {
        case kTiles256: return body(Form<8, 4, 2, 4, 2>{});
        case kTiles128: return body(Form<2, 4, 4, 2, 4>{});
        case kTiles96: return body(Form<3, 4, 2, 2, 5>{});
        case kTiles64: return body(Form<2, 4, 2, 2, 6>{});
        default: return body(Form<1, 4, 4, 1, 4>{});
    }
}

}  // namespace

int launch_byte_tiles_i8(const Product& p, int form, bool swiglu, uint32_t blocks, hipStream_t s) {
    return with_form(form, [&](auto which) {
        using FORM = decltype(which);
        if (p.type == mx::F32) return swiglu ? launch_one<FORM, true, true>(p, blocks, s) : launch_one<FORM, true, false>(p, blocks, s);
        return swiglu ? launch_one<FORM, false, true>(p, blocks, s) : launch_one<FORM, false, false>(p, blocks, s);
    });
}
TilesShape byte_tiles_shape(int kind, int form, bool grouped) {
    if (form == kWide128 || form == kWide64) {
        auto shape = [](auto wide) {
            using WIDE = decltype(wide);
            return TilesShape{WIDE::bm, WIDE::bn, 64 * WIDE::waves, WIDE::lds, WIDE::to_a_cu};
        };
        if (kind != I8) return form == kWide128 ? shape(Wide<F16, 8, true>{}) : shape(Wide<F16, 4, true>{});
        if (!grouped) return shape(Wide<I8, 8, false>{});
        return form == kWide128 ? shape(Wide<I8, 8, true>{}) : shape(Wide<I8, 4, true>{});
    }
    return with_form(form, [&](auto which) {
        using FORM = decltype(which);
        return TilesShape{FORM::bm, FORM::bn, 64 * FORM::waves, FORM::lds, 160 * 1024 / FORM::lds};
    });
}

}  // namespace orx
