// Products of many rows with weights by byte tiles, dense and routed experts: tiles of the output from LDS.
//
// DOWN x ACROSS waves share a tile, each ROWS x CHANNELS blocks of 16 x 16 of it; K goes in steps of 128 bytes.  Rows and weights come from memory to LDS without passing a register, two
// or three stages.  Weights and dense rows arrive as they are laid out, a kilobyte to a request; of an expert's row, which lies anywhere, the 128 bytes of a step keep their 16-byte piece p at p ^ ((row >> 1) & 7), so that the
// sixteen rows of a read meet different banks.  A workgroup goes through its tiles as one sequence of steps: the next tile's first steps are on their way while the last ones are multiplied, and
// results drain under the next multiplies.
#pragma once
#include "byte_tiles.h"
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
    static constexpr int rows = ROWS, channels = CHANNELS, down = DOWN, across = ACROSS, stages = STAGES;
    static constexpr int bm = 16 * ROWS * DOWN, bn = 16 * CHANNELS * ACROSS, waves = DOWN * ACROSS;
    static constexpr int stage = (bm + bn) * kStep;
    // what a tile's rows and channels have, for the results: scales, and of dense rows zero points, sums and biases; of the tile that is multiplied and of as many as there are stages
    template <bool GROUPED>
    static constexpr int scales() { return 4 * (GROUPED ? bm + bn : 2 * bm + 3 * bn); }
    template <int KIND, bool GROUPED>
    static constexpr int lds() { return STAGES * stage + (KIND == I8 ? (STAGES + 1) * scales<GROUPED>() : 0) + (GROUPED ? 2 * 4 * bm : 0); }
};

template <int KIND, typename FORM, bool WIDE, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(64 * FORM::waves, 2) void byte_tiles_kernel(Product p) {
    using Sum = typename Operands<KIND>::Sum;
    constexpr int ROWS = FORM::rows, CHANNELS = FORM::channels, DOWN = FORM::down, WAVES = FORM::waves, STAGES = FORM::stages, BM = FORM::bm, BN = FORM::bn;
    constexpr bool TILED = !GROUPED;  // the rows' layout
    constexpr int A_REQUESTS = BM / (TILED ? 16 : 8) / WAVES, W_REQUESTS = BN / 16 / WAVES;  // of a wave and step: a tile of rows or eight rows, a tile
    constexpr int kAll = A_REQUESTS + W_REQUESTS, kLoads = (TILED ? 2 : 1) * A_REQUESTS + 2 * W_REQUESTS;
    constexpr int kW = BM * kStep, kStage = FORM::stage;
    constexpr int kScales = STAGES * kStage, kScaleBytes = FORM::template scales<GROUPED>(), kTokens = kScales + (KIND == I8 ? (STAGES + 1) * kScaleBytes : 0);
    constexpr int kZeros = 4 * BM, kChannels = GROUPED ? 4 * BM : 8 * BM;  // of a tile's scales
    extern __shared__ __align__(128) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wave_m = wave % DOWN, wave_n = wave / DOWN;

    // ---- which results: tiles blockIdx.x, blockIdx.x + gridDim.x, .. of an order in which every XCD has one run ----
    const int groups = (p.tiles + BN / 16 - 1) / (BN / 16);
    const int row_tiles = GROUPED ? min(__builtin_amdgcn_readfirstlane(*p.unit_count), p.most_units) : (p.m + BM - 1) / BM;
    const int total = row_tiles * groups;
    const int my_tiles = __builtin_amdgcn_readfirstlane((total - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x);
    if (my_tiles <= 0) return;
    struct Tile {
        int first_row, rows, group, expert;
    };
    // (units through the scalar cache: a vector load would be waited for behind all requests)
    typedef int int4v __attribute__((ext_vector_type(4)));
    const auto units = reinterpret_cast<const __attribute__((address_space(4))) int4v*>(reinterpret_cast<uint64_t>(p.units));
    auto tile_of = [&](int number) __attribute__((always_inline)) {
        const int at = (int)blockIdx.x + number * (int)gridDim.x, xcd = at & 7;
        const int id = xcd * (total >> 3) + min(xcd, total & 7) + (at >> 3);
        Tile t;
        if (GROUPED) {
            const int4v u = units[__builtin_amdgcn_readfirstlane(id / groups)];
            t.group = id % groups, t.first_row = __builtin_amdgcn_readfirstlane(u[1]), t.rows = __builtin_amdgcn_readfirstlane(u[2]), t.expert = __builtin_amdgcn_readfirstlane(u[0]);
        } else {
            // eight tiles of rows for each tile of channels, so that an L2 holds what neighbours share
            const int band = id / (8 * groups), in_band = min(8, row_tiles - 8 * band), within = id % (8 * groups);
            t.first_row = (8 * band + within % in_band) * BM, t.group = within / in_band;
            t.rows = min(BM, p.m - t.first_row), t.expert = 0;
        }
        return t;
    };
    const uint32_t lds_base = lds_asm::lds_address_of(lds);
    const bool gather = GROUPED && p.slot_token != nullptr;
    // Rows that are not there repeat the last: their sums go nowhere.
    auto slot_of = [&](const Tile& t, int local) __attribute__((always_inline)) { return max(t.first_row + min(local, t.rows - 1), 0); };
    // A tile's tokens come to LDS while the tile in front of it is requested (a load would be waited for behind all requests).
    auto row_of = [&](const Tile& t, int local, int number) __attribute__((always_inline)) -> int64_t {
        return gather ? *reinterpret_cast<const int*>(lds + kTokens + (number & 1) * (4 * BM) + 4 * local) : slot_of(t, local);
    };
    auto request_tokens = [&](int number) __attribute__((always_inline)) {
        if (!gather || number >= my_tiles) return;
        const Tile t = tile_of(number);
#pragma unroll
        for (int c = 0; c < (BM / 64 + WAVES - 1) / WAVES; ++c) {
            const int chunk = wave + c * WAVES;
            request_4_from(reinterpret_cast<const uint8_t*>(p.slot_token + slot_of(t, chunk * 64 + lane)), __builtin_amdgcn_readfirstlane(lds_base + kTokens + (number & 1) * (4 * BM) + chunk * 256), __builtin_amdgcn_readfirstlane(BM / 64 - chunk));
        }
    };

    // ---- requests ----
    const uint8_t* a_from[A_REQUESTS];  // a tile, or this lane's piece of eight rows
    const uint8_t* w_from[W_REQUESTS];  // a tile
    auto piece_of = [&](int b) __attribute__((always_inline)) { return (lane & 7) ^ ((((wave * A_REQUESTS + b) * 8 + (lane >> 3)) >> 1) & 7); };
    // 16-bit rows may end within a step: the pieces behind come from the weights' padding, which is 0
    const int last_pieces = KIND == I8 ? 0 : (p.row_bytes % kStep) / 16, partial_step = last_pieces ? p.steps - 1 : -1;
    const int64_t step_bytes = (int64_t)p.tiles * kTileBytes;  // of the weights of one expert
    const uint8_t* const zeros = p.w + (p.steps - 1) * step_bytes + last_pieces * 256;
    int load_tile = 0, load_step = 0, load_scales = 0, scales = 0;  // the tile and step whose requests come next, and where its scales and those of the tile that is multiplied lie
    auto turn = [&](int& at) __attribute__((always_inline)) { at = at == STAGES * kScaleBytes ? 0 : at + kScaleBytes; };
    Tile load_at;
    auto aim = [&]() __attribute__((always_inline)) {
        load_at = tile_of(load_tile);
        const Tile& t = load_at;
#pragma unroll
        for (int b = 0; b < A_REQUESTS; ++b) {
            if constexpr (TILED) a_from[b] = uniform_pointer(p.a + (int64_t)min(t.first_row / 16 + wave * A_REQUESTS + b, (p.m - 1) / 16) * p.steps * kTileBytes);
            else a_from[b] = p.a + row_of(t, (wave * A_REQUESTS + b) * 8 + (lane >> 3), load_tile) * p.pitch + piece_of(b) * 16;
        }
        const int64_t expert = (int64_t)t.expert * p.steps * p.tiles;
#pragma unroll
        for (int b = 0; b < W_REQUESTS; ++b) w_from[b] = uniform_pointer(p.w + (expert + min(t.group * (BN / 16) + wave * W_REQUESTS + b, p.tiles - 1)) * kTileBytes);
        request_tokens(load_tile + 1);
    };
    auto request_scales = [&]() __attribute__((always_inline)) {  // in front of a tile's first step
        const Tile& t = load_at;
        if constexpr (KIND == I8) {
            constexpr int R = BM / 64, C = BN / 64, CHUNKS = GROUPED ? R + C : 2 * R + 3 * C;
            const uint32_t to = __builtin_amdgcn_readfirstlane(lds_base + kScales + load_scales);
#pragma unroll
            for (int c = 0; c < (CHUNKS + WAVES - 1) / WAVES; ++c) {
                const int chunk = wave + c * WAVES;  // (uniform)
                const bool of_rows = chunk < (GROUPED ? R : 2 * R);
                const int64_t row = row_of(t, chunk % R * 64 + lane, load_tile);
                const int64_t channel = (int64_t)t.expert * p.tiles * 16 + min((t.group * C + (chunk - (GROUPED ? R : 2 * R)) % C) * 64 + lane, p.tiles * 16 - 1);
                const int kind = GROUPED ? (of_rows ? 0 : 2) : of_rows ? chunk / R : 2 + (chunk - 2 * R) / C;
                const uint8_t* const base = reinterpret_cast<const uint8_t*>(kind == 0 ? (const void*)p.scale : kind == 1 ? (const void*)p.zero : kind == 2 ? (const void*)p.w_scale : kind == 3 ? (const void*)p.w_sum : (const void*)p.bias);
                request_4_from(base + (of_rows ? row : channel) * 4, to + chunk * 256, __builtin_amdgcn_readfirstlane(base == nullptr ? 0 : CHUNKS - chunk));
            }
            turn(load_scales);
        }
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
        if constexpr (ID < A_REQUESTS && TILED) {
            request_tile(lane * 16, a_from[ID], to + (wave * A_REQUESTS + ID) * kTileBytes, take);
            a_from[ID] += kTileBytes;
        } else if constexpr (ID < A_REQUESTS) {
            const uint8_t* from = a_from[ID];
            if constexpr (KIND != I8) from = load_step == partial_step && piece_of(ID) >= last_pieces ? zeros : from;
            request_16_from(from, to + (wave * A_REQUESTS + ID) * 1024, take);
            a_from[ID] += kStep;
        } else {
            constexpr int B = ID - A_REQUESTS;
            request_tile(lane * 16, w_from[B], to + kW + (wave * W_REQUESTS + B) * kTileBytes, take);
            w_from[B] += step_bytes;
        }
    };

    // ---- operands: halves of a step, 64 bytes of K ----
    const int r = lane & 15, piece = lane >> 4;  // row or channel of a block; pieces `piece` and 4 behind of a step
    const uint32_t a_at = TILED ? wave_m * ROWS * kTileBytes + lane * 16 : (wave_m * 16 * ROWS + r) * kStep + (piece ^ ((r >> 1) & 7)) * 16;
    const uint32_t w_at = kW + wave_n * CHANNELS * kTileBytes + lane * 16;
    // A half's operands are read while the half before is multiplied.  Rows, where there are many, into the registers whose last multiply has just been issued.
    constexpr int kHeldRows = ROWS > 4 ? 1 : 2;
    v4i fa[kHeldRows][ROWS], fw[2][CHANNELS];
    auto read_row = [&](auto half, auto i, uint32_t stage) __attribute__((always_inline)) {
        constexpr int H = decltype(half)::value, I = decltype(i)::value;
        fa[H % kHeldRows][I] = *reinterpret_cast<const v4i*>(lds + ((TILED ? a_at : a_at ^ (H * 64)) + stage) + I * (16 * kStep) + (TILED ? H * 1024 : 0));
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
    const int patient = gather && p.steps == 1 ? left : STAGES - 1;  // (tokens are requested behind a tile's last step, and a tile of one step reads them behind the next one's requests)
    auto next_stage_is_there = [&]() __attribute__((always_inline)) {
        if constexpr (STAGES == 2) everybody_arrived();
        else everybody_arrived_but<(STAGES - 2) * kLoads>(left - patient);
        if (KIND == I8 && load_step == 0 && left > STAGES) request_scales();
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
                sum[I][J] = multiply<KIND>(fw[H][J], fa[H % kHeldRows][I], decltype(fresh)::value ? Sum{} : sum[I][J]);
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
    auto store = [&](const Tile& t) __attribute__((always_inline)) {
        const int first_col = (t.group * (BN / 16) + wave_n * CHANNELS) / KINDS * 16;
        const uint8_t* const values = lds + kScales + scales;
        auto channel_of = [&](int block) {  // block of the weights
            Channels c = {};
            if constexpr (KIND == I8) {
                const uint8_t* const at = values + kChannels + ((wave_n * CHANNELS + block) * 16 + 4 * piece) * 4;
                c.scale = *reinterpret_cast<const v4f*>(at);
                if (!GROUPED && p.w_sum != nullptr) c.sum = *reinterpret_cast<const v4i*>(at + 4 * BN);
                if (!GROUPED && p.bias != nullptr) c.bias = *reinterpret_cast<const v4f*>(at + 8 * BN);
            }
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
                RowScale row = {};
                if constexpr (KIND == I8) {
                    row.scale = *reinterpret_cast<const float*>(values + 4 * local);
                    if (!GROUPED && p.zero != nullptr) row.zero = *reinterpret_cast<const int*>(values + kZeros + 4 * local);
                }
                v4f y[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    y[b] = scaled<KIND, !GROUPED>(sum[I][(J0 + b) * KINDS], channel[b * KINDS], row);
                    if constexpr (SWIGLU) {
                        const v4f up = scaled<KIND, !GROUPED>(sum[I][(J0 + b) * KINDS + KINDS - 1], channel[b * KINDS + KINDS - 1], row);
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

    if (gather) {
        request_tokens(0);
        everybody_arrived();
    }
    aim();
#pragma unroll 1
    for (int s = 0; s < STAGES; ++s) {
        if (KIND == I8 && load_step == 0 && left > s) request_scales();
        Each<kAll>::run([&](auto q) { request(q, s * kStage, left - s); });
        if (gather && p.steps <= STAGES) everybody_arrived();  // (the next tile's tokens)
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
        if constexpr (KIND == I8) turn(scales);
    }
}

template <int KIND, typename FORM, bool WIDE, bool GROUPED, bool SWIGLU>
int launch_one(const Product& p, uint32_t blocks, hipStream_t s) {
    constexpr uint32_t kLds = FORM::template lds<KIND, GROUPED>();
    static_assert(kLds <= 160 * 1024, "a CU's LDS");
    constexpr auto kernel = &byte_tiles_kernel<KIND, FORM, WIDE, GROUPED, SWIGLU>;
    static DeviceOnce ready;
    const int code = ready.run([] { return hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds), "hipFuncSetAttribute"); });
    if (code != ORX_OK) return code;
    ORX_LAUNCH(kernel, dim3(blocks), dim3(64 * FORM::waves), kLds, s, p);
    return hip_check(hipGetLastError(), "launch byte tiles");
}
template <int KIND, bool GROUPED>
struct Launch {
    template <typename FORM>
    int operator()(FORM, const Product& p, bool swiglu, uint32_t blocks, hipStream_t s) const {
        if (p.type == mx::F32) return swiglu ? launch_one<KIND, FORM, true, GROUPED, true>(p, blocks, s) : launch_one<KIND, FORM, true, GROUPED, false>(p, blocks, s);
        return swiglu ? launch_one<KIND, FORM, false, GROUPED, true>(p, blocks, s) : launch_one<KIND, FORM, false, GROUPED, false>(p, blocks, s);
    }
};
// The forms by their numbers (byte_tiles.h).
template <typename BODY>
int with_form(int form, BODY body) {
    switch (form) {
        case kTiles256: return body(Form<8, 4, 2, 4, 2>{});
        case kTiles128x256: return body(Form<4, 4, 2, 4, 3>{});
        case kTiles128: return body(Form<4, 4, 2, 2, 2>{});
        default: return body(Form<2, 4, 2, 2, 2>{});
    }
}

}  // namespace
}  // namespace orx
