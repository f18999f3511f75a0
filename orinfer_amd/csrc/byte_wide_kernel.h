// Products of many rows with weights by byte tiles, dense and routed experts: rows through LDS, weights straight into registers.
//
// A workgroup of four waves takes 128 rows x 256 channels (units of 64 rows: two waves, 128 channels, four workgroups to a CU, which even out better: 16 experts of 4096 x 1536 in fp16, 400 routes, 49
// -> 44 us), each wave all of these rows and 64 of the channels; K goes in steps of 128 bytes.  Waves that share rows and channels both read
// more from LDS than it gives: with 64 x 64 results to a wave a step's reads and writes take 1.4 times its multiplies (128 x 256 results to eight waves, all operands through LDS, three
// stages: 0.84 us a step where the multiplies are 0.43).  Here a wave's weights are its own, so they pass no LDS: four half-steps of them are held or on their way in registers, whole kilobytes a
// load.  Rows come from memory to LDS without passing a register, four stages; a step's LDS traffic is 0.6 of the multiplies' time, the L1's 0.75.  Two workgroups share a CU: one multiplies
// while the other waits or stores.  Of a row of experts, which lies anywhere, the 128 bytes of a step keep their 16-byte piece p at p ^ ((row >> 1) & 7), so that the sixteen rows of a read
// meet different banks; dense rows arrive by tiles.  A workgroup goes through its tiles as one sequence of steps: the next tile's first steps are on their way while the last ones are multiplied.
// us of 128 experts, 32768 routes: gate | up 1024 x 2048 98-105 int8, 185-206 in bf16, down 2048 x 512 98-106 and 140-148.  Bound by memory at 4.6 to 5.1 TB/s, a large copy's 5.1: they read 463 and 919
// MB and 238 and 482 beside 268 of fp32 results, of which an expert's weights come about one and a half times (the list has its short last unit far from its full ones, and at the ends of runs two
// XCDs share an expert); the pipe is busy in 0.38 and 0.42, 0.18 and 0.26 of the cycles.
// The int8 form of 128 rows with a gather and SwiGLU to 16 bits leaves 32 bytes to scratch (of request_tokens, read again where a tile is aimed at), to fp32 8; the dense ones with SwiGLU 44 and 108, around
// the results (1024 and 2048 rows of 17408 x 5120: 99 and 173 us, without SwiGLU 95 and 177).
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

template <int KIND, int ROWS, bool GROUPED>
struct Wide {
    static constexpr int waves = ROWS <= 4 ? 2 : 4, to_a_cu = ROWS <= 4 ? 4 : 2, stages = 4, channels = 4, bm = 16 * ROWS, bn = 16 * channels * waves, stage = bm * kStep;
    // what a tile's rows and channels have, for the results: scales, and of dense rows zero points, sums and biases; of the tile that is multiplied and of two more
    static constexpr int scale_bytes = 4 * (GROUPED ? bm + bn : 2 * bm + 3 * bn), ring = KIND == I8 ? 3 * scale_bytes : 0;
    static constexpr int tokens = GROUPED ? 2 * 4 * bm : 0;
    static constexpr int lds = stages * stage + ring + tokens;
    static_assert(to_a_cu * lds <= 160 * 1024 && to_a_cu * waves == 8, "a CU's LDS, two waves to a SIMD");
};

template <int KIND, int ROWS, bool WIDE, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(ROWS <= 4 ? 128 : 256, 2) void byte_wide_kernel(Product p) {
    using Sum = typename Operands<KIND>::Sum;
    using FORM = Wide<KIND, ROWS, GROUPED>;
    constexpr int WAVES = FORM::waves, CHANNELS = FORM::channels, BM = FORM::bm, BN = FORM::bn, kStage = FORM::stage, kStages = FORM::stages * kStage;
    constexpr bool TILED = !GROUPED;  // the rows' layout
    constexpr int A_REQUESTS = BM / (TILED ? 16 : 8) / WAVES;  // of a wave and step: a tile of rows, or eight rows
    constexpr int kScaleBytes = FORM::scale_bytes, kTokens = kStages + FORM::ring;
    constexpr int kZeros = 4 * BM, kChannels = GROUPED ? 4 * BM : 8 * BM;  // of a tile's scales
    extern __shared__ __align__(128) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);

    // ---- which results: tiles blockIdx.x, blockIdx.x + gridDim.x, .. of an order in which every XCD has p.runs runs (and one of the last few tiles) ----
    const int groups = (p.tiles + BN / 16 - 1) / (BN / 16);
    const int row_tiles = GROUPED ? min(__builtin_amdgcn_readfirstlane(*p.unit_count), p.most_units) : (p.m + BM - 1) / BM;
    const int total = row_tiles * groups;
    const int of_xcd = total >> 3, run = (of_xcd + p.runs - 1) / p.runs;
    const int my_tiles = __builtin_amdgcn_readfirstlane((total - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x);
    if (my_tiles <= 0) return;
    struct Tile {
        int first_row, rows, group, expert;
    };
    // (units through the scalar cache: a vector load would be waited for behind all requests)
    typedef int int4v __attribute__((ext_vector_type(4)));
    const auto units = reinterpret_cast<const __attribute__((address_space(4))) int4v*>(reinterpret_cast<uint64_t>(p.units));
    auto tile_of = [&](int number) __attribute__((always_inline)) {
        const int at = (int)blockIdx.x + number * (int)gridDim.x, xcd = at & 7, nth = at >> 3;
        const int before = run == 0 ? 0 : nth / run * run;  // tiles of this XCD in earlier runs
        const int id = nth < of_xcd ? before * 8 + xcd * min(run, of_xcd - before) + nth - before : at;
        Tile t;
        if (GROUPED) {
            const int4v u = units[__builtin_amdgcn_readfirstlane(id / groups)];
            t.group = __builtin_amdgcn_readfirstlane(id % groups), t.first_row = __builtin_amdgcn_readfirstlane(u[1]), t.rows = __builtin_amdgcn_readfirstlane(u[2]);
            t.expert = __builtin_amdgcn_readfirstlane(u[0]);
        } else {
            // eight tiles of rows for each tile of channels, so that an L2 holds what neighbours share
            const int band = id / (8 * groups), in_band = min(8, row_tiles - 8 * band), within = id % (8 * groups);
            t.first_row = __builtin_amdgcn_readfirstlane((8 * band + within % in_band) * BM), t.group = __builtin_amdgcn_readfirstlane(within / in_band);
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
        request_4_from(reinterpret_cast<const uint8_t*>(p.slot_token + slot_of(t, wave * 64 + lane)), __builtin_amdgcn_readfirstlane(lds_base + kTokens + (number & 1) * (4 * BM) + wave * 256),
                       __builtin_amdgcn_readfirstlane(BM / 64 - wave));
    };

    // ---- requests of rows ----
    const uint8_t* a_from[A_REQUESTS];  // a tile, or this lane's piece of eight rows
    auto piece_of = [&](int b) __attribute__((always_inline)) { return (lane & 7) ^ ((((wave * A_REQUESTS + b) * 8 + (lane >> 3)) >> 1) & 7); };
    // 16-bit rows may end in front of the last step's end: the pieces behind come from the weights' padding, which is 0
    const int64_t step_bytes = (int64_t)p.tiles * kTileBytes;  // of the weights of one expert
    const uint8_t* const zeros = p.w + (p.steps - 1) * step_bytes + 7 * 256;
    int load_tile = 0, load_step = 0, load_scales = 0, scales = 0;  // the tile and step whose requests come next, and where its scales and those of the tile that is multiplied lie
    auto turn = [&](int& at) __attribute__((always_inline)) { at = at == 2 * kScaleBytes ? 0 : at + kScaleBytes; };
    Tile load_at;
    auto aim = [&]() __attribute__((always_inline)) {
        load_at = tile_of(load_tile);
#pragma unroll
        for (int b = 0; b < A_REQUESTS; ++b) {
            if constexpr (TILED) a_from[b] = uniform_pointer(p.a + (int64_t)min(load_at.first_row / 16 + wave * A_REQUESTS + b, (p.m - 1) / 16) * p.steps * kTileBytes);
            else a_from[b] = p.a + row_of(load_at, (wave * A_REQUESTS + b) * 8 + (lane >> 3), load_tile) * p.pitch + piece_of(b) * 16;
        }
        request_tokens(load_tile + 1);
    };
    auto request_scales = [&]() __attribute__((always_inline)) {  // in front of a tile's first step
        if constexpr (KIND == I8) {
            constexpr int R = BM / 64, C = BN / 64, CHUNKS = GROUPED ? R + C : 2 * R + 3 * C;
            const uint32_t to = __builtin_amdgcn_readfirstlane(lds_base + kStages + load_scales);
#pragma unroll
            for (int c = 0; c < (CHUNKS + WAVES - 1) / WAVES; ++c) {
                const int chunk = wave + c * WAVES;  // (uniform)
                const bool of_rows = chunk < (GROUPED ? R : 2 * R);
                const int64_t row = row_of(load_at, chunk % R * 64 + lane, load_tile);
                const int64_t channel = (int64_t)load_at.expert * p.tiles * 16 + min((load_at.group * C + (chunk - (GROUPED ? R : 2 * R)) % C) * 64 + lane, p.tiles * 16 - 1);
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
        if constexpr (TILED) {
            request_tile(lane * 16, a_from[ID], to + (wave * A_REQUESTS + ID) * kTileBytes, take);
            a_from[ID] += kTileBytes;
        } else {
            const uint8_t* from = a_from[ID];
            if constexpr (KIND != I8) from = load_step * kStep + piece_of(ID) * 16 >= p.row_bytes ? zeros : from;
            request_16_from(from, to + (wave * A_REQUESTS + ID) * 1024, take);
            a_from[ID] += kStep;
        }
    };

    // ---- weights: half-steps of 64 bytes of K, three ahead of the one that is multiplied ----
    struct Weights {
        const uint8_t* base;  // of the tile's expert
        uint32_t offset;      // of this wave's channels in a step
    };
    int w_tile = 0, w_step = 0;
    uint32_t w_first = 0;
    const uint32_t expert_bytes = (uint32_t)(step_bytes * p.steps);  // (the host gives no more to this kernel)
    const uint8_t* w_base = p.w;
    auto weights_of = [&]() __attribute__((always_inline)) {  // of the step that comes next (behind the last tile its first steps once more, which nobody multiplies)
        if (w_step == 0 && w_tile < my_tiles) {
            const Tile t = tile_of(w_tile);
            const int first = t.group * (BN / 16) + wave * CHANNELS;  // (there are whole fours of tiles; a wave without channels takes the first ones)
            w_base = uniform_pointer(p.w + (int64_t)t.expert * p.steps * step_bytes);
            w_first = __builtin_amdgcn_readfirstlane((uint32_t)(first < p.tiles ? first : 0) * kTileBytes);
        }
        const Weights w = {w_base, w_first + (uint32_t)w_step * (uint32_t)step_bytes};
        if (++w_step == p.steps) w_step = 0, ++w_tile;
        return w;
    };
    v4i fw[4][CHANNELS];
    const int w_lane = lane * 16;
    auto load_weight = [&](auto slot, auto half, auto j, const Weights& from) __attribute__((always_inline)) {
        constexpr int SLOT = decltype(slot)::value, H = decltype(half)::value, J = decltype(j)::value;
        const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(from.base), 0, expert_bytes, 0x00027000);
        fw[SLOT][J] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(buffer, w_lane + (J % 2 * kTileBytes + H * 1024), from.offset + J / 2 * (2 * kTileBytes), 0));
    };

    // ---- rows' operands: four blocks of 16 rows ahead ----
    const int r = lane & 15, piece = lane >> 4;  // row or channel of a block; pieces `piece` and 4 behind of a step
    const uint32_t a_at = TILED ? lane * 16 : r * kStep + (piece ^ ((r >> 1) & 7)) * 16;
    v4i fa[4];
    auto read_row = [&](auto half, auto i, uint32_t stage) __attribute__((always_inline)) {
        constexpr int H = decltype(half)::value, I = decltype(i)::value;
        fa[I % 4] = *reinterpret_cast<const v4i*>(lds + ((TILED ? a_at : a_at ^ (H * 64)) + stage) + I * (16 * kStep) + (TILED ? H * 1024 : 0));
    };
    Sum sum[ROWS][CHANNELS];
    using N0 = std::integral_constant<int, 0>;
    using N1 = std::integral_constant<int, 1>;
    using N2 = std::integral_constant<int, 2>;
    uint32_t stage = 0;
    int left = my_tiles * p.steps;  // steps, with this one
    bool is_short = false;          // the tile's rows are at most 64
    Weights next_w, after_w;        // of the next step and of the one behind it
    // Half H of a step of parity PARITY; behind every multiply stands at most a read, a load or a request.  In the second half, once the first row's multiplies are on
    // their way, the next step's rows are there, and nobody reads the last step's any more.  (Of the requests and loads of a wave at least sixteen are newer than those rows' requests, which
    // were made two steps before: the loads of weights of four half-steps.)
    auto half_step = [&](auto parity, auto half) __attribute__((always_inline)) {
        constexpr int H = decltype(half)::value, SLOT = 2 * decltype(parity)::value + H;
        using Other = std::integral_constant<int, 1 - H>;
        using Refilled = std::integral_constant<int, (SLOT + 3) % 4>;
        const uint32_t next = (stage + kStage) & (kStages - 1);
        // Rows behind a short tile's 64 are not multiplied: the first four blocks' registers then get the next half's rows.
        constexpr int FULL = ROWS == 8 && GROUPED ? 4 : ROWS;
        const uint32_t behind = FULL == ROWS ? 0 : (a_at ^ ((is_short ? 1 - H : H) * 64)) + (is_short ? (H == 0 ? stage : next) : stage + FULL * 16 * kStep);
        auto one_row = [&](auto i) __attribute__((always_inline)) {
            constexpr int I = decltype(i)::value;
            Each<CHANNELS>::run([&](auto jj) {
                constexpr int JJ = decltype(jj)::value, J = I & 1 ? CHANNELS - 1 - JJ : JJ;  // one operand changes between neighbours
                multiply_in_place<KIND>(sum[I][J], fw[SLOT][J], fa[I % 4]);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (H == 1 && I == 0 && JJ == CHANNELS - 1) {
                    everybody_arrived_but<16>(1);
                    if (KIND == I8 && load_step == 0 && left > 3) request_scales();
                    __builtin_amdgcn_sched_barrier(0);
                }
                // Loads of weights behind the first row's second multiply and later ones; requests behind the barrier, and in front of the loads: the compiler does not count them where it waits for
                // weights, so a wait is for as many loads more (the other way round, of older loads: half of their time on the way).
                constexpr int AT = I * CHANNELS + JJ, FIRST = H == 1 ? CHANNELS : 1, EVERY = (FULL * CHANNELS - FIRST) / (H == 1 ? CHANNELS + A_REQUESTS : CHANNELS);
                if constexpr (AT >= FIRST && (AT - FIRST) % EVERY == 0) {
                    constexpr int Q = (AT - FIRST) / EVERY;
                    constexpr int W = H == 1 ? Q - A_REQUESTS : Q;
                    if constexpr (H == 1 && Q < A_REQUESTS) request(std::integral_constant<int, Q>{}, (stage + 3 * kStage) & (kStages - 1), left - 3);
                    else if constexpr (W < CHANNELS) load_weight(Refilled{}, Other{}, std::integral_constant<int, W>{}, H == 0 ? next_w : after_w);
                }
                if constexpr (JJ == CHANNELS - 1) {
                    if constexpr (FULL < ROWS && I < FULL) fa[I] = *reinterpret_cast<const v4i*>(lds + behind + I * (16 * kStep));
                    else if constexpr (I + 4 < ROWS) read_row(half, std::integral_constant<int, I + 4>{}, stage);
                    else read_row(Other{}, std::integral_constant<int, I + 4 - ROWS>{}, H == 0 ? stage : next);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        Each<FULL>::run([&](auto i) { one_row(i); });
        if constexpr (FULL < ROWS)
            if (!is_short) Each<ROWS - FULL>::run([&](auto i) { one_row(std::integral_constant<int, FULL + decltype(i)::value>{}); });
    };

    // ---- results: block (i, j) has channels 4 piece .. of row r; pairs of blocks change rows of lanes, and a lane has eight neighbours ----
    constexpr int KINDS = SWIGLU ? 2 : 1, BLOCKS = CHANNELS / KINDS;  // of results
    auto store = [&](const Tile& t) __attribute__((always_inline)) {
        int own = threadIdx.x & 63;
        asm volatile("" : "+v"(own));  // (opaque: or the addresses of all results are made in front of the loop and held through it)
        const int r = own & 15, piece = own >> 4;
        const int first_col = (t.group * (BN / 16) + wave * CHANNELS) / KINDS * 16;
        const uint8_t* const values = lds + kStages + scales;
        auto channel_of = [&](int block) __attribute__((always_inline)) {  // block of the weights
            Channels c = {};
            if constexpr (KIND == I8) {
                const uint8_t* const at = values + kChannels + ((wave * CHANNELS + block) * 16 + 4 * piece) * 4;
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
                if (I * 16 >= t.rows) return;
                const int local = I * 16 + r;
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
                if (WIDE && whole) {
                    // Lanes eight rows apart change values, so that a store is whole lines of 128 bytes (268 MB of slots: 16-bit product 159 -> 155 us, int8 114 -> 110; past the caches besides
                    // 145 and 103, but the sum that reads them takes as much longer).
                    typedef float four __attribute__((ext_vector_type(4), aligned(4)));
                    const bool upper = r & 8;
                    v4f low, high;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float given = upper ? y[0][e] : y[1][e];
                        const float got = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, given), 0x128, 0xf, 0xf, false));  // row_ror:8
                        low[e] = upper ? got : y[0][e], high[e] = upper ? y[1][e] : got;
                    }
                    const int at = I * 16 + (r & 7);
                    float* const to = reinterpret_cast<float*>(p.out) + (int64_t)(t.first_row + at) * p.cols + first_col + J0 * 16 + (upper ? 16 : 0) + 4 * piece;
                    if (at < t.rows) *reinterpret_cast<four*>(to) = low;
                    if (at + 8 < t.rows) *reinterpret_cast<four*>(to + 8 * (int64_t)p.cols) = high;
                } else if (WIDE || !whole) {
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
    for (int s = 0; s < 3; ++s) {
        if (KIND == I8 && load_step == 0 && left > s) request_scales();
        Each<A_REQUESTS>::run([&](auto q) { request(q, s * kStage, left - s); });
        if (gather && p.steps <= 4) everybody_arrived();  // (the next tile's tokens)
        advance();
    }
    next_w = weights_of();
    Each<CHANNELS>::run([&](auto j) { load_weight(N0{}, N0{}, j, next_w); });
    Each<CHANNELS>::run([&](auto j) { load_weight(N1{}, N1{}, j, next_w); });
    next_w = weights_of();
    Each<CHANNELS>::run([&](auto j) { load_weight(N2{}, N0{}, j, next_w); });
    after_w = weights_of();
    everybody_arrived();
    Each<4>::run([&](auto i) { read_row(N0{}, i, 0); });
    auto one_step = [&](auto parity) __attribute__((always_inline)) {
        half_step(parity, N0{});
        half_step(parity, N1{});
        advance();
        next_w = after_w, after_w = weights_of();
        stage = (stage + kStage) & (kStages - 1);
        --left;
    };
#pragma unroll 1
    for (int tile = 0; tile < my_tiles; ++tile) {
        is_short = ROWS == 8 && GROUPED && tile_of(tile).rows <= 64;
        // (the first step as one of its own, whose sums start at 0, takes the registers of a second set of sums)
        Each<ROWS * CHANNELS>::run([&](auto at) {
            Sum& one = sum[decltype(at)::value / CHANNELS][decltype(at)::value % CHANNELS];
            one = Sum{};
            lds_asm::keep(one);
        });
        settle();
        // (K is padded to pairs of steps, so that a step's weights lie in the same registers whatever the tile)
#pragma unroll 1
        for (int step = 0; step < p.steps; step += 2) {
            one_step(N0{});
            one_step(N1{});
        }
        settle();
        Each<ROWS * CHANNELS>::run([&](auto at) { lds_asm::keep(sum[decltype(at)::value / CHANNELS][decltype(at)::value % CHANNELS]); });
        store(tile_of(tile));
        if constexpr (KIND == I8) turn(scales);
    }
}

template <int KIND, int ROWS, bool WIDE, bool GROUPED, bool SWIGLU>
int launch_wide(const Product& p, uint32_t blocks, hipStream_t s) {
    constexpr uint32_t kLds = Wide<KIND, ROWS, GROUPED>::lds;
    constexpr auto kernel = &byte_wide_kernel<KIND, ROWS, WIDE, GROUPED, SWIGLU>;
    static DeviceOnce ready;
    const int code = ready.run([] { return hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds), "hipFuncSetAttribute"); });
    if (code != ORX_OK) return code;
    ORX_LAUNCH(kernel, dim3(blocks), dim3(64 * Wide<KIND, ROWS, GROUPED>::waves), kLds, s, p);
    return hip_check(hipGetLastError(), "launch byte product");
}
template <int KIND, int ROWS, bool GROUPED>
int launch_wide(const Product& p, bool swiglu, uint32_t blocks, hipStream_t s) {
    if (p.type == mx::F32) return swiglu ? launch_wide<KIND, ROWS, true, GROUPED, true>(p, blocks, s) : launch_wide<KIND, ROWS, true, GROUPED, false>(p, blocks, s);
    return swiglu ? launch_wide<KIND, ROWS, false, GROUPED, true>(p, blocks, s) : launch_wide<KIND, ROWS, false, GROUPED, false>(p, blocks, s);
}

}  // namespace
}  // namespace orx
