// Products of many rows with MXFP4 weights, dense and routed experts: tiles of the output from LDS.
//
// DOWN x ACROSS waves share a tile, each 32 ROWS x 32 CHANNELS of it in blocks of 32 x 32; K goes in steps of 256.  Codes and powers come from memory to LDS without passing a
// register (16 or 4 bytes a lane), two stages.  Weights and dense rows arrive as they are laid out, a kilobyte to a request; of an expert's rows, which lie anywhere, the 128 bytes of a
// step keep their 16-byte piece p at p ^ ((row >> 1) & 7), so that the sixteen rows of a read meet different banks.  A workgroup goes through its tiles as one sequence of steps: the next
// tile's first steps are on their way while the last ones are multiplied, and results drain under the next multiplies.
// HALVES 2: as many waves again take the second half of K, for launches whose tiles do not fill the CUs (7168 x 5120, weights out of cache, us with / without: 333 rows in tiles of 128
// 20.4 / 23.1, 200 rows in tiles of 64 17.0 / 19.6; 5120 x 17408, 333 rows, 64: 45 / 57).
// LOOK: quarters of a step that operands are read ahead, two where the registers hold them (128 x 128: 333 rows 17.6 / 17.9, experts of 2048 x 512 70.2 / 74.0).
//
// v_mfma_scale_f32_32x32x64 takes 32 cycles, 16 x 16 x 128 18, so the former: 6.2 PFLOP/s on random codes straight from registers, 5.4 the latter.  The multipliers do not run out of
// work there, the chip runs into its power: 1.5 GHz with random codes, 2.35 with zeros (9.6 PFLOP/s).  The account of 8192 x 17408 x 5120, 2176 tiles of 256 x 256, eight or nine to a CU,
// by the time at each tile's steps and results in a launch of 377 us: 1.9 before the first step, 33.0 for the first tile's 20 steps (1.65 each), 39.3 for those of each later tile (1.95; with
// all CUs at it, 4.4 PFLOP/s, and taken for power, which was not measured apart), 2.7 for the results of each; the CUs with eight tiles end 41 before the others.  Launches behind one another take
// 360-395 (3.7-4.05 PFLOP/s).  8192 x 4096 x 4096, two tiles to a CU: 1.4, then 16 steps of 1.6-1.8 and 2-3 of results each, all ended at 62-71, the launch 66-76 (3.6-4.15).
// A 128 x 128 step alone on a CU takes 0.5-0.65 us, 0.3 without its requests, 0.15 without its multiplies either.
// Tried: four waves of 128 x 128 results (a third less from LDS, 1.63 us a step, but sums come out of accumulation registers by moves, 4.4-6.2 us a tile against 2.1: the same in
// all); results by lines of 128 bytes through LDS (more instructions, and not faster: what a tile's end took was its instructions); three to six stages, a CU then holding one workgroup
// (305 units of 128 expert rows, 1024 x 2048: 64 us with two stages and two workgroups, 80 with four and one); requests masked instead of branched around (level); barriers that do not
// wait for the last tile's stores (no faster, and 256 x 256 spills); results past the caches (8192 x 4096 x 4096 75 -> 103 us: an instruction stores 32 bytes of a row, the L2 joins
// them).  Without its requests that product of experts takes 46 us, without results 55.
#include "lds_asm.h"
#include "mx_device.h"
#include "mx_tiles.h"
#include "orx_internal.h"

namespace orx {
namespace {

using namespace mx;
using lds_asm::Each;

// Requests to LDS where `wanted` is above 0, by a branch inside the statement: the K loop stays one block.  16 or 4 bytes a lane, one lane behind the other.
#define ORX_WANTED(BODY) "s_cmp_gt_i32 %2, 0\n\ts_cbranch_scc0 .Lskipped%=\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t" BODY "\n.Lskipped%=:"
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is reserved: it holds nothing of the compiler's from one statement to the next)
__device__ __forceinline__ void request_16_from(const uint8_t* lane_address, uint32_t lds_wave_base, int wanted) {
    asm volatile(ORX_WANTED("global_load_lds_dwordx4 %0, off") ::"v"(lane_address), "s"(lds_wave_base), "s"(wanted) : "memory", "m0", "scc");
}
__device__ __forceinline__ const uint8_t* uniform_pointer(const uint8_t* pointer) {
    const uint64_t bits = reinterpret_cast<uint64_t>(pointer);
    const uint32_t low = __builtin_amdgcn_readfirstlane((uint32_t)bits), high = __builtin_amdgcn_readfirstlane((uint32_t)(bits >> 32));
    return reinterpret_cast<const uint8_t*>(((uint64_t)high << 32) | low);
}
__device__ __forceinline__ void request_4_from(const uint8_t* lane_address, uint32_t lds_wave_base, int wanted) {
    asm volatile(ORX_WANTED("global_load_lds_dword %0, off") ::"v"(lane_address), "s"(lds_wave_base), "s"(wanted) : "memory", "m0", "scc");
}
// two kilobytes that lie together on both sides
__device__ __forceinline__ void request_tile(uint32_t lane_offset, const uint8_t* uniform_base, uint32_t lds_wave_base, int wanted) {
    asm volatile(ORX_WANTED("global_load_lds_dwordx4 %0, %3\n\tglobal_load_lds_dwordx4 %0, %3 offset:1024") ::"v"(lane_offset), "s"(lds_wave_base), "s"(wanted), "s"(uniform_base)
                 : "memory", "m0", "scc");
}
#pragma clang diagnostic pop
#undef ORX_WANTED
// All requests and LDS reads of this wave have ended, and those of the others.  (The builtin, not a statement: the compiler then knows that its reads are there.)
__device__ __forceinline__ void everybody_arrived() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int ROWS, int CHANNELS, int DOWN, int ACROSS, int LOOK, int HALVES, bool WIDE, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(64 * DOWN * ACROSS * HALVES, 2) void mx_tiles_kernel(Product p) {
    constexpr int BM = 32 * ROWS * DOWN, BN = 32 * CHANNELS * ACROSS, WAVES = DOWN * ACROSS;
    constexpr int A_REQUESTS = BM / (GROUPED ? 8 : 16) / WAVES, W_REQUESTS = BN / 16 / WAVES;  // of a wave and step: eight rows or a tile, a tile
    constexpr int POWERS = BM / 32 + BN / 32;                                                   // of all waves
    constexpr int kW = BM * 128, kAS = kW + BN * 128, kWS = kAS + BM * 8, kStage = kWS + BN * 8;
    constexpr int kSmall = (POWERS + WAVES - 1) / WAVES;
    extern __shared__ __align__(128) uint8_t whole_lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) % WAVES, half = HALVES == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) / WAVES;
    uint8_t* const lds = whole_lds + half * (2 * kStage);
    // of K, two halves of equal steps: of an odd number both have the middle one, and the second half drops it
    const int steps = HALVES == 1 ? p.steps : (p.steps + 1) / 2, first_step = half ? p.steps - steps : 0;
    const int wave_m = wave % DOWN, wave_n = wave / DOWN;

    // ---- which results: tiles blockIdx.x, blockIdx.x + gridDim.x, .. of an order in which every XCD has one run ----
    const int groups = (p.tiles + BN / 16 - 1) / (BN / 16);
    const int row_tiles = GROUPED ? min(__builtin_amdgcn_readfirstlane(*p.unit_count), p.most_units) : (p.m + BM - 1) / BM;
    const int total = row_tiles * groups;
    const int my_tiles = (total - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    if (my_tiles <= 0) return;
    struct Tile {
        int first_row, rows, group, expert;
    };
    auto tile_of = [&](int number) {
        const int at = (int)blockIdx.x + number * (int)gridDim.x, xcd = at & 7;
        const int id = xcd * (total >> 3) + min(xcd, total & 7) + (at >> 3);
        Tile t;
        if (GROUPED) {
            const int4 u = p.units[id / groups];
            t.group = id % groups, t.first_row = __builtin_amdgcn_readfirstlane(u.y), t.rows = __builtin_amdgcn_readfirstlane(u.z);
            t.expert = __builtin_amdgcn_readfirstlane(u.x);
        } else {
            // eight tiles of rows for each tile of channels, so that an L2 holds what neighbours share
            const int band = id / (8 * groups), in_band = min(8, row_tiles - 8 * band), within = id % (8 * groups);
            t.first_row = (8 * band + within % in_band) * BM, t.group = within / in_band;
            t.rows = min(BM, p.m - t.first_row), t.expert = 0;
        }
        return t;
    };

    // ---- requests ----
    const uint32_t lds_base = lds_asm::lds_address_of(lds);
    const uint8_t* a_from[A_REQUESTS];  // a tile, or this lane's piece of eight rows
    const uint8_t* w_from[W_REQUESTS];
    // powers: request j < BM / 32 is 32 rows of 8 bytes or two tiles of 128, the others two tiles
    const uint8_t* power_from[kSmall];
    int power_step[kSmall], power_to[kSmall];
    auto aim = [&](const Tile& t) {
#pragma unroll
        for (int b = 0; b < A_REQUESTS; ++b) {
            if constexpr (GROUPED) {
                const int local = (wave * A_REQUESTS + b) * 8 + (lane >> 3);
                int64_t row = t.first_row + min(local, t.rows - 1);
                if (p.slot_token != nullptr) row = p.slot_token[row];
                a_from[b] = p.a + row * p.pitch + first_step * 128 + ((lane & 7) ^ ((local >> 1) & 7)) * 16;
            } else {
                a_from[b] = uniform_pointer(p.a + ((int64_t)min(t.first_row / 16 + wave * A_REQUESTS + b, (p.m - 1) / 16) * p.steps + first_step) * kTileBytes);
            }
        }
        const int64_t expert = (int64_t)t.expert * p.tiles;
#pragma unroll
        for (int b = 0; b < W_REQUESTS; ++b) w_from[b] = uniform_pointer(p.w + ((expert + min(t.group * (BN / 16) + wave * W_REQUESTS + b, p.tiles - 1)) * p.steps + first_step) * kTileBytes);
#pragma unroll
        for (int i = 0; i < kSmall; ++i) {
            const int j = wave + WAVES * i;
            if (j < BM / 32) {
                power_to[i] = kAS + j * 256;
                if constexpr (GROUPED) {
                    int64_t row = t.first_row + min(j * 32 + (lane >> 1), t.rows - 1);
                    if (p.slot_token != nullptr) row = p.slot_token[row];
                    power_from[i] = p.as + row * (p.pitch / 16) + (lane & 1) * 4;
                    power_step[i] = 8;
                } else {
                    power_from[i] = p.as + (int64_t)min(t.first_row / 16 + j * 2 + (lane >> 5), (p.m - 1) / 16) * p.steps * kTilePowers + (lane & 31) * 4;
                    power_step[i] = kTilePowers;
                }
            } else {
                const int64_t tile = expert + min(t.group * (BN / 16) + (j - BM / 32) * 2 + (lane >> 5), p.tiles - 1);
                power_from[i] = p.ws + tile * p.steps * kTilePowers + (lane & 31) * 4;
                power_step[i] = kTilePowers, power_to[i] = kWS + (j - BM / 32) * 256;
            }
            power_from[i] += first_step * power_step[i];
        }
    };
    int load_tile = 0, load_step = 0;
    auto advance = [&]() {
        if (++load_step < steps) return;
        load_step = 0;
        if (++load_tile < my_tiles) aim(tile_of(load_tile));
    };
    constexpr int kAll = A_REQUESTS + W_REQUESTS + kSmall;  // requests of a step
    auto request = [&](int id, uint32_t stage, int wanted) {  // the next step's; in order
        const uint32_t to = lds_base + stage;
        if (id < A_REQUESTS) {
            if constexpr (GROUPED) request_16_from(a_from[id], to + (wave * A_REQUESTS + id) * 1024, wanted);
            else request_tile(lane * 16, a_from[id], to + (wave * A_REQUESTS + id) * 2048, wanted);
            a_from[id] += GROUPED ? 128 : kTileBytes;
        } else if (id < A_REQUESTS + W_REQUESTS) {
            const int b = id - A_REQUESTS;
            request_tile(lane * 16, w_from[b], to + kW + (wave * W_REQUESTS + b) * 2048, wanted);
            w_from[b] += kTileBytes;
        } else {
            const int i = id - A_REQUESTS - W_REQUESTS;
            request_4_from(power_from[i], to + power_to[i], min(wanted, POWERS - wave - WAVES * i));
            power_from[i] += power_step[i];
        }
    };

    // ---- operands ----
    const int r = lane & 31, low = lane >> 5;  // row or channel of a block; blocks 2 t + low of a step's eight
    const uint32_t a_at = GROUPED ? (wave_m * 32 * ROWS + r) * 128 + ((low ^ ((r >> 1) & 7)) * 16) : (wave_m * 2 * ROWS + (r >> 4)) * 2048 + low * 256 + (r & 15) * 16;
    const uint32_t w_at = kW + (wave_n * 2 * CHANNELS + (r >> 4)) * 2048 + low * 256 + (r & 15) * 16;
    const uint32_t as_at = GROUPED ? kAS + (wave_m * 32 * ROWS + r) * 8 : kAS + (wave_m * 2 * ROWS + (r >> 4)) * 128 + (r & 15) * 8 + low * 4;
    const uint32_t ws_at = kWS + (wave_n * 2 * CHANNELS + (r >> 4)) * 128 + (r & 15) * 8 + low * 4;
    constexpr int kHeld = LOOK == 1 ? 2 : 4;  // quarters' operands
    v4i fa[kHeld][ROWS], fw[kHeld][CHANNELS];
    uint2 read_a[ROWS];  // of the next step
    int read_w[CHANNELS], powers_a[ROWS], powers_w[CHANNELS];
    const uint32_t select = low ? 0x07050301u : 0x06040200u;  // a row's eight powers, those of this lane's four blocks
    constexpr int kSet = ROWS + CHANNELS;  // reads of a quarter's operands, and of a step's powers
    // read number `at` of the operands of quarter t
    auto read_operand = [&](auto t, auto at, uint32_t stage) {
        constexpr int T = decltype(t)::value, AT = decltype(at)::value;
        if constexpr (AT < ROWS)
            fa[T % kHeld][AT] = *reinterpret_cast<const v4i*>(lds + ((GROUPED ? a_at ^ (T * 32) : a_at) + stage) + (AT * 4096 + (GROUPED ? 0 : T * 512)));
        else
            fw[T % kHeld][AT - ROWS] = *reinterpret_cast<const v4i*>(lds + (w_at + stage) + ((AT - ROWS) * 4096 + T * 512));
    };
    auto read_power = [&](auto at, uint32_t stage) {
        constexpr int AT = decltype(at)::value;
        if constexpr (AT < ROWS && GROUPED)
            read_a[AT] = *reinterpret_cast<const uint2*>(lds + (as_at + stage) + AT * 256);
        else if constexpr (AT < ROWS)
            read_a[AT].x = *reinterpret_cast<const uint32_t*>(lds + (as_at + stage) + AT * 256);
        else
            read_w[AT - ROWS] = *reinterpret_cast<const int*>(lds + (ws_at + stage) + (AT - ROWS) * 256);
    };
    auto take_powers = [&]() {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) powers_a[i] = GROUPED ? (int)__builtin_amdgcn_perm(read_a[i].y, read_a[i].x, select) : (int)read_a[i].x;
#pragma unroll
        for (int j = 0; j < CHANNELS; ++j) powers_w[j] = read_w[j];
        __builtin_amdgcn_sched_barrier(0);
    };
    v16f sum[ROWS][CHANNELS];
    // One multiply of K 64 t.. of a step, the at-th of them; FRESH: the first of a tile, whose sums are 0.
    auto multiply = [&](auto t, auto at, auto fresh) {
        constexpr int T = decltype(t)::value, I = decltype(at)::value / CHANNELS, JJ = decltype(at)::value % CHANNELS;
        constexpr int J = I & 1 ? CHANNELS - 1 - JJ : JJ;  // one operand changes between neighbours
        if constexpr (decltype(fresh)::value)
            sum[I][J] = multiply_32<T, T>(fw[T % kHeld][J], fa[T % kHeld][I], v16f{}, powers_w[J], powers_a[I]);
        else
            sum[I][J] = multiply_32<T, T>(fw[T % kHeld][J], fa[T % kHeld][I], sum[I][J], powers_w[J], powers_a[I]);
    };
    using Fresh = std::true_type;
    using Added = std::false_type;
    using T0 = std::integral_constant<int, 0>;
    using T1 = std::integral_constant<int, 1>;
    using T2 = std::integral_constant<int, 2>;
    using T3 = std::integral_constant<int, 3>;
    // A wave cannot issue anything while an LDS read or a request waits for its slot, and with one wave to a SIMD the multiplier then runs dry: behind every multiply stands at most
    // a read or two.  A step's requests go out in three parts, behind the barrier that frees their stage and in the two quarters of the next step behind it.
    constexpr int kPart0 = kAll * 8 / 20, kPart1 = (kAll - kPart0 + 1) / 2;
    constexpr int kAtOnce = LOOK == 1 ? kPart0 : kPart0 + kPart1;  // in front of the next step
    // Multiplies FIRST.. of quarter t with `other(0)` .. `other(COUNT - 1)` among them.
    auto multiply_among = [&](auto t, auto first, auto fresh, auto count, auto other) {
        constexpr int FIRST = decltype(first)::value, LEFT = ROWS * CHANNELS - FIRST, COUNT = decltype(count)::value;
        Each<LEFT>::run([&](auto at) {
            constexpr int AT = decltype(at)::value;
            multiply(t, std::integral_constant<int, AT + FIRST>{}, fresh);
            __builtin_amdgcn_sched_barrier(0);
            Each<COUNT>::run([&](auto q) {
                if constexpr (decltype(q)::value * LEFT / COUNT == AT) other(q);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    constexpr int FOURS = SWIGLU ? 2 : 4;  // results of a block and lane, by four
    uint32_t stage = 0;
    int left = my_tiles * steps;  // steps, with this one
    // Quarter t, with the reads of quarter t + LOOK's operands, of the next step's powers in the last one, and a part of the requests.  In quarter 4 - LOOK, after one multiply to go on
    // with, the next stage is whole and nobody reads this one any more.
    auto quarter = [&](auto t, auto fresh, uint32_t next) {
        constexpr int T = decltype(t)::value, PART = (T + LOOK) % 4, kFirst = PART == 0 ? 1 : 0, kPowers = T == 3 ? kSet : 0;
        constexpr int kBegin = PART == 0 ? 0 : PART == 1 ? kPart0 : kPart0 + kPart1, kRequests = PART == 0 ? kPart0 : PART == 1 ? kPart1 : PART == 2 ? kAll - kPart0 - kPart1 : 0;
        if constexpr (PART == 0) {
            multiply(t, T0{}, fresh);
            __builtin_amdgcn_sched_barrier(0);
            everybody_arrived();
            __builtin_amdgcn_sched_barrier(0);
        }
        multiply_among(t, std::integral_constant<int, kFirst>{}, fresh, std::integral_constant<int, kSet + kPowers + kRequests>{}, [&](auto q) {
            constexpr int Q = decltype(q)::value;
            if constexpr (Q < kSet) read_operand(std::integral_constant<int, (T + LOOK) % 4>{}, q, T + LOOK < 4 ? stage : next);
            else if constexpr (Q < kSet + kPowers) read_power(std::integral_constant<int, Q - kSet>{}, next);
            else if constexpr (T + LOOK < 4) request(kBegin + Q - kSet - kPowers, next, left - 1);
            else request(kBegin + Q - kSet - kPowers, stage, left - 2);
        });
    };

    // ---- results: block (i, j) has channels 8 (e / 4) + 4 low + e % 4 of row r; pairs of fours change halves, and a lane has eight neighbours ----
    auto results = [&](v16f& s, v4f(&four)[FOURS]) {
#pragma unroll
        for (int q = 0; q < FOURS; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) four[q][e] = SWIGLU ? swiglu(s[4 * q + e], s[8 + 4 * q + e]) : s[4 * q + e];
    };
    // Two halves of K: each hands half of its blocks over in LDS, adds what it gets to the others, and stores those.
    auto kept = [&](int at) { return HALVES == 1 || (at < ROWS * CHANNELS / 2) == (half == 0); };
    auto store = [&](const Tile& t) {
        const int first_col = (t.group * ACROSS + wave_n) * CHANNELS * (8 * FOURS);
        if (first_col + CHANNELS * 8 * FOURS <= p.cols) {
            Each<ROWS * CHANNELS>::run([&](auto at) {
                constexpr int I = decltype(at)::value / CHANNELS, J = decltype(at)::value % CHANNELS;
                if (!kept(decltype(at)::value)) return;
                const int row = (wave_m * ROWS + I) * 32 + r;
                v16f& s = sum[I][J];
                v4f four[FOURS];
                results(s, four);
                if constexpr (WIDE) {
                    float* const to = reinterpret_cast<float*>(p.out) + (int64_t)(t.first_row + row) * p.cols + first_col + 4 * low;
                    if (row < t.rows) {
#pragma unroll
                        for (int q = 0; q < FOURS; ++q) *reinterpret_cast<floats4*>(to + J * 8 * FOURS + 8 * q) = four[q];
                    }
                } else {
                    unsigned short* const to = reinterpret_cast<unsigned short*>(p.out) + (int64_t)(t.first_row + row) * p.cols + first_col + 8 * low;
                    uint32_t pairs[2 * FOURS];
                    if (p.type == F16) {
#pragma unroll
                        for (int q = 0; q < 2 * FOURS; ++q) pairs[q] = two_values(four[q / 2][q % 2 * 2], four[q / 2][q % 2 * 2 + 1], F16);
                    } else {
#pragma unroll
                        for (int q = 0; q < 2 * FOURS; ++q) pairs[q] = two_values(four[q / 2][q % 2 * 2], four[q / 2][q % 2 * 2 + 1], BF16);
                    }
                    v4u eight[FOURS / 2];
#pragma unroll
                    for (int q = 0; q < FOURS; q += 2) {
                        auto first = __builtin_amdgcn_permlane32_swap(pairs[2 * q], pairs[2 * q + 2], false, false);
                        auto second = __builtin_amdgcn_permlane32_swap(pairs[2 * q + 1], pairs[2 * q + 3], false, false);
                        eight[q / 2] = v4u{first[0], second[0], first[1], second[1]};
                    }
                    if (row < t.rows) {
#pragma unroll
                        for (int q = 0; q < FOURS / 2; ++q) *reinterpret_cast<words4*>(to + J * 8 * FOURS + 16 * q) = eight[q];
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            return;
        }
        // the last channels: one piece of code for all blocks, column by column where they end
#pragma unroll 1
        for (int at = 0; at < ROWS * CHANNELS; ++at) {
            if (!kept(at)) continue;
            v16f s;
            Each<ROWS * CHANNELS>::run([&](auto which) {
                v16f& block = sum[decltype(which)::value / CHANNELS][decltype(which)::value % CHANNELS];
                if (at == decltype(which)::value) {
                    // (volatile: or the moves of all blocks are made in front of the loop)
                    asm volatile("" : "+v"(block));
                    s = block;
                }
            });
            v4f four[FOURS];
            results(s, four);
            const int row = (wave_m * ROWS + at / CHANNELS) * 32 + r;
            if (row < t.rows) {
#pragma unroll
                for (int q = 0; q < FOURS; ++q) store_four(p.out, WIDE ? F32 : p.type, (int64_t)(t.first_row + row) * p.cols, first_col + at % CHANNELS * 8 * FOURS + 8 * q + 4 * low, p.cols, four[q]);
            }
        }
    };

    aim(tile_of(0));
#pragma unroll
    for (int q = 0; q < kAll; ++q) request(q, 0, 1);
    advance();
    everybody_arrived();
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) request(q, kStage, left - 1);
    Each<kSet>::run([&](auto at) { read_operand(T0{}, at, 0); });
    if constexpr (LOOK > 1) Each<kSet>::run([&](auto at) { read_operand(T1{}, at, 0); });
    Each<kSet>::run([&](auto at) { read_power(at, 0); });
    // One sequence of steps over all tiles: the next tile's first steps are on their way while this one's last are multiplied.  (The last step of all reads a stage that nobody filled.)
    auto one_step = [&](auto fresh) {
        const uint32_t next = kStage - stage;
        take_powers();
        quarter(T0{}, fresh, next);
        if constexpr (LOOK > 1) advance();
        quarter(T1{}, Added{}, next);
        if constexpr (LOOK == 1) advance();
        quarter(T2{}, Added{}, next);
        quarter(T3{}, Added{}, next);
        stage = next;
        --left;
    };
    if constexpr (HALVES == 1) {
#pragma unroll 1
        for (int tile = 0; tile < my_tiles; ++tile) {
            one_step(Fresh{});
#pragma unroll 1
            for (int step = 1; step < steps; ++step) one_step(Added{});
            store(tile_of(tile));
        }
    } else {  // one tile
        one_step(Fresh{});
        int step = 1;
        if (half && (p.steps & 1)) one_step(Fresh{}), ++step;
#pragma unroll 1
        for (; step < steps; ++step) one_step(Added{});
        constexpr int kGiven = ROWS * CHANNELS / 2;
        v4f(*const given)[WAVES][kGiven * 4][64] = reinterpret_cast<v4f(*)[WAVES][kGiven * 4][64]>(whole_lds);
        Each<ROWS * CHANNELS>::run([&](auto at) {
            constexpr int AT = decltype(at)::value;
            const v16f& s = sum[AT / CHANNELS][AT % CHANNELS];
            if (!kept(AT)) {
#pragma unroll
                for (int q = 0; q < 4; ++q) given[half][wave][AT % kGiven * 4 + q][lane] = v4f{s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
            }
        });
        __syncthreads();
        Each<ROWS * CHANNELS>::run([&](auto at) {
            constexpr int AT = decltype(at)::value;
            v16f& s = sum[AT / CHANNELS][AT % CHANNELS];
            if (kept(AT)) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const v4f other = given[1 - half][wave][AT % kGiven * 4 + q][lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[4 * q + e] += other[e];
                }
            }
        });
        store(tile_of(0));
    }
}

template <int ROWS, int CHANNELS, int DOWN, int ACROSS, int LOOK, int HALVES, bool WIDE, bool GROUPED, bool SWIGLU>
int launch_one(const Product& p, uint32_t blocks, hipStream_t s) {
    constexpr uint32_t kLds = HALVES * 2 * (32 * ROWS * DOWN + 32 * CHANNELS * ACROSS) * 136;
    constexpr auto kernel = &mx_tiles_kernel<ROWS, CHANNELS, DOWN, ACROSS, LOOK, HALVES, WIDE, GROUPED, SWIGLU>;
    static DeviceOnce ready;
    const int code = ready.run([] { return hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds), "hipFuncSetAttribute"); });
    if (code != ORX_OK) return code;
    ORX_LAUNCH(kernel, dim3(blocks), dim3(64 * DOWN * ACROSS * HALVES), kLds, s, p);
    return hip_check(hipGetLastError(), "launch mxfp4 tiles");
}
template <int ROWS, int CHANNELS, int DOWN, int ACROSS, int LOOK, int HALVES, bool WIDE>
int launch_of_type(const Product& p, bool grouped, bool swiglu, uint32_t blocks, hipStream_t s) {
    if constexpr (HALVES == 1)
        if (grouped) return swiglu ? launch_one<ROWS, CHANNELS, DOWN, ACROSS, LOOK, HALVES, WIDE, true, true>(p, blocks, s) : launch_one<ROWS, CHANNELS, DOWN, ACROSS, LOOK, HALVES, WIDE, true, false>(p, blocks, s);
    return swiglu ? launch_one<ROWS, CHANNELS, DOWN, ACROSS, LOOK, HALVES, WIDE, false, true>(p, blocks, s) : launch_one<ROWS, CHANNELS, DOWN, ACROSS, LOOK, HALVES, WIDE, false, false>(p, blocks, s);
}
template <int ROWS, int CHANNELS, int DOWN, int ACROSS, int LOOK, int HALVES>
int launch(const Product& p, bool grouped, bool swiglu, uint32_t blocks, hipStream_t s) {
    return p.type == F32 ? launch_of_type<ROWS, CHANNELS, DOWN, ACROSS, LOOK, HALVES, true>(p, grouped, swiglu, blocks, s) : launch_of_type<ROWS, CHANNELS, DOWN, ACROSS, LOOK, HALVES, false>(p, grouped, swiglu, blocks, s);
}

}  // namespace

int launch_mx_tiles(const mx::Product& p, int rows, int channels, int halves, bool grouped, bool swiglu, uint32_t blocks, hipStream_t s) {
    if (rows == 256 && channels == 256) return launch<4, 2, 2, 4, 1, 1>(p, grouped, swiglu, blocks, s);
    if (halves == 2) return rows == 128 ? launch<2, 2, 2, 2, 2, 2>(p, false, swiglu, blocks, s) : launch<1, 2, 2, 2, 1, 2>(p, false, swiglu, blocks, s);
    if (rows == 128 && channels == 128) return launch<2, 2, 2, 2, 2, 1>(p, grouped, swiglu, blocks, s);
    return launch<1, 2, 2, 2, 1, 1>(p, grouped, swiglu, blocks, s);
}

}  // namespace orx
