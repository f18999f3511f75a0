// Products of many rows with weights by byte tiles, dense and routed experts: tiles of the output from LDS.
//
// DOWN x ACROSS waves share a tile, each ROWS x CHANNELS blocks of 16 x 16 of it; K goes in steps of 128 bytes.  Rows and weights come from memory to LDS without passing a register, two
// stages.  Weights arrive as they are laid out, a kilobyte to a request; of a row, which lies anywhere, the 128 bytes of a step keep their 16-byte piece p at p ^ ((row >> 1) & 7), so that the
// sixteen rows of a read meet different banks.  A workgroup goes through its tiles as one sequence of steps: the next tile's first steps are on their way while the last ones are multiplied, and
// results drain under the next multiplies.
#include "byte_tiles.h"
#include "lds_asm.h"
#include "orx_internal.h"
#include "tile_requests.h"

namespace orx {
namespace {

using namespace bytes;
using namespace tile_requests;
using lds_asm::Each;

template <int KIND, int ROWS, int CHANNELS, int DOWN, int ACROSS, bool WIDE, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(64 * DOWN * ACROSS, 2) void byte_tiles_kernel(Product p) {
    using Sum = typename Operands<KIND>::Sum;
    constexpr int BM = 16 * ROWS * DOWN, BN = 16 * CHANNELS * ACROSS, WAVES = DOWN * ACROSS;
    constexpr int A_REQUESTS = BM / 8 / WAVES, W_REQUESTS = BN / 16 / WAVES;  // of a wave and step: eight rows, a tile
    constexpr int kAll = A_REQUESTS + W_REQUESTS;
    constexpr int kW = BM * kStep, kStage = kW + BN * kStep;
    extern __shared__ __align__(128) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
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
    auto row_of = [&](const Tile& t, int local) {
        int64_t row = max(t.first_row + min(local, t.rows - 1), 0);  // (rows that are not there repeat the last: their sums go nowhere)
        if (GROUPED && p.slot_token != nullptr) row = p.slot_token[row];
        return row;
    };

    // ---- requests ----
    const uint32_t lds_base = lds_asm::lds_address_of(lds);
    const uint8_t* a_from[A_REQUESTS];  // this lane's piece of eight rows
    const uint8_t* w_from[W_REQUESTS];  // a tile
    auto piece_of = [&](int b) { return (lane & 7) ^ ((((wave * A_REQUESTS + b) * 8 + (lane >> 3)) >> 1) & 7); };
    // 16-bit rows may end within a step: the pieces behind come from the weights' padding, which is 0
    const int last_pieces = KIND == I8 ? 0 : (p.row_bytes % kStep) / 16, partial_step = last_pieces ? p.steps - 1 : -1;
    const uint8_t* const zeros = p.w + (int64_t)(p.steps - 1) * kTileBytes + last_pieces * 256;
    auto aim = [&](const Tile& t) {
#pragma unroll
        for (int b = 0; b < A_REQUESTS; ++b) a_from[b] = p.a + row_of(t, (wave * A_REQUESTS + b) * 8 + (lane >> 3)) * p.pitch + piece_of(b) * 16;
        const int64_t expert = (int64_t)t.expert * p.tiles;
#pragma unroll
        for (int b = 0; b < W_REQUESTS; ++b) w_from[b] = uniform_pointer(p.w + (expert + min(t.group * (BN / 16) + wave * W_REQUESTS + b, p.tiles - 1)) * p.steps * kTileBytes);
    };
    int load_tile = 0, load_step = 0;
    auto advance = [&]() {
        if (++load_step < p.steps) return;
        load_step = 0;
        if (++load_tile < my_tiles) aim(tile_of(load_tile));
    };
    auto request = [&](auto id, uint32_t stage, int wanted) {  // the next step's; in order
        constexpr int ID = decltype(id)::value;
        const uint32_t to = lds_base + stage;
        if constexpr (ID < A_REQUESTS) {
            const uint8_t* from = a_from[ID];
            if constexpr (KIND != I8) from = load_step == partial_step && piece_of(ID) >= last_pieces ? zeros : from;
            request_16_from(from, to + (wave * A_REQUESTS + ID) * 1024, wanted);
            a_from[ID] += kStep;
        } else {
            constexpr int B = ID - A_REQUESTS;
            request_tile(lane * 16, w_from[B], to + kW + (wave * W_REQUESTS + B) * kTileBytes, wanted);
            w_from[B] += kTileBytes;
        }
    };

    // ---- operands: halves of a step, 64 bytes of K ----
    const int r = lane & 15, piece = lane >> 4;  // row or channel of a block; pieces `piece` and 4 behind of a step
    const uint32_t a_at = (wave_m * 16 * ROWS + r) * kStep + (piece ^ ((r >> 1) & 7)) * 16;
    const uint32_t w_at = kW + wave_n * CHANNELS * kTileBytes + lane * 16;
    // A half's operands are read while the half before is multiplied.  Rows, where there are many, into the registers whose last multiply has just been issued.
    constexpr int kHeldRows = ROWS > 4 ? 1 : 2;
    v4i fa[kHeldRows][ROWS], fw[2][CHANNELS];
    auto read_row = [&](auto half, auto i, uint32_t stage) {
        constexpr int H = decltype(half)::value, I = decltype(i)::value;
        fa[H % kHeldRows][I] = *reinterpret_cast<const v4i*>(lds + ((a_at ^ (H * 64)) + stage) + I * (16 * kStep));
    };
    auto read_weight = [&](auto half, auto j, uint32_t stage) {
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
    // Half H of a step; behind every multiply stands at most a read or a request.  In the second half, once the first row's multiplies are on their way, the next stage is whole and nobody reads
    // this one any more.  FRESH: the first of a tile, whose sums are 0.
    auto half_step = [&](auto half, auto fresh, uint32_t next) {
        constexpr int H = decltype(half)::value;
        using Other = std::integral_constant<int, 1 - H>;
        Each<ROWS>::run([&](auto i) {
            constexpr int I = decltype(i)::value;
            Each<CHANNELS>::run([&](auto jj) {
                constexpr int JJ = decltype(jj)::value, J = I & 1 ? CHANNELS - 1 - JJ : JJ;  // one operand changes between neighbours
                sum[I][J] = multiply<KIND>(fw[H][J], fa[H % kHeldRows][I], decltype(fresh)::value ? Sum{} : sum[I][J]);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (H == 1 && I == 0 && JJ == CHANNELS - 1) {
                    everybody_arrived();
                    __builtin_amdgcn_sched_barrier(0);
                }
                // reads of weights 0 .. CHANNELS - 1 and requests 0 .. kAll - 1 spread over the rows' multiplies
                constexpr int AT = I * CHANNELS + JJ - (H == 1 ? CHANNELS - 1 : 0), COUNT = ROWS * CHANNELS - (H == 1 ? CHANNELS - 1 : 0);
                if constexpr (AT >= 0) {
                    Each<CHANNELS>::run([&](auto w) {
                        if constexpr ((2 * decltype(w)::value) * COUNT / (2 * ROWS * CHANNELS) == AT) read_weight(Other{}, w, H == 0 ? stage : next);
                    });
                    if constexpr (H == 1)
                        Each<kAll>::run([&](auto q) {
                            if constexpr ((2 * decltype(q)::value + 1) * COUNT / (2 * kAll) == AT) request(q, stage, left - 2);
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
    auto store = [&](const Tile& t) {
        RowScale rows[ROWS];
        if constexpr (KIND == I8) {
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const int64_t row = row_of(t, (wave_m * ROWS + i) * 16 + r);
                rows[i] = {p.scale[row], !GROUPED && p.zero != nullptr ? p.zero[row] : 0};
            }
        }
        const int first_tile = t.group * (BN / 16) + wave_n * CHANNELS, first_col = first_tile / KINDS * 16;
        const int64_t channels = (int64_t)t.expert * p.tiles * 16;
        auto result = [&](auto i, auto j) {  // of block j of the results
            constexpr int I = decltype(i)::value, J = decltype(j)::value;
            const int64_t at = channels + min(first_tile + J * KINDS, p.tiles - KINDS) * 16 + 4 * piece;
            v4f y = scaled<KIND, GROUPED>(p, sum[I][J * KINDS], at, rows[I]);
            if constexpr (SWIGLU) {
                const v4f up = scaled<KIND, GROUPED>(p, sum[I][J * KINDS + 1], at + 16, rows[I]);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = mx::swiglu(y[e], up[e]);
            }
            return y;
        };
        const bool whole = first_col + BLOCKS * 16 <= p.cols;
        Each<BLOCKS / 2>::run([&](auto pair) {
            using J0 = std::integral_constant<int, 2 * decltype(pair)::value>;
            using J1 = std::integral_constant<int, J0::value + 1>;
            Each<ROWS>::run([&](auto i) {
                const int local = (wave_m * ROWS + decltype(i)::value) * 16 + r;
                const int64_t row_start = (int64_t)(t.first_row + local) * p.cols;
                const v4f y0 = result(i, J0{}), y1 = result(i, J1{});
                if (WIDE || !whole) {
                    if (local < t.rows) {
                        mx::store_four(p.out, WIDE ? mx::F32 : p.type, row_start, first_col + J0::value * 16 + 4 * piece, p.cols, y0);
                        mx::store_four(p.out, WIDE ? mx::F32 : p.type, row_start, first_col + J1::value * 16 + 4 * piece, p.cols, y1);
                    }
                } else {
                    uint32_t a[2], b[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (p.type == mx::F16) a[e] = mx::two_values(y0[2 * e], y0[2 * e + 1], mx::F16), b[e] = mx::two_values(y1[2 * e], y1[2 * e + 1], mx::F16);
                        else a[e] = mx::two_values(y0[2 * e], y0[2 * e + 1], mx::BF16), b[e] = mx::two_values(y1[2 * e], y1[2 * e + 1], mx::BF16);
                    }
                    // lanes of an even `piece` get the first block's eight channels 2 piece .., of an odd one the second's
                    auto low = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
                    auto high = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
                    const int col = first_col + (J0::value + (piece & 1)) * 16 + (piece >> 1) * 8;
                    if (local < t.rows) *reinterpret_cast<mx::words4*>(reinterpret_cast<unsigned short*>(p.out) + row_start + col) = v4u{low[0], high[0], low[1], high[1]};
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        });
    };

    aim(tile_of(0));
    Each<kAll>::run([&](auto q) { request(q, 0, 1); });
    advance();
    everybody_arrived();
    Each<kAll>::run([&](auto q) { request(q, kStage, left - 1); });
    advance();
    Each<ROWS>::run([&](auto i) { read_row(H0{}, i, 0); });
    Each<CHANNELS>::run([&](auto j) { read_weight(H0{}, j, 0); });
    // One sequence of steps over all tiles: the next tile's first steps are on their way while this one's last are multiplied.  (The last step of all reads a stage that nobody filled.)
    auto one_step = [&](auto fresh) {
        const uint32_t next = kStage - stage;
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
    }
}

template <int KIND, int ROWS, int CHANNELS, int DOWN, int ACROSS, bool WIDE, bool GROUPED, bool SWIGLU>
int launch_one(const Product& p, uint32_t blocks, hipStream_t s) {
    constexpr uint32_t kLds = 2 * 16 * (ROWS * DOWN + CHANNELS * ACROSS) * kStep;
    constexpr auto kernel = &byte_tiles_kernel<KIND, ROWS, CHANNELS, DOWN, ACROSS, WIDE, GROUPED, SWIGLU>;
    static DeviceOnce ready;
    const int code = ready.run([] { return hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds), "hipFuncSetAttribute"); });
    if (code != ORX_OK) return code;
    ORX_LAUNCH(kernel, dim3(blocks), dim3(64 * DOWN * ACROSS), kLds, s, p);
    return hip_check(hipGetLastError(), "launch byte tiles");
}
template <int KIND, int ROWS, int CHANNELS, int DOWN, int ACROSS, bool GROUPED>
int launch_of(const Product& p, bool swiglu, uint32_t blocks, hipStream_t s) {
    if (p.type == mx::F32)
        return swiglu ? launch_one<KIND, ROWS, CHANNELS, DOWN, ACROSS, true, GROUPED, true>(p, blocks, s) : launch_one<KIND, ROWS, CHANNELS, DOWN, ACROSS, true, GROUPED, false>(p, blocks, s);
    return swiglu ? launch_one<KIND, ROWS, CHANNELS, DOWN, ACROSS, false, GROUPED, true>(p, blocks, s) : launch_one<KIND, ROWS, CHANNELS, DOWN, ACROSS, false, GROUPED, false>(p, blocks, s);
}
template <int KIND, bool GROUPED>
int launch(const Product& p, int rows, bool swiglu, uint32_t blocks, hipStream_t s) {
    return rows == 256   ? launch_of<KIND, 8, 4, 2, 4, GROUPED>(p, swiglu, blocks, s)
           : rows == 128 ? launch_of<KIND, 4, 4, 2, 2, GROUPED>(p, swiglu, blocks, s)
                         : launch_of<KIND, 2, 4, 2, 2, GROUPED>(p, swiglu, blocks, s);
}

}  // namespace

int launch_byte_tiles(const bytes::Product& p, int kind, int rows, int channels, bool grouped, bool swiglu, uint32_t blocks, hipStream_t s) {
    if (kind == F16) return launch<F16, true>(p, rows, swiglu, blocks, s);
    if (kind == BF16) return launch<BF16, true>(p, rows, swiglu, blocks, s);
    return grouped ? launch<I8, true>(p, rows, swiglu, blocks, s) : launch<I8, false>(p, rows, swiglu, blocks, s);
}

}  // namespace orx
