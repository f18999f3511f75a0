// Host side of the products of many rows with weights by byte tiles (k_byte_tiles.hip; byte_wide_kernel.h, k_byte_wide_*.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "byte_device.h"

namespace orx {

// rows x channels: 256 x 256, 128 x 128, 96 x 128, 64 x 128, 64 x 64 (dense); 128 x 256 with weights straight to registers; 64 x 256 of those (experts)
enum { kTiles256, kTiles128, kTiles96, kTiles64, kTiles64x64, kWide128, kWide64 };

struct TilesShape {
    int rows, channels, threads, lds, to_a_cu;  // to_a_cu: workgroups that a CU holds, by its LDS and registers
};
TilesShape byte_tiles_shape(int kind, int form, bool grouped);
// `blocks` workgroups, each of which takes every blocks-th tile
int launch_byte_tiles_i8(const bytes::Product& p, int form, bool swiglu, uint32_t blocks, hipStream_t s);
int launch_byte_wide_i8(const bytes::Product& p, int form, bool grouped, bool swiglu, uint32_t blocks, hipStream_t s);
int launch_byte_wide_f16(const bytes::Product& p, int form, bool swiglu, uint32_t blocks, hipStream_t s);  // (experts)
int launch_byte_wide_bf16(const bytes::Product& p, int form, bool swiglu, uint32_t blocks, hipStream_t s);
inline int launch_byte_tiles(const bytes::Product& p, int kind, int form, bool grouped, bool swiglu, uint32_t blocks, hipStream_t s) {
    if (kind == bytes::F16) return launch_byte_wide_f16(p, form, swiglu, blocks, s);
    if (kind == bytes::BF16) return launch_byte_wide_bf16(p, form, swiglu, blocks, s);
    return form == kWide128 || form == kWide64 ? launch_byte_wide_i8(p, form, grouped, swiglu, blocks, s) : launch_byte_tiles_i8(p, form, swiglu, blocks, s);
}

}  // namespace orx
