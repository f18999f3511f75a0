// Host side of the products by byte tiles from LDS (k_byte_tiles.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "byte_device.h"

namespace orx {

// Tiles of 256 x 256, 128 x 128 or 64 x 128 rows x channels; `blocks` workgroups, each of which takes every blocks-th tile.
int launch_byte_tiles(const bytes::Product& p, int kind, int rows, int channels, bool grouped, bool swiglu, uint32_t blocks, hipStream_t s);
inline uint32_t byte_tiles_lds(int rows, int channels) { return 2u * (rows + channels) * bytes::kStep; }
inline uint32_t byte_tiles_threads(int rows) { return rows == 256 ? 512 : 256; }
// workgroups that a CU holds (its LDS)
inline uint32_t byte_tiles_to_a_cu(int rows) { return rows == 256 ? 1 : rows == 128 ? 2 : 3; }

}  // namespace orx
