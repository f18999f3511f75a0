// Host side of the MXFP4 products from LDS (k_mx_tiles.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "mx_device.h"

namespace orx {

// Tiles of 256 x 256, 128 x 128 or 64 x 128 rows x channels; `blocks` workgroups, each of which takes every blocks-th tile.  Two halves of K (not 256 x 256, not experts, K of two steps
// and more): a workgroup to a tile.
int launch_mx_tiles(const mx::Product& p, int rows, int channels, int halves, bool grouped, bool swiglu, uint32_t blocks, hipStream_t s);
inline uint32_t mx_tiles_lds(int rows, int channels, int halves) { return 2u * halves * (rows + channels) * 136u; }
inline uint32_t mx_tiles_threads(int rows, int halves) { return rows == 256 ? 512 : 256 * halves; }
// workgroups that a CU holds (its LDS)
inline uint32_t mx_tiles_to_a_cu(int rows) { return rows == 256 ? 1 : rows == 128 ? 2 : 3; }

}  // namespace orx
