// Internal interface of the piles (cw_piles.hip): picks sorted by expert, and the tiles of neighbouring positions that the experts'
// products take.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>

#include "cw_common.h"

namespace cw {

// A tile: m positions from pos0, all of one expert, which has `of` tiles, the first of them tile `first`. Expert E: positions of no
// expert.
struct PileTile {
    int expert, pos0, m, first, of;
};
constexpr int PILE_TILE = 128;  // positions of a tile, at most
constexpr int PILE_MAX_EXPERTS = 1024;
inline int64_t pile_max_tiles(int64_t picks, int experts) { return (picks + PILE_TILE - 1) / PILE_TILE + std::min<int64_t>(experts + 1, picks); }
// the tiles' buffer: their count, then (from byte 16) the tiles
inline int64_t pile_tiles_bytes(int64_t picks, int experts) { return 16 + pile_max_tiles(picks, experts) * (int64_t)sizeof(PileTile); }
__host__ __device__ __forceinline__ const PileTile *pile_tiles(const void *tiles) { return (const PileTile *)((const uint8_t *)tiles + 16); }

// out (of type dtype) = sum_j w y of f32 rows (w not NULL)
int from_piles_f32(int dtype, const float *rows, const float *w, int64_t T, int K, int E, int64_t h, const int *place, const int *offsets, void *out,
                   hipStream_t s);

}  // namespace cw
