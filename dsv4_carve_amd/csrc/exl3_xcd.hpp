// Which workgroup has which piece of work, so that the workgroups of an XCD have
// neighbouring ones.
#pragma once

#include <hip/hip_runtime.h>

namespace exl3 {

// Workgroups go to the XCDs in turn (workgroup b to XCD b % 8), and what one reads its
// neighbours on the XCD find in L2: so an XCD's workgroups take neighbouring work.
constexpr int XCDS = 8;

// Workgroup b's place where each XCD's workgroups are next to each other.
__host__ __device__ __forceinline__ int by_xcd(int b, int n) {
    const int x = b % XCDS, each = n / XCDS, more = n % XCDS;
    return x * each + (x < more ? x : more) + b / XCDS;
}

// A workgroup a tile: a head's tiles in turn on the XCDs that the head has, or an XCD's heads one after another.  False
// for the workgroups that a launch of tile_grid has more than tiles of all heads.
__host__ __device__ __forceinline__ unsigned tile_grid(int tiles, int heads) { return (unsigned)((tiles + XCDS - 1) / XCDS * XCDS) * heads; }
__host__ __device__ __forceinline__ bool tile_by_xcd(int b, int tiles, int heads, int& tile, int& head) {
    const int x = b % XCDS, i = b / XCDS;
    if (heads < XCDS && XCDS % heads == 0) {
        const int of = XCDS / heads;
        head = x / of;
        tile = i * of + x % of;
    } else if (heads % XCDS == 0) {
        head = x * (heads / XCDS) + i / tiles;
        tile = i % tiles;
        return i / tiles < heads / XCDS;
    } else {
        head = b / tiles;
        tile = b % tiles;
    }
    return tile < tiles && head < heads;
}

}  // namespace exl3
