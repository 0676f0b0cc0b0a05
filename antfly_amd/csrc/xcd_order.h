// Which workgroup has which share of an attention over the 8-bit cache.  Workgroups go round the eight XCDs in turn; a chunk of
// neighbouring shares lies on one of them, whose L2 then holds the keys that they have in common.
#pragma once

#include <stdint.h>

namespace afhip {

// Shares of a chunk, of `total`, that are numbered by row tiles, within key heads, within parts or requests.  The row tiles of a key head read the
// same keys, the heads of a part lines of scales together, so a part is a chunk while parts are small or many (64 requests of 100 to
// 4000 keys, 8 key heads: 67 us, 71 a head by itself).  Beyond that a part would fill an XCD while others idle: 4000 new tokens of one
// request, 8 key heads, 2896 us as one chunk, 396 head by head, 402 tile by tile; 1 token on 700 keys, 64 key heads, 28 and 13 us; 20
// requests of 17 tokens on 3000 keys 108 and 73.  Heads fill the XCDs evenly by eights, otherwise tiles do (2000 tokens, 4 key heads: 874
// us, 234 by heads, 140 by tiles).
constexpr uint64_t xcd_chunk(uint64_t row_tiles, uint64_t heads, uint64_t total) {
    const uint64_t part = row_tiles * heads;
    if (part <= 16 || (row_tiles == 1 && total >= 32 * part)) return part;
    return heads % 8 == 0 ? row_tiles : 1;
}

constexpr uint32_t xcd_share(uint32_t workgroup, uint32_t chunk) {
    const uint32_t turn = workgroup >> 3;
    return (turn / chunk * 8 + (workgroup & 7)) * chunk + turn % chunk;
}

}  // namespace afhip
