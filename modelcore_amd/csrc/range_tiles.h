// Where the key ranges of a block begin among its tiles. Standard C++ alone, on the device (constexpr) as on the
// host.
#pragma once

#include <cstdint>

namespace mcamd {

// Tile from which on range `part` of `ranges` (at most 65535) lies, of `tiles`: part * tiles / ranges, rounded down.
// That product alone passes 31 bits: a row of 2^30 keys is 2^25 tiles of 32, and there may be 512 ranges.
constexpr int range_tile(int part, int tiles, int ranges) {
  const uint32_t each = uint32_t(tiles) / uint32_t(ranges), rest = uint32_t(tiles) - each * uint32_t(ranges);
  return int(each * uint32_t(part) + rest * uint32_t(part) / uint32_t(ranges));
}

}  // namespace mcamd
