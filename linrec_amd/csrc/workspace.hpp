// How a look-back workspace is laid out, a function of its size alone: shared by every launch that uses one.
#pragma once
#include <cstddef>
#include <cstdint>

#include "tile_kernel.hpp"  // CarryHeader

namespace linrec {

// Workspace = header | completion counters | descriptors.  The counter tree of T tiles needs
// sum_l ceil(T / 32^l) < T/31 + 8 words; T/16 + 64 words are reserved.
struct WorkspaceLayout {
  size_t counters_offset, desc_offset;
  int64_t tiles;  // descriptors (and tiles of one launch) the workspace has room for
};

inline size_t counter_bytes_for(int64_t tiles) { return ((size_t(tiles) / 16 + 64) * 4 + 15) & ~size_t(15); }

// (All of this in the lower half of the buffer; the upper half is scratch without a life beyond
// one call: the maps of the segmented column launches.  A map must never land where a later launch
// reads descriptors, whose validity is a bit pattern.)
inline WorkspaceLayout workspace_layout(size_t whole_bytes) {
  const size_t bytes = whole_bytes / 2;
  WorkspaceLayout lay{sizeof(CarryHeader), 0, 0};
  const size_t fixed = sizeof(CarryHeader) + 64 * 4 + 16;
  if (bytes <= fixed) return lay;
  // 16 bytes of descriptors and a quarter byte of counters per tile
  int64_t tiles = int64_t((bytes - fixed) * 4 / 65);
  while (tiles > 0 && sizeof(CarryHeader) + counter_bytes_for(tiles) + size_t(tiles) * 16 > bytes) --tiles;
  lay.tiles = tiles;
  lay.desc_offset = sizeof(CarryHeader) + counter_bytes_for(tiles);
  return lay;
}

}  // namespace linrec
