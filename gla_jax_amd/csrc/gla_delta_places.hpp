// Places in what the passes of the gated delta rule leave for each other.  Plain arithmetic, which a host program can go through without a GPU.
#pragma once

#include <stdint.h>

namespace gla {

// 16 features each, in pairs (of features pi: gla_chunk_common.hpp)
constexpr int delta_state_tiles(int64_t DK) { return (int)((DK + 31) / 32 * 2); }

// A state lies as [columns / 16][tiles][256] floats.  Of those of a workgroup's columns col0 .. the lines of 128 bytes that a lane of wave w touches, two tiles
// a wave and 16 columns for 16 lanes: bytes from the state's beginning, or a place behind any state.  (Columns behind the last lie behind the state's end as well.)
constexpr unsigned delta_touched_line(int DK, int col0, int columns, int w, int lane)
{
    return 2 * w < delta_state_tiles(DK) && 16 * (lane >> 4) < columns
               ? 4u * (unsigned)(((col0 >> 4) + (lane >> 4)) * delta_state_tiles(DK) * 256 + 512 * w + 32 * (lane & 15))
               : 0x7fffff00u;
}

}  // namespace gla
