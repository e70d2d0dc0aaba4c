"""Which lines of the states the backward walk of chunk_delta touches ahead, gone through on the host from the header that the kernels take them from."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gla_jax_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "gla_delta_places.hpp"
int main()
{
    for (int DK = 16; DK <= 128; DK += 16)
        for (int DV = 16; DV <= 256; DV += 16)
            for (int columns = 16; columns <= 32; columns += 16) {
                const unsigned bytes = 16u * gla::delta_state_tiles(DK) * DV * 4;      // of a state
                std::vector<int> touched(bytes / 128);
                for (int col0 = 0; col0 < DV; col0 += columns) {
                    // the workgroup's columns lie in one piece
                    const unsigned first = bytes / DV * col0, end = first + bytes / DV * columns;
                    for (int w = 0; w < 4; ++w)
                        for (int lane = 0; lane < 64; ++lane) {
                            const unsigned at = PLACE;
                            if (at + 4 > bytes) continue;       // the load is bounded by the state: nothing is read
                            if (at < first || at >= end || at % 128) return printf("%d %d %d: %u outside of %u .. %u\n", DK, DV, columns, at, first, end), 1;
                            ++touched[at / 128];
                        }
                }
                for (unsigned i = 0; i < touched.size(); ++i)
                    if (touched[i] != 1) return printf("%d %d %d: line %u touched %d times\n", DK, DV, columns, i, touched[i]), 1;
            }
    return puts("each line once"), 0;
}
"""


# without a lane's own group of columns: columns 2r and 2r + 1 of 32 belong to the group behind for r >= 8
OWN_COLUMN = """2 * w < gla::delta_state_tiles(DK) ? 4u * (unsigned)((((col0 + columns / 16 * (lane & 15)) >> 4) * gla::delta_state_tiles(DK)) * 256
              + ((columns / 16 * (lane & 15) & 15) - (lane & 15)) * 4 + 512 * w + 32 * (lane & 15)) : 0x7fffff00u"""


def gone_through(tmp_path, place):
    if not shutil.which("g++"):
        pytest.skip("needs a C++ compiler")
    (tmp_path / "places.cpp").write_text(PROGRAM.replace("PLACE", place))
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, str(tmp_path / "places.cpp"), "-o", str(tmp_path / "places")], check=True)
    r = subprocess.run([str(tmp_path / "places")], capture_output=True, text=True)
    return r.returncode, r.stdout.strip()


def test_every_line_of_a_state_is_touched_once_and_nothing_else(tmp_path):
    assert gone_through(tmp_path, "gla::delta_touched_line(DK, col0, columns, w, lane)") == (0, "each line once")


def test_places_by_a_lanes_own_column_are_seen(tmp_path):
    code, said = gone_through(tmp_path, OWN_COLUMN)
    assert code == 1 and ("outside" in said or "touched" in said)
