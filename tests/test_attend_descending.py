"""Steps whose starts do not ascend: units of the work can pass 32 bits then, so that two requests have the same one (no GPU)."""
import subprocess
from pathlib import Path

import pytest

import test_mma_waitcounts as wc

PROGRAM = """
#include "attend_plan.hpp"
#include <cstdio>
#include <vector>
using namespace splosh;
int main() {
    // 4096 requests of up to 4096 rows and 32768 tokens, four key/value heads of six queries each, tiles of 16 and units of 128 keys.
    const int requests = 4096, rows = 4096, page = 256, pages = 128;
    const TileShape t = tile_shape(16, 128, 3, 6, 4, 256);
    for (int down = 0; down < 3; ++down) {
        std::vector<int32_t> starts(requests + 1), lengths(requests, page * pages);
        for (int r = 0; r <= requests; ++r) starts[r] = down == 1 ? (r % 2 ? rows : 0) : down == 2 ? (r < 9 ? -r : r < 99 ? r : 3 * rows - r) : r;
        const PackedView p{starts.data(), lengths.data(), nullptr, pages, pages, requests, rows};
        int64_t total = 0;
        bool sound = true;
        for (int r = 0; r < requests; ++r) {
            const Span s = own_span(p, page, 0, r);
            total += (int64_t)t.heads * units_before(s, t, tiles_of(s, t));
            sound &= ascends(p, r);
        }
        const int64_t segments = most_segments(requests, rows, 24, 4, 16);
        // what the host asks of a call (attend_fits), whether the units fit, and whether the kernels compute such a step
        printf("%d %d %d\\n", (int)(segments * (page * pages / t.keys + 2 + t.extra) < INT32_MAX), (int)(total < INT32_MAX), (int)sound);
    }
}
"""


@pytest.mark.skipif(not Path(wc.HIPCC).exists(), reason="needs hipcc")
def test_units_of_descending_starts(tmp_path):
    source, program = tmp_path / "descending.cpp", tmp_path / "descending"
    source.write_text(PROGRAM)
    subprocess.run([wc.HIPCC, "-x", "hip", "--offload-arch=gfx950", "-O1", "-std=c++17", f"-I{wc.ROOT / 'include'}", f"-I{wc.ROOT / 'splosh_amd/csrc'}",
                    str(source), "-o", str(program)], check=True, capture_output=True)
    up, down, outside = (tuple(map(int, line.split())) for line in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert up == (1, 1, 1)
    assert down == (1, 0, 0)
    assert outside == (1, 1, 1)  # (below 0 and past the rows, in any order, they are all the same)
