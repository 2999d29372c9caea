"""Where rows stand, from the host and device functions that the operators share: attention's spans and the cache's rows agree (no GPU)."""
import random
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
    int requests, rows;
    while (scanf("%d %d", &requests, &rows) == 2) {
        std::vector<int32_t> starts(requests + 1), lengths(requests);
        for (auto &x : starts) if (scanf("%d", &x) != 1) return 1;
        for (auto &x : lengths) if (scanf("%d", &x) != 1) return 1;
        const PackedView p{starts.data(), lengths.data(), nullptr, 1 << 20, 1 << 20, requests, rows};
        for (int r = 0; r < requests; ++r) {
            const Span s = own_span(p, 32, 0, r);
            for (int row = s.begin; row < s.begin + s.n; ++row) printf("%d %d %d %d\\n", r, row, position_in(p, r, row), s.first + row - s.begin);
        }
        puts("-");
    }
}
"""


@pytest.mark.skipif(not Path(wc.HIPCC).exists(), reason="needs hipcc")
def test_positions(tmp_path):
    source, program = tmp_path / "positions.cpp", tmp_path / "positions"
    source.write_text(PROGRAM)
    subprocess.run([wc.HIPCC, "-x", "hip", "--offload-arch=gfx950", "-O1", "-std=c++17", f"-I{wc.ROOT / 'include'}", f"-I{wc.ROOT / 'splosh_amd/csrc'}",
                    str(source), "-o", str(program)], check=True, capture_output=True)
    rng, steps = random.Random(2), []
    for _ in range(200):
        requests = rng.choice([1, 2, 5])
        starts = [0]
        for _ in range(requests):
            starts.append(starts[-1] + rng.choice([0, 1, 4, 30]))
        rows = max(1, starts[-1] + rng.choice([0, 3, -1, -2, -10]))
        if rng.random() < 0.2:
            starts[0] = -3
        lengths = [rng.choice([rng.randint(0, 2000), rng.randint(0, 2000), -5, 2 ** 31 - 1, -2 ** 31, -2 ** 31 + 7]) for _ in range(requests)]
        steps.append((starts, lengths, rows))
    text = "\n".join(" ".join(map(str, [len(lengths), rows, *starts, *lengths])) for starts, lengths, rows in steps)
    blocks = subprocess.run([str(program)], input=text, check=True, capture_output=True, text=True).stdout.split("-\n")
    for (starts, lengths, rows), block in zip(steps, blocks):
        clipped = [min(max(s, 0), rows) for s in starts]
        lines = [tuple(map(int, line.split())) for line in block.splitlines()]
        assert [line[:2] for line in lines] == [(r, m) for r in range(len(lengths)) for m in range(clipped[r], clipped[r + 1])]
        for r, m, position, span in lines:
            want = lengths[r] - clipped[r + 1] + m
            assert position == max(want, -2 ** 31), (starts, lengths, rows, r, m)
            # (Attention takes a length past either end of what a table holds as one that sees nothing, or everything.)
            assert span == position or (want < 0 and span < 0) or (want > 2 ** 30 and span > 2 ** 30), (starts, lengths, rows, r, m)
