"""How attention shares a step's work out: every unit of every segment belongs to one workgroup, shares are even, a workgroup
begins in the middle of one segment at most, and the slots hold all segments (no GPU)."""
import random
import subprocess
from pathlib import Path

import pytest

import test_mma_waitcounts as wc

PROGRAM = """
#include "attend_plan.hpp"
#include <cstdio>
#include <vector>
#include <climits>
using namespace splosh;
int main() {
    long long wrong = 0;  // of the divisions
    for (int d : {1, 2, 3, 5, 6, 7, 8, 12, 16, 31, 33, 48, 64, 96, 100, 255, 256, 257, 1023, 1024, 1000000, (1 << 25) - 1, 1 << 25})
        for (int64_t x : {(int64_t)0, (int64_t)1, (int64_t)2, (int64_t)d - 1, (int64_t)d, (int64_t)d + 1, (int64_t)7 * d - 1, (int64_t)7 * d, (int64_t)(1 << 30) - 1, (int64_t)1 << 30,
                          (int64_t)INT32_MAX / d * d - 1, (int64_t)INT32_MAX / d * d, (int64_t)INT32_MAX})
            if (x >= 0 && x <= INT32_MAX && divisor(d).of((int)x) != (int)x / d) ++wrong;
    printf("%lld\\n", wrong);
    int requests, rows, shared, table_pages, page, group, heads, tile_rows, keys, extra, workgroups;
    while (scanf("%d %d %d %d %d %d %d %d %d %d %d", &requests, &rows, &shared, &table_pages, &page, &group, &heads, &tile_rows, &keys, &extra, &workgroups) == 11) {
        std::vector<int32_t> starts(requests + 1), lengths(requests);
        for (auto &x : starts) if (scanf("%d", &x) != 1) return 1;
        for (auto &x : lengths) if (scanf("%d", &x) != 1) return 1;
        const PackedView p{starts.data(), lengths.data(), nullptr, table_pages, table_pages, requests, rows};
        const TileShape t = tile_shape(tile_rows, keys, extra, group, heads, workgroups);
        std::vector<int> units;  // of each segment
        long long bad = 0;
        for (int part = 0; part < (shared ? 2 : 1); ++part) {
            units.clear();
            for (int r = 0; r < (part ? 1 : requests); ++r) {
                const Span s = part ? prefix_span(p, shared) : own_span(p, page, shared, r);
                if (s.begin < 0 || s.n < 0 || s.begin + s.n > rows) ++bad;
                for (int h = 0; h < heads; ++h)
                    for (int i = 0; i < tiles_of(s, t); ++i) {
                        units.push_back(tile_units(s, t, i));
                        if (tile_end(s, t, i) > s.to || (tile_end(s, t, i) > s.from && (int64_t)(units.back() - extra) * keys < tile_end(s, t, i) - s.from)) ++bad;
                    }
                if (heads * units_before(s, t, tiles_of(s, t)) < 0) ++bad;
            }
            if ((int64_t)units.size() > most_segments(part ? 1 : requests, rows, (int64_t)heads * group, heads, tile_rows)) ++bad;
            for (int u : units) if (u <= extra) ++bad;
            int64_t sum = 0;
            for (int u : units) sum += u;
            if (sum > INT32_MAX) continue;  // (such a call is refused)
            const int total = (int)sum;
            if (total == 0) continue;
            int begin = 0, most = 0;
            const int sharers = sharers_of(total, workgroups);
            for (int w = 0; w < sharers; ++w) {
                const int a = first_unit(total, sharers, w), b = first_unit(total, sharers, w + 1);
                if (a != begin || b <= a) ++bad;
                for (int u = a; u < b; ++u) if (owner_of(total, sharers, u) != w) ++bad;
                most = b - a > most ? b - a : most;
                begin = b;
            }
            if (begin != total || most > (sum + workgroups - 1) / workgroups) ++bad;
        }
        printf("%lld\\n", bad);
    }
}
"""


@pytest.mark.skipif(not Path(wc.HIPCC).exists(), reason="needs hipcc")
def test_shares(tmp_path):
    source, program = tmp_path / "shares.cpp", tmp_path / "shares"
    source.write_text(PROGRAM)
    subprocess.run([wc.HIPCC, "-x", "hip", "--offload-arch=gfx950", "-O1", "-std=c++17", f"-I{wc.ROOT / 'include'}", f"-I{wc.ROOT / 'splosh_amd/csrc'}",
                    str(source), "-o", str(program)], check=True, capture_output=True)
    rng, lines = random.Random(1), []
    for _ in range(400):
        requests, page = rng.choice([1, 2, 7, 64, 300]), 32 * rng.randint(1, 8)
        table_pages = rng.randint(1, 40)
        shared = page * rng.choice([0, 0, rng.randint(1, table_pages)])
        runs = [rng.choice([0, 1, 1, 4, rng.randint(0, 90)]) for _ in range(requests)]
        starts = [sum(runs[:i]) for i in range(requests + 1)]
        rows = max(1, starts[-1] + rng.randint(0, 5))
        lengths = [max(0, n + rng.choice([0, -1, -5, rng.randint(0, table_pages * page), rng.randint(-2 ** 31 + 100, 2 ** 31 - 400)])) for n in runs]
        lengths = [min(n, 2 ** 31 - 1) for n in lengths]
        shape = [rng.randint(1, 12), rng.randint(1, 8), rng.choice([16, 32, 48, 64, 256]), rng.choice([64, 96, 128]), rng.choice([0, 1, 3]), rng.choice([8, 64, 256, 512])]
        lines.append(" ".join(map(str, [requests, rows, shared, table_pages, page, *shape, *starts, *lengths])))
    got = subprocess.run([str(program)], input="\n".join(lines), check=True, capture_output=True, text=True).stdout.split()
    assert got.pop(0) == "0" and len(got) == len(lines)
    for line, bad in zip(lines, got):
        assert bad == "0", line
