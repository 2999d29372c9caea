"""How a segment of attention's work is cut over workgroups: the pieces with keys tile them exactly, the first of them knows their count, and no two pieces
that are joined leave their results in one slot (no GPU)."""
import random
import subprocess
from pathlib import Path

import pytest

import test_mma_waitcounts as wc

PROGRAM = """
#include "attend_plan.hpp"
#include <cstdio>
#include <set>
#include <vector>
using namespace splosh;
int main() {
    int requests, rows, shared, table_pages, page, group, heads, tile_rows, keys, extra, workgroups, partial, prefix;
    while (scanf("%d %d %d %d %d %d %d %d %d %d %d %d %d", &requests, &rows, &shared, &table_pages, &page, &group, &heads, &tile_rows, &keys, &extra, &workgroups, &partial, &prefix) == 13) {
        std::vector<int32_t> starts(requests + 1), lengths(requests);
        for (auto &x : starts) if (scanf("%d", &x) != 1) return 1;
        for (auto &x : lengths) if (scanf("%d", &x) != 1) return 1;
        const PackedView p{starts.data(), lengths.data(), nullptr, table_pages, table_pages, requests, rows};
        const TileShape t = tile_shape(tile_rows, keys, extra, group, heads, workgroups);
        struct Segment { Span span; int tile; };
        std::vector<Segment> all;
        for (int r = 0; r < (prefix ? 1 : requests); ++r) {
            const Span s = prefix ? prefix_span(p, shared) : own_span(p, page, shared, r);
            for (int h = 0; h < heads; ++h)
                for (int i = 0; i < tiles_of(s, t); ++i) all.push_back({s, i});
        }
        int total = 0;
        for (auto &x : all) total += tile_units(x.span, t, x.tile);
        const int64_t most = most_segments(prefix ? 1 : requests, rows, (int64_t)heads * group, heads, tile_rows), first_slots = partial ? most : workgroups;
        const int sharers = sharers_of(total, workgroups);
        long long bad = (int64_t)all.size() > most;
        std::vector<int> blocks(all.size(), 0), pieces(all.size(), 0), count(all.size(), -1), first_workgroup(all.size(), -1), last_workgroup(all.size(), -1);
        std::set<int> slots;
        size_t segment = 0;
        int offset = 0;
        for (int w = 0; w < sharers; ++w) {
            int unit = first_unit(total, sharers, w);
            const int end = first_unit(total, sharers, w + 1);
            while (unit < end) {
                const Segment &x = all[segment];
                const Cut c = cut_of(x.span, t, x.tile, (int)segment, offset, unit, end, w, sharers, total, partial, first_slots);
                if (c.take <= 0) { printf("stuck\\n"); return 1; }
                if (c.any) {
                    const bool first = pieces[segment] == 0;
                    if (c.first_block != blocks[segment]) ++bad;                  // where the last piece ended
                    blocks[segment] += c.blocks;
                    if (first != (c.count > 0)) ++bad;
                    if (first) count[segment] = c.count, first_workgroup[segment] = w;
                    else if (w != last_workgroup[segment] + 1) ++bad;             // their workgroups are consecutive, ...
                    last_workgroup[segment] = w, ++pieces[segment];
                    if (!c.direct) {
                        const int64_t want = first ? (partial ? (int64_t)segment : w) : first_slots + first_workgroup[segment] + pieces[segment] - 1;
                        if (c.slot != want || c.slot < 0 || c.slot >= first_slots + workgroups) ++bad;  // ... which is how the joining launch finds their slots
                        if (!slots.insert(c.slot).second) ++bad;
                    } else if (partial || c.count != 1) ++bad;
                } else if (c.blocks) ++bad;
                unit += c.take, offset += c.take;
                if (offset == tile_units(x.span, t, x.tile)) offset = 0, ++segment;
            }
        }
        if (segment != all.size() || offset) ++bad;
        for (size_t i = 0; i < all.size(); ++i) {
            const int seen = tile_end(all[i].span, t, all[i].tile) - all[i].span.from;
            if (blocks[i] != (seen > 0 ? (seen + kBlock - 1) / kBlock : 0) || count[i] != pieces[i] || pieces[i] < 1) ++bad;
        }
        printf("%lld\\n", bad);
    }
}
"""


@pytest.mark.skipif(not Path(wc.HIPCC).exists(), reason="needs hipcc")
def test_cuts(tmp_path):
    source, program = tmp_path / "cuts.cpp", tmp_path / "cuts"
    source.write_text(PROGRAM)
    subprocess.run([wc.HIPCC, "-x", "hip", "--offload-arch=gfx950", "-O1", "-std=c++17", f"-I{wc.ROOT / 'include'}", f"-I{wc.ROOT / 'splosh_amd/csrc'}",
                    str(source), "-o", str(program)], check=True, capture_output=True)
    rng, lines = random.Random(3), []
    # (rows, keys of a unit, units beside the keys, workgroups) as the kernels are launched, and others
    shapes = [(16 * n, 128, 3, w) for n in (1, 2, 3, 4) for w in (256, 512)] + [(256, 64, 5, 256), (256, 64, 1, 256), (256, 128, 3, 256), (256, 128, 1, 256)]
    for turn in range(600):
        requests, page = rng.choice([1, 2, 7, 64, 300]), 32 * rng.randint(1, 8)
        table_pages = rng.randint(1, 60)
        shared = page * rng.choice([0, rng.randint(1, table_pages)])
        runs = [rng.choice([0, 1, 1, 4, rng.randint(0, 90), rng.randint(0, 900) if requests < 8 else 0]) for _ in range(requests)]
        runs[0] = max(runs[0], 1)
        starts = [sum(runs[:i]) for i in range(requests + 1)]
        rows = max(1, starts[-1] + rng.randint(-2, 5))
        lengths = [min(max(-3, shared * (rng.random() < 0.8) + n + rng.choice([0, -1, rng.randint(0, table_pages * page)])), 2 ** 30) for n in runs]
        tile, keys, extra, workgroups = rng.choice(shapes) if turn % 4 else (rng.choice([16, 48, 256]), rng.choice([64, 96, 128]), rng.choice([0, 1, 3, 5, 9]), rng.choice([8, 64, 304]))
        prefix = shared > 0 and rng.random() < 0.5
        partial = prefix or shared > 0
        lines.append(" ".join(map(str, [requests, rows, shared, table_pages, page, rng.randint(1, 12), rng.randint(1, 8), tile, keys, extra, workgroups, int(partial), int(prefix),
                                        *starts, *lengths])))
    got = subprocess.run([str(program)], input="\n".join(lines), check=True, capture_output=True, text=True).stdout.split()
    assert len(got) == len(lines)
    for line, bad in zip(lines, got):
        assert bad == "0", line
