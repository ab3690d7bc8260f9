"""The chunk attention's places of tiles, stages and ranges
(mlx_amd/csrc/chunk_places.h), compiled for the host, against whole numbers of
any size: up to lengths of 2^31 - 1, whose last stages end behind 2^31."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "mlx_amd", "csrc", "chunk_places.h")
STAGES = [32, 64, 128]


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("places")
    (d / "t.cpp").write_text(f"""#include "{HEADER}"
#include <stdio.h>
#include <string.h>
using namespace lxq::chunk;
static void places() {{
    int s0, s1, pos, n, tile, tb, window, st, u, off, len, row;
    while (scanf("%d %d %d %d %d %d %d %d %d %d %d %d", &s0, &s1, &pos, &n, &tile, &tb, &window, &st, &u, &off, &len, &row) == 12) {{
        const Tile t = tile_at(s0, s1, pos, n, tile, tb, window, st);
        int from, to, a, b;
        seen_by(t, row, window, from, to);
        const uint32_t at = stage_at(t, u, st) + (uint32_t)off;
        steps_inside(stage_at(t, 0, st) + (uint32_t)off, len, st, from, to, a, b);
        printf("%d %d %d %d %d %d %d %d %u %u %d %d %d %d %d %d %d\\n", t.first, t.m, t.base, t.end, t.units, from, to,
               (int)t.pos, stage_at(t, u, st), stages_end(t, u, st), is_whole(t, at, len), is_seen(at, len, from, to),
               is_inside(at, len, from, to), or_last(t, at), or_last_run(t, at, 8), a, b);
    }}
}}
static void cuts() {{
    unsigned long long units, u;
    int log;
    while (scanf("%llu %d %llu", &units, &log, &u) == 3) {{
        const Ranges r(units, log);
        const int w = r.of(u);
        printf("%d %d %llu %llu\\n", r.log, w, (unsigned long long)r.first(w), (unsigned long long)r.first(w + 1));
    }}
}}
int main(int, char** v) {{
    strcmp(v[1], "cuts") ? places() : cuts();
}}
""")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", str(d / "t.cpp"),
                    "-o", str(d / "t")], check=True)
    return str(d / "t")


def ask(program, what, cases):
    out = subprocess.run([program, what], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True).stdout
    got = [tuple(map(int, line.split())) for line in out.splitlines()]
    assert len(got) == len(cases)
    return zip(cases, got)


def cases():
    rng = random.Random(1)
    for below in [*range(1, 300), 5000, 2 ** 20, 2 ** 30, 2 ** 31 - 1, 2 ** 31 - 100]:
        for st in STAGES:
            for window in (0, 1, 16, 100, 2 ** 31 - 1):
                tb, new = rng.choice([1, 7, 64, 256]), rng.choice([1, 1, 2, 60, 300])
                n = 2 ** 31 - below
                new = min(new, n)
                tile = rng.randrange(-(-new // tb) + 1)
                # the last stages, and any
                m = min(tb, max(0, new - tile * tb))
                end, first = min(n - new + tile * tb + m, n), n - new + tile * tb
                base = (first + 1 - window) & ~15 if window and first + 1 > window else 0
                units = max(1, -(-(end - base) // st))
                for u in {units - 1, units, max(0, units - 3), rng.randrange(units + 1)}:
                    yield (5, 5 + new, n - new, n, tile, tb, window, st, u, rng.choice([0, 32, 64, 96]) % st, rng.choice([32, 64]), rng.randrange(max(1, m)))


def test_places(program):
    for c, got in ask(program, "places", list(cases())):
        s0, s1, pos, n, tile, tb, window, st, u, off, length, row = c
        m = min(tb, max(0, s1 - s0 - tile * tb))
        if m == 0:
            assert got[1] == 0 and got[4] == 1 and got[3] <= 0, c
            continue
        p = pos + tile * tb
        end = min(p + m, n)
        base = (p + 1 - window) & ~15 if window and p + 1 > window else 0
        units = -(-(end - base) // st) if end > base else 1
        start, to = max(0, p + row + 1 - window) if window else 0, min(p + row + 1, n)
        at = base + u * st + off
        assert got[:8] == (s0 + tile * tb, m, base, end, units, start, to, p), c
        assert got[8] == base + u * st and got[9] == min(base + u * st, end), c
        assert got[10] == (at + length <= end) and got[11] == (at < to and at + length > start) and got[12] == (at >= start and at + length <= to), c
        assert got[13] == (at if at < end else end - 1) and got[14] == (at if at < end else (end - 1) // 8 * 8), c
        inside = [j for j in {0, 1, units - 1, units, got[15] - 1, got[15], got[16] - 1, got[16], (got[15] + got[16]) // 2} if j >= 0]
        for j in inside:
            t0 = base + off + j * st
            assert (got[15] <= j < got[16]) == (t0 >= start and t0 + length <= to), (c, j, got)


def test_cuts(program):
    """The range of a unit is the one that holds it."""
    rng = random.Random(2)
    units = [1, 2, 3, 5, 255, 256, 257, 1000, 2 ** 24, 2 ** 31 - 1, (2 ** 31 - 1) * 1024, *(rng.randrange(1, 2 ** rng.randrange(1, 42)) for _ in range(300))]
    every = [(n, log, u) for n in units for log in (0, 3, 8) for u in {0, n - 1, n // 2, rng.randrange(n)}]
    for (n, log, u), (cut, w, lo, hi) in ask(program, "cuts", every):
        assert cut == min(log, n.bit_length() - 1)
        assert 0 <= w < 2 ** cut and lo == n * w >> cut and hi == n * (w + 1) >> cut and lo <= u < hi, (n, log, u)


def test_units_behind_all(program):
    """Starts that decrease, which no call may have, lay tiles behind the last unit: their parts are taken for the last
    range's, so that none is looked for behind the workspace."""
    rng = random.Random(3)
    every = [(n, log, n + more) for n in (1, 3, 256, 1000, 2 ** 31 - 1) for log in (0, 3, 8) for more in (0, 1, 100, 2 ** 31, rng.randrange(2 ** 40))]
    for (n, log, u), (cut, w, lo, hi) in ask(program, "cuts", every):
        assert w == 2 ** cut - 1 and hi == n, (n, log, u)
