"""The serving operators' size arithmetic (mlx_amd/csrc/extent.h), compiled for
the host, against whole numbers of any size."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "mlx_amd", "csrc", "extent.h")
MOST = 2 ** 64 - 1


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("extent")
    (d / "t.cpp").write_text(f"""#include "{HEADER}"
#include <stdio.h>
int main() {{
    long long rows, stride, row; unsigned long long esz, size, skip;
    while (scanf("%lld %lld %lld %llu %llu %llu", &rows, &stride, &row, &esz, &size, &skip) == 6) {{
        const size_t n = lxh::extent(rows, stride, row, esz);
        printf("%zu %d\\n", n, lxh::holds(size, skip, n));
    }}
}}
""")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", str(d / "t.cpp"),
                    "-o", str(d / "t")], check=True)
    return str(d / "t")


def test_extents_and_buffers(program):
    rng = random.Random(1)
    cases = [(2 ** 22 + 1, 2 ** 40, 16, 4, 64, 0), (2 ** 23 + 1, 2 ** 40, 16, 2, 32, 0), (2 ** 31 - 1, 2 ** 40, 2 ** 31 - 1, 4, 2 ** 40, 0),
             (0, 5, 5, 4, 0, 0), (0, 5, 5, 4, 0, 1), (1, 2 ** 40, 7, 2, 14, 0), (1, 9, 7, 2, 14, 2), (3, 9, 7, 2, 52, 2), (3, 9, 7, 2, 51, 2),
             (5, 9, 0, 2, 0, 0)]
    for _ in range(500):
        row = 2 ** rng.randrange(31) + rng.randrange(3)
        stride = max(row, min(2 ** 40, 2 ** rng.randrange(41) + rng.randrange(3)))
        esz, rows = rng.choice([2, 4]), max(0, 2 ** rng.randrange(31) + rng.randrange(3) - 2)
        n = ((rows - 1) * stride + row) * esz if rows else 0
        skip = rng.choice([0, 0, 2 ** rng.randrange(42) * esz])
        cases.append((rows, stride, row, esz, max(0, min(2 ** 62, n + skip + rng.choice([-1, 0, 1, -(2 ** 64)]))), skip))
    out = subprocess.run([program], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True).stdout
    got = [tuple(map(int, line.split())) for line in out.splitlines()]
    assert len(got) == len(cases)
    for c, (n, held) in zip(cases, got):
        rows, stride, row, esz, size, skip = c
        want = ((rows - 1) * stride + row) * esz if rows and row else 0
        big = (rows - 1) * stride + row >= 2 ** 63 or want > MOST
        assert n == (MOST if big else want), c
        assert held == (skip + want <= size), c
