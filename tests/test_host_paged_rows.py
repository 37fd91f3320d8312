"""Which token a thread of a cache write takes, up to the largest grids: the kernels' own
arithmetic, compiled for the host."""

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "dit_sparse_atten_amd" / "csrc"

MAIN = """
#include <cstdio>
#include <cstdlib>
#include "paged_rows.h"
int main(int argc, char** argv) {
  for (int i = 1; i + 3 < argc; i += 4)
    std::printf("%d\\n", paged::token_of((uint32_t)std::strtoul(argv[i], nullptr, 10),
                                        std::atoi(argv[i + 1]), std::atoi(argv[i + 2]),
                                        std::atoi(argv[i + 3])));
}
"""


@pytest.fixture(scope="module")
def token_of(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    folder = tmp_path_factory.mktemp("rows")
    (folder / "main.cpp").write_text(MAIN)
    program = folder / "main"
    subprocess.run([compiler, "-std=c++17", "-I", str(CSRC), "-o", str(program),
                    str(folder / "main.cpp")], check=True)

    def run(cases):
        args = [str(x) for case in cases for x in case]
        out = subprocess.run([str(program), *args], check=True, capture_output=True, text=True)
        return [int(x) for x in out.stdout.split()]

    return run


def _groups(tokens, rows):
    return -(-tokens // rows)


@pytest.mark.parametrize("tokens", [1, 63, 64, 257, 57600, (1 << 29) + 1, (1 << 30) - 64])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 96, 128])
def test_tokens_of_a_packing_write(token_of, tokens, dim):
    """The grid counts workgroups of the packing walk; the queries' walk takes more tokens a
    workgroup.  Every token once, none outside the call."""
    packing = 256 // (4 * -(-dim // 32))
    turning = 256 // ((dim // 8 + 1) // 2)
    groups = _groups(tokens, packing)
    assert turning >= packing
    for rows in (packing, turning):
        last = _groups(tokens, rows) - 1
        at = sorted({0, last // 2, last, min(last + 1, groups - 1), groups // 2, groups - 1,
                     min(1 << 23, groups - 1), min((1 << 23) + 1, groups - 1)})
        cases = [(g, rows, row, tokens) for g in at for row in (0, 1, rows - 1, rows, 255)]
        for (g, _, row, _), got in zip(cases, token_of(cases)):
            token = g * rows + row
            assert got == (token if row < rows and token < tokens else -1), (g, rows, row)


def test_the_last_token_of_all(token_of):
    most = (1 << 31) - 1
    cases = [((1 << 23) - 1, 256, 254, most), ((1 << 23) - 1, 256, 255, most),
             (1 << 23, 256, 0, most), ((1 << 24) - 1, 256, 255, most), ((1 << 32) - 1, 256, 0, 5)]
    assert token_of(cases) == [most - 1, -1, -1, -1, -1]
