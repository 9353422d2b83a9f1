"""How the work on shared beginnings is cut, by the header that the kernels use, compiled for the host: a (tile, kv head) never has more
units than attention_rows.cu has room to weigh, and the units of a launch are never more than the partial results have room for."""
import random
import subprocess

import pytest

from holon_b200.kernels.build import BuildError, CSRC, nvcc_path

try:
    nvcc_path()
except BuildError:
    pytest.skip("nvcc is not installed", allow_module_level=True)

PROGRAM = r"""
#include <cstdio>
#include "prefix_units.cuh"
int main() {                                                          // lines of: tiles blocks longest each -> least most
    int tiles, blocks, longest, each;
    printf("%d\n", PU_MOST_PARTS);
    while (scanf("%d %d %d %d", &tiles, &blocks, &longest, &each) == 4) {
        const PrefixChunks c(tiles, blocks, longest, each);
        printf("%d %d\n", c.least, c.most);
    }
}
"""


@pytest.fixture(scope="module")
def chunks(tmp_path_factory):
    folder = tmp_path_factory.mktemp("units")
    (folder / "units.cu").write_text(PROGRAM)
    subprocess.run([nvcc_path(), "-std=c++17", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a", "-I", str(CSRC), "-o",
                    str(folder / "units"), str(folder / "units.cu")], check=True, capture_output=True)

    def ask(cases):
        out = subprocess.run([str(folder / "units")], input="\n".join(" ".join(map(str, c)) for c in cases), check=True, capture_output=True, text=True)
        numbers = list(map(int, out.stdout.split()))
        return numbers[0], list(zip(numbers[1::2], numbers[2::2]))
    return ask


def cut(groups, rows_per_tile):
    """(tiles, blocks of 64 keys) of each group of (rows, shared tokens)."""
    return [(-(-rows // rows_per_tile), -(-tokens // 64)) for rows, tokens in groups]


def test_units_are_bounded(chunks):
    rng = random.Random(7)
    shapes = [([(8, n)], 8, 296) for n in (64, 128, 15360, 30656, 31488, 37888, 88064, 90000, 1 << 20)]      # (one kv head of 64, eight query heads)
    shapes += [([(2, 40000), (2, 64), (9, 640)], 64 // g, each) for g in (1, 8, 64) for each in (296, 148, 18, 1)]
    for _ in range(3000):
        n = rng.randint(1, 40)
        shapes.append(([(rng.randint(2, 70), max(1, int(2 ** rng.uniform(0, 20)))) for _ in range(n)], rng.choice((1, 2, 8, 64, 256)),
                       rng.choice((296, 148, 74, 37, 18, 9, 4, 1, 0))))
    tiled = [cut(groups, per) for groups, per, _ in shapes]
    most_parts, got = chunks([(sum(t for t, _ in x), sum(t * b for t, b in x), max(b for _, b in x), each) for x, (_, _, each) in zip(tiled, shapes)])
    # what the smallest form of the join has room for: the tiles of 64 keys of 64 codes, two stages of keys and values, less the four warps'
    # sums of eight heads; four pieces of the row's own beside the shared ones
    assert most_parts <= (2 * 2 * 64 * 64 - 4 * 8 * (64 + 2) * 4) // (4 * 8) - 4
    for x, (_, _, each), (least, most) in zip(tiled, shapes, got):
        assert 2 <= least <= most
        units = lambda chunk: sum(t * -(-b // chunk) for t, b in x)                    # noqa: E731
        for chunk in (least, most):
            assert all(-(-b // chunk) <= most_parts for _, b in x)
        assert units(most) <= max(each, sum(t for t, _ in x))
