"""Where key ranges begin (csrc/range_tiles.h), compiled for the host."""
from test_split_rules_host import _run

SOURCE = """
#include "range_tiles.h"
#include <cstdio>
#include <cstdlib>
int main(int argc, char **argv) {
  for (int i = 1; i + 1 < argc; i += 2) {
    const int tiles = atoi(argv[i]), ranges = atoi(argv[i + 1]);
    for (int part = 0; part <= ranges; ++part) printf("%d\\n", mcamd::range_tile(part, tiles, ranges));
  }
}
"""


def test_ranges_of_the_longest_rows(tmp_path):
    """Every range of rows of up to 2^30 keys in tiles of 16 to 128, cut into as many as any chip holds: part * tiles
    / ranges in whole numbers of any size, so that the ranges follow one another from the first tile to the last."""
    cases = [(max(1, -(-keys // tile)), ranges)
             for keys in (1, 700, 16385, (1 << 27) - 1, 1 << 27, 134_500_000, 140_000_001, 1 << 29, 1 << 30)
             for tile in (16, 32, 64, 128) for ranges in (1, 2, 31, 32, 255, 256, 304, 511, 512, 2047, 65535)]
    got = iter(_run(tmp_path, SOURCE, [x for c in cases for x in c]))
    for tiles, ranges in cases:
        assert [next(got) for _ in range(ranges + 1)] == [part * tiles // ranges for part in range(ranges + 1)]
