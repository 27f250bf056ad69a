"""Where attention of few queries reads keys and values, on the CPU: never behind the array, whatever the heads' length, and all that it needs."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinyflow_amd", "csrc")

# Every load of a step's 16 keys from key j0 on: as the hardware does it, four bytes at a time, those outside of the buffer as zero.
PROGRAM = r"""
#include "few_rows.h"
#include <cstdio>
#include <cstdlib>
#include <algorithm>
using namespace tf::attention;
int main(int, char **argv) {
  const int64_t batch = atoll(argv[1]), keys = atoll(argv[2]), heads = atoll(argv[3]), dim = atoll(argv[4]);
  const int64_t all = batch * keys * heads * dim, step = heads * dim;
  int64_t behind = 0, missing = 0;
  for (int64_t b : {(int64_t)0, batch - 1})
    for (int64_t g : {(int64_t)0, heads - 1})
      for (int64_t j0 = std::max<int64_t>(0, (keys - 1) / 16 * 16 - 32); j0 < keys; j0 += 16) {
        const int64_t from = (b * keys + j0) * step + g * dim;
        const uint32_t bytes = (uint32_t)buffer_bytes(all, from);
        for (int row = 0; row < std::min<int64_t>(16, keys - j0); ++row)
          for (int column = 0; column < 256; column += 4)
            for (int e = 0; e < 4; ++e) {
              const uint64_t at = (uint64_t)buffer_offset(row, step, column, (int)dim) + 4u * e;
              const bool read = at + 4 <= bytes;
              if (read && from + (int64_t)at / 4 >= all) ++behind;
              if (column + e < dim && !(read && at == ((uint64_t)row * step + column + e) * 4)) ++missing;
            }
      }
  printf("%lld %lld\n", (long long)behind, (long long)missing);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    folder = tmp_path_factory.mktemp("few_rows")
    source, binary = folder / "reads.cpp", folder / "reads"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(source), "-o", str(binary)], check=True)
    return str(binary)


# a cache whose bytes fill whole blocks of memory (4 096 rows of 4 heads of 66, 8 192 of one), the shortest, the widest rows, and more than 2^31 bytes
@pytest.mark.parametrize("batch,keys,heads,dim", [(1, 4096, 4, 66), (1, 8192, 1, 66), (2, 1, 1, 1), (1, 1, 1, 255), (3, 17, 2, 5), (2, 40, 3, 63),
                                                  (1, 33, 7, 64), (2, 100, 131071, 127), (1, 1 << 24, 1, 254), (8, 1 << 20, 4, 129)])
def test_reads_stay_inside(program, batch, keys, heads, dim):
    out = subprocess.run([program] + [str(n) for n in (batch, keys, heads, dim)], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["0", "0"]
