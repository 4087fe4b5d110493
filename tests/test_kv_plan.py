"""The arithmetic by which the cache's attention cuts a tile's slots into parts, on the host: the join's tables hold every part of
every row."""
import ctypes
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "rtq_kargs.h"
// the most rows x parts that one workgroup joins, over tiles of `rows` rows and lengths from..to, every shortest range of 128 to 2048
extern "C" int most(int rows, int from, int to, int step, int fused) {
  int64_t top = 0;
  for (int64_t total = from; total <= to; total += step)
    for (int least = 128; least <= 2048; least += 128) {
      const int c = kv_range((int)total, rows, least, fused), ns = kv_parts((int)total, c);
      if (c % 128 || c < least || (int64_t)c * ns < total || (ns > 1 && (int64_t)c * (ns - 1) >= total) || ns < 1) return -1;
      const int64_t mine = fused ? rows : (rows + ns - 1) / ns;  // a kernel's workgroups, one a part, share the rows
      if (!fused && ns > RTQ_KV_JOIN) return -1;
      if (mine * ns > top) top = mine * ns;
    }
  return (int)top;
}
extern "C" int tables() { return RTQ_KV_JOINED; }
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "rust_trainer_amd", "csrc"), str(d / "plan.cpp"), "-o",
                    str(d / "plan.so")], check=True)
    return ctypes.CDLL(str(d / "plan.so"))


@pytest.mark.parametrize("fused", [1, 0])
def test_a_joins_tables_hold_every_length(plan, fused):
    for rows in list(range(1, 18)) + [31, 33, 60, 64, 65, 100, 113, 127, 128]:
        top = plan.most(rows, 0, 16384, 1, fused)
        assert 1 <= top <= plan.tables(), (rows, top)


@pytest.mark.parametrize("fused", [1, 0])
def test_a_joins_tables_hold_the_longest(plan, fused):
    for rows in (1, 3, 7, 9, 13, 15, 16, 100, 127, 128):
        for lo, hi, step in ((16384, 2 ** 20, 997), (2 ** 20, 2 ** 30, 2 ** 20 - 3), (2 ** 30 - 4, 2 ** 30, 1)):
            top = plan.most(rows, lo, hi, step, fused)
            assert 1 <= top <= plan.tables(), (rows, top)


def test_lengths_that_need_more_than_the_quotient(plan):
    """Rows that do not divide the tables' entries: a part more than the whole quotient."""
    assert plan.most(12, 10900, 10900, 1, 1) == 86 * 12 and plan.most(14, 9360, 9360, 1, 1) == 74 * 14
    assert plan.most(13, 10082, 10082, 1, 1) == 79 * 13 and plan.most(15, 8720, 8720, 1, 1) == 69 * 15
