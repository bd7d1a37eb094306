"""csrc/kv4_plan.h on the CPU: the spans of a sequence's keys and the workspace laid out for the largest lengths agree
for every size, so no part of a row is written outside its place, none is left out of the join and no key is read twice."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "deciax_amd" / "csrc"
GXX = shutil.which("g++")

PRELUDE = r"""
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <vector>
#include "kv4_plan.h"
using namespace kv4;
#define CHECK(...) do { if (!(__VA_ARGS__)) { \
  std::printf("%s\n  ctx %d n %d group %d window %d in a batch of %d tokens over %d\n", #__VA_ARGS__, ctx, n, group, window, \
              max_n, max_ctx); return 1; } } while (0)
// one sequence in a batch whose longest have max_n new tokens and max_ctx slots
static int check(int ctx, int n, int group, int window, int max_n, int max_ctx) {
  const int slots = std::min(window, max_ctx), rows = n * group;  // a window beyond the longest sequence is cut to it
  const Spans s = spans(ctx, n, rows, slots);
  const Plan p = attn_plan(max_n, max_ctx, group, slots);
  CHECK(s.count >= 1 && s.count <= p.max_splits && s.count <= MAX_SPANS);
  CHECK(s.count == 1 || (int64_t)s.count * rows <= p.part_rows);  // where the parts stand in the workspace
  CHECK(s.count == 1 || rows <= MOST_SPLIT_ROWS);                 // the rows that are joined
  CHECK(rows <= p.max_rows);
  CHECK(s.lo % 64 == 0 && s.keys > 0 && s.keys % 128 == 0);
  // [lo, ctx) once: the last span reaches the end, and the one before does not
  CHECK(s.lo <= ctx && s.lo + (int64_t)s.count * s.keys >= ctx);
  CHECK(s.count == 1 || s.lo + (int64_t)(s.count - 1) * s.keys < ctx);
  // every slot that some row may see
  CHECK(s.lo == 0 || (slots > 0 && s.lo <= (int64_t)ctx - n - slots + 1));
  CHECK(p.score_rows >= std::min(rows, SCORE_ROWS) && p.score_slots >= (ctx + 31) / 32 * 32);
  return 0;
}
"""

SWEEP = r"""
int main() {
  const std::vector<int> contexts{0, 1, 63, 64, 65, 500, 511, 512, 513, 575, 1023, 1024, 1025, 1300, 2047, 2048, 2111, 3000, 4097,
                                  8192, 9000, 16383, 16384, 16385, 16500, 40000, 1 << 20, (1 << 30) - 1, 1 << 30};
  const std::vector<int> rows{0, 1, 15, 16, 17, 32, 33, 48, 49, 64, 127, 128, 129, 1023, 1024, 1025, 1300, 1364, 1365, 1366, 1367,
                              2040, 2047, 2048, 2049, 2050, 2200, 2400, 4095, 4096, 4097, 4800, 8191, 8192, 8200, 65536, 1 << 25};
  long done = 0;
  for (int group : {1, 2, 3, 4, 5, 6, 7, 8, 16})
    for (int r : rows)
      for (int ctx : contexts)
        for (int window : {0, 1, 70, 128, 700, 4096, 1 << 20, 0x7fffffff}) {
          const int n = r / group;
          for (int max_n : {n, n + 1, std::max(n, 300), std::max(n, 2500 / group)})
            for (int max_ctx : {ctx, std::max(ctx, 513), std::max(ctx, 9000), std::max(ctx, 1 << 20)}) {
              if ((int64_t)max_n * group > 1 << 25) continue;  // refused by the entry point
              if (check(ctx, n, group, window, max_n, max_ctx)) return 1;
              ++done;
            }
        }
  std::printf("%ld\n", done);
  return done < 1000000;
}
"""

SMALL = r"""
int main() {
  for (int rows = 1; rows <= 4200; ++rows)
    for (int ctx = 1; ctx <= 18000; ctx += ctx < 2200 ? 61 : 997)
      for (int window : {0, 128, 4096})
        if (check(ctx, rows, 1, window, rows, ctx)) return 1;
  return 0;
}
"""


@pytest.mark.skipif(GXX is None, reason="no g++")
@pytest.mark.parametrize("name,body", [pytest.param("sweep", SWEEP, id="sweep"), pytest.param("small", SMALL, id="small")])
def test_spans_and_workspace_agree(tmp_path: Path, name: str, body: str) -> None:
    src, exe = tmp_path / f"{name}.cpp", tmp_path / name
    src.write_text(PRELUDE + body)
    subprocess.run([GXX, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}", str(src), "-o",
                    str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
