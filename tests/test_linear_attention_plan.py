"""How linear attention cuts sequences into segments: compiled from the kernels' own header and swept on the CPU."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "deciax_amd" / "csrc"

PROGRAM = r'''
#include <cstdio>
#include <initializer_list>
#include "linear_attention_plan.h"
int sweep(int limit) {
  int most = 0;
  for (long len = 0; len <= (1L << 30); len += len < 70000 ? 1 : len / 977) {
    const la::Segments s = la::segments((int)len, limit);
    if (s.count < 1 || s.tokens < 64 || s.tokens % 64) return printf("%ld: %d segments of %d\n", len, s.count, s.tokens);
    // every token in a segment, none of them empty but that of no tokens
    if ((long)s.tokens * s.count < len || (s.count > 1 && (long)s.tokens * (s.count - 1) >= len))
      return printf("%ld: %d segments of %d\n", len, s.count, s.tokens);
    most = s.count > most ? s.count : most;
    const int room = la::most_segments((int)len, limit);
    if (most > room || room > limit) return printf("%ld: %d, room for %d\n", len, most, room);
  }
  return 0;
}
int main() {
  if (la::limit(64) != la::limit(128) || sweep(la::limit(64)) || sweep(la::limit(256))) return 1;
  for (int len : {0, 1, la::STEP, la::ONE, la::ONE + 1, 1 << 30}) {
    const la::Segments s = la::segments(len, la::limit(128));
    printf("%d %d %d %d\n", len, s.tokens, s.count, la::most_segments(len, la::limit(128)));
  }
  return 0;
}
'''


def test_segments_cover_every_length(tmp_path: Path) -> None:
    compiler = shutil.which("g++") or shutil.which("clang++")
    if compiler is None:
        pytest.skip("no host compiler")
    (tmp_path / "plan.cc").write_text(PROGRAM)
    subprocess.run([compiler, "-std=c++17", "-O1", f"-I{CSRC}", str(tmp_path / "plan.cc"), "-o", str(tmp_path / "plan")],
                   check=True)
    res = subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout
    lines = [list(map(int, line.split())) for line in res.stdout.splitlines()]
    assert [x[2] for x in lines[:4]] == [1, 1, 1, 1] and lines[5][2] == lines[5][3]
