"""CPU: every byte that the adapters' rings ask for lies in its row, at every width from the smallest on.

The kernel's own arithmetic (``csrc/mi_adapter_ring.h``) is compiled for the host and walked over a row's steps and
the eight chunks of a step, steps behind the last among them."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "minimal-inference_amd" / "csrc"

# %s: the place of a chunk.  Prints a line for each width that reads outside its row or a wrong place of it.
PROGRAM = r"""
#include <cstdio>
#include "mi_adapter_ring.h"
static bool good(int width, int lots) {  // lots: steps of 128 bytes of this row to one of x's
  const int steps = (width + 128 * lots - 1) / (128 * lots);
  for (int step = 0; step < steps + 64; ++step) {
    const int off = step < steps ? step * 128 : 0;
    for (int l = 0; l < lots; ++l)
      for (int chunk = 0; chunk < 128; chunk += 16) {
        const int at = off * lots + l * 128, place = %s;
        if (place < 0 || place + 16 > width) return false;
        if (step < steps && at + chunk < width && place != at + chunk) return false;
      }
  }
  return true;
}
int main() {
  for (int k = 32; k <= 4096; k += 32) {
    if (!good(2 * k, 1)) std::printf("bf16 %%d\n", k);   // x, A beside it
    if (!good(k, 1)) std::printf("codes %%d\n", k);      // x in 8 bits
    if (!good(2 * k, 2)) std::printf("factor %%d\n", k); // A beside 8-bit x
  }
}
"""


def _run(tmp_path, place):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    source, binary = tmp_path / "ring.cpp", tmp_path / "ring"
    source.write_text(PROGRAM % place)
    subprocess.run([cxx, "-std=c++20", f"-I{CSRC}", str(source), "-o", str(binary)], check=True)
    return subprocess.run([str(binary)], check=True, capture_output=True, text=True).stdout.split("\n")[:-1]


def test_ring_reads_within_its_rows(tmp_path):
    assert _run(tmp_path, "mi::adapter::ring_place(at, chunk, width)") == []
    assert "ring_place(" in (CSRC / "mi_adapter.hip").read_text()


def test_the_walk_sees_a_chunk_past_a_short_row(tmp_path):
    """A lane that keeps its chunk where the row ends before it."""
    seen = _run(tmp_path, "(at + chunk < width ? at : 0) + chunk")
    assert seen == ["bf16 32", "codes 32", "factor 32", "codes 64", "codes 96"]
