"""Loads that end with a row, compiled for the host: the row ends where readable memory does."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parents[1] / "autosage_amd" / "csrc" / "raw_vec.h"

PROGRAM = r"""
#include <cstdio>
#include <cstring>
#include <sys/mman.h>
#include <unistd.h>
#include "raw_vec.h"

static unsigned char* fence;  // the first byte that cannot be read

// Every run of a row of `count` elements that ends at the fence.
template <typename E, int N>
__attribute__((noinline)) int check(int count) {
  const E* row = reinterpret_cast<const E*>(fence) - count;
  for (int at = 0; at < count; at += N) {
    const int left = count - at;
    const auto got = as::load_up_to<E, N>(row + at, left);
    unsigned char want[sizeof(got)] = {};
    std::memcpy(want, row + at, sizeof(E) * (left < N ? left : N));
    if (std::memcmp(&got, want, sizeof(got)) != 0) return 1;
  }
  return 0;
}

int main() {
  const long page = sysconf(_SC_PAGESIZE);
  auto* pages = static_cast<unsigned char*>(
      mmap(nullptr, 2 * page, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
  for (long i = 0; i < page; ++i) pages[i] = static_cast<unsigned char>(1 + i * 37 % 255);
  fence = pages + page;
  mprotect(fence, page, PROT_NONE);
  for (int width = 2; width <= 256; width += 2) {
    std::printf("width %d\n", width);
    std::fflush(stdout);
    if (check<uint8_t, 2>(width / 2) || check<uint8_t, 4>(width / 2) || check<uint16_t, 8>(width) ||
        check<uint32_t, 8>(width))
      return 1;
  }
  return 0;
}
"""


@pytest.mark.parametrize("level", ["-O0", "-O2"])
def test_a_row_is_read_to_its_end_and_no_further(tmp_path, level):
    """The runs of 4-bit rows of every even width: two bytes of codes for four numbers of float32, four for eight of the
    16-bit types; and the rows of tokens."""
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    (tmp_path / "rows.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", level, f"-I{HEADER.parent}", "rows.cpp", "-o", "rows"], cwd=tmp_path, check=True)
    done = subprocess.run([str(tmp_path / "rows")], capture_output=True, text=True)
    assert done.returncode == 0, (done.returncode, done.stdout[-20:])
