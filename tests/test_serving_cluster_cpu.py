"""Which cluster the 4-bit cache attention launches where a device has no room for the planned one."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "oct_b200" / "csrc"
CUDA = Path("/usr/local/cuda/include")
PROGRAM = """
#include <cstdio>
#include "serving.h"
int main() {
  for (uint32_t room = 0; room <= 32; ++room)
    for (uint32_t wanted = 1; wanted <= 16; wanted *= 2) {
      uint32_t asked = 0;
      const uint32_t got = oct::kv4_cluster_to_launch(wanted, [&](uint32_t n) { ++asked; return n <= room; });
      std::printf("%u %u %u %u\\n", room, wanted, got, asked);
    }
}
"""


@pytest.mark.skipif(not (CUDA / "cuda_runtime.h").exists(), reason="needs the CUDA headers")
def test_a_cluster_without_room_is_halved_until_it_fits(tmp_path):
    src = tmp_path / "cluster.cpp"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), "-I", str(CUDA), "-o", str(tmp_path / "cluster"), str(src)], check=True)
    lines = subprocess.run([str(tmp_path / "cluster")], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(lines) == 33 * 5
    for line in lines:
        room, wanted, got, asked = map(int, line.split())
        fitting = [n for n in (1, 2, 4, 8, 16) if n <= min(wanted, max(room, 1))]
        assert got == fitting[-1]  # one block needs no room of a cluster's
        assert asked <= 4
