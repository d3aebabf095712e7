"""What a kernel asks of a device once: kept per device, and not kept where the question failed (csrc/device_counts.h)."""
import shutil
import subprocess
from pathlib import Path

import pytest

import hibana_b200

CSRC = Path(hibana_b200.__file__).parent / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <thread>
#include <vector>
#include "device_counts.h"

static int asked = 0;
int main() {
  static hb::DeviceCounts<17> table;
  auto answer = [](int n) { return [n] { ++asked; return n; }; };
  auto got = [&](int device, int index, int would) { std::printf("%d ", table.get(device, index, answer(would))); };
  got(0, 4, 18); got(0, 4, 99);        // kept
  got(1, 4, 12); got(0, 4, 99);        // another device has its own
  got(0, 5, -1); got(0, 5, 7); got(0, 5, 99);      // a failed question is asked again
  got(0, 6, 0); got(0, 6, 99);         // an answer of none is one
  got(hb::kMaxDevices - 1, 16, 3); got(0, 16, 2); got(0, 0, 1);
  std::printf("%d\n", asked);
  std::vector<std::thread> many;
  int wrong[8] = {};
  for (int t = 0; t < 8; ++t)
    many.emplace_back([&, t] { for (int i = 0; i < 100000; ++i) wrong[t] += table.get(i % 2, 7, [i] { return 5 + i % 2; }) != 5 + i % 2; });
  int sum = 0;
  for (auto& t : many) t.join();
  for (int w : wrong) sum += w;
  std::printf("%d\n", sum);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_counts_are_kept_per_device_cpu(tmp_path):
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", str(CSRC), str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout.splitlines()
    assert out[0].split() == ["18", "18", "12", "18", "0", "7", "7", "0", "0", "3", "2", "1", "8"] and out[1] == "0"


def test_cluster_counts_are_asked_of_the_current_device_cpu():
    """Every kernel that asks how many clusters fit keeps the answer in such a table, by the current device."""
    for src in CSRC.glob("*.cu"):
        text = src.read_text()
        if "cudaOccupancyMaxActiveClusters(" in text:
            assert "DeviceCounts<" in text and ".get(device_index()," in text, src.name
