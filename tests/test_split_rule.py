"""How many CTAs share a tile's range of k: by fixed numbers of clusters, so that a row's sum runs in the same order on every GPU, whatever
clusters of it the device's GPCs happen to fit. The rule is compiled for the host and asked; that both kernels go by it is read from the sources."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen38-3090-cuda-server_b200", "csrc")

HARNESS = r"""
#include <cstdio>
#include "ragged.cuh"
int main() {
  const int room[9] = {0, 296, 148, 93, 71, 56, 45, 37, 33};
  for (int most = 1; most <= 8; ++most)
    for (int tiles = 1; tiles <= 300; ++tiles) {
      int same = -1;
      for (int delta = -40; delta <= 40; delta += 5) {
        int runs[9];
        for (int n = 0; n < 9; ++n) runs[n] = room[n] + delta > 1 ? room[n] + delta : 1;
        const int s = w4a16::splits_at_once(tiles, most, room, runs);
        if (same >= 0 && s != same) return 1;
        same = s;
      }
      if (same < 1 || same > most || (same > 1 && tiles > room[same]) || (same < most && tiles <= room[same + 1])) return 2;
    }
  int none[9] = {0, 148, 74, 46, 0, 0, 0, 0, 0};
  if (w4a16::splits_at_once(20, 8, room, none) != 3) return 3;  // what the device cannot run at all
  return 0;
}
"""


def test_the_rule(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not found")
    (tmp_path / "rule.cu").write_text(HARNESS)
    exe = str(tmp_path / "rule")
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, "-o", exe, str(tmp_path / "rule.cu")], check=True)
    assert subprocess.run([exe]).returncode == 0


@pytest.mark.parametrize("name,function,table", [("ragged.cu", "int launch_ragged(", "kRoom"), ("prefill.cu", "PrefillPlan plan_single(", "kClusters")])
def test_both_kernels_go_by_it(name, function, table):
    with open(os.path.join(CSRC, name)) as f:
        body = f.read().split(function, 1)[1].split("\n}\n", 1)[0]
    assert re.search(r"constexpr int " + table + r"\[", body)
    assert len(re.findall(r"splits_at_once\([^;]*\b" + table + r",", body)) == 1
    assert not re.search(r"<= (fit|device_clusters)\[", body)
