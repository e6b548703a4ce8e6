"""The host-side table of what devices were asked: one answer for each device and key (compiled and run here)."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / 'deepep_trn_b200' / 'csrc'
MAIN = r'''
#include <cstdio>
#include <stdexcept>
#include "device_table.h"
int main() {
  static b200ep::DeviceTable<9> t;
  int asked = 0;
  auto get = [&](int device, int key) { return t.get(device, key, [&] { ++asked; return 100 * device + key + 1; }); };
  for (int round = 0; round < 2; ++round)
    for (int device = 0; device < 70; ++device)
      for (int key = 1; key < 9; ++key)
        if (get(device, key) != 100 * device + key + 1) return 1;
  if (asked != 64 * 8 + 2 * 6 * 8) return 2;              // past the table: every time
  if (get(3, 9) != 310 || get(3, -1) != 300 || get(-1, 2) != -97) return 3;
  try {
    t.get(0, 0, []() -> int { throw std::runtime_error("no"); });
    return 4;
  } catch (const std::runtime_error&) {
  }
  return t.get(0, 0, [] { return 7; }) == 7 && t.get(0, 0, [] { return 8; }) == 7 ? 0 : 5;
}
'''


@pytest.mark.skipif(shutil.which('g++') is None, reason='needs g++')
def test_each_device_has_its_own_answers(tmp_path):
    src, exe = tmp_path / 'main.cpp', tmp_path / 'main'
    src.write_text(MAIN)
    subprocess.run(['g++', '-std=c++17', '-O1', '-Wall', '-Werror', f'-I{CSRC}', str(src), '-o', str(exe)], check=True)
    assert subprocess.run([str(exe)]).returncode == 0
