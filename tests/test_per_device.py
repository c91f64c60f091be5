"""What launchers ask the CUDA runtime once for each device of the process (csrc/per_device.h), on fake devices; and no
launcher asks for a kernel's shared memory in any other way."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "grxcp_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "per_device.h"
static grx::PerDevice a, b;
int main() {
  int asked[3] = {0, 0, 0};
  auto on = [&](grx::PerDevice& p, int device, int answer) {
    return p.get(device, [&] { ++asked[device % 3]; return answer; });
  };
  if (on(a, 0, 7) != 7 || on(a, 0, 8) != 7 || asked[0] != 1) return 1;  // once a device
  if (on(a, 1, 9) != 9 || asked[1] != 1 || on(a, 0, 8) != 7) return 2;  // the other device is asked for itself
  if (on(b, 0, 5) != 5 || asked[0] != 2) return 3;                      // and the other launcher
  if (on(a, 2, -1) != -1 || on(a, 2, 4) != 4 || on(a, 2, 3) != 4) return 4;  // a failure is not kept
  if (on(a, 300, 6) != 6 || on(a, 300, 5) != 5) return 5;               // past the last device: every time
  return 0;
}
"""


def test_asked_once_for_each_device(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    (tmp_path / "p.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(tmp_path / "p.cpp"), "-o", str(tmp_path / "p")], check=True)
    assert subprocess.run([str(tmp_path / "p")]).returncode == 0


def test_no_kernel_attribute_is_set_for_the_first_device_alone():
    for src in sorted(CSRC.glob("*.c*")):
        assert not re.search(r"cudaFuncSetAttribute", src.read_text()), src.name
