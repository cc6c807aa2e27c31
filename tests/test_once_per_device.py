"""What a process asks of a device once (``csrc/once_per_device.h``): a request that failed is made again, and devices do not answer for one another."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "innova_b200", "csrc")
PROGRAM = r"""
#include "once_per_device.h"
#include <cstdio>
int main() {
  inv::OncePerDevice once;
  int asked = 0, answer = 2;
  auto request = [&] { ++asked; return answer; };
  if (once.ask(3, request) != 2 || once.ask(3, request) != 2 || asked != 2) return 1;      // failed: asked again
  answer = 0;
  if (once.ask(3, request) != 0 || asked != 3) return 2;
  answer = 5;
  if (once.ask(3, request) != 0 || asked != 3) return 3;                                    // granted: not asked again
  if (once.ask(4, request) != 5 || once.ask(67, request) != 5 || once.ask(-61, request) != 5 || asked != 6) return 4;
  answer = 0;
  if (once.ask(67, request) != 0 || once.ask(67, request) != 0 || once.ask(3, request) != 0 || asked != 8) return 5;
  inv::OncePerDevice other;
  return other.ask(3, request) == 0 && asked == 9 ? 0 : 6;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_a_failed_request_is_made_again(tmp_path):
    (tmp_path / "p.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, "-o", str(tmp_path / "p"), str(tmp_path / "p.cpp")], check=True)
    assert subprocess.run([str(tmp_path / "p")]).returncode == 0
