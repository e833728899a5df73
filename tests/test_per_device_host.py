"""What the driver is asked once per device: each device's own answer, and no refusal kept, on the CPU."""
import shutil
import subprocess

import pytest

from llm_pytorch_inference_b200.build import CSRC

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "per_device.h"

int main() {
  static mvb::PerDevice known[2];
  int asked = 0, bad = 0;
  auto of = [&](int answer) { return [&asked, answer] { return ++asked, answer; }; };
  auto expect = [&](int got, int want, int times) { bad += got != want || asked != times; };
  expect(known[0].get(0, of(74), 1), 74, 1);
  expect(known[0].get(1, of(60), 1), 60, 2);  // another device: its own
  expect(known[0].get(0, of(99), 1), 74, 2);  // kept
  expect(known[0].get(1, of(99), 1), 60, 2);
  expect(known[1].get(0, of(33), 1), 33, 3);  // another size: its own
  expect(known[0].get(2, of(0), 1), 1, 4);    // refused: the fallback, which is not kept
  expect(known[0].get(2, of(-3), 1), 1, 5);
  expect(known[0].get(2, of(15), 1), 15, 6);
  expect(known[0].get(2, of(99), 1), 15, 6);
  for (int device : {-1, 64, 1 << 20}) {      // not kept, and nothing written out of range
    const int before = asked;
    expect(known[0].get(device, of(7), 1), 7, before + 1);
    expect(known[0].get(device, of(8), 1), 8, before + 2);
  }
  const int before = asked;
  expect(known[0].get(63, of(5), 1), 5, before + 1);
  printf("%d\n", bad);
  return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_each_device_has_its_own_answer(tmp_path):
    (tmp_path / "known.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", "-o", tmp_path / "known", tmp_path / "known.cpp"],
                   check=True)
    done = subprocess.run([tmp_path / "known"], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
