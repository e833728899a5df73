"""The order of the few-row product's copies, run on the CPU with copies that come late or not in time."""
import shutil
import subprocess

import pytest

from llm_pytorch_inference_b200.build import CSRC

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "w4_ring.h"

// A place's barrier: an arrival with bytes, and a phase that is over when they have come.
struct Place {
  int asked = 0, landed = 0, item = -1;
  bool under_way() const { return asked > landed; }
};

int run(int stages, int items, int gives_up, int late) {
  mvb::W4Ring ring(0);
  int lost = -1;
  std::vector<Place> places(stages);
  std::vector<int> to_come;  // places of copies that have not come, in order
  int next = 0, waits = 0, bad = 0;
  auto ask = [&] {
    if (next >= items || ring.stopped()) return;
    Place& p = places[ring.fill];
    if (p.under_way()) return void(++bad);  // an arrival on a phase that is not over
    p.item = next++;
    ++p.asked;
    to_come.push_back(ring.fill);
    ring.asked(stages);
  };
  auto come = [&](int n) {
    for (; n > 0 && !to_come.empty(); --n) ++places[to_come.front()].landed, to_come.erase(to_come.begin());
  };
  // A wait for parity `phase`: over when the place's completed phases have passed it.
  auto over = [&](const Place& p, unsigned phase) { return p.landed > 0 && ((p.landed - 1) & 1u) == phase; };
  for (int s = 0; s < stages; ++s) ask();
  for (int i = 0; i < items; ++i) {
    bool came = true;
    if (!ring.stopped()) {
      ++waits;
      if (i == gives_up) came = false;  // its copy has not come
      else {
        while (!over(places[ring.read], ring.phase) && !to_come.empty()) come(1);
        if (!over(places[ring.read], ring.phase)) ++bad;
        if (places[ring.read].item != i) ++bad;  // the item's own records
      }
    } else {
      came = i % 2;  // whatever the waits after that say
    }
    if (!came) ring.stop(lost);
    ask();
    ring.next(stages);
    if (i % 3 == 0 && !(gives_up >= 0 && i >= gives_up && i < gives_up + late)) come(1);
  }
  if (ring.stopped()) {
    ring.back(lost);
    do {
      Place& p = places[ring.read];
      while (!over(p, ring.phase) && !to_come.empty()) come(1);
      if (!over(p, ring.phase)) ++bad;  // would run to its limit
    } while (ring.more(stages));
  }
  for (auto& p : places) bad += p.under_way();  // a copy that comes after the block has ended
  if (!to_come.empty()) ++bad;
  if (gives_up < 0 && (next != items || waits != items)) ++bad;
  return bad;
}

int main() {
  int bad = 0, runs = 0;
  for (int stages = 1; stages <= 8; ++stages)
    for (int items = 0; items <= 40; ++items)
      for (int gives_up = -1; gives_up < items; ++gives_up)
        for (int late : {0, 1, 3, 100}) ++runs, bad += run(stages, items, gives_up, late) != 0;
  printf("%d of %d\n", bad, runs);
  return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_no_copy_is_asked_for_twice_or_left_behind(tmp_path):
    (tmp_path / "ring.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", "-o", tmp_path / "ring", tmp_path / "ring.cpp"],
                   check=True)
    done = subprocess.run([tmp_path / "ring"], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
