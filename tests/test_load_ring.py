"""The attention kernel's ring of loads, on the host: the loads in flight when a wait runs out
are exactly the ones that the unwinding then waits for."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "co-alibi_b200", "csrc")

# Steps and loads in the kernel's order: NBUF - 1 loads ahead, then per step a wait and, where
# there is one, the next load; items follow one another.  The wait of step `stop` runs out.
PROGRAM = """
#include <cstdio>
#include <vector>
#include "load_ring.h"
template <int NBUF> int run(int items, int nsteps, int stop) {
  coalibi::LoadRing<NBUF> ring;
  std::vector<int> slot_load(NBUF, -1), slot_phases(NBUF, 0);  // load in the slot, loads it has had
  int issued = 0, awaited = 0, step = 0;
  auto load = [&] { slot_load[ring.fill] = issued++; slot_phases[ring.fill]++; ring.issue(); };
  auto expect = [&] {  // the cursor names the oldest load that has not been awaited, and its phase
    return slot_load[ring.drain] == awaited && (int)ring.phase == (slot_phases[ring.drain] - 1) % 2;
  };
  for (int item = 0; item < items; ++item) {
    bool ok = true;
    for (int a = 1; a < NBUF; ++a) if (nsteps - a >= 0) load();
    for (int st = nsteps - 1; st >= 0; --st, ++step) {
      if (!ok || step == stop) { ok = false; continue; }
      if (!expect()) return 1;
      ++awaited;
      ring.landed();
      if (st - (NBUF - 1) >= 0) load();
    }
    if (!ok) {
      for (; ring.in_flight(); ring.landed(), ++awaited) if (!expect()) return 2;
      return awaited == issued ? 0 : 3;
    }
    if (ring.in_flight()) return 4;
  }
  return 0;
}
int main() {
  for (int items = 1; items < 4; ++items)
    for (int nsteps = 0; nsteps < 9; ++nsteps)
      for (int stop = 0; stop <= items * nsteps; ++stop) {
        int rc = run<2>(items, nsteps, stop);
        if (!rc) rc = run<3>(items, nsteps, stop);
        if (rc) { printf("%d items of %d steps, stop %d: %d\\n", items, nsteps, stop, rc); return 1; }
      }
  return 0;
}
"""


def test_the_loads_in_flight_when_a_wait_runs_out(tmp_path):
    cxx = os.environ.get("CXX") or shutil.which("g++")
    if not cxx:
        pytest.skip("no C++ compiler")
    src, exe = tmp_path / "ring.cpp", tmp_path / "ring"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
