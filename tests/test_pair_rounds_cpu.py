"""A pair of CTAs that gives up: every copy that either of them issued has landed before shared memory is released.

The barrier of a stage (two arrivals a phase, bytes counted), the two copiers and the products are modelled on the host and
stopped at every combination of places; what is left is settled as csrc/pair_rounds.h, compiled here, says."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "psgd_pro_b200", "csrc")
MODEL = r"""
#include <cstdio>
#include "pair_rounds.h"

struct Barrier {  // a phase ends when nobody's arrival is pending and no byte is expected
  int pending = 2, bytes = 0;
  unsigned phase = 0;
  void settle() { if (pending == 0 && bytes == 0) pending = 2, ++phase; }
  void arrive() { --pending; settle(); }
  void expect(int n) { bytes += n; --pending; settle(); }
  void land(int n) { bytes -= n; settle(); }
  bool done(unsigned parity) const { return (phase & 1u) != parity; }  // as mbarrier.try_wait.parity
};

static unsigned state = 1;
static unsigned draw(unsigned n) {
  state = state * 1664525u + 1013904223u;
  return (state >> 8) % n;
}

int main() {
  long cases = 0, apart = 0;
  for (unsigned stages = 1; stages <= 4; ++stages)
    for (unsigned stop0 = 0; stop0 <= 13; ++stop0)
      for (unsigned stop1 = 0; stop1 <= 13; ++stop1)
        for (int turn = 0; turn < 20; ++turn) {
          Barrier full[4];
          unsigned used[4] = {0, 0, 0, 0};  // phases that the products used up, by stage
          unsigned rounds[2] = {0, 0}, stop[2] = {stop0, stop1}, consumed = 0;
          struct { unsigned stage; } flight[64];
          int flying = 0;
          for (int step = 0; step < 400; ++step) {
            const unsigned what = draw(4);
            if (what < 2) {  // a copier's next round, unless it gave up: its stage has to be free
              const unsigned r = rounds[what], s = r % stages;
              if (r < stop[what] && used[s] >= r / stages && flying < 64) {
                full[s].expect(1);
                flight[flying++].stage = s;
                ++rounds[what];
              }
            } else if (what == 2 && flying) {  // some copy lands
              const int k = draw(flying);
              full[flight[k].stage].land(1);
              flight[k] = flight[--flying];
            } else if (what == 3) {  // the products take the next round, in order
              const unsigned s = consumed % stages;
              if (full[s].phase > consumed / stages) ++used[s], ++consumed;
            }
          }
          // both have stopped; some copies may still be on their way
          bool open[4] = {};
          for (unsigned i = 0; i < stages; ++i) {
            const psgd::StageLeft left = psgd::stage_left(rounds[0], rounds[1], stages, i);
            const psgd::StageLeft same = psgd::stage_left(rounds[1], rounds[0], stages, i);
            if (left.arrive != same.arrive || left.wait != same.wait || left.parity != same.parity) return puts("asymmetric"), 1;
            if (left.arrive) full[i].arrive(), ++apart;
            bool inflight = false;
            for (int k = 0; k < flying; ++k) inflight |= flight[k].stage == i;
            open[i] = left.wait && !full[i].done(left.parity);
            if (open[i] != inflight) return printf("stages %u stops %u %u: stage %u waits %d, copies %d\n", stages, stop0, stop1, i, (int)open[i], (int)inflight), 1;
          }
          while (flying) full[flight[--flying].stage].land(1);
          for (unsigned i = 0; i < stages; ++i) {
            const psgd::StageLeft left = psgd::stage_left(rounds[0], rounds[1], stages, i);
            if (left.wait && !full[i].done(left.parity)) return printf("stages %u stops %u %u: stage %u never ends\n", stages, stop0, stop1, i), 1;
          }
          ++cases;
        }
  if (!apart) return puts("the two were never apart"), 1;
  printf("%ld cases\n", cases);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_copies_of_both_ctas_land_before_a_pair_leaves(tmp_path):
    src, exe = tmp_path / "model.cpp", tmp_path / "model"
    src.write_text(MODEL)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout
