"""The bounded wait of the 8-bit products and the end of their rings (csrc/lcg_wait.h) compiled for the host, with a clock and a barrier of its own."""
import shutil
import subprocess

import pytest

from conftest import PKG

PROGRAM = r"""
#include <cstdio>
#include "lcg_wait.h"

struct Fake {
  uint32_t flag = 0;
  uint64_t clock = 1000, tries = 0, met_at = ~0ull;     // the barrier is met at this try
  int reports = 0;
  void wait(uint64_t limit) {
    lcg::bounded_wait(&flag, limit, [&] { clock += 10000; return ++tries >= met_at; }, [&] { return clock; },
                      [&] { ++reports; });
  }
};

int main() {
  Fake fine;                                 // an ordinary wait: met after some tries, nothing reported
  fine.met_at = 1000;
  fine.wait(1000000000ull);
  std::printf("%llu %d %u\n", (unsigned long long)fine.tries, fine.reports, fine.flag);

  Fake f;                                    // never met: gives up after its limit, once
  f.wait(1500000000ull);
  const uint64_t elapsed = f.clock - 1000;
  std::printf("%llu %d %u\n", (unsigned long long)elapsed, f.reports, f.flag);
  f.tries = 0;                               // the waits that follow, as many as a long product has
  for (int i = 0; i < 5000; ++i) f.wait(1500000000ull);
  std::printf("%llu %d\n", (unsigned long long)f.tries, f.reports);

  Fake late;                                 // the flag goes up while a wait is under way
  lcg::bounded_wait(&late.flag, 1500000000ull, [&] { if (++late.tries == 5) late.flag = 1; return false; },
                    [&] { return late.clock; }, [&] { ++late.reports; });
  std::printf("%llu %d\n", (unsigned long long)late.tries, late.reports);

  // A ring of `stages` filled `fills` times.  The releases land late, each when a wait asks for it; a wait for
  // parity p is met while the number of releases that landed in its stage is of the other parity.
  int left = 0, stuck = 0;
  for (uint32_t stages = 4; stages <= 7; ++stages) {
    for (int fills = 1; fills < 40; ++fills) {
      int landed[8] = {}, pending[8] = {};
      auto wait = [&](uint32_t s, uint32_t p) {
        if ((landed[s] & 1) != (int)p) return;
        if (pending[s] == 0) ++stuck;
        else --pending[s], ++landed[s];
      };
      uint32_t stage = 0, parity = 1;
      for (int i = 0; i < fills; ++i) {
        wait(stage, parity);
        ++pending[stage];
        if (++stage == stages) stage = 0, parity ^= 1u;
      }
      lcg::drain_ring(stages, stage, parity, wait);
      for (int p : pending) left += p;
    }
  }
  std::printf("%d %d\n", left, stuck);
}
"""


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    where = tmp_path_factory.mktemp("wait")
    (where / "wait.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{PKG / 'csrc'}", "-o", str(where / "wait"), str(where / "wait.cpp")], check=True)
    out = subprocess.run([str(where / "wait")], check=True, capture_output=True, text=True).stdout
    return [[int(v) for v in line.split()] for line in out.splitlines()]


def test_a_wait_that_is_met_reports_nothing(lines):
    assert lines[0] == [1000, 0, 0]


def test_a_wait_that_is_not_met_gives_up_after_its_limit(lines):
    elapsed, reports, flag = lines[1]
    # the timer is read once in 64 tries, and the first reading starts it
    assert 1500000000 < elapsed <= 1500000000 + 2 * 64 * 10000 + 10000
    assert (reports, flag) == (1, 1)


def test_once_one_has_run_out_every_later_wait_returns_at_once(lines):
    assert lines[2] == [5000, 1]             # one try each, and no second report
    assert lines[3] == [5, 0]


def test_a_drained_ring_has_every_release(lines):
    assert lines[4] == [0, 0]                # none outstanding, and no wait for one that never comes
