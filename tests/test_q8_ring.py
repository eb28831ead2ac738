"""The decode kernel's ring of copies (csrc/q8_ring.h, the code that the kernel runs) on the CPU,
against barriers that complete, and against waits that run out: whatever is under way then is
waited for, nothing more is copied or used, and the walk says so."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "hive-limited_b200" / "csrc"

MAIN = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "q8_ring.h"
#define CHECK(x) do { if (!(x)) { std::printf("%s: stages %d, %d..%d by %d, bad wait %d\n", #x, \
                                              kStages, b0, end, step, bad); std::exit(1); } } while (0)

// the bad'th wait runs out (never: -1); with `late` the copy has not arrived by the second wait either
template <int kStages>
void run(int b0, int end, int step, int bad, bool late) {
  int flying[kStages], phase[kStages];         // block on its way to a place; phases completed there
  for (int i = 0; i < kStages; ++i) flying[i] = -1, phase[i] = 0;
  auto copy = [&](int b, int place) {
    if (b >= end) return;
    CHECK(flying[place] == -1);                // no copy on top of another
    flying[place] = b;
  };
  for (int i = 0; i < kStages; ++i) copy(b0 + i * step, i);
  int waits = 0, failed_at = -1, drained = 0;
  std::vector<int> used;
  int ready = -1;
  auto wait = [&](int place, int parity) {
    CHECK(flying[place] != -1);                // never for a copy that nobody started
    CHECK((phase[place] & 1) == parity);       // the phase under way
    const int n = waits++;
    if (failed_at >= 0) ++drained;
    if (n == bad) { failed_at = place; return false; }
    if (late && failed_at == place) return false;
    ready = flying[place];
    flying[place] = -1;
    ++phase[place];
    return true;
  };
  auto fetch = [&](int b, int place) { CHECK(failed_at == -1); copy(b, place); };
  auto use = [&](int b, int) { CHECK(failed_at == -1); CHECK(b == ready); used.push_back(b); };
  const bool ok = hv::ring_walk<kStages>(b0, end, step, wait, fetch, use);
  CHECK(ok == (failed_at == -1));
  size_t n = 0;
  for (int b = b0; b < end; b += step, ++n)
    if (ok) CHECK(n < used.size() && used[n] == b);
  CHECK(ok ? used.size() == n : used.size() == (size_t)bad);
  for (int i = 0; i < kStages; ++i) CHECK(flying[i] == -1 || (late && i == failed_at));
  CHECK(ok || drained >= 1);
}

template <int kStages>
void all() {
  for (int step : {1, 8})
    for (int b0 = 0; b0 < 9; b0 += 4)
      for (int end = 0; end < 60; ++end)
        for (int bad = -1; bad < 12; ++bad)
          for (bool late : {false, true}) run<kStages>(b0, end, step, bad, late);
}

int main() { all<1>(); all<2>(); all<3>(); std::puts("ok"); }
"""


def test_ring_walk(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not found")
    (tmp_path / "main.cc").write_text(MAIN)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined",
                    f"-I{CSRC}", str(tmp_path / "main.cc"), "-o", str(tmp_path / "main")], check=True)
    r = subprocess.run([str(tmp_path / "main")], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
