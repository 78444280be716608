"""The meetings of the 8-bit product's scheduler warp and MMA issuer when waits give up.

Both warps meet on a barrier without a time limit, so a wait that gives up at any point (an
accumulator that is never freed, a K block that never lands) must leave both with the same number
of meetings and tell the issuer to stop. The kernel's control flow (csrc/pq8_schedule.h) is compiled for
the CPU and run with one wait failing at every possible point."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / 'parakeet_cuda_b200' / 'csrc'

PROGRAM = r'''
#include <cstdio>
#include <utility>
#include <vector>
#include "pq8_schedule.h"

// Wait number `fail` (from 0; -1: none) gives up. Returns what went wrong, or NULL.
const char* check(int tiles, int k_blocks, int step, int fail) {
  const int stride = 3, first = 2, kb0 = 5;
  const pq8::ScheduleRange range{first, first + tiles * stride, stride, kb0, kb0 + k_blocks};
  std::vector<bool> met;
  int waits = 0, freed = 0, blocks = 0, after = 0;
  bool failed = false;
  auto wait = [&] {
    if (failed) ++after;
    const bool ok = waits++ != fail;
    failed = failed || !ok;
    return ok;
  };
  pq8::schedule_products(
      range, step,
      [&](int tile) { return tile == freed++ && wait(); },
      [&](int n, bool ok) { blocks += ok ? n : 0; return ok && wait(); },
      [&](bool bad) { met.push_back(bad); return bad; });
  if (after) return "a wait after one that gave up";
  size_t at = 0;
  bool alone = false;
  std::vector<std::pair<int, int>> issued;  // tile, K block
  const bool stop = pq8::issue_products(
      range, step,
      [&](bool) {
        if (at == met.size()) { alone = true; return true; }  // the scheduler never comes
        return static_cast<bool>(met[at++]);
      },
      [&](int tile, int kb, int n) { for (int i = 0; i < n; ++i) issued.emplace_back(tile, kb - kb0 + i); });
  if (alone) return "the issuer waits for a meeting that never comes";
  if (at != met.size()) return "the scheduler waits for a meeting that never comes";
  if (stop != failed) return "the issuer is not told";
  for (size_t i = 0; i < issued.size(); ++i)
    if (issued[i] != std::make_pair(static_cast<int>(i) / k_blocks, static_cast<int>(i) % k_blocks)) return "order";
  if (!failed && issued.size() != static_cast<size_t>(tiles) * k_blocks) return "products left out";
  if (failed && issued.size() >= static_cast<size_t>(tiles) * k_blocks) return "products issued that were not released";
  if (blocks < static_cast<int>(issued.size())) return "products before their operands";
  return nullptr;
}

int main() {
  for (int tiles = 0; tiles <= 4; ++tiles)
    for (int k_blocks = 1; k_blocks <= 7; ++k_blocks)
      for (int step = 1; step <= 3; ++step) {
        const int all = tiles * (1 + (k_blocks + step - 1) / step);  // waits of a run without failures
        for (int fail = -1; fail < all; ++fail)
          if (const char* what = check(tiles, k_blocks, step, fail)) {
            std::printf("%d tiles of %d K blocks, %d a meeting, wait %d: %s\n", tiles, k_blocks, step, fail, what);
            return 1;
          }
      }
  std::puts("meets");
}
'''


def test_scheduler_and_issuer_meet_whatever_fails(tmp_path):
    cxx = shutil.which('g++') or shutil.which('c++')
    if cxx is None:
        pytest.skip('no C++ compiler')
    source = tmp_path / 'schedule.cpp'
    source.write_text(PROGRAM)
    subprocess.run([cxx, '-std=c++17', '-O1', '-I', str(CSRC), str(source), '-o', str(tmp_path / 'schedule')], check=True)
    run = subprocess.run([str(tmp_path / 'schedule')], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and 'meets' in run.stdout, run.stdout
