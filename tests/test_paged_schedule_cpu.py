"""CPU test of the arithmetic behind the paged attention's schedule (csrc/paged_schedule.h): the closed forms that
the blocks locate their work with, against sums over every unit."""
import re
import subprocess
from pathlib import Path

import fav4_bshd as F

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "paged_schedule.h"
using namespace fav4;
int main() {
  srand(1);
  const int groups[] = {1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 32, 100, 128};
  long checked = 0;
  for (int it = 0; it < 20000; ++it) {
    SeqView s;
    s.q0 = 0;
    s.sq = 1 + rand() % (it % 3 ? 300 : 5000);
    s.len = it % 5 == 0 ? rand() % (s.sq + 1) : it % 7 == 0 ? s.sq : s.sq + rand() % 6000;
    if (it % 11 == 0) s.len = -rand() % 500;  // all rows before the first key
    const int bt = 128 / groups[rand() % 13] * (1 + rand() % 2), causal = it % 4 != 0;
    const int units = (s.sq + bt - 1) / bt;
    long sum = 0;
    for (int r = 0; r <= units; ++r, ++checked) {
      if (units_steps(s, causal, bt, r) != sum) {
        printf("sq %d len %d bt %d causal %d: %ld steps before unit %d, not %ld\n", s.sq, s.len, bt, causal, sum, r,
               (long)units_steps(s, causal, bt, r));
        return 1;
      }
      if (r == units) break;
      const long end = (r + 1L) * bt < s.sq ? (r + 1L) * bt : s.sq, keys = causal ? (long)s.len - s.sq + end : s.len;
      const long want = keys <= 0 ? 1 : (keys + 127) / 128;
      if (unit_steps(s, causal, bt, r) != want) return 2;
      sum += want;
    }
    if (tile_seq_work(s, causal, bt) != sum + kUnitExtra * units) return 3;
  }
  // units on a line, cut into stretches as the blocks do it, each from the unit that holds its begin to the last
  // one that begins before its end: every step is taken once, in order, by consecutive blocks
  for (int it = 0; it < 20000; ++it) {
    const int per = 1 + rand() % (it % 4 ? 9 : 60), units = 1 + rand() % 12;
    long first[13] = {0};
    int n[12], done[12] = {0}, opened[12], last[12];
    for (int u = 0; u < units; ++u) {
      n[u] = 1 + rand() % (it % 5 ? 12 : 200);
      if (it % 2 && rand() % 2) n[u] = 1;
      first[u + 1] = first[u] + kUnitExtra + n[u];
      opened[u] = last[u] = -1;
    }
    for (long c = 0; c * per < first[units]; ++c) {
      const long begin = c * per, end = begin + per < first[units] ? begin + per : first[units];
      for (int u = 0; u < units; ++u) {
        if (first[u + 1] <= begin || first[u] >= end) continue;
        const long step0 = first[u] + kUnitExtra;
        const int from = steps_before(begin - step0, n[u]), to = steps_before(end - step0, n[u]);
        if (to <= from) continue;
        if (from != done[u] || (last[u] >= 0 && c != last[u] + 1)) return 5;
        if (from == 0) opened[u] = (int)c;
        done[u] = to;
        last[u] = (int)c;
      }
    }
    for (int u = 0; u < units; ++u) {
      const long step0 = first[u] + kUnitExtra;
      if (done[u] != n[u] || opened[u] != step0 / per || last[u] != (step0 + n[u] - 1) / per) return 6;
    }
  }
  if (quotient(1L << 40, 3) != (1L << 40) / 3 || quotient(7, 1L << 33) != 0 || quotient(4294967295L, 2) != 2147483647L) return 4;
  printf("%ld\n", checked);
  return 0;
}
"""


def test_closed_forms(tmp_path):
    src, exe = tmp_path / "schedule.cpp", tmp_path / "schedule"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", f"-I{F.PKG_ROOT / 'csrc'}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout)
    assert int(r.stdout) > 100000


KERNELS = r"""
#include <cstdio>
#include "paged_schedule.h"
using namespace fav4;
int main() {
  const int heads_of[] = {1, 2, 7, 8, 16, 40, 128, 160, 256, 1024}, batches[] = {1, 2, 5, 33, 64, 1000};
  const long tokens_of[] = {1, 2, 3, 4, 5, 8, 15, 16, 17, 64, 127, 128, 129, 257, 1023, 1024, 5000};
  const long tables[] = {16, 64, 400, 2048, 8192, 1 << 20};
  int seen[3] = {0};
  for (int heads : heads_of)
    for (int kv = 1; kv <= heads; ++kv) {
      if (heads % kv) continue;
      for (long tokens : tokens_of)
        for (int batch : batches)
          for (long keys : tables) {
            const int tiles = q_tiles(tokens, batch, heads / kv, kv, keys);
            if (tiles < 0 || tiles > q_tiles_bound(tokens, heads)) {
              printf("heads %d kv %d tokens %ld batch %d keys %ld: %d tiles\n", heads, kv, tokens, batch, keys, tiles);
              return 1;
            }
            ++seen[tiles];
          }
    }
  return seen[0] && seen[1] && seen[2] ? 0 : 2;
}
"""


def test_workspaces_have_room_for_every_choice_of_kernel(tmp_path):
    src, exe = tmp_path / "kernels.cpp", tmp_path / "kernels"
    src.write_text(KERNELS)
    subprocess.run(["g++", "-O1", "-std=c++17", f"-I{F.PKG_ROOT / 'csrc'}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout)


def test_an_aborted_block_waits_for_every_copy_it_issued():
    # a block that gives up must not leave shared memory while a copy is on its way there: each barrier that a TMA
    # load of the tile kernel signals is waited for where its load warps leave early
    code = (F.PKG_ROOT / "csrc" / "paged_tile_sm100.cuh").read_text()
    barriers = set(re.findall(r"tma_load_\dd\([^;]*?(bar\(L::\w+\)|\bfb\b)", code))
    assert barriers == {"bar(L::kQFull)", "fb"} and "fb = bar(L::kKVFull + ring.stage)" in code
    abort = code[code.index("if (*abort_flag) {"):]
    abort = abort[:abort.index("__syncwarp();")]
    assert re.search(r"wait_phase\(bar\(L::kKVFull \+ s\)", abort) and re.search(r"wait_phase\(bar\(L::kQFull\)", abort)


def test_parity_of_the_last_query_load():
    # LoadState's q_empty is 1 before the first load and turns with each; a barrier's phases complete in order, and
    # waiting for parity p passes once the phase of that parity has (a new one has parity 1 behind it)
    for loads in range(6):
        q_empty = 1
        for _ in range(loads):
            q_empty ^= 1
        for complete in {loads, max(loads - 1, 0)}:
            passes = (complete - 1) % 2 == q_empty  # the phase before the current one
            assert passes == (complete == loads)
