"""Which slots of a paged cache the lanes of the attention kernels address
(sym_amd/csrc/attend_share.h), gone through on the CPU: pages are whole groups of
sixteen slots there, and a group may be the cache's last."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sym_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "attend_share.h"

template <int DP, int CELL, int W, bool TURNS> void walk() {
  constexpr int NT = TURNS ? 32 : 32 / W; // turns: a wave brings whole tiles
  using S = relx::Share<DP, CELL, NT>;
  int past = 0, past_bare = 0, brought = 0;
  for (int wave = 0; wave < (TURNS ? 1 : W); ++wave)
    for (int i = 0; i < S::LOADS; ++i)
      for (int lane = 0; lane < 64; ++lane) {
        const int t0 = wave * NT + i * S::TPI; // of the load's first token in the tile
        past += (t0 & 15) + S::token(lane) > 15;
        past_bare += (t0 & 15) + lane / S::TL > 15;
        if (S::brings(lane)) {
          if (S::token(lane) != lane / S::TL)
            ++past;
          brought += lane % S::TL == 0;
        }
      }
  std::printf("%d %d %d %d %d %d %d\n", DP, CELL, W, TURNS, past, past_bare, brought);
}

template <int DP, int CELL> void widths() {
  walk<DP, CELL, 4, true>();
  walk<DP, CELL, 4, false>();
  walk<DP, CELL, 8, false>();
}

int main() {
  widths<64, 1>(), widths<64, 2>(), widths<128, 1>(), widths<128, 2>(), widths<256, 1>(), widths<256, 2>();
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_lanes_stay_in_their_group_of_slots(tmp_path):
    source, exe = tmp_path / "share.cpp", str(tmp_path / "share")
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I" + CSRC, str(source), "-o", exe], check=True)
    rows = [[int(x) for x in line.split()] for line in subprocess.run([exe], check=True, capture_output=True, text=True)
            .stdout.splitlines()]
    assert len(rows) == 18
    for width, cell, waves, turns, past, _, brought in rows:
        assert past == 0, (width, cell, waves, turns)
        assert brought == 32, "every token of a tile, once"
    # by its bare number a lane would pass the end of the group in these forms
    assert [(w, c, n) for w, c, n, t, _, bare, _ in rows if bare] == [(64, 1, 4), (64, 1, 8), (64, 2, 8), (128, 1, 8)]
