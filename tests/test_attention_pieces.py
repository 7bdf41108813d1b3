"""The rule that cuts the scored attention of many queries into pieces
(csrc/fattn_pieces.h, which the kernel's workgroups evaluate), compiled for the
host: the pieces of all query blocks have a place in the launch's grid, whatever
the span. No device is needed."""

import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include "fattn_pieces.h"
using namespace mi355x;
static uint64_t state = 1;
static int below(int n) { state = state * 6364136223846793005ull + 1442695040888963407ull; return (int) ((state >> 33) % (uint64_t) n); }
int main() {
    static_assert(fs_pieces(0, 4, 9) == 1 && fs_pieces(8, 4, 9) == 2 && fs_pieces(9, 4, 9) == 3 && fs_pieces(100, 4, 9) == 9, "");
    static int open[512];
    long cases = 0;
    for (int slots : {256, 304, 64})
        for (int tiles = 1; tiles <= 16384; tiles++) {
            // (all short spans, the borders of the steps, and some between)
            const bool border = tiles < 600 || tiles % 511 < 6 || tiles % 512 < 6 || tiles % 511 > 508 || tiles % 512 > 508 || tiles % 61 == 0;
            if (!border) continue;
            if (fs_length(0, tiles) != 4 || fs_length(kFsLengths - 1, tiles) < tiles) return printf("%d tiles: lengths\n", tiles), 1;
            for (int like : {1, 8})
                for (int units : {1, 5, slots / 2 + 1, slots - 1}) {
                    const int n_units = units / like;
                    if (n_units < 1) continue;
                    const int split = slots < tiles / 4 ? slots : tiles / 4;
                    if (split < 2) continue;
                    for (int kind = 0; kind < 3; kind++) {  // everything seen, a causal mask, anything
                        for (int u = 0; u < n_units; u++)
                            open[u] = kind == 0 ? tiles : kind == 1 ? 1 + (int) ((int64_t) (tiles - 1) * (u + 1) / n_units) : below(tiles + 1);
                        int first = -1, total = 0;
                        for (int i = 0; i < kFsLengths; i++) {
                            total = 0;
                            for (int u = 0; u < n_units; u++) total += like * fs_pieces(open[u], fs_length(i, tiles), split);
                            if (total <= slots) { first = i; break; }
                        }
                        if (first < 0) return printf("%d tiles, %d blocks: %d pieces of %d\n", tiles, like * n_units, total, slots), 1;
                        cases++;
                    }
                }
        }
    printf("%ld\n", cases);
    return 0;
}
"""


def test_every_piece_has_a_place(tmp_path):
    src, exe = tmp_path / "pieces.cpp", tmp_path / "pieces"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", f"-I{ROOT / 'openasr_amd' / 'csrc'}", str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
    assert int(run.stdout) > 10000
