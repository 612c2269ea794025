"""The page numbers that a walk over a paged cache looks up: replayed on the CPU with the kernels' own rule (csrc/dsa_paged_ring.h), for every place among the pages that a piece
of keys may begin at.  Runs without a GPU."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vlm_training_amd", "csrc")

# A number on its way is counted as none at all for three steps.  Steps, look-ups and requests in the order of dsa_paged_walk.h: tiles 0 to 5 in front of the walk, then, in step t, K of
# tile t + 6 and V of tile t + 4 behind the request for more numbers.
REPLAY = r"""
#include "dsa_paged_ring.h"
#include <cstdio>
#include <cstdlib>
int main(int, char **argv) {
    const bool early = std::atoi(argv[1]);
    long looked = 0, wrong = 0, pieces = 0;
    for (int pshift = 4; pshift <= 8; ++pshift) {
        const int batch_tiles = 64 << pshift >> 5;
        for (int base = 0; base < 2 * batch_tiles + 3; ++base, ++pieces) {
            const PageRing ring{base, pshift};
            int number[128], there[128];                // which page's, and from which step on
            for (int i = 0; i < 128; ++i) number[i] = -1, there[i] = 0;
            auto load = [&](int batch, int step) {
                for (int i = 0; i < 64; ++i) number[(batch & 1) * 64 + i] = batch * 64 + i, there[(batch & 1) * 64 + i] = step;
            };
            auto look = [&](int tile, int step) {
                for (int wave = 0; wave < 4; ++wave, ++looked) {
                    const int page = ((base + tile) * 32 + 8 * wave) >> pshift, at = PageRing::place(page);
                    wrong += number[at] != page || there[at] > step;
                }
            };
            load(ring.batch(0), -1);
            load(ring.batch(0) + 1, -1);
            for (int tile = 0; tile <= 5; ++tile) look(tile, -1);
            if (early && ring.due_early()) load(ring.batch(2) + 1, 3);
            for (int t = 0; t < 4 * batch_tiles; ++t) {
                if (ring.due(t + 3)) load(ring.batch(t + 3) + 1, t + 3);
                look(t + 6, t);
                look(t + 4, t);
            }
        }
    }
    std::printf("%ld %ld %ld\n", pieces, looked, wrong);
}
"""


def _replay(tmp_path, early):
    source, program = tmp_path / "replay.cpp", tmp_path / "replay"
    source.write_text(REPLAY)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(source), "-o", str(program)], check=True)
    return [int(n) for n in subprocess.run([str(program), str(int(early))], check=True, capture_output=True, text=True).stdout.split()]


def test_every_page_number_is_there_when_it_is_looked_up(tmp_path):
    pieces, looked, wrong = _replay(tmp_path, True)
    assert pieces == sum(2 * (64 << s >> 5) + 3 for s in range(4, 9)) and looked > 10 ** 6 and wrong == 0


def test_replay_sees_a_batch_that_is_never_asked_for(tmp_path):
    assert _replay(tmp_path, False)[2] > 0
