"""csrc/heads_index.h compiled for the host: over all head and rotary sizes that each form
takes, 16 and 64 lanes place every value of a head once, and a lane's pairs are the
rotation's."""
import os
import subprocess

import pytest

from pixelina_amd import build

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "heads_index.h"
using namespace pixhip;

static int bad(const char* form, int lanes, int dim, int rotary, int lane)
{
    std::printf("%s of %d lanes: head of %d, rotary %d, lane %d\n",form,lanes,dim,rotary,lane);
    return 1;
}

template <int G, int MODE>
int wide()
{
    const char* form = MODE == kTurnAdjacent? "adjacent" : "halves";
    for (int dim = 4; dim <= 8 * G; dim += 4)
        for (int rotary = 0; rotary <= dim; rotary += 8) {
            std::vector<int> seen(dim / 4);
            for (int lane = 0; lane < G; lane++) {
                int o[2] = {-1,-1};
                turn_quads<MODE>(lane,rotary,o[0],o[1]);
                for (int q : o) {
                    if (q < 0 || q % 4) return bad(form,G,dim,rotary,lane);
                    if (q < dim) seen[q / 4]++;
                }
                // pairs 4 lane .. + 3
                if (4 * lane < rotary / 2 && (MODE == kTurnAdjacent? o[0] != 8 * lane || o[1] != o[0] + 4 : o[0] != 4 * lane || o[1] != rotary / 2 + 4 * lane))
                    return bad(form,G,dim,rotary,lane);
            }
            for (int n : seen)
                if (n != 1) return bad(form,G,dim,rotary,-1);
        }
    return 0;
}

template <int G>
int scalar()
{
    for (int dim = 1; dim <= 8 * G; dim++)
        for (int rotary = 0; rotary <= dim; rotary += 2)
            for (int interleaved = 0; interleaved < 2; interleaved++) {
                std::vector<int> seen(dim);
                for (int lane = 0; lane < G; lane++)
                    for (int j = 0; j < 4; j++) {
                        int a = -1, b = -1;
                        turn_pair<G>(lane,j,rotary,interleaved != 0,a,b);
                        if (a < 0 || b < 0) return bad("scalar",G,dim,rotary,lane);
                        const int pair = lane + G * j;
                        if (pair < rotary / 2 && (interleaved? a != 2 * pair || b != a + 1 : a != pair || b != pair + rotary / 2)) return bad("scalar",G,dim,rotary,lane);
                        if (a < dim) seen[a]++;
                        if (b < dim) seen[b]++;
                    }
                for (int n : seen)
                    if (n != 1) return bad("scalar",G,dim,rotary,-1);
            }
    return 0;
}

int main()
{
    return wide<16,kTurnHalves>() || wide<16,kTurnAdjacent>() || wide<64,kTurnHalves>() || wide<64,kTurnAdjacent>() || scalar<16>() || scalar<64>();
}
"""


@pytest.fixture(scope="module")
def compiled(tmp_path_factory):
    def make(header):
        d = tmp_path_factory.mktemp("heads")
        (d / "heads_index.h").write_text(header)
        (d / "check.cpp").write_text(PROGRAM)
        subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", str(d / "check.cpp"), "-o", str(d / "check")], check=True)
        return subprocess.run([str(d / "check")], capture_output=True, text=True)
    return make


def source():
    with open(os.path.join(build.HERE, "csrc", "heads_index.h")) as f:
        return f.read()


def test_every_value_is_placed_once(compiled):
    done = compiled(source())
    assert done.returncode == 0, done.stdout


@pytest.mark.parametrize("right,wrong", [("o2 = rotary / 2 + 4 * lp", "o2 = rotary / 4 + 4 * lp"), ("o1 = rotary + 8 * (lp - rotary / 8)", "o1 = rotary + 4 * (lp - rotary / 8)"),
                                         ("ia = rotary + 2 * (p - half)", "ia = rotary + p - half")])
def test_a_misplaced_value_is_found(compiled, right, wrong):
    assert right in source()
    assert compiled(source().replace(right, wrong)).returncode == 1
