"""Which kernels the shapes of operator_shapes.py reach, asked of the rules the library itself uses (csrc/kernels/forms.h, which is
host code): every form has to be among them, so that a later change of a rule cannot leave one untested in silence.  No GPU."""
import os
import shutil
import subprocess

import pytest

from tests import operator_shapes as shapes

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "infmoe_amd", "csrc")
PROGRAM = r"""
#include <cstdio>
#include "kernels/forms.h"
using namespace infmoe::forms;
int main() {
    char what;
    int v[6];
    while (std::scanf(" %c %d %d %d %d %d %d", &what, v, v + 1, v + 2, v + 3, v + 4, v + 5) == 7) {
        if (what == 'l') {  // T d n r size aligned
            const Project p = project_form(v[0], v[1], v[2], v[4], v[5]);
            const int each = 16 / v[4];
            std::printf("%d %d %d %d %d\n", (int)shrink_form(v[0], (v[3] + each - 1) / each * each), (int)p.kind, p.fm, p.fn, p.splits);
        } else {  // slots E d h size aligned
            const Experts f = experts_form(v[0], v[1], v[2], v[3], v[4], v[5]);
            std::printf("%d %d %d %d %d %d\n", (int)f.kind, f.blocks, f.mini, stream_blocks(f.max_tiles, v[3], false),
                        stream_blocks(f.max_tiles, v[3], true), stream_blocks(f.max_tiles, v[2], false));
        }
    }
}
"""
STREAM, TALL, TILES = 0, 1, 2


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    gxx = shutil.which("g++")
    assert gxx is not None, "g++ is needed to build the query"
    at = tmp_path_factory.mktemp("forms")
    (at / "q.cpp").write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", f"-I{CSRC}", str(at / "q.cpp"), "-o", str(at / "q")], check=True)

    def run(lines):
        text = "\n".join(" ".join(str(v) for v in line) for line in lines)
        out = subprocess.run([str(at / "q")], input=text, capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return run


@pytest.mark.parametrize("size", [2, 4])
def test_adapters_shapes_reach_every_form(ask, size):
    whole = ask([("l", T, d, n, r, size, 1) for T, d, n, r in shapes.LORA[size]])
    odd = ask([("l", T, d, n, r, size, 0) for T, d, n, r in shapes.LORA_ODD])
    assert all(d * size % 16 == 0 for _, d, _, _ in shapes.LORA[size]) and all(d * size % 16 for _, d, _, _ in shapes.LORA_ODD)
    assert {f[0] for f in whole} == {f[0] for f in odd} == {0, 1, 2}
    # tall tiles of every height, with K whole and cut
    assert {(f[2], f[4] > 1) for f in whole if f[1] == TALL} == {(fm, cut) for fm in range(2, 9) for cut in (False, True)}
    assert {f[2:4] for f in whole if f[1] == STREAM} == {(1, 1), (1, 2)}
    assert not any(f[1] == TILES for f in whole)
    assert {f[2:4] for f in odd if f[1] == STREAM} == {(1, 1), (1, 2), (2, 1), (2, 2), (4, 1), (4, 2), (4, 4)}
    assert {f[1] for f in odd} == {STREAM, TILES} and all(f[4] == 1 for f in odd)


@pytest.mark.parametrize("size", [2, 4])
def test_experts_shapes_reach_every_form(ask, size):
    whole = ask([("e", T * k, E, d, h, size, 1) for T, k, E, d, h in shapes.EXPERTS])
    odd = ask([("e", T * k, E, d, h, size, 0) for T, k, E, d, h in shapes.EXPERTS_ODD])
    assert {f[0] for f in whole} == {STREAM, TALL, TILES} and {f[0] for f in odd} == {STREAM, TILES}
    for forms in (whole, odd):
        streams = [f for f in forms if f[0] == STREAM]
        assert {f[2] for f in streams if f[1] == 1} == {0, 1}
        for blocks in (1, 2):  # of rows: the first product, the gated one, the second product
            assert {f[3] for f in streams if f[1] == blocks} == {1, 2, 4}, blocks
            assert {f[4] for f in streams if f[1] == blocks} == {2, 4}, blocks
            assert {f[5] for f in streams if f[1] == blocks} == {1, 2, 4}, blocks
