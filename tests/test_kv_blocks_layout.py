"""The block cache's layout (csrc/kv_blocks.h) as plain arithmetic: every (token, dim) has a byte of its own
inside its slice, at the place the matrix instruction's operands are read from, and the scale's exponent is the
smallest that fits."""

import math
import struct
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "gguf_train_amd" / "csrc"

PROGRAM = r"""
#include "kv_blocks.h"
#include <cstdio>
#include <cstring>
#include <vector>
using namespace gtkvb;
int main(int argc, char **argv) {
    for (int Dp : {64, 128, 256}) {
        const int64_t tokens = 192;
        for (int which = 0; which < 2; ++which) {
            std::vector<int> seen(tokens * Dp, 0);
            for (int64_t t = 0; t < tokens; ++t)
                for (int d = 0; d < Dp; ++d) {
                    const int64_t at = which ? v_at(t, d, Dp) : k_at(t, d, Dp);
                    if (at < 0 || at >= tokens * Dp || seen[at]++) return 1;
                    // a unit's bytes stay in the unit
                    if (at / (kUnit * Dp) != t / kUnit) return 2;
                }
        }
        // lane 16 g + m of KiB i: dims 16 (4i + g) .. of token m; dim 16 i + m of tokens 16 kb + 4 g + r
        for (int64_t tile = 0; tile < 12; ++tile)
            for (int i = 0; i < Dp / 64; ++i)
                for (int lane = 0; lane < 64; ++lane)
                    for (int e = 0; e < 16; ++e)
                        if (k_at(16 * tile + lane % 16, 16 * (4 * i + lane / 16) + e, Dp) != tile * 16 * Dp + 1024 * i + 16 * lane + e) return 3;
        for (int64_t unit = 0; unit < 3; ++unit)
            for (int i = 0; i < Dp / 16; ++i)
                for (int lane = 0; lane < 64; ++lane)
                    for (int e = 0; e < 16; ++e)
                        if (v_at(64 * unit + 16 * (e / 4) + 4 * (lane / 16) + e % 4, 16 * i + lane % 16, Dp) != unit * 64 * Dp + 1024 * i + 16 * lane + e) return 4;
    }
    // a tail row is read inside the tail, whatever span of tokens a workgroup looks at
    for (int shift = 5; shift <= 7; ++shift)
        for (int held = 0; held < 300; ++held)
            for (int p = 0; p < 512; ++p) {
                const int row = p - (held >> shift << shift);
                const bool want = p < held && p / (1 << shift) == held / (1 << shift);
                if (in_tail(p, held, shift) != want) return 6;
                if (want && (row < 0 || row >= 1 << shift || row >= held % (1 << shift))) return 7;
            }
    if (padded_dim(1) != 64 || padded_dim(64) != 64 || padded_dim(65) != 128 || padded_dim(129) != 256 || padded_dim(256) != 256) return 5;
    for (int i = 1; i < argc; ++i) {
        unsigned bits;
        sscanf(argv[i], "%u", &bits);
        printf("%d %d\n", scale_exponent(bits, false), scale_exponent(bits, true));
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("layout")
    (d / "p.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(d / "p.cpp"), "-o", str(d / "p")], check=True)
    return d / "p"


def test_every_value_has_its_place(program):
    assert subprocess.run([program]).returncode == 0


def test_scale_exponents(program):
    values = [127.0, 126.99999, 127.00001, 448.0, 447.99997, 448.00003, 1.0, 0.9921875, 0.992188, 1e-30, 1e30, 3.4e38,
              1.17549435e-38, 1e-42, 63.5, 63.500004, 2.0 ** -119 * 127 / 128, 0.0]
    bits = [struct.unpack("<I", struct.pack("<f", v))[0] for v in values]
    out = subprocess.run([program, *map(str, bits)], capture_output=True, text=True, check=True).stdout.split("\n")
    for v, line in zip(values, out):
        v = struct.unpack("<f", struct.pack("<f", v))[0]
        for e, top in zip(map(int, line.split()), (127.0, 448.0)):
            want = -126
            while v > top * math.ldexp(1.0, want):
                want += 1
            assert e == want, (v, top, e, want)
