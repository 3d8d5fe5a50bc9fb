"""Which pieces of memory share a byte (rt/overlap.hpp), against a count of their bytes; and that
the row operators' entry points, which refuse such calls, look at all of them. No GPU."""

import os
import re
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

HARNESS = r"""
#include <cstdio>
#include "rt/overlap.hpp"
using namespace ovvs::rt;
int main() {
  long long a, ar, ac, al, b, br, bc, bl;
  while (std::scanf("%lld %lld %lld %lld %lld %lld %lld %lld", &a, &ar, &ac, &al, &b, &br, &bc, &bl) == 8)
    std::printf("%d\n", overlap(span_of(reinterpret_cast<void*>(a), ar, ac, al, 2),
                                span_of(reinterpret_cast<void*>(b), br, bc, bl, 2)) ? 1 : 0);
  Span none{}, one = span_of(reinterpret_cast<void*>(4096), 8, 4);
  Span two = span_of(reinterpret_cast<void*>(4096 + 32), 8, 4);
  Span in = span_of(reinterpret_cast<void*>(4096 + 28), 1, 8);
  std::printf("%d%d%d%d%d\n", clash({one, two}, {none}), clash({one, none}, {two}),
              clash({one}, {in}), clash({none, two, in}, {none}), clash({none}, {one}));
}
"""


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("needs g++")
    d = tmp_path_factory.mktemp("overlap")
    src = d / "overlap.cpp"
    src.write_text(HARNESS)
    subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "ovvs_b200", "csrc"), str(src), "-o",
                    str(d / "overlap")], check=True)
    return str(d / "overlap")


def bytes_of(at, rows, cols, ld):
    return {at + 2 * (r * ld + c) + i for r in range(rows) for c in range(cols) for i in (0, 1)}


def test_overlap_against_the_bytes(harness):
    rng = np.random.default_rng(1)
    cases, want = [], []
    while len(cases) < 4000:
        a, b = (int(v) for v in 1000 + 2 * rng.integers(0, 60, 2))
        ar, br = (int(v) for v in rng.integers(1, 6, 2))
        ac, bc = (int(v) for v in rng.integers(1, 12, 2))
        al = ac + int(rng.integers(0, 8))
        bl = bc + int(rng.integers(0, 8))
        kind = len(cases) % 4
        if kind == 0:
            bl = bc  # b in one piece
        elif kind == 1:
            al = ac
        elif kind == 2:
            bl = al  # one pitch
            if bl < bc:
                continue
        got = bool(bytes_of(a, ar, ac, al) & bytes_of(b, br, bc, bl))
        if kind == 3 and al != bl and ar > 1 and br > 1 and al != ac and bl != bc:
            if got:
                continue  # two pitches: may be overlooked, but what shares nothing is not refused
        cases.append((a, ar, ac, al, b, br, bc, bl))
        want.append(int(got))
    out = subprocess.run([harness], input="\n".join(" ".join(map(str, c)) for c in cases),
                         check=True, capture_output=True, text=True).stdout.split()
    assert out[-1] == "00110"
    wrong = [(c, w) for c, w, g in zip(cases, want, out) if int(g) != w]
    assert not wrong, wrong[:5]
    assert 500 < sum(want) < 3500


def test_every_pointer_of_the_row_operators_is_looked_at():
    src = open(os.path.join(ROOT, "ovvs_b200", "csrc", "rt", "rows_abi.cpp")).read()
    bodies = re.findall(r"^ovvsStatus (ovvs\w+)\((.*?)\) \{\n(.*?)^\}", src, re.S | re.M)
    assert len(bodies) == 4
    for name, args, body in bodies:
        for p in re.findall(r"\bd_\w+", args):
            assert f"span_of({p}," in body, (name, p)
