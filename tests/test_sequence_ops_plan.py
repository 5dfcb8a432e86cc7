"""How embedding_grad shares out the zeros of rows without a token: the host's
plan, compiled from its header, against a replay of what the kernels do with
it (no GPU)."""

import os
import random
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "macmetalpy_b200", "csrc")

PROGRAM = """
#include <cstdio>
#include "mmp_embedding_plan.h"
int main() {
  long long rows, row;
  int beside;
  while (std::scanf("%lld %lld %d", &rows, &row, &beside) == 3) {
    const mmp::EmbZeroPlan p = mmp::emb_zero_plan(rows, row, beside != 0);
    std::printf("%u %u %u\\n", p.first, p.second, p.unit);
  }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """plan([(rows, row bytes, beside the sort), ...]) -> [(first, second, unit), ...]"""
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-I", CSRC, str(d / "plan.cpp"), "-o", str(d / "plan")], check=True)

    def call(cases):
        text = "".join("%d %d %d\n" % c for c in cases)
        out = subprocess.run([str(d / "plan")], input=text, capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return call


def taken_for_empty(first, end, unit, tokens):
    """The rows with tokens that a walk over [first, end) writes zeros to: a
    warp takes `unit` rows from r on and reads their bits from the word of row
    r alone, into whose upper end a shift brings zeros."""
    bad = []
    for r in range(first, end, unit):
        word = 0
        for row in range(r // 32 * 32, r // 32 * 32 + 32):
            word |= (row in tokens) << (row % 32)
        word >>= r % 32
        bad += [r + k for k in range(min(unit, end - r)) if not word >> k & 1 and r + k in tokens]
    return bad


def test_the_replay_sees_a_start_inside_a_word():
    """With the first row where 32 MB end, not rounded, tokens are lost."""
    assert taken_for_empty(21845, 22000, 4, set(range(22000)))
    assert not taken_for_empty(21824, 22000, 4, set(range(22000)))


def test_units_stay_in_their_word(plan):
    rng = random.Random(5)
    cases = [(50257, 1536, True), (50257, 2560, True), (50257, 3200, True), (50257, 2000, True), (1500000, 24, True),
             (100000, 1200, True), (131072, 400, True), (50257, 4096, True), (8192, 512, True), (1, 2, True),
             (1 << 30, 2, True), (20, 3 << 20, True), (27, 3 << 20, True), (3, 30 << 20, True), (81, 1 << 20, True)]
    cases += [(100003, 2 * w, True) for w in range(1, 4200)]
    cases += [(rng.randint(1, 1 << rng.randint(1, 30)), 2 * rng.randint(1, 1 << rng.randint(1, 13)), b)
              for _ in range(4000) for b in (True, False)]
    for (rows, row, beside), (first, second, unit) in zip(cases, plan(cases), strict=True):
        what = (rows, row, beside, first, second, unit)
        assert 0 <= first <= second <= rows, what          # three ranges that together are the table
        assert beside or first == 0, what
        assert unit in (1, 2, 4, 8, 16, 32), what
        for start in (first, second):                       # a walk that begins at a word's edge stays in words
            assert start % 32 == 0 or start == rows, what


def test_no_row_with_a_token_is_zeroed(plan):
    """The walk itself round both borders, every row a token's, and every row
    that is a multiple of 32."""
    cases = [(50257, 1536, True), (50257, 2560, True), (1500000, 24, True), (131072, 400, True), (50257, 2000, False)]
    for (rows, row, _), (first, second, unit) in zip(cases, plan(cases), strict=True):
        for start, end in ((first, second), (second, rows)):
            end = min(end, start + 700)
            assert not taken_for_empty(start, end, unit, set(range(start, end)))
            assert not taken_for_empty(start, end, unit, set(range(start // 32 * 32, end, 32)))
