"""The walk over the tokens that no sequence covers (gdn_ops.h), compiled for
the host: it ends for every content of starts, also where they decrease, and
gives the uncovered tokens where they do not."""
import os
import random
import subprocess

import pytest

from gateddeltanet_b200 import build

PROGRAM = r"""
#include "gdn_ops.h"
#include <stdio.h>
#include <vector>
int main() {
    int tokens, entries;
    while (scanf("%d %d", &tokens, &entries) == 2) {
        std::vector<int32_t> starts(entries);
        for (int &s : starts) scanf("%d", &s);
        gdn::ops::DeltaParams p = {};
        p.starts = starts.data();
        p.N = entries - 1;
        p.tokens = tokens;
        const gdn::ops::Covered c = gdn::ops::covered_tokens(p);
        uint32_t steps = 0, t = c.first_outside();
        for (; t < p.tokens && steps <= p.tokens; t = c.next_outside(t), ++steps) printf("%u ", t);
        puts(t < p.tokens ? "-1" : "");
    }
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    (d / "walk.cu").write_text(PROGRAM)
    subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "-I", build.CSRC, "-I", os.path.join(build.REPO, "include"),
                    "-o", str(d / "walk"), str(d / "walk.cu")], check=True)

    def run(cases):
        text = "".join(f"{tokens} {len(starts)} {' '.join(map(str, starts))}\n" for tokens, starts in cases)
        out = subprocess.run([str(d / "walk")], input=text, capture_output=True, text=True, check=True, timeout=60).stdout
        return [list(map(int, line.split())) for line in out.splitlines()]
    return run


def test_decreasing_starts_end(walk):
    rng = random.Random(1)
    cases = [(20, [10, 3, 5]), (10, [4, 8, 0, 0]), (10, [5, 8, 3, 2]), (10, [0, 5, 9, 0, 0]), (7, [2 ** 31 - 1, -5]),
             (5, [5, 0]), (1, [1, 0])]
    cases += [(rng.randint(0, 40), [rng.randint(-3, 45) for _ in range(rng.randint(2, 6))]) for _ in range(300)]
    for (tokens, starts), outside in zip(cases, walk(cases)):
        assert -1 not in outside, (tokens, starts)
        assert outside == sorted(set(outside)) and all(0 <= t < tokens for t in outside), (tokens, starts)


def test_uncovered_tokens(walk):
    rng = random.Random(2)
    cases = [(tokens, sorted(rng.randint(-2, tokens + 2) for _ in range(rng.randint(2, 6))))
             for tokens in (rng.randint(0, 40) for _ in range(300))]
    for (tokens, starts), outside in zip(cases, walk(cases)):
        first, end = (max(0, min(x, tokens)) for x in (starts[0], starts[-1]))
        assert outside == [t for t in range(tokens) if not first <= t < end], (tokens, starts)
