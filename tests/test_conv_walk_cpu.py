"""The walk of the short convolution over its tiles (conv_part of gdn_ops.h),
compiled for the host: whatever starts holds, no row outside x is read; where
it does not decrease, every token is computed once, by the tile that may."""
import os
import subprocess

import pytest

from gateddeltanet_b200 import build

PROGRAM = r"""
#include "gdn_ops.h"
#include <algorithm>
#include <stdio.h>
#include <stdlib.h>
#include <vector>
using namespace gdn::ops;

long long tokens, checked, sorted_walks, far;
void row(long long t, const char *what) {
    ++checked;
    if ((t < 0 || t >= tokens) && ++far <= 20) printf("row %lld of %lld tokens: %s\n", t, tokens, what);
}
uint32_t clamped(int s) { return s < 0 ? 0u : std::min<uint32_t>(s, tokens); }

/* the rows that conv_kernel reads and writes of one sequence from the walk's token t on; returns the walk's next token */
uint32_t rows_of(uint32_t bound, uint32_t end, uint32_t t, uint32_t t0, uint32_t t1, uint32_t back, std::vector<int> *done) {
    const ConvPart part = conv_part(bound, end, t, t0, t1, back);
    t = part.t;
    auto take = [&](uint32_t i) {
        row(i, "taken");
        if (done != nullptr && i < done->size()) ++(*done)[i];
    };
    if (part.begins) {
        const uint32_t few = std::min(back, end - t);
        for (uint32_t i = 0; i < few; ++i) take(t + i);
        if (end - t > back)
            for (uint32_t j = 0; j < back; ++j) row((long long)end - back + j, "of the slot's new content");
        t += few;
    }
    if (t < part.stop)
        for (uint32_t j = 0; j < back; ++j) row((long long)t - back + j, "of the window");
    for (; t < part.stop; ++t) take(t);
    return part.stop;
}

int main(int, char **argv) {
    const int most = atoi(argv[1]), entries = atoi(argv[2]), tiles[] = {1, 2, 4, 22, 128};
    std::vector<int> starts(entries);
    for (tokens = 1; tokens <= most; ++tokens) {
        long long arrays = 1;
        for (int i = 0; i < entries; ++i) arrays *= tokens + 1;
        for (long long a = 0; a < arrays; ++a) {
            long long rest = a;
            for (int &s : starts) s = (int)(rest % (tokens + 1)), rest /= tokens + 1;
            const bool up = std::is_sorted(starts.begin(), starts.end());
            for (uint32_t back = 1; back <= 3; ++back)
                for (int tile : tiles) {
                    std::vector<int> done(tokens, 0);
                    for (uint32_t t0 = 0; t0 < tokens; t0 += tile) {
                        const uint32_t t1 = std::min<uint32_t>(t0 + tile, tokens);
                        /* the walk may come to any sequence at any token */
                        for (int n = 1; n < entries; ++n)
                            for (uint32_t t = t0; t < t1; ++t)
                                if (clamped(starts[n]) > t) rows_of(clamped(starts[n - 1]), clamped(starts[n]), t, t0, t1, back, nullptr);
                        if (!up) continue;
                        uint32_t t = t0;
                        int n = (int)(std::upper_bound(starts.begin(), starts.end(), (int)t0) - starts.begin());
                        while (t < t1) {
                            const uint32_t end = n < entries ? clamped(starts[n]) : tokens;
                            if (n < entries && end <= t) {
                                ++n;
                            } else if (n == 0 || n == entries) {
                                for (const uint32_t stop = std::min(end, t1); t < stop; ++t) ++done[t];
                                ++n;
                            } else {
                                t = rows_of(clamped(starts[n - 1]), end, t, t0, t1, back, &done);
                                ++n;
                            }
                        }
                    }
                    if (up) {
                        ++sorted_walks;
                        for (int n : done)
                            if (n != 1 && ++far <= 20) printf("a token taken %d times\n", n);
                    }
                }
        }
    }
    printf("%lld %lld %lld\n", checked, sorted_walks, far);
    return far != 0;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    (d / "walk.cu").write_text(PROGRAM)
    subprocess.run([build.nvcc(), *build.ARCH, "-O2", "-std=c++17", "-I", build.CSRC, "-I", os.path.join(build.REPO, "include"),
                    "-o", str(d / "walk"), str(d / "walk.cu")], check=True)
    return str(d / "walk")


@pytest.mark.parametrize("most,entries", [(9, 4), (30, 3), (6, 5)])
def test_every_starts_of_few_tokens(walk, most, entries):
    """All arrays of so many entries over up to `most` tokens, tiles of 1 to 128 tokens, widths 2 to 4."""
    run = subprocess.run([walk, str(most), str(entries)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout
    checked, sorted_walks, far = map(int, run.stdout.split())
    assert checked > 100000 and sorted_walks > 1000 and far == 0
