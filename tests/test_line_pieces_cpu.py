"""How a line of units is cut into pieces (goml_b200/csrc/fa_line_pieces.h), asked without a GPU."""
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ASK = r"""
#include <cstdio>
#include "fa_line_pieces.h"
int main() {
    long long total, u, n;
    int pieces;
    while (std::scanf("%lld %d %lld %lld", &total, &pieces, &u, &n) == 4) {
        const fa_sm100::Pieces x(total, pieces);
        const fa_sm100::Pieces::Span s = x.pieces_of(u, n, pieces);
        std::printf("%d %d %lld %lld\n", s.first, s.count, x.begin(s.first), x.begin(s.first + s.count));
    }
}
"""


@pytest.fixture(scope="module")
def pieces(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    exe = str(tmp_path_factory.mktemp("pieces") / "ask")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "goml_b200", "csrc"), "-x", "c++", "-", "-o", exe],
                       input=ASK, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def ask(calls):
        r = subprocess.run([exe], input="\n".join(" ".join(map(str, c)) for c in calls), capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        lines = r.stdout.split("\n")[:-1]
        assert len(lines) == len(calls)
        return [tuple(map(int, x.split())) for x in lines]

    return ask


def test_pieces_that_hold_units_of_the_line(pieces):
    r = random.Random(1)
    calls = []
    for _ in range(3000):
        count = r.choice([1, 2, 3, 148, 592, r.randint(1, 700)])
        total = r.choice([1, count, r.randint(1, 3 * count), r.randint(1, 10 ** 6), r.randint(1, 2 ** 45)])
        u = r.randrange(total)
        calls.append((total, count, u, r.randint(1, min(total - u, 2 ** 31 - 1))))
    for (total, count, u, n), (first, parts, begin, end) in zip(calls, pieces(calls)):
        # the pieces that begin and end there are the nearest ones around the units, and equal to within a unit
        small, more = divmod(total, count)
        starts = [i * small + min(i, more) for i in (first, first + 1, first + parts - 1, first + parts)]
        assert 0 <= first and first + parts <= count and (begin, end) == (starts[0], starts[3])
        assert starts[0] <= u < starts[1] and starts[2] <= u + n - 1 < starts[3]


def test_units_that_are_not_on_the_line_have_pieces_that_there_are(pieces):
    # lengths that change while a call runs, which its header forbids, can put a pair anywhere: its states' places must be those of CTAs of the launch all the same
    r = random.Random(2)
    calls = []
    for _ in range(3000):
        count = r.choice([1, 2, 148, 592])
        total = r.choice([1, 2, count, count + 1, r.randint(1, 10 ** 6)])
        u = r.choice([-1, total - 1, total, total + r.randint(1, 10 ** 6), r.randint(-2 ** 40, 2 ** 40), 2 ** 62, -2 ** 62])
        calls.append((total, count, u, r.choice([1, 2, r.randint(1, 2 ** 31 - 1), 0, -5])))
    for call, (first, parts, _, _) in zip(calls, pieces(calls)):
        assert first >= 0 and parts >= 1 and first + parts <= call[1], call
