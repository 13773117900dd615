"""Which teams and plan fa_decode_fp4 chooses (goml_b200/csrc/fa_decode_fp4_layout.h), asked without a GPU: the forms that the GPU tests are to reach, and that what is chosen can be launched."""
import os
import shutil
import subprocess

import numpy as np
import pytest

from tests.fp4_forms import FORMS, form_of

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SMS = 148

ASK = r"""
#include <cstdio>
#include "fa_decode_fp4_layout.h"
int main() {
    int batch, hq, hkv, span, sms;
    long long rows;
    while (std::scanf("%d %d %d %d %lld %d", &batch, &hq, &hkv, &span, &rows, &sms) == 6) {
        const fa_fp4::Layout x = fa_fp4::layout_of(batch, hq, hkv, span, rows, sms);
        std::printf("%s %s %d %d %d %d\n", x.plan == fa_fp4::LINE ? "line" : "pair", x.alone ? "warps" : "ctas", x.grid, x.rows, x.pieces(), x.slots());
    }
}
"""


@pytest.fixture(scope="module")
def layout(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    exe = str(tmp_path_factory.mktemp("layout") / "ask")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "goml_b200", "csrc"), "-x", "c++", "-", "-o", exe], input=ASK, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def ask(calls):
        text = "\n".join(" ".join(map(str, (*c, SMS))) for c in calls)
        lines = subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout.split("\n")[:-1]
        assert len(lines) == len(calls)
        return [(x[0], x[1], *map(int, x[2:])) for x in map(str.split, lines)]

    return ask


@pytest.mark.parametrize("name", FORMS)
def test_the_gpu_tests_reach_the_forms_they_are_for(layout, name):
    f = FORMS[name]
    (plan, teams, grid, rows, pieces, _), = layout([form_of(f)])
    assert (plan, teams) == (f["plan"], f["teams"]) and rows == (8 if f["hq"] // f["kv"] <= 8 else 16)
    chunks = [-(-n // 64) for n in f["lens"]]
    per_step = 4 if teams == "ctas" else 1
    if plan == "pair":
        piece = max(chunks)
    else:   # as the kernel cuts the line
        least, more = (12, 5) if teams == "ctas" else (2, 1)
        piece = f["kv"] * sum(c + max(more, least - c) for c in chunks if c) / pieces
        assert max(chunks) / piece >= f["cuts"] + 1
    if "steps" in f:
        assert piece / per_step > f["steps"] + (6 if plan == "line" else 0)    # less what a pair costs beyond its chunks


def test_whatever_is_chosen_can_be_launched(layout):
    r = np.random.default_rng(0)
    calls = []
    for _ in range(3000):
        kv = int(r.choice([1, 2, 4, 8, 32, 128]))
        batch = int(np.exp(r.uniform(0, np.log(100000))))
        span = int(np.exp(r.uniform(0, np.log(2 ** 31 - 64)))) // 16 * 16
        share = int(np.exp(r.uniform(0, np.log(span + 2))))
        calls.append((batch, kv * int(r.integers(1, 17)), kv, span, batch * share))
    for (batch, hq, kv, span, _), (plan, teams, grid, rows, pieces, slots) in zip(calls, layout(calls)):
        per_cta = 4 if teams == "warps" else 1
        assert rows == (8 if hq // kv <= 8 else 16) and grid > 0 and pieces == grid * per_cta
        if plan == "pair":
            assert (grid - 1) * per_cta < batch * kv <= grid * per_cta
        else:
            assert grid <= SMS * (3 if rows == 8 else 2) and batch * kv * (-(-span // 64) + 12) < 2 ** 31 and slots >= 2 * pieces + 2 * -(-pieces // 8)
