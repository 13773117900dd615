"""fa_decode_fp4 where scores are far larger than any model's."""
import numpy as np
import pytest
import torch

from oracle import fp4
from tests.test_fp4_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [16, 20, 23, 24, 25, 26, 28, 40, 80])
@pytest.mark.parametrize("hd,hq,kv,n", [(128, 4, 4, 300), (64, 16, 1, 700)])
def test_decode_of_scores_of_any_size(fa_ctx, hd, hq, kv, n, power, sign):
    # One key is 50 times 2^power ahead of all others (their differences are lost in 32 bits from 2^24 on): O is its value, rounded once, LSE its score.  With the sign turned it is as far behind, and
    # another key is far ahead of the rest: one whose dims are all negative.
    c = Case(hd + power, 1, hq, kv, hd, [n], page=64, q_type="fp16")
    at = {1: n // 2, -1: n - 2}
    c.cache["ks"] = np.where(c.cache["ks"] == 0x7F, 0x7F, np.minimum(c.cache["ks"], 0x40)).astype(np.uint8)
    for s, place in at.items():
        page, row = c.table[0, place // 64], place % 64
        c.cache["k"][page, :, row], c.cache["ks"][page, :, row] = (0x77 if s > 0 else 0xFF), 0x70      # every dim 6 or -6, 128 and the tensor scale
    c.qd = torch.full_like(c.qd, 1.0)
    c.load()
    c.scale *= sign * 2.0 ** power
    c.call(fa_ctx)
    ro, rl, _, _ = c.reference()
    page, row = c.table[0, at[sign] // 64], at[sign] % 64
    v = (fp4.values(c.cache["v"], fp4.natural(c.cache["vs"]), c.cache["v_scale"]))[page, :, row].astype(np.float64)
    assert (np.abs(ro - np.repeat(v, hq // kv, axis=0)[None]) <= 2.0 ** -20 * np.abs(v).max()).all()
    o, l = c.o.double().cpu().numpy(), c.lse.double().cpu().numpy()
    # weights below 2^-39 of the largest are nothing; the largest one is rounded to fp16, and O once more
    assert (np.abs(o - ro) <= 2.0 ** -10 * np.abs(ro) + 2.0 ** -20 * np.abs(v).max() + 2.0 ** -24).all(), np.abs(o).max()
    assert (np.abs(l - rl) <= (hd + 16) * 2.0 ** -23 * np.abs(rl)).all()
