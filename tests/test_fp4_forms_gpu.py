"""fa_decode_fp4 in every form of its kernel (tests/fp4_forms.py; that each call takes the form that it is for is asked in test_fp4_layout_cpu.py), against the restatement in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import fp4
from tests.fp4_forms import FORMS, _pages
from tests.test_fp4_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", FORMS)
def test_decode_forms(fa_ctx, name):
    f = FORMS[name]
    c = Case(len(name), len(f["distinct"]), f["hq"], f["kv"], f["hd"], f["distinct"], page=64)
    assert c.pages == _pages(f["distinct"]) <= f["pool"]
    order = torch.tensor(f["order"], device="cuda")
    table = torch.full((len(order), f["table"]), 2 ** 30, dtype=torch.int32, device="cuda")     # entries behind what a sequence has are not looked at
    wide = min(f["table"], c.max_pages)
    table[:, :wide] = c.table_d[order][:, :wide]
    q, lens = c.q[order].contiguous(), c.lens_d[order].contiguous()
    o = torch.full((len(order), c.hq, c.hd), 7.0, dtype=torch.float16, device="cuda")
    lse = torch.full((len(order), c.hq), 7.0, device="cuda")

    def call():
        c.call(fa_ctx, out=o, lOut=lse.data_ptr(), q=q.data_ptr(), seq_lens=lens.data_ptr(), block_table=table.data_ptr(), max_pages_per_seq=f["table"], batch=len(order), num_pages=f["pool"])
        return o.clone(), lse.clone()

    first, second = call(), call()
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    ro, rl, spread, size = (x[f["order"]] for x in c.reference())
    n = np.asarray(f["lens"])[:, None].astype(np.float64)
    # A score: hd products, of which each addition may lose 2^-23 of the largest partial sum, and twelve more operations; both sums of the quotient see it.  Weights are rounded to fp16, by 2^-11
    # at most; those below fp16's normal range, 2^-28 of the largest, by 2^-39 of it.  A sum over n keys is one of at most n / 8 additions of a lane, or n / 16 products, each of which may
    # lose 2^-23, and of a few dozen more where states are added up.  O is rounded once more.
    ds = (c.hd + 12) * 2.0 ** -23 * np.maximum(size, 1.0)
    sums = (n / 8 + 64) * 2.0 ** -23
    vmax = float(np.nanmax(np.abs(fp4.values(c.cache["v"], fp4.natural(c.cache["vs"]), c.cache["v_scale"]))))
    tol = (2.0 ** -11 + 2 * ds + 2 * sums)[..., None] * spread + 2.0 ** -11 * np.abs(ro) + n[..., None] * 2.0 ** -39 * vmax + 2.0 ** -24
    o, l = first[0].double().cpu().numpy(), first[1].double().cpu().numpy()
    assert np.isfinite(o).all() and (np.abs(o - ro) <= tol).all(), float((np.abs(o - ro) / tol).max())
    assert np.array_equal(np.isneginf(l), np.isneginf(rl)) and np.array_equal(np.isneginf(rl), np.broadcast_to(n == 0, rl.shape))
    live = np.isfinite(rl)
    assert (np.abs(l[live] - rl[live]) <= (2 * ds + sums + 2.0 ** -20 + 2.0 ** -22 * np.abs(rl))[live]).all()
