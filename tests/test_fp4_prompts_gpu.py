"""Prompts into a 4-bit pool whose sequences are not all without keys."""
import pytest
import torch

import oracle as O
from tests.test_decoder_block_gpu import _make_block

pytestmark = pytest.mark.gpu


def test_a_prompt_behind_cached_keys_is_not_taken(cuda, built_libs):
    # a prompt's attention counts positions from 0 and does not see the cache: sequences that have keys keep them as they are, and the others' prompts are what they are alone
    from goml_b200 import nn
    B, d, H, Fh, S = 3, 256, 4, 704, 70
    blk, _, _, _, t = _make_block("fp4behind", d, H, Fh)
    pages = nn.KVPages(B, 12, 64, 4)
    pools = [nn.FP4KVPool(pages, H, d // H) for _ in range(2)]
    first = t(O.seeded_normal("first", (B * 20, d), config="fp4behind"))
    pages.plan(torch.tensor([20, 0, 0], dtype=torch.int32, device="cuda"), tokens_per_seq=20)
    for pool in pools:
        blk(first, B, 20, pool)
    before = [pool.rows() for pool in pools]
    slots = pages.slots.clone()
    x = t(O.seeded_normal("x", (B * S, d), config="fp4behind"))
    pages.plan(torch.tensor([S, S, 0], dtype=torch.int32, device="cuda"), tokens_per_seq=S)
    assert pages.taken.tolist() == [0, S, 0] and pages.lens.tolist() == [20, S, 0]
    y = x
    for pool in pools:
        y = blk(y, B, S, pool)
    for pool, (k, v) in zip(pools, before):
        now = pool.rows(slots)
        assert k[:20].any() and torch.equal(now[0], k) and torch.equal(now[1], v)
        k, v = pool.rows()
        assert not k[:S].any() and not v[:S].any() and k[S:2 * S].any() and v[S:2 * S].any()
    # the first goes on by steps
    pages.plan(1)
    assert pages.taken.tolist() == [1, 1, 1] and pages.lens.tolist() == [21, S + 1, 1]
    assert torch.isfinite(blk.decode_step(x[:B], pools[0])).all()
    # one token of prompts is planned as such, and begins the sequences that have ended
    pages.plan(torch.tensor([0, -1, -1], dtype=torch.int32, device="cuda"), tokens_per_seq=1)
    pages.plan(1, prompts=True)
    assert pages.taken.tolist() == [0, 1, 1] and pages.lens.tolist() == [21, 1, 1]
    assert torch.equal(blk(x[:B], B, 1, pools[0]), blk(x[:B], B, 1))
    blk.close()
