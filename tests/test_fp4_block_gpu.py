"""The decoder block on a KV cache held in 4 bits: plan, append and attention together, as a server's steps are, against the CPU restatement with the same quantisation points
(bars of tests/test_decoder_block_gpu.py)."""
import numpy as np
import pytest
import torch

import oracle as O
from oracle import fp4
from oracle.decoder_block import decoder_block_decode_step_fp4
from tests.test_decoder_block_gpu import _make_block

pytestmark = pytest.mark.gpu


def state_of(pool):
    get = lambda x: x.cpu().numpy().copy()   # noqa: E731
    s = get(pool.scales)
    return dict(k=get(pool.k), ks=get(pool.ks), v=get(pool.v), vs=get(pool.vs), k_scale=s[0], v_scale=s[1])


@pytest.mark.parametrize("d,H,Fh,page", [(512, 4, 1376, 64), (256, 4, 704, 128)])
def test_a_server_prompt_and_steps(cuda, built_libs, d, H, Fh, page):
    from goml_b200 import nn
    B, S, hd = 3, 61, d // H
    cfg = f"fp4block{d}"
    blk, w, g1, g2, t = _make_block(cfg, d, H, Fh)
    pages = nn.KVPages(B, 9, page, 3)
    pool = nn.FP4KVPool(pages, H, hd, k_scale=0.011, v_scale=0.013)
    x = O.seeded_normal("x", (B * S, d), config=cfg)
    xd = t(x)
    pages.plan(S)
    assert pages.taken.tolist() == [S] * B and pages.lens.tolist() == [S] * B
    y = blk(xd, B, S, pool)
    assert torch.equal(y, blk(xd, B, S))             # the prompt's own output is that without a cache
    # what the prompt has left in the pool is its projections, rotated and in 4 bits
    cache = state_of(pool)
    k, v = pool.rows()
    assert k.shape == (B * S, H, hd) and torch.isfinite(k).all() and k.float().abs().mean() > 0.01 and v.float().abs().mean() > 0.01
    lens = np.full(B, S)
    ended = np.zeros(B, bool)
    for step in range(6):
        fresh = np.array([1, 1, 1], np.int32)
        if step == 2:
            fresh[1] = 0                              # waits
        if step == 4:
            fresh[2] = -1                             # ends, and its place is vacant for a step
        pages.plan(torch.from_numpy(fresh).cuda(), tokens_per_seq=1)
        positions = np.where(fresh > 0, lens, -1)
        lens = np.where(fresh < 0, 0, lens + np.maximum(fresh, 0))
        assert np.array_equal(pages.positions.cpu().numpy(), positions) and np.array_equal(pages.lens.cpu().numpy(), lens)
        x = O.seeded_normal(f"x{step}", (B, d), config=cfg)
        tables = pages.table.cpu().numpy()
        ref = decoder_block_decode_step_fp4(x, positions, cache, tables, lens, H, w["wqkv"], w["wo"], w["wgate_up"], w["wdown"], g1, g2)
        got = blk.decode_step(t(x), pool).double().cpu().numpy()
        blk.fa.DeviceStatus()
        maxabs, meanrel = O.error_stats(got, ref)
        assert maxabs <= 2e-2 and meanrel <= 1e-2, (step, maxabs, meanrel)
        maxabs_d, meanrel_d = O.error_stats(got - x, ref - x)
        assert maxabs_d <= 2e-2 and meanrel_d <= 5e-2, (step, maxabs_d, meanrel_d)
        # the cache's bytes up to isolated neighbouring codes, where the projection's rounding went the other way
        now = state_of(pool)
        for n in ("k", "v", "ks", "vs"):
            assert (now[n] != cache[n]).mean() < 1e-3, n
        cache = now
        ended |= fresh < 0
    assert ended.any()
    blk.close()


def test_steps_replayed_from_a_graph(cuda, built_libs):
    # plan and two layers in one graph, replayed: pages are taken up as the sequences grow over a page's end; the same calls eagerly give the same bits
    from goml_b200 import nn
    B, d, H, Fh, S = 4, 256, 4, 704, 62
    blk, _, _, _, t = _make_block("fp4graph", d, H, Fh)
    outs = []
    for graphed in (False, True):
        pages = nn.KVPages(B, 10, 64, 3)
        pools = [nn.FP4KVPool(pages, H, d // H) for _ in range(2)]
        x = t(O.seeded_normal("x", (B * S, d), config="fp4graph"))
        pages.plan(S)
        for pool in pools:
            blk(x, B, S, pool)
        x = t(O.seeded_normal("xs", (B, d), config="fp4graph"))

        def step():
            pages.plan(1, tokens_per_seq=1)
            return blk.decode_step(blk.decode_step(x, pools[0]), pools[1])

        run = step
        if graphed:
            saved = [a.clone() for a in (pages.table, pages.lens, pages.ring, pages.state)]
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step()                       # set-up of what a first call sets up
            torch.cuda.synchronize()
            for a, b in zip((pages.table, pages.lens, pages.ring, pages.state), saved):
                a.copy_(b)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=torch.cuda.Stream()):
                y = step()

            def run():
                g.replay()
                return y
        outs.append([run().clone() for _ in range(5)])
        assert pages.lens.tolist() == [S + 5] * B and (pages.table[:, 1] >= 0).all() and pages.state[1] == 2
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    blk.close()


def test_a_captured_step_outlives_other_plans(cuda, built_libs):
    # between replays other steps are planned, with more rows and fewer, and what they leave behind them is written over: the graph's plan writes where it did
    from goml_b200 import nn
    B, d, H, Fh, S = 2, 256, 4, 704, 30
    blk, _, _, _, t = _make_block("fp4outlive", d, H, Fh)
    x = t(O.seeded_normal("x", (B * S, d), config="fp4outlive"))
    token = t(O.seeded_normal("t", (B, d), config="fp4outlive"))
    end = torch.full((B,), -1, dtype=torch.int32, device="cuda")

    def prompt(pages, pool, s):
        pages.plan(end, tokens_per_seq=1)
        pages.plan(s)
        blk(x[:B * s], B, s, pool)

    outs = []
    for graphed in (False, True):
        pages = nn.KVPages(B, 8, 64, 2)
        pool = nn.FP4KVPool(pages, H, d // H)
        prompt(pages, pool, S)

        def step():
            pages.plan(1, tokens_per_seq=1)
            return blk.decode_step(token, pool)

        run = step
        if graphed:
            step()
            prompt(pages, pool, S)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=torch.cuda.Stream()):
                y = step()

            def run():
                g.replay()
                return y
        got, keep = [], []
        for s in (S, 3, 20):
            prompt(pages, pool, s)
            for n in (2, 4, 60, 64, 128, 1024):      # memory that was freed would be among these
                keep.append([torch.full((n,), 2 ** 30, dtype=torch.int32, device="cuda") for _ in range(20)])
            got += [run().clone() for _ in range(2)]
            assert pages.lens.tolist() == [s + 2] * B
        assert all((a == 2 ** 30).all() for k in keep for a in k)
        outs.append(got)
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    blk.close()


@pytest.mark.parametrize("fresh,num_pages,taken", [((0, 70, 70, 20), 3, (0, 70, 0, 0)),     # the third asks for pages that are not there, and the fourth comes after it
                                                   ((0, 70, 1, 20), 4, (0, 70, 1, 20)), ((64, 0, 65, 0), 3, (64, 0, 65, 0))])
def test_prompts_padded_and_not_taken(cuda, built_libs, fresh, num_pages, taken):
    # rows keep their places whatever is taken, and the pool holds what the same prompt leaves in one with room for all
    from goml_b200 import nn
    d, H, Fh, S, B = 256, 4, 704, 70, 4
    blk, _, _, _, t = _make_block("fp4pad", d, H, Fh)
    x = t(O.seeded_normal("x", (B * S, d), config="fp4pad"))
    pages = nn.KVPages(B, num_pages, 64, 2)
    pool = nn.FP4KVPool(pages, H, d // H)
    pages.plan(torch.tensor(fresh, dtype=torch.int32, device="cuda"), tokens_per_seq=S)
    assert pages.taken.tolist() == pages.lens.tolist() == list(taken)
    blk(x, B, S, pool)
    k, v = (a.view(B, S, H, -1) for a in pool.rows())
    full = nn.KVPages(B, 2 * B, 64, 2)
    other = nn.FP4KVPool(full, H, d // H)
    full.plan(S)
    blk(x, B, S, other)
    fk, fv = (a.view(B, S, H, -1) for a in other.rows())
    for a, f in ((k, fk), (v, fv)):
        for b, n in enumerate(taken):
            assert torch.equal(a[b, :n], f[b, :n]) and f[b].any() and not a[b, n:].any()
    blk.close()


def test_pools_and_pages_are_looked_at(cuda, built_libs):
    from goml_b200 import nn
    blk, _, _, _, t = _make_block("fp4refuse", 256, 4, 704)
    pages = nn.KVPages(2, 6, 64, 3)
    x = torch.zeros(2, 256, device="cuda")
    for pool in (nn.FP4KVPool(pages, 2, 64), nn.FP4KVPool(pages, 4, 128), nn.FP4KVPool(nn.KVPages(3, 6, 64, 3), 4, 64), nn.FP4KVPool(pages, 4, 64)):
        with pytest.raises(ValueError, match="the pool must"):   # the last one: no step planned
            blk.decode_step(x, pool)
    pages.plan(1, tokens_per_seq=1)
    pool = nn.FP4KVPool(pages, 4, 64)
    assert torch.isfinite(blk.decode_step(x, pool)).all()
    with pytest.raises(ValueError, match="the pool must"):
        blk(torch.zeros(2 * 10, 256, device="cuda"), 2, 10, pool)
    pages.plan(torch.zeros(2, dtype=torch.int32, device="cuda"), rows=2)     # as many rows, but packed
    with pytest.raises(ValueError, match="the pool must"):
        blk.decode_step(x, pool)
    k, v = pool.rows(torch.tensor([-1, 0], dtype=torch.int32, device="cuda"))
    assert not k[0].any() and k.shape == (2, 4, 64)
    with pytest.raises(ValueError, match="rows: slots"):
        pool.rows(torch.zeros(2, device="cuda"))
    blk.close()
