"""RoPE tables of the blocks on one KVPages."""
import numpy as np
import pytest
import torch

import oracle as O
from tests.test_decoder_block_gpu import _make_block

pytestmark = pytest.mark.gpu


def test_layers_share_their_tables(cuda, built_libs):
    # tables of all pages' tokens, as KVPages has them by default: once, not for each layer
    from goml_b200 import nn
    B, d, H, Fh = 2, 256, 4, 704
    blocks = [_make_block(f"fp4rope{i}", d, H, Fh) for i in range(3)]
    t = blocks[0][-1]
    pages = nn.KVPages(B, 1 << 12, 64)
    pools = [nn.FP4KVPool(pages, H, d // H) for _ in blocks]
    x = t(O.seeded_normal("x", (B, d), config="fp4rope"))
    pages.plan(1)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for (blk, *_), pool in zip(blocks, pools):
        assert torch.isfinite(blk.decode_step(x, pool)).all()
    assert torch.cuda.memory_allocated() - before < 1.5 * pages.capacity * 4 * (d // H)
    for blk, *_ in blocks:
        blk.close()


def test_a_step_captured_before_any_other(cuda, built_libs):
    # what a graph writes when it is replayed is not there for the calls before that
    from goml_b200 import nn
    B, d, H, Fh = 2, 256, 4, 704
    blk, _, _, _, t = _make_block("fp4first", d, H, Fh)
    x = t(O.seeded_normal("x", (B, d), config="fp4first"))

    def step(pages, pool):
        pages.plan(1)
        return blk.decode_step(x, pool)

    def fresh(num_pages):
        pages = nn.KVPages(B, num_pages, 64, num_pages // B)
        return pages, nn.FP4KVPool(pages, H, d // H)

    step(*fresh(4))            # set-up of what a first call sets up
    ref = fresh(8)
    want = [step(*ref) for _ in range(4)]
    other = fresh(8)
    blk._rope.clear()          # no tables of this many rows from the calls above
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        y = step(*other)
    assert torch.equal(step(*other), want[0])
    assert torch.equal(step(*other), want[1])      # the first step with two keys to choose between
    graph.replay()
    assert torch.equal(y, want[2])
    assert torch.equal(step(*other), want[3])
    blk.close()


@pytest.mark.parametrize("rows,hd", [((1 << 25) - 1, 128), ((1 << 25) + 3, 128)])
def test_tables_whose_entries_pass_31_bits(cuda, built_libs, rows, hd):
    # as long as a table of pages may be wide: the last index, and a step of the grid past it, are beyond an int
    from goml_b200 import block_glue as BG
    half = hd // 2
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.fail("this test takes 17 GB of the GPU")
    tables = torch.full((2, rows, half), 7.0, device="cuda")
    BG.RopeTable(tables[0].data_ptr(), tables[1].data_ptr(), rows, hd, 10000.0, torch.cuda.current_stream().cuda_stream)
    at = np.unique(np.concatenate([[0, 1, 2, 4095, rows // 2, (1 << 24) + 1, rows - 2, rows - 1], np.random.default_rng(0).integers(0, rows, 200)]))
    got = tables[:, torch.from_numpy(at).cuda()].double().cpu().numpy()
    angle = at[:, None] * 10000.0 ** (-2.0 * np.arange(half) / hd)
    # rounded to 32 bits; angles up to 2^25 that are off by a few of their last bits in 64 (2^-28 together)
    for x, want in zip(got, (np.cos(angle), np.sin(angle))):
        assert (np.abs(x - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -25).all()
    assert not (tables[:, -1] == 7).any()
