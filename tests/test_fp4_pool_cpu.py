"""KVPages, FP4KVPool and the block's calls on them, without a GPU: what they refuse, and where and with what they launch."""
import ctypes
import types

import pytest
import torch

from goml_b200 import nn


@pytest.mark.parametrize("scale", [float("inf"), 1e39, 7.7e35, 1e-46, 0.0, -1.0, float("nan")])
def test_scales_that_the_cache_cannot_have(scale):
    # 448 of a scale have to be a number of 32 bits, and the scale itself one above zero
    pages = nn.KVPages(2, 8, 64, 3, device="cpu")
    for name in ("k_scale", "v_scale"):
        with pytest.raises(ValueError, match="FP4KVPool"):
            nn.FP4KVPool(pages, 2, 64, **{name: scale})


@pytest.mark.parametrize("scale", [2.0 ** -149, 1e-40, 1 / 32, 7.5e35])
def test_scales_that_it_can(scale):
    pool = nn.FP4KVPool(nn.KVPages(2, 8, 64, 3, device="cpu"), 2, 64, k_scale=scale, v_scale=scale)
    assert (pool.scales > 0).all() and torch.isfinite(448 * pool.scales).all()


CPU = torch.device("cpu")
current = ["another device"]     # the thread's current device, as a stack


class On:
    """torch.cuda.device"""

    def __init__(self, device):
        self.device = device

    def __enter__(self):
        current.append(self.device)

    def __exit__(self, *_):
        current.pop()


def ints(pointer, n):
    return list((ctypes.c_int32 * n).from_address(pointer))


@pytest.fixture
def planned(monkeypatch):
    """What KVPages.plan hands to the planner, call by call: the binding's arguments, with the new tokens read through their pointer."""
    calls = []

    def plan(lens, fresh, *rest):
        calls.append(dict(lens=lens, fresh=ints(fresh, rest[9]), rows=rest[13], tokens_per_seq=rest[14], stream=rest[15]))

    monkeypatch.setattr(nn.BG, "KVPagePlan", plan)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=("stream of", device or current[-1])))
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return calls


def test_sequences_that_have_keys_take_no_prompt(planned):
    pages = nn.KVPages(4, 16, 64, 4, device="cpu")
    pages.lens.copy_(torch.tensor([61, 0, 3, 0]))
    fresh = torch.tensor([10, 10, -1, 0], dtype=torch.int32)
    pages.plan(fresh, tokens_per_seq=10)
    assert planned[-1]["fresh"] == [0, 10, -1, 0] and pages.prompts and fresh.tolist() == [10, 10, -1, 0]
    pages.plan(7)
    assert planned[-1]["fresh"] == [0, 7, 0, 7] and pages.prompts
    # tokens that go on behind what is there, and steps of one
    pages.plan(fresh, tokens_per_seq=10, prompts=False)
    assert planned[-1]["fresh"] == [10, 10, -1, 0] and not pages.prompts
    pages.plan(1)
    assert planned[-1]["fresh"] == [1, 1, 1, 1] and not pages.prompts
    pages.plan(1, prompts=True)
    assert planned[-1]["fresh"] == [0, 1, 0, 1] and pages.prompts
    pages.plan(fresh, rows=20)
    assert planned[-1]["fresh"] == [10, 10, -1, 0] and not pages.prompts
    with pytest.raises(ValueError, match="KVPages.plan: packed"):
        pages.plan(fresh, rows=20, prompts=True)


def block(hd=64, heads=2):
    blk = nn.FP8DecoderBlock.__new__(nn.FP8DecoderBlock)   # no weights: nothing here gets as far as a kernel
    blk.d, blk.H, blk.hd, blk.F, blk.fused = heads * hd, heads, hd, 128, True
    return blk


def test_prompts_need_a_plan_of_prompts(planned):
    pages = nn.KVPages(2, 8, 64, 3, device="cpu")
    pool = nn.FP4KVPool(pages, 2, 64)
    for fresh, S, how in ((5, 5, dict(prompts=False)), (1, 1, {})):
        pages.plan(fresh, **how)
        with pytest.raises(ValueError, match="the pool must .* rows of prompts"):
            block()(torch.zeros(2 * S, 128), 2, S, pool)


def test_launches_are_on_the_tensors_device(planned, monkeypatch):
    # whatever device is current: a launch goes to that one, and pointers and stream are those of the pages' device
    pages = nn.KVPages(2, 8, 64, 3, device="cpu")
    pool = nn.FP4KVPool(pages, 2, 64)
    seen = []
    plan = nn.BG.KVPagePlan
    monkeypatch.setattr(nn.BG, "KVPagePlan", lambda *a: (seen.append(("plan", current[-1], a[-1])), plan(*a)))
    monkeypatch.setattr(nn.BG, "FP4CacheRows", lambda *a: seen.append(("rows", current[-1], a[-1])))
    pages.plan(3)
    pool.rows()
    assert seen == [(name, CPU, ("stream of", CPU)) for name in ("plan", "rows")] and current == ["another device"]


def test_the_block_launches_on_its_inputs_device(planned, monkeypatch):
    class Stop(Exception):
        pass

    def first_launch(*a):
        assert current[-1] == CPU and a[-1] == ("stream of", CPU)
        raise Stop

    pages = nn.KVPages(2, 8, 64, 3, device="cpu")
    pool = nn.FP4KVPool(pages, 2, 64)
    blk = block()
    blk.norm1, blk.eps, blk.theta = torch.ones(128), 1e-5, 10000.0
    monkeypatch.setattr(nn.BG, "RopeTable", lambda *a: None)
    monkeypatch.setattr(nn.BG, "RMSNormQuantizeInto", first_launch)
    pages.plan(1)
    with pytest.raises(Stop):
        blk.decode_step(torch.zeros(2, 128), pool)
    assert current == ["another device"]
    blk.norm1 = torch.ones(128, device="meta")
    with pytest.raises(ValueError, match="the pool must lie on"):
        blk.decode_step(torch.zeros(2, 128), pool)


def test_one_pair_of_rope_tables_for_all_blocks(planned, monkeypatch):
    made, capturing = [], [False]
    monkeypatch.setattr(nn.BG, "RopeTable", lambda cos, sin, rows, hd, theta, stream: made.append((rows, hd, theta, current[-1], stream)))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    pages = nn.KVPages(2, 8, 64, 3, device="cpu")
    capturing[0] = True
    graph = pages.rope_tables(64, 10000.0)     # nobody else is given what only a replay writes
    capturing[0] = False
    a = pages.rope_tables(64, 10000.0)
    assert a is not graph and a is pages.rope_tables(64, 10000) and a[0].shape == a[1].shape == (192, 32)
    assert pages.rope_tables(64, 500000.0) is not a and pages.rope_tables(128, 10000.0)[0].shape == (192, 64)
    assert made == [(192, 64, 10000.0, CPU, ("stream of", CPU))] * 2 + [(192, 64, 500000.0, CPU, ("stream of", CPU)), (192, 128, 10000.0, CPU, ("stream of", CPU))]
