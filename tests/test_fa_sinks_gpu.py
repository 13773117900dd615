"""fa_forward_sinks on the GPU against attention in 64 bits where the first tokens stay visible behind the window."""
import numpy as np
import pytest
import torch

from oracle import parts
from tests.parts_util import codes

pytestmark = pytest.mark.gpu
SCALE, V_SCALE = 1 / (60 * 60 * 11.0), 1 / 50.0


def call(ctx, q, k, v, window, sinks, scale=SCALE, lse=True, entry="sinks"):
    bh, s, hd = q.shape
    o = torch.full((bh * s * hd + 64,), 5.0, dtype=torch.float16, device="cuda")
    le = torch.full((bh * s + 16,), 5.0, device="cuda")
    t = [torch.from_numpy(x).cuda() for x in (q, k, v)]
    tail = (scale, V_SCALE, 0, 0, 0, torch.cuda.current_stream().cuda_stream)
    args = [x.data_ptr() for x in t] + [o.data_ptr(), le.data_ptr() if lse else 0, bh, s, hd]
    if entry == "sinks":
        ctx.ForwardSinks(*args, window, sinks, *tail)
    else:
        ctx.ForwardEx(*args, 1, window, *tail)
    torch.cuda.synchronize()
    ctx.DeviceStatus()
    assert (o[bh * s * hd:] == 5).all() and (le[bh * s:] == 5).all()
    return o[:bh * s * hd].reshape(bh, s, hd), le[:bh * s].reshape(bh, s)


def inputs(seed, bh, s, hd):
    r = np.random.default_rng(seed)
    return codes(r, (bh, s, hd)), codes(r, (bh, s, hd)), codes(r, (bh, s, hd), 50.0)


def check(got, q, k, v, window, sinks, scale=SCALE, rows=None):
    bh, s, hd = q.shape
    o, lse = (x.double().cpu().numpy() for x in got)
    rows = np.arange(s) if rows is None else rows
    j = np.arange(s)
    seen = (j <= rows[:, None]) & ((j > rows[:, None] - window) | (j < sinks))
    for h in range(bh):
        want, want_l, tol, tol_l = parts.attend(q[h, rows], k[h], v[h], seen, scale, V_SCALE)
        assert (np.abs(o[h, rows] - want) <= tol).all(), (h, (np.abs(o[h, rows] - want) / tol).max())
        assert (np.abs(lse[h, rows] - want_l) <= tol_l).all(), (h, (np.abs(lse[h, rows] - want_l) / tol_l).max())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("s,window,sinks", [(1, 1, 1), (2, 1, 1), (64, 1, 1), (65, 1, 64), (129, 64, 4), (300, 7, 3), (300, 64, 64), (300, 64, 65), (300, 64, 100), (300, 130, 128), (300, 100, 199),
                                            (300, 100, 200), (300, 300, 4), (300, 0, 4), (500, 33, 130), (500, 33, 1), (500, 400, 20)])
def test_small(fa_ctx, s, window, sinks, hd):
    q, k, v = inputs(s + window + sinks, 2, s, hd)
    check(call(fa_ctx, q, k, v, window, sinks), q, k, v, window or s, sinks)


@pytest.mark.parametrize("bh,s,hd,window,sinks", [(40, 2500, 128, 300, 4), (400, 700, 64, 100, 70), (3, 6000, 128, 1000, 200), (300, 1100, 128, 129, 5), (24, 3001, 64, 512, 4), (600, 300, 128, 64, 4)])
def test_every_form_of_the_kernel(fa_ctx, bh, s, hd, window, sinks):
    # V converted ahead and in the kernel, one tile to a CTA and several: some rows of some heads
    q, k, v = inputs(bh, bh, s, hd)
    o, lse = call(fa_ctx, q, k, v, window, sinks)
    rows = np.unique(np.concatenate([np.random.default_rng(1).integers(0, s, 40), [0, s - 1, window, min(s - 1, window + sinks), min(s - 1, window + 127)]]))
    heads = [0, bh // 2, bh - 1]
    check((o[heads], lse[heads]), q[heads], k[heads], v[heads], window, sinks, rows=rows)


@pytest.mark.parametrize("hd", [64, 128])
def test_the_same_bits_as_without(fa_ctx, hd):
    q, k, v = inputs(3, 3, 500, hd)
    for window, sinks in ((100, 0), (0, 5), (500, 5), (0, 0)):
        a, b = call(fa_ctx, q, k, v, window, sinks), call(fa_ctx, q, k, v, window, 0, entry="ex")
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # a window and sinks that leave out nothing
    a, b = call(fa_ctx, q, k, v, 300, 200), call(fa_ctx, q, k, v, 0, 0, entry="ex")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_negative_scale_and_scores_far_apart(fa_ctx):
    q, k, v = inputs(4, 2, 400, 128)
    for scale in (-SCALE, 30 * SCALE):
        check(call(fa_ctx, q, k, v, 70, 6, scale), q, k, v, 70, 6, scale)


def test_captured(fa_ctx):
    q, k, v = inputs(5, 30, 1500, 128)
    want = call(fa_ctx, q, k, v, 200, 4)
    t = [torch.from_numpy(x).cuda() for x in (q, k, v)]
    o = torch.empty((30, 1500, 128), dtype=torch.float16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fa_ctx.ForwardSinks(*[x.data_ptr() for x in t], o.data_ptr(), 0, 30, 1500, 128, 200, 4, SCALE, V_SCALE, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0])


def test_refusals(fa_ctx):
    from goml_b200 import fa_forward as F
    q, k, v = inputs(6, 1, 64, 64)
    with pytest.raises(F.FAError, match="sinks must be >= 0"):
        call(fa_ctx, q, k, v, 5, -1)
    for window in (-1, 65):
        with pytest.raises(F.FAError, match="window must be in"):
            call(fa_ctx, q, k, v, window, 1)
    with pytest.raises(F.FAError, match="head_dim"):
        call(fa_ctx, *inputs(6, 1, 64, 96), 5, 1)
    a = F.ForwardArgs(causal=0)
    assert F.FALoad() and F._forward_sinks(fa_ctx.ptr, bytes(a), 1) == F.FA_ERR_INVALID_ARG and F._forward_sinks(None, bytes(a), 1) == F.FA_ERR_INVALID_ARG
    with pytest.raises(F.FAError, match="nil ctx"):
        F.FAContext(0).ForwardSinks(*[0] * 11)


def test_only_causal_prompts(fa_ctx):
    from goml_b200 import fa_forward as F
    t = [torch.from_numpy(x).cuda() for x in inputs(7, 2, 200, 64)]
    o = torch.full((2, 200, 64), 5.0, dtype=torch.float16, device="cuda")
    a = F.ForwardArgs(q=t[0].data_ptr(), k=t[1].data_ptr(), v=t[2].data_ptr(), o=o.data_ptr(), batch_heads=2, seq_len=200, head_dim=64, causal=1, window=70, scale=SCALE, v_descale=1.0,
                      stream=torch.cuda.current_stream().cuda_stream)
    for causal in (0, 2, -1):
        a.causal = causal
        assert F._forward_sinks(fa_ctx.ptr, bytes(a), 4) == F.FA_ERR_INVALID_ARG and fa_ctx._msg() == "fa_forward_sinks: causal must be 1"
    torch.cuda.synchronize()
    assert (o == 5).all()
    a.causal = 1
    assert F._forward_sinks(fa_ctx.ptr, bytes(a), 4) == F.FA_OK
    torch.cuda.synchronize()
    assert (o != 5).any()
