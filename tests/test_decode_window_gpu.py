"""fa_decode_window on the GPU against attention in 64 bits over the keys that a window and the first tokens leave."""
import numpy as np
import pytest
import torch

from tests.parts_util import Cache

pytestmark = pytest.mark.gpu
SCALE, V_SCALE = 1 / (60 * 60 * 11.0), 1 / 50.0


def call(ctx, c, hq, window, sinks, scale=SCALE, v_scale=V_SCALE, lens=True, seq_len=0, stream=None, scales=(0, 0, 0)):
    d = c.d
    ctx.DecodeWindow(d["q"].data_ptr(), d["k"].data_ptr(), d["v"].data_ptr(), c.o.data_ptr(), c.lse.data_ptr(), d["lens"].data_ptr() if lens else 0, len(c.lens), hq, c.kv, c.hd,
                     c.s_max, seq_len, window, sinks, scale, v_scale, *scales, torch.cuda.current_stream().cuda_stream if stream is None else stream,
                     d["table"].data_ptr() if c.page else 0, c.page, c.width if c.page else 0, c.pages if c.page else 0)


def keys(n, window, sinks):
    return set(range(min(n, sinks))) | set(range(max(0, n - window) if window else 0, n))


LENS = [[1], [64], [65], [700], [0, 1, 2, 63, 64, 65, 127, 128, 129, 1000, 333, 0]]


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (64, 4), (100, 0), (130, 4), (37, 100), (200, 64), (1, 700), (5000, 3), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("hd,kv,group", [(128, 2, 4), (64, 2, 1), (128, 1, 16), (64, 1, 9)])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("page", [0, 64, 192])
def test_window(fa_ctx, lens, hd, kv, group, page, window, sinks):
    c = Cache(len(lens) + window % 97 + sinks % 31, lens, kv, hd, page)
    hq = c.to_gpu(group)
    call(fa_ctx, c, hq, window, sinks)
    o, lse = c.results(hq)
    fa_ctx.DeviceStatus()
    c.check(o, lse, lambda b: keys(lens[b], window, sinks), SCALE, V_SCALE)


def test_many_pieces_and_many_pairs(fa_ctx):
    # pairs that are cut into many pieces; more sequences than a warp keeps lengths of
    for lens, kv, group, hd, window, sinks in [([9000], 1, 5, 128, 7001, 70), ([int(n) for n in np.random.default_rng(2).integers(0, 300, 300)], 2, 2, 64, 90, 4)]:
        c = Cache(3, lens, kv, hd, 64)
        hq = c.to_gpu(group)
        for _ in range(3):   # the counts of arrivals are zero again behind every call
            call(fa_ctx, c, hq, window, sinks)
        o, lse = c.results(hq)
        c.check(o, lse, lambda b: keys(lens[b], window, sinks), SCALE, V_SCALE)


def test_pages_that_the_window_has_passed_are_not_looked_at(fa_ctx):
    lens = [1000, 640, 129]
    c = Cache(5, lens, 2, 128, 64)
    for b, n in enumerate(lens):
        for j in range(c.width):
            if j * 64 >= 4 and (j + 1) * 64 <= n - 200:
                c.table[b, j] = -1 if b else 2 ** 31 - 1
    hq = c.to_gpu(2)
    call(fa_ctx, c, hq, 200, 4)
    c.check(*c.results(hq), lambda b: keys(lens[b], 200, 4), SCALE, V_SCALE)


def test_entries_outside_the_pool_count_as_zeros(fa_ctx):
    lens = [300, 200]
    c = Cache(6, lens, 2, 64, 64)
    c.table[0, 4], c.table[1, 0], c.table[0, 0] = -1, c.pages, -2 ** 31
    hq = c.to_gpu(3)
    call(fa_ctx, c, hq, 100, 4)
    c.check(*c.results(hq), lambda b: keys(lens[b], 100, 4), SCALE, V_SCALE)


def test_one_length_for_all_and_lengths_out_of_range(fa_ctx):
    c = Cache(7, [500, 500], 2, 128, 0, s_max=500)
    hq = c.to_gpu(4)
    call(fa_ctx, c, hq, 90, 5, lens=False, seq_len=333)
    c.check(*c.results(hq), lambda b: keys(333, 90, 5), SCALE, V_SCALE)
    c.d["lens"].copy_(torch.tensor([2 ** 31 - 1, -4]))   # clamped to the cache
    call(fa_ctx, c, hq, 90, 5)
    c.check(*c.results(hq), lambda b: keys((500, 0)[b], 90, 5), SCALE, V_SCALE)


def test_scales_on_the_device_and_negative_ones(fa_ctx):
    lens = [400, 77]
    c = Cache(8, lens, 1, 64, 64)
    hq = c.to_gpu(8)
    s = torch.tensor([1 / 60, -1 / 60, 1 / 50], device="cuda")
    call(fa_ctx, c, hq, 128, 4, 1 / 11.0, 1.0, scales=[s.data_ptr() + 4 * i for i in range(3)])
    f = np.float32
    c.check(*c.results(hq), lambda b: keys(lens[b], 128, 4), float(f(1 / 60)) * float(f(-1 / 60)) * float(f(1 / 11.0)), float(f(1 / 50)))


def test_scores_far_apart(fa_ctx):
    # weights from one to nothing: the running maximum moves often
    lens = [900]
    c = Cache(9, lens, 2, 128, 64)
    hq = c.to_gpu(4)
    call(fa_ctx, c, hq, 500, 4, scale=SCALE * 40)
    c.check(*c.results(hq), lambda b: keys(900, 500, 4), SCALE * 40, V_SCALE)


def test_a_nan_that_is_seen_stays_one(fa_ctx):
    c = Cache(10, [200, 200, 200], 1, 128, 64)
    for b, key in ((0, 150), (1, 60)):   # the second lies between the sinks and the window
        c.k[c.table[b, key // 64], 0, key % 64, 5] = 127
    hq = c.to_gpu(4)
    call(fa_ctx, c, hq, 100, 4)
    o, lse = c.results(hq)
    assert np.isnan(o[0]).all() and np.isnan(lse[0]).all() and np.isfinite(o[1:]).all() and np.isfinite(lse[1:]).all()


def test_no_lse_and_an_output_of_two_byte_alignment(fa_ctx):
    lens = [130, 0, 64]
    c = Cache(11, lens, 2, 64, 64)
    hq = c.to_gpu(2)
    whole, c.o = c.o, torch.full((len(lens) * hq * 64 + 65,), 5.0, dtype=torch.float16, device="cuda")[1:]
    d = c.d
    fa_ctx.DecodeWindow(d["q"].data_ptr(), d["k"].data_ptr(), d["v"].data_ptr(), c.o.data_ptr(), 0, d["lens"].data_ptr(), 3, hq, 2, 64, 0, 0, 100, 4, SCALE, V_SCALE, 0, 0, 0, 0,
                    d["table"].data_ptr(), 64, c.width, c.pages)
    torch.cuda.synchronize()
    got = c.o.clone()
    c.o = whole
    call(fa_ctx, c, hq, 100, 4)
    torch.cuda.synchronize()
    n = len(lens) * hq * 64
    assert torch.equal(got[:n], c.o[:n]) and (got[n:] == 5).all()


def test_captured_on_two_streams_and_the_same_bits(fa_ctx):
    # eager, in a graph, replayed on another stream beside an eager call of other inputs
    lens = [3000, 150, 0, 700]
    c, e = Cache(12, lens, 2, 128, 64), Cache(13, [2500, 64], 2, 128, 64)
    hq = c.to_gpu(4)
    e.to_gpu(4)
    call(fa_ctx, c, hq, 1500, 4)
    call(fa_ctx, e, hq, 1500, 4)
    torch.cuda.synchronize()
    want, want_l, other = c.o.clone(), c.lse.clone(), e.o.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(fa_ctx, c, hq, 1500, 4)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        c.o.zero_()
        e.o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            call(fa_ctx, e, hq, 1500, 4)
        torch.cuda.synchronize()
        n = want.numel() - 64
        assert torch.equal(c.o[:n], want[:n]) and torch.equal(c.lse, want_l) and torch.equal(e.o[:other.numel() - 64], other[:-64])


def test_refusals(fa_ctx):
    from goml_b200 import fa_forward as F
    c = Cache(14, [100], 2, 64, 64)
    c.to_gpu(2)
    for window, sinks in ((-1, 0), (0, -1)):
        with pytest.raises(F.FAError, match="window and sinks must be >= 0"):
            call(fa_ctx, c, 4, window, sinks)
    q = c.d["q"]
    c.d["q"] = torch.zeros(q.numel() + 16, dtype=torch.uint8, device="cuda")[4:]
    with pytest.raises(F.FAError, match="16-byte aligned"):
        call(fa_ctx, c, 4, 5, 0)
    c.d["q"], c.pages = q, 2 ** 31 - 1
    with pytest.raises(F.FAError, match="2\\^31"):
        call(fa_ctx, c, 4, 5, 0)
    with pytest.raises(F.FAError, match="nil ctx"):
        F.FAContext(0).DecodeWindow(*[0] * 15)


def test_calls_behind_a_wait_that_ran_out(fa_ctx):
    # the status says so once; the words that calls keep between them are zero behind it, on every stream, and calls give the same bits as before
    from goml_b200 import fa_forward as F
    c = Cache(23, [3000, 2500], 2, 128, 64)
    hq = c.to_gpu(4)
    streams = [torch.cuda.Stream() for _ in range(3)]
    call(fa_ctx, c, hq, 2000, 4)
    want = [x.copy() for x in c.results(hq)]
    for status in (fa_ctx.DeviceStatus, None):
        for s in streams:
            call(fa_ctx, c, hq, 2000, 4, stream=s.cuda_stream)
        fa_ctx.SelftestWaitExpiry()
        if status:
            with pytest.raises(F.FAError, match="0x2f0"):
                status()
        else:
            assert F.FANoAllocDeviceStatus() == 0x2F0
        for s in streams:
            c.o.fill_(5)
            c.lse.fill_(5)
            torch.cuda.synchronize()
            for _ in range(2):
                call(fa_ctx, c, hq, 2000, 4, stream=s.cuda_stream)
            for x, y in zip(want, c.results(hq)):
                assert np.array_equal(x, y)
    fa_ctx.DeviceStatus()
