"""fa_decode_shared on the GPU against attention in 64 bits over each sequence's own keys."""
import numpy as np
import pytest
import torch

from tests.parts_util import Cache

pytestmark = pytest.mark.gpu
SCALE, V_SCALE = 1 / (60 * 60 * 11.0), 1 / 50.0


def ints(x):
    return torch.tensor([int(i) for i in x], dtype=torch.int32, device="cuda")


def call(ctx, c, hq, starts, shared, scale=SCALE, v_scale=V_SCALE, scales=(0, 0, 0)):
    d = c.d
    if "starts" not in d:
        d["starts"], d["shared"] = ints(starts), ints(shared)
    ctx.DecodeShared(d["q"].data_ptr(), d["k"].data_ptr(), d["v"].data_ptr(), c.o.data_ptr(), c.lse.data_ptr(), d["lens"].data_ptr(), d["shared"].data_ptr(), d["starts"].data_ptr(),
                     len(starts) - 1, len(c.lens), hq, c.kv, c.hd, c.s_max, scale, v_scale, *scales, torch.cuda.current_stream().cuda_stream, d["table"].data_ptr() if c.page else 0,
                     c.page, c.width if c.page else 0, c.pages if c.page else 0)


def room(lens, kv, hd, groups=1):
    """Keys that every sequence can have so that the call does not leave each to read its own: 1.9 10^8 bytes (of head dim 64 10^8) that sharing can save (of groups of one it saves none)."""
    return int((1.91e8 if hd == 128 else 1.01e8) / (max(len(lens) - groups, 1) * kv * hd * 2)) + 1


def run(ctx, seed, lens, starts, shared, kv, group, hd, page, calls=1, small=False, **kw):
    c = Cache(seed, lens, kv, hd, page, room=0 if small else room(lens, kv, hd, len(starts) - 1))
    c.share(starts, shared)
    hq = c.to_gpu(group)
    for _ in range(calls):
        call(ctx, c, hq, starts, shared, **kw)
    o, lse = c.results(hq)
    ctx.DeviceStatus()
    c.check(o, lse, lambda b: range(lens[b]), kw.get("scale", SCALE), kw.get("v_scale", V_SCALE))


# lengths, groups' starts, lengths in common
SMALL = [
    ([1], [0, 1], [1]), ([1], [0, 1], [0]), ([0], [0, 1], [0]), ([0], [0, 1], [5]), ([70], [0, 1], [64]), ([64, 64], [0, 2], [64, 64]), ([64, 65], [0, 2], [64, 64]),
    ([300, 200, 131, 130, 0, 129], [0, 6], [130, 130, 130, 130, 130, 128]),            # of different lengths, one empty, one with nothing of its own
    ([300, 300, 300, 300], [0, 1, 2, 4], [0, 299, 64, 64]),                            # groups of one
    ([200, 50, 200, 70, 200], [0, 5], [200, 40, 199, 70, 1]),                          # different parts in common with the first
    ([100, 100, 90], [0, 0, 3, 3], [63, 63, 63]),                                      # groups without sequences
    ([40, 500, 60], [0, 3], [40, 40, 1000]),                                           # above its own length: counts as that
]


@pytest.mark.parametrize("hd,kv,group", [(128, 2, 4), (64, 2, 1), (128, 1, 16), (64, 1, 9), (64, 3, 2), (128, 8, 1)])
@pytest.mark.parametrize("case", SMALL)
@pytest.mark.parametrize("page", [0, 64, 192])
@pytest.mark.parametrize("small", [False, True])
def test_small(fa_ctx, case, hd, kv, group, page, small):
    # small: few keys in all, which the call has every sequence read for itself
    lens, starts, shared = case
    if case is SMALL[-1]:
        lens = [70, 500, 60]
    run(fa_ctx, len(lens) + hd, lens, starts, shared, kv, group, hd, page, small=small)


@pytest.mark.parametrize("hd,kv,group,page", [(128, 2, 4, 64), (64, 1, 16, 128), (128, 1, 5, 0)])
def test_more_rows_than_a_tile_and_long_prefixes(fa_ctx, hd, kv, group, page):
    r = np.random.default_rng(4)
    shared = [1990] * 70 + [700] * 3 + [0] * 2
    lens = [n + int(x) for n, x in zip(shared, r.integers(0, 200, 75))]
    run(fa_ctx, 5, lens, [0, 70, 73, 75], shared, kv, group, hd, page, calls=3)


def test_many_groups(fa_ctx):
    # more pieces than CTAs are resident: a CTA takes several, and slots, rings and tensor memory go on from one to the next
    r = np.random.default_rng(6)
    sizes = r.integers(1, 6, 150)
    starts = [0, *np.cumsum(sizes).tolist()]
    base = r.integers(1, 200, 150)
    shared = [int(x) for x, n in zip(base, sizes) for _ in range(n)]
    lens = [n + int(x) for n, x in zip(shared, r.integers(0, 70, len(shared)))]
    run(fa_ctx, 7, lens, starts, shared, 4, 2, 64, 64, calls=2)


def test_scores_far_apart_and_scales_on_the_device(fa_ctx):
    lens, shared = [900, 850, 840, 835], [800, 800, 799, 800]
    run(fa_ctx, 8, lens, [0, 4], shared, 2, 4, 128, 64, scale=SCALE * 40)
    c = Cache(9, lens, 2, 64, 64, room=room(lens, 2, 64))
    c.share([0, 4], shared)
    hq = c.to_gpu(4)
    s = torch.tensor([1 / 60, -1 / 60, 1 / 50], device="cuda")
    call(fa_ctx, c, hq, [0, 4], shared, 1 / 11.0, 1.0, scales=[s.data_ptr() + 4 * i for i in range(3)])
    f = np.float32
    c.check(*c.results(hq), lambda b: range(lens[b]), float(f(1 / 60)) * float(f(-1 / 60)) * float(f(1 / 11.0)), float(f(1 / 50)))


def test_nans_stay_with_those_who_see_them(fa_ctx):
    # behind a prefix, between what two sequences have of it, and inside it; among keys and among values
    lens, shared = [400, 400, 150, 400], [300, 300, 100, 300]
    for where in ("k", "v"):
        for key, hit in ((120, (True, True, False, True)), (20, (True,) * 4), (310, (True, False, False, False))):
            c = Cache(10, lens, 1, 128, 64, room=room(lens, 1, 128))
            c.share([0, 4], shared)
            x = c.k if where == "k" else c.v
            x[c.table[0, key // 64], 0, key % 64, 77] = 127 if key == 20 else 255
            if key < 100:   # the copies of a page that is not whole keep what they have: this one is whole for all
                assert (c.table[:, key // 64] == c.table[0, key // 64]).all()
            hq = c.to_gpu(4)
            for _ in range(2):   # of a call before, nothing is left
                call(fa_ctx, c, hq, [0, 4], shared)
            o, lse = c.results(hq)
            for b in range(4):
                # (a NaN among values makes NaN of all of O where it is common to the group, of its own dim where it is not)
                assert np.isnan(o[b]).any() == hit[b] and (np.isnan(o[b]).all(1) | np.isnan(o[b][:, 77]) | ~np.isnan(o[b]).any(1)).all(), (where, key, b)
            free = [b for b in range(4) if not hit[b]]
            assert np.isfinite(lse[free]).all()


@pytest.mark.parametrize("small", [False, True])
def test_entries_outside_the_pool_count_as_zeros(fa_ctx, small):
    lens, shared = [300, 250], [200, 200]
    c = Cache(11, lens, 2, 64, 64, room=0 if small else room(lens, 2, 64))
    c.share([0, 2], shared)
    c.table[0, 1] = c.table[1, 1] = -1
    c.table[0, 4] = -2 ** 31
    hq = c.to_gpu(3)
    call(fa_ctx, c, hq, [0, 2], shared)
    c.check(*c.results(hq), lambda b: range(lens[b]), SCALE, V_SCALE)


def test_starts_that_do_not_ascend_stay_inside_the_buffers(fa_ctx):
    lens = [200, 180, 170, 160]
    c = Cache(12, lens, 2, 128, 64, room=room(lens, 2, 128, 3))
    hq = c.to_gpu(4)
    for starts in ([0, 4, 0, 4, 0], [9, -3, 2 ** 31 - 1, -2 ** 31, 4], [4, 3, 2, 1, 0]):
        c.d.pop("starts", None)
        call(fa_ctx, c, hq, starts, [150] * 4)
        c.results(hq)   # what lies behind O and LSE is untouched
        fa_ctx.DeviceStatus()
    c.d.pop("starts")
    call(fa_ctx, c, hq, [0, 1, 2, 3, 4], [150] * 4)
    c.check(*c.results(hq), lambda b: range(lens[b]), SCALE, V_SCALE)


def test_captured_on_two_streams_and_the_same_bits(fa_ctx):
    lens, shared = [1100, 1030, 1000, 1200, 5], [1000, 1000, 1000, 900, 5]
    c, e = Cache(13, lens, 2, 128, 64, room=room(lens, 2, 128, 2)), Cache(14, [500, 470], 2, 128, 64, room=room([0, 0], 2, 128))
    c.share([0, 4, 5], shared)
    e.share([0, 2], [460, 460])
    hq = c.to_gpu(4)
    e.to_gpu(4)
    call(fa_ctx, c, hq, [0, 4, 5], shared)
    call(fa_ctx, e, hq, [0, 2], [460, 460])
    torch.cuda.synchronize()
    want, want_l, other = c.o.clone(), c.lse.clone(), e.o.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(fa_ctx, c, hq, [0, 4, 5], shared)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        c.o.zero_()
        e.o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            call(fa_ctx, e, hq, [0, 2], [460, 460])
        torch.cuda.synchronize()
        assert torch.equal(c.o[:want.numel() - 64], want[:-64]) and torch.equal(c.lse, want_l) and torch.equal(e.o[:other.numel() - 64], other[:-64])


def test_behind_the_kernel_that_has_just_written_what_it_reads(fa_ctx):
    # lengths, lengths in common, queries and the cache come from kernels ahead on the stream
    lens, shared = [700, 650, 640], [600, 600, 512]
    c = Cache(15, lens, 2, 128, 64, room=room(lens, 2, 128))
    c.share([0, 3], shared)
    hq = c.to_gpu(4)
    good = {k: v.clone() for k, v in c.d.items()}
    call(fa_ctx, c, hq, [0, 3], shared)
    good["shared"], good["starts"] = c.d["shared"].clone(), c.d["starts"].clone()
    torch.cuda.synchronize()
    want = c.o.clone()
    for _ in range(10):
        for k in ("k", "v", "q", "table", "lens", "shared"):
            c.d[k].zero_()
        for k in ("table", "lens", "shared", "q", "v", "k"):
            c.d[k].copy_(good[k])
        call(fa_ctx, c, hq, [0, 3], shared)
    torch.cuda.synchronize()
    assert torch.equal(c.o, want)


def test_refusals(fa_ctx):
    from goml_b200 import fa_forward as F
    c = Cache(16, [100, 90], 2, 64, 64)
    hq = c.to_gpu(2)
    s = ints([0, 2])
    args = lambda **kw: {**dict(q=c.d["q"].data_ptr(), k_cache=c.d["k"].data_ptr(), v_cache=c.d["v"].data_ptr(), o=c.o.data_ptr(), lOut=0, seq_lens=s.data_ptr(), shared_lens=s.data_ptr(),   # noqa: E731
                                group_starts=s.data_ptr(), groups=1, batch=2, q_heads=hq, kv_heads=2, hd=64, s_max=0, scale=1.0, block_table=c.d["table"].data_ptr(), page_size=64,
                                max_pages_per_seq=c.width, num_pages=c.pages), **kw}
    for bad, text in ((dict(seq_lens=0), "are needed"), (dict(shared_lens=0), "are needed"), (dict(group_starts=0), "are needed"), (dict(groups=0), "are needed"),
                      (dict(groups=3), "more groups than sequences"), (dict(shared_lens=s.data_ptr() + 2), "4-byte aligned"), (dict(lOut=2), "4-byte aligned"), (dict(hd=96), "head_dim"),
                      (dict(q_heads=34), "16 query heads"), (dict(num_pages=2 ** 31 - 1), "2\\^31"), (dict(k_cache=c.d["k"].data_ptr() + 8), "16-byte aligned"), (dict(q=0), "null pointer")):
        with pytest.raises(F.FAError, match=text):
            fa_ctx.DecodeShared(**args(**bad))
    with pytest.raises(F.FAError, match="nil ctx"):
        F.FAContext(0).DecodeShared(**args())


def test_the_most_groups(fa_ctx):
    from goml_b200.fa_forward import FAError
    run(fa_ctx, 1, [2] * 2049, [*range(2048), 2049], [1] * 2049, 1, 1, 64, 64)
    c = Cache(1, [1] * 2049, 1, 64)
    with pytest.raises(FAError, match="at most 2048 groups"):
        call(fa_ctx, c, c.to_gpu(1), list(range(2050)), [0] * 2049)


@pytest.mark.parametrize("small", [False, True])
def test_no_lse_and_an_output_of_two_byte_alignment(fa_ctx, small):
    lens, starts, shared = [200, 150, 3], [0, 2, 3], [100, 100, 3]
    c = Cache(17, lens, 2, 128, 64, room=0 if small else room(lens, 2, 128, 2))
    c.share(starts, shared)
    hq = c.to_gpu(4)
    call(fa_ctx, c, hq, starts, shared)
    want = c.results(hq)[0]
    d, odd = c.d, torch.full((3 * hq * 128 + 9,), 5.0, dtype=torch.float16, device="cuda")
    fa_ctx.DecodeShared(d["q"].data_ptr(), d["k"].data_ptr(), d["v"].data_ptr(), odd.data_ptr() + 2, 0, d["lens"].data_ptr(), d["shared"].data_ptr(), d["starts"].data_ptr(), 2, 3, hq, 2, 128,
                        c.s_max, SCALE, V_SCALE, 0, 0, 0, torch.cuda.current_stream().cuda_stream, d["table"].data_ptr(), c.page, c.width, c.pages)
    torch.cuda.synchronize()
    assert np.array_equal(odd[1:-8].double().cpu().numpy().reshape(want.shape), want) and odd[0] == 5 and (odd[-8:] == 5).all()


@pytest.mark.parametrize("small", [False, True])
def test_pages_far_into_a_pool(fa_ctx, small):
    # offsets of bytes that pass 32 bits; the calls read the same wherever the pages lie
    from goml_b200 import block_glue as BG
    kv, hd, page, lens, starts, shared = 8, 128, 64, [300, 170], [0, 2], [150, 150]
    c = Cache(18, lens, kv, hd, page, room=0 if small else room(lens, kv, hd))
    c.share(starts, shared)
    hq = c.to_gpu(2)
    call(fa_ctx, c, hq, starts, shared)
    near = [x.copy() for x in c.results(hq)]
    d, pages = c.d, 70000     # 4.6 10^9 bytes
    k, v = (torch.zeros((pages, kv, page, hd), dtype=torch.uint8, device="cuda") for _ in range(2))
    k[:c.pages], v[:c.pages] = d["k"], d["v"]
    n = c.pages
    frm, to, copies = ints(range(n)), ints(range(pages - n, pages)), ints([n])
    BG.KVPageCopy([(k.data_ptr(), k.stride(0)), (v.data_ptr(), v.stride(0))], frm.data_ptr(), to.data_ptr(), copies.data_ptr(), n, pages, torch.cuda.current_stream().cuda_stream)
    k[:c.pages], v[:c.pages] = 127, 127
    d["k"], d["v"] = k, v
    inside = (d["table"] >= 0) & (d["table"] < c.pages)
    d["table"] = torch.where(inside, d["table"] + (pages - n), -1)
    c.pages = pages
    c.o.fill_(5)
    c.lse.fill_(5)
    call(fa_ctx, c, hq, starts, shared)
    for x, y in zip(near, c.results(hq)):
        assert np.array_equal(x, y)
    fa_ctx.DecodeWindow(d["q"].data_ptr(), k.data_ptr(), v.data_ptr(), c.o.data_ptr(), c.lse.data_ptr(), d["lens"].data_ptr(), 2, hq, kv, hd, 0, 0, 0, 0, SCALE, V_SCALE, 0, 0, 0,
                        torch.cuda.current_stream().cuda_stream, d["table"].data_ptr(), page, c.width, pages)
    o, lse = c.results(hq)
    c.page, c.pages = 0, n      # (every entry that matters is inside)
    c.check(o, lse, lambda b: range(lens[b]), SCALE, V_SCALE)
    fa_ctx.DeviceStatus()


@pytest.mark.parametrize("hd,kv,group,page", [(128, 2, 4, 64), (64, 1, 9, 0)])
@pytest.mark.parametrize("small", [False, True])
def test_a_nan_among_values_leaves_the_lse(fa_ctx, hd, kv, group, page, small):
    # in the first, in a middle and in the last block of what is common, and behind it: the weights do not see it, so the LSE is that of clean values, bit for bit
    lens, shared = [700, 700, 640, 300], [600, 600, 600, 250]
    for key in (3, 270, 599, 650):
        got = []
        for value in (None, 127, 255):
            c = Cache(19, lens, kv, hd, page, room=0 if small else room(lens, kv, hd))
            c.share([0, 4], shared)
            if value is not None:
                for b in range(4):   # wherever a sequence has that key of the first one's
                    if key < (lens[0] if b == 0 else min(shared[b], lens[b])):
                        c.v[c.table[b, key // c.k.shape[2]], :, key % c.k.shape[2], hd // 2 + 1] = value
            hq = c.to_gpu(group)
            call(fa_ctx, c, hq, [0, 4], shared)
            o, lse = c.results(hq)
            got.append(lse)
            if value is None:
                c.check(o, lse, lambda b: range(lens[b]), SCALE, V_SCALE)
                assert np.isfinite(o).all()
            for b in range(4):
                sees = value is not None and key < (lens[0] if b == 0 else min(shared[b], lens[b]))
                assert np.isnan(o[b, :, hd // 2 + 1]).all() if sees else np.isfinite(o[b]).all()
        assert np.isfinite(got[0]).all() and np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
