"""Pages that change hands, on the GPU, against the restatement that goes one sequence and one page at a time: whole numbers, all equal."""
import numpy as np
import pytest
import torch

from oracle import pages as P

pytestmark = pytest.mark.gpu
GUARD = 77   # words behind every array, which stay


class Dev:
    """An int32 array on the GPU with words behind it that nothing may write."""

    def __init__(self, values):
        a = np.asarray(values, np.int32)
        self.shape = a.shape
        self.t = torch.full((a.size + GUARD,), -12345, dtype=torch.int32, device="cuda")
        self.t[:a.size] = torch.from_numpy(np.ascontiguousarray(a).reshape(-1)).cuda()
        self.n = a.size

    @property
    def ptr(self):
        return self.t.data_ptr()

    def get(self):
        assert (self.t[self.n:] == -12345).all()
        return self.t[:self.n].cpu().numpy().reshape(self.shape)


def world(seed, batch, pages, width, page, lens=None, free=0.3, sinks=0, gone=False, corrupt=False):
    """Sequences with pages of a pool, some of them shared, and a ring with some of the others."""
    r = np.random.default_rng(seed)
    lens = r.integers(0, width * page + 1, batch) if lens is None else np.array(lens)
    table = np.full((batch, width), -1, np.int32)
    order, at = r.permutation(pages), 0
    shares = np.zeros(pages, np.int32)
    gone_of = np.array([r.integers(0, max(1, n // page + 1)) if gone else 0 for n in lens], np.int32)
    for b, n in enumerate(lens):
        for j in range(-(-int(n) // page)):
            if not P._has(j, int(n), gone_of[b], sinks, page):
                table[b, j] = r.integers(-3, pages + 3)   # what has gone names anything
            elif b and j < n // page and j < lens[b - 1] // page and r.random() < 0.3 and P._has(j, int(lens[b - 1]), gone_of[b - 1], sinks, page):
                table[b, j] = table[b - 1, j]
                shares[table[b, j]] += 1
            else:
                assert at < pages
                table[b, j], at = order[at], at + 1
    n_free = int((pages - at) * free)
    head = int(r.integers(0, pages))
    ring = np.full(pages, -9, np.int32)
    for i in range(n_free):
        ring[(head + i) % pages] = order[at + i]
    if corrupt:   # entries that name no page, or one that others have too
        table[r.random(table.shape) < 0.1] = pages + 5
        table[r.random(table.shape) < 0.1] = -7
        table[r.random(table.shape) < 0.1] = order[0]
        ring[r.random(pages) < 0.1] = 2 ** 31 - 1
        lens = lens.copy()
        lens[0], lens[-1] = -5, 2 ** 31 - 1
    return dict(lens=lens.astype(np.int32), table=table, shares=shares, gone=gone_of, ring=ring, state=np.array([head, n_free, 0, 0], np.int32), page=page, pages=pages, sinks=sinks, r=r)


WORLDS = [dict(batch=1, pages=1, width=1, page=1), dict(batch=1, pages=40, width=9, page=16), dict(batch=7, pages=120, width=13, page=64), dict(batch=33, pages=999, width=24, page=128),
          dict(batch=300, pages=4000, width=11, page=16), dict(batch=9000, pages=30000, width=3, page=3), dict(batch=3, pages=5000, width=1500, page=64), dict(batch=64, pages=1, width=2, page=16, lens=[0] * 64)]


def fork_call(w, parent, keep, in_place, gone):
    from goml_b200 import block_glue as BG
    batch, width = w["table"].shape
    d = {k: Dev(w[k]) for k in ("lens", "table", "shares", "ring", "state")}
    d["gone"] = Dev(w["gone"]) if gone else None
    d["parent"], d["keep"] = Dev(parent), None if keep is None else Dev(keep)
    new = lambda n: Dev(np.full(n, -1))   # noqa: E731
    for k in ("lens", "shares", "state", "gone"):
        d[k + "_out"] = d[k] if in_place or d[k] is None else new(d[k].n)
    d |= dict(taken=new(batch), copy_from=new(batch), copy_to=new(batch), copies=new(1))
    at = lambda k: d[k].ptr if d[k] is not None else 0   # noqa: E731
    BG.KVPageFork(at("lens"), at("parent"), at("keep"), at("table"), at("ring"), at("state"), at("shares"), at("gone"), at("lens_out"), at("state_out"), at("shares_out"), at("gone_out"),
                  at("taken"), at("copy_from"), at("copy_to"), at("copies"), batch, width, w["page"], w["pages"], w["sinks"], torch.cuda.current_stream().cuda_stream)
    return d


def release_call(w, keep, in_place, gone, window):
    from goml_b200 import block_glue as BG
    batch, width = w["table"].shape
    d = {k: Dev(w[k]) for k in ("lens", "table", "shares", "ring", "state")}
    d["gone"] = Dev(w["gone"]) if gone else None
    d["keep"] = None if keep is None else Dev(keep)
    for k in ("lens", "shares", "state", "gone"):
        d[k + "_out"] = d[k] if in_place or d[k] is None else Dev(np.full(d[k].n, -1))
    at = lambda k: d[k].ptr if d[k] is not None else 0   # noqa: E731
    BG.KVPageRelease(at("lens"), at("keep"), at("table"), at("ring"), at("state"), at("shares"), at("gone"), at("lens_out"), at("state_out"), at("shares_out"), at("gone_out"), batch, width,
                     w["page"], w["pages"], window, w["sinks"], torch.cuda.current_stream().cuda_stream)
    return d


def compact_call(w, in_place):
    from goml_b200 import block_glue as BG
    batch, width = w["table"].shape
    d = {k: Dev(w[k]) for k in ("lens", "table", "shares", "ring", "state")}
    for k in ("table", "shares", "ring", "state"):
        d[k + "_out"] = d[k] if in_place else Dev(w[k])
    new = lambda n: Dev(np.full(n, -1))   # noqa: E731
    d |= dict(moved_to=new(w["pages"]), copy_from=new(w["pages"] // 2), copy_to=new(w["pages"] // 2), copies=new(1))
    at = lambda k: d[k].ptr   # noqa: E731
    BG.KVPageCompact(at("lens"), at("table"), at("ring"), at("state"), at("shares"), at("table_out"), at("ring_out"), at("state_out"), at("shares_out"), at("moved_to"), at("copy_from"),
                     at("copy_to"), at("copies"), batch, width, w["page"], w["pages"], torch.cuda.current_stream().cuda_stream)
    return d


def moves_of(d):
    n = int(d["copies"].get()[0])
    a, b = d["copy_from"].get(), d["copy_to"].get()
    assert (a[n:] == -1).all() and (b[n:] == -1).all()
    return list(zip(a[:n].tolist(), b[:n].tolist()))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("gone", [False, True])
@pytest.mark.parametrize("spec", WORLDS)
@pytest.mark.parametrize("corrupt", [False, True])
def test_fork(cuda, built_libs, spec, gone, in_place, corrupt):
    batch = spec["batch"]
    if corrupt and in_place and gone:
        pytest.skip("one of the corrupt ones is enough")
    r = np.random.default_rng(5)
    empty = r.random(batch) < 0.5
    lens = np.where(empty, 0, r.integers(0, spec["width"] * spec["page"] + 1, batch)) if "lens" not in spec else spec["lens"]
    w = world(11, sinks=spec["page"] + 1 if gone else 0, gone=gone, corrupt=corrupt, free=0.3 if batch < 1000 else 0.01, **spec | dict(lens=lens))
    parent = np.where(r.random(batch) < 0.8, r.integers(-2, batch + 2, batch), -1)
    parent[0] = 0   # itself
    keep = np.where(r.random(batch) < 0.5, r.integers(-2, spec["width"] * spec["page"] + 9, batch), 2 ** 31 - 1)
    for k in (None, keep):
        want = P.fork(w["lens"], parent, k, w["table"], w["ring"], w["state"][0], w["state"][1], w["shares"], w["gone"] if gone else None, w["page"], w["sinks"])
        d = fork_call(w, parent, k, in_place, gone)
        assert d["lens_out"].get().tolist() == want["lens"] and d["taken"].get().tolist() == want["taken"]
        assert np.array_equal(d["table"].get(), want["table"]) and np.array_equal(d["shares_out"].get(), want["shares"])
        assert tuple(d["state_out"].get()[:2]) == want["state"] and np.array_equal(d["ring"].get(), w["ring"]) and moves_of(d) == want["moves"]
        if gone:
            assert d["gone_out"].get().tolist() == want["gone"]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("window", [None, 0, 1, 40, 1000])
@pytest.mark.parametrize("spec", WORLDS)
@pytest.mark.parametrize("corrupt", [False, True])
def test_release(cuda, built_libs, spec, window, in_place, corrupt):
    batch, gone = spec["batch"], window is not None
    window = window or 0
    w = world(12, sinks=spec["page"] + 1 if window > 1 else 0, gone=gone and window != 40, corrupt=corrupt, free=1.0 if window == 1000 else 0.3, **spec)
    r = w["r"]
    keep = np.where(r.random(batch) < 0.5, r.integers(-2, spec["width"] * spec["page"] + 9, batch), 2 ** 31 - 1)
    for k in (None, keep):
        want = P.release(w["lens"], k, w["table"], w["ring"], w["state"][0], w["state"][1], w["shares"], w["gone"] if gone else None, w["page"], window, w["sinks"])
        d = release_call(w, k, in_place, gone, window)
        assert d["lens_out"].get().tolist() == want["lens"] and np.array_equal(d["shares_out"].get(), want["shares"])
        assert np.array_equal(d["ring"].get(), want["ring"]) and tuple(d["state_out"].get()[:2]) == want["state"] and np.array_equal(d["table"].get(), w["table"])
        if gone:
            assert d["gone_out"].get().tolist() == want["gone"]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("free", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("spec", WORLDS)
@pytest.mark.parametrize("corrupt", [False, True])
def test_compact(cuda, built_libs, spec, free, in_place, corrupt):
    w = world(13, free=free, corrupt=corrupt, **spec)
    want = P.compact(w["lens"], w["table"], w["ring"], w["state"][0], w["state"][1], w["shares"], w["page"])
    d = compact_call(w, in_place)
    assert np.array_equal(d["table_out"].get(), want["table"]) and d["ring_out"].get().tolist() == want["ring"] and tuple(d["state_out"].get()[:2]) == want["state"]
    assert np.array_equal(d["shares_out"].get(), want["shares"]) and d["moved_to"].get().tolist() == want["moved_to"] and moves_of(d) == want["moves"]


@pytest.mark.parametrize("sizes", [[16], [1024, 48], [65536, 65536, 4096, 16384 + 16], [32] * 70])
@pytest.mark.parametrize("copies,most", [(0, 5), (1, 5), (5, 5), (9, 5), (-3, 5), (400, 400)])
def test_copy(cuda, built_libs, sizes, copies, most):
    from goml_b200 import block_glue as BG
    pages = 1000
    g = torch.Generator(device="cuda").manual_seed(1)
    pools = [torch.randint(0, 256, (pages, n), generator=g, device="cuda", dtype=torch.uint8) for n in sizes]
    order = torch.randperm(pages, generator=g, device="cuda").int()
    a, b = order[:most].clone(), order[most:2 * most].clone()
    if most > 4:
        a[3], b[2] = -1, pages   # nothing is copied
    want = [p.clone() for p in pools]
    n = min(max(copies, 0), most)
    for p in want:
        for x, y in zip(a[:n].tolist(), b[:n].tolist()):
            if 0 <= x < pages and 0 <= y < pages:
                p[y] = p[x]
    count = torch.tensor([copies], dtype=torch.int32, device="cuda")
    BG.KVPageCopy([(p.data_ptr(), p[0].numel()) for p in pools], a.data_ptr(), b.data_ptr(), count.data_ptr(), most, pages, torch.cuda.current_stream().cuda_stream)
    assert all(torch.equal(p, q) for p, q in zip(pools, want))


def test_a_captured_fork_and_release_on_another_stream(cuda, built_libs):
    # fork, copy, release and compaction in one graph, in place: every replay goes on from what the one before has left, as calls do
    from goml_b200 import block_glue as BG
    w = world(3, 12, 90, 6, 16, lens=[90, 40, 33, 0, 0, 0, 17, 0, 64, 96, 0, 5], free=0.8)
    batch, width, page, pages = 12, 6, 16, 90
    parent = np.array([-1, -1, -1, 0, 1, 9, -1, 8, -1, -1, 2, -1])
    keep = np.where(np.arange(batch) % 2, 2 ** 31 - 1, 20)
    names = ("lens", "table", "ring", "state", "shares")
    t = {k: torch.from_numpy(np.ascontiguousarray(w[k])).cuda() for k in names}
    t |= {k: torch.full((n,), -1, dtype=torch.int32, device="cuda") for k, n in (("taken", batch), ("from", 45), ("to", 45), ("copies", 1), ("moved", pages))}
    t["parent"], t["keep"] = (torch.from_numpy(x.astype(np.int32)).cuda() for x in (parent, keep))
    pool = torch.arange(pages, dtype=torch.int32, device="cuda")[:, None].repeat(1, 64).contiguous()
    p = {k: x.data_ptr() for k, x in t.items()}

    def step():
        s = torch.cuda.current_stream().cuda_stream
        BG.KVPageFork(p["lens"], p["parent"], 0, p["table"], p["ring"], p["state"], p["shares"], 0, p["lens"], p["state"], p["shares"], 0, p["taken"], p["from"], p["to"], p["copies"],
                      batch, width, page, pages, 0, s)
        BG.KVPageCopy([(pool.data_ptr(), 256)], p["from"], p["to"], p["copies"], 45, pages, s)
        BG.KVPageRelease(p["lens"], p["keep"], p["table"], p["ring"], p["state"], p["shares"], 0, p["lens"], p["state"], p["shares"], 0, batch, width, page, pages, 0, 0, s)
        BG.KVPageCompact(p["lens"], p["table"], p["ring"], p["state"], p["shares"], p["table"], p["ring"], p["state"], p["shares"], p["moved"], p["from"], p["to"], p["copies"], batch,
                         width, page, pages, s)
        BG.KVPageCopy([(pool.data_ptr(), 256)], p["from"], p["to"], p["copies"], 45, pages, s)

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    step()   # the libraries are loaded before the capture
    for k in names:
        t[k].copy_(torch.from_numpy(np.ascontiguousarray(w[k])))
    pool.copy_(torch.arange(pages, dtype=torch.int32, device="cuda")[:, None].expand(-1, 64))
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    x = {k: w[k].copy() for k in names}
    held = np.arange(pages)
    for _ in range(3):
        f = P.fork(x["lens"], parent, None, x["table"], x["ring"], *x["state"][:2], x["shares"], None, page)
        for a, b in f["moves"]:
            held[b] = held[a]
        q = P.release(f["lens"], keep, f["table"], x["ring"], *f["state"], f["shares"], None, page)
        c = P.compact(q["lens"], f["table"], q["ring"], *q["state"], q["shares"], page)
        for a, b in c["moves"]:
            held[b] = held[a]
        x = dict(lens=np.array(q["lens"]), table=c["table"], ring=np.array(c["ring"], np.int32), state=np.array(c["state"]), shares=c["shares"])
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        assert all(np.array_equal(t[k].cpu().numpy().reshape(-1)[:x[k].size], x[k].reshape(-1)) for k in names)
        assert np.array_equal(pool[:, 0].cpu().numpy(), held) and (pool == pool[:, :1]).all()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("spec", [dict(batch=7, pages=120, width=13, page=64), dict(batch=300, pages=4000, width=11, page=16), dict(batch=9000, pages=30000, width=3, page=3)])
def test_forks_through_windows(cuda, built_libs, spec, in_place):
    from goml_b200 import block_glue as BG
    batch, page, width = spec["batch"], spec["page"], spec["width"]
    for window, sinks in ((1, 0), (page, 1), (2 * page + 1, page + 1), (width * page, 0), (2 ** 31 - 1, 2 ** 31 - 1)):
        r = np.random.default_rng(window % 1000)
        lens = np.where(r.random(batch) < 0.5, 0, r.integers(0, width * page + 1, batch))
        w = world(12, sinks=sinks, gone=True, free=0.9, **spec | dict(lens=lens))
        # windows give back at most what they have passed; some parents have given back less
        w["gone"] = np.where(r.random(batch) < 0.8, np.maximum(w["lens"] + 1 - window, 0) // page, w["gone"]).astype(np.int32)
        parent = np.where(lens == 0, r.integers(0, batch, batch), -1)
        keep = np.where(r.random(batch) < 0.7, lens[np.maximum(parent, 0)] - r.integers(0, 3 * page, batch), r.integers(0, width * page + 1, batch))
        want = P.fork(w["lens"], parent, keep, w["table"], w["ring"], w["state"][0], w["state"][1], w["shares"], w["gone"], page, sinks, window)
        blind = P.fork(w["lens"], parent, keep, w["table"], w["ring"], w["state"][0], w["state"][1], w["shares"], w["gone"], page, sinks)
        if batch >= 300 and 1 < window <= width * page:
            assert want["taken"] != blind["taken"] and any(want["taken"])
        d = {k: Dev(w[k]) for k in ("lens", "table", "shares", "ring", "state", "gone")}
        d["parent"], d["keep"] = Dev(parent), Dev(keep)
        for k in ("lens", "shares", "state", "gone"):
            d[k + "_out"] = d[k] if in_place else Dev(np.full(d[k].n, -1))
        d |= {k: Dev(np.full(n, -1)) for k, n in (("taken", batch), ("copy_from", batch), ("copy_to", batch), ("copies", 1))}
        names = ("lens", "parent", "keep", "table", "ring", "state", "shares", "gone", "lens_out", "state_out", "shares_out", "gone_out", "taken", "copy_from", "copy_to", "copies")
        BG.KVPageFork(*(d[k].ptr for k in names), batch, width, page, w["pages"], sinks, torch.cuda.current_stream().cuda_stream, window)
        for k in ("lens", "gone"):
            assert d[k + "_out"].get().tolist() == want[k]
        assert d["taken"].get().tolist() == want["taken"] and tuple(d["state_out"].get()[:2]) == want["state"] and moves_of(d) == want["moves"]
        assert np.array_equal(d["table"].get(), want["table"]) and np.array_equal(d["shares_out"].get(), want["shares"])
