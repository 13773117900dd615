"""The 4-bit KV cache on the GPU: append, rows, decode attention and the page plan against the restatement in 64 bits (oracle/fp4.py)."""
import math

import numpy as np
import pytest
import torch

from oracle import fp4
from oracle.glue import rope_table

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def stream():
    return torch.cuda.current_stream().cuda_stream


def bf16(x):
    return torch.from_numpy(np.asarray(x, np.float32)).bfloat16().float().numpy()


# ------------------------------------------------------------------------------------------------------------ append and rows
def empty_cache(pages, kv, page, hd, k_scale, v_scale, fill=0x5A):
    full = lambda *shape: np.full(shape, fill, np.uint8)   # noqa: E731
    return dict(k=full(pages, kv, page, hd // 2), ks=full(pages, kv, page, hd // 16), v=full(pages, kv, page, hd // 2), vs=full(pages, kv, page // 16, hd // 16, 16),
                k_scale=np.float32(k_scale), v_scale=np.float32(v_scale))


def on_device(cache):
    return {n: dev(np.array([x]) if np.ndim(x) == 0 else x) for n, x in cache.items()}


def run_append(qkv, cos, sin, positions, slots, hq, cache, want_q=True):
    """(Q as the kernel leaves it, the cache on the device)."""
    from goml_b200 import block_glue as BG
    c = on_device(cache)
    pages, kv, page, half = cache["k"].shape
    tokens = len(qkv)
    x = dev(qkv.reshape(tokens, -1)).bfloat16()
    q = torch.full((tokens, hq, 2 * half), float("nan"), dtype=torch.bfloat16, device="cuda")
    t = [dev(np.asarray(a, np.int32)) for a in (positions, slots)]
    tables = dev(cos), dev(sin)
    BG.FP4RopeAppend(x.data_ptr(), tables[0].data_ptr(), tables[1].data_ptr(), t[0].data_ptr(), t[1].data_ptr(), q.data_ptr() if want_q else 0, c["k"].data_ptr(), c["ks"].data_ptr(),
                     c["v"].data_ptr(), c["vs"].data_ptr(), c["k_scale"].data_ptr(), c["v_scale"].data_ptr(), tokens, hq, kv, 2 * half, len(cos), page, pages, stream())
    torch.cuda.synchronize()
    return q, c


def same_cache(c, cache):
    """Bytes as the restatement has them, wherever a block scale is a number (a NaN's codes say nothing)."""
    for codes, scales, want in (("k", "ks", cache["ks"]), ("v", "vs", fp4.natural(cache["vs"]))):
        got = c[scales].cpu().numpy()
        got = fp4.natural(got) if scales == "vs" else got
        assert np.array_equal(got, want), scales
        number = np.repeat((want & 0x7F) != 0x7F, 8, -1)
        assert np.array_equal(c[codes].cpu().numpy()[number], cache[codes][number]), codes


def tokens_of(r, tokens, heads, hd, kind):
    x = r.normal(size=(tokens, heads, hd)).astype(np.float32)
    if kind == "few bits":   # many values halfway between two codes
        x = (r.integers(-24, 25, size=x.shape) / 4).astype(np.float32)
    if kind == "wild":
        x *= np.exp2(r.integers(-30, 30, size=(tokens, heads, 1))).astype(np.float32)
        x[r.random(x.shape) < 0.02] = 0
        x[0, -1, :17] = np.nan
        if tokens > 2:
            x[1, -1, 5], x[2, -1, 40] = np.inf, -np.inf
            x[2, 0, 3] = np.nan
    return bf16(x)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens,hq,kv,page,kind", [(1, 1, 1, 16, "normal"), (3, 4, 4, 64, "wild"), (17, 5, 1, 16, "few bits"), (65, 8, 2, 48, "normal"), (300, 16, 2, 64, "few bits"),
                                                    (300, 2, 3, 128, "wild"), (2100, 8, 8, 64, "normal"), (2101, 8, 8, 64, "few bits"), (2100, 4, 8, 64, "wild")])
def test_append(cuda, built_libs, tokens, hq, kv, page, kind, hd):
    r = np.random.default_rng(tokens + hd)
    qkv = tokens_of(r, tokens, hq + 2 * kv, hd, kind)
    rope_rows = 513
    cos, sin = rope_table(rope_rows, hd, 10000.0)
    positions = r.integers(0, rope_rows, tokens)
    positions[r.random(tokens) < 0.2] = 0    # no rotation: halfway stays halfway
    pages = -(-tokens // page) + 2
    slots = r.permutation(pages * page)[:tokens]
    if tokens > 10:
        positions[[2, 5]] = -1, rope_rows
        slots[[3, 7, 9]] = -1, pages * page, 2 ** 31 - 1
    # scales of a calibrated cache, of few bits and not
    cache = empty_cache(pages, kv, page, hd, 1 / 32 if kind == "few bits" else 0.0123, 1 / 4 if kind == "few bits" else 0.0077)
    q, c = run_append(qkv, cos, sin, positions, slots, hq, cache)
    want = fp4.append(qkv, cos, sin, positions, slots, hq, cache)
    same_cache(c, cache)                     # rows that no token has among them: left as they were
    want = torch.from_numpy(want).bfloat16()
    assert torch.equal(torch.nan_to_num(q.cpu(), nan=77.0), torch.nan_to_num(want, nan=77.0))


@pytest.mark.parametrize("k_scale,v_scale", [(1.0, 2.0 ** -20), (1e-5, 3e4), (2.0 ** -120, 2.0 ** -140), (7.7e-39, 1e30)])
def test_append_at_the_ends_of_the_scales(cuda, built_libs, k_scale, v_scale):
    r = np.random.default_rng(5)
    qkv = tokens_of(r, 40, 6, 64, "normal") * np.float32(1.5)
    qkv[:, -2:] *= np.exp2(r.integers(-60, 60, size=(40, 2, 1))).astype(np.float32)
    cos, sin = rope_table(64, 64, 10000.0)
    cache = empty_cache(4, 2, 16, 64, k_scale, v_scale)
    q, c = run_append(bf16(qkv), cos, sin, np.arange(40), np.arange(40), 2, cache)
    fp4.append(bf16(qkv), cos, sin, np.arange(40), np.arange(40), 2, cache)
    same_cache(c, cache)


def test_append_without_queries_and_twice_the_same_slot(cuda, built_libs):
    r = np.random.default_rng(7)
    qkv = tokens_of(r, 2, 4, 64, "normal")
    qkv[1] = qkv[0]
    cos, sin = rope_table(4, 64, 10000.0)
    cache = empty_cache(2, 1, 16, 64, 0.01, 0.01)
    q, c = run_append(qkv, cos, sin, [3, 3], [20, 20], 2, cache, want_q=False)
    fp4.append(qkv, cos, sin, [3, 3], [20, 20], 2, cache)
    assert q.isnan().all()
    same_cache(c, cache)


@pytest.mark.parametrize("hd,kv,page,tokens", [(64, 1, 16, 1), (128, 8, 64, 100), (64, 3, 48, 1000)])
def test_rows(cuda, built_libs, hd, kv, page, tokens):
    from goml_b200 import block_glue as BG
    r = np.random.default_rng(hd + tokens)
    pages = 9
    cache = empty_cache(pages, kv, page, hd, 0.0123, 7.7)
    for n in ("k", "ks", "v", "vs"):
        cache[n] = r.integers(0, 256, cache[n].shape).astype(np.uint8)   # every byte, NaN scales and signed ones among them
    slots = r.integers(0, pages * page, tokens)
    slots[::7] = -1
    if tokens > 3:
        slots[1], slots[2] = pages * page, 2 ** 31 - 1
    c = on_device(cache)
    out = [torch.full((tokens, kv, hd), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    s = dev(slots.astype(np.int32))
    BG.FP4CacheRows(s.data_ptr(), c["k"].data_ptr(), c["ks"].data_ptr(), c["v"].data_ptr(), c["vs"].data_ptr(), c["k_scale"].data_ptr(), c["v_scale"].data_ptr(), out[0].data_ptr(),
                    out[1].data_ptr(), tokens, kv, hd, page, pages, stream())
    torch.cuda.synchronize()
    inside = (slots >= 0) & (slots < pages * page)
    at = np.where(inside, slots, 0)
    for got, x in zip(out, (fp4.values(cache["k"], cache["ks"], 1.0), fp4.values(cache["v"], fp4.natural(cache["vs"]), 1.0))):
        scale = cache["k_scale"] if got is out[0] else cache["v_scale"]
        want = (x[at // page, :, at % page].astype(np.float32) * scale).astype(np.float32)
        want = torch.from_numpy(np.where(inside[:, None, None], want, 0)).bfloat16()
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=77.0), torch.nan_to_num(want, nan=77.0))
    assert all(torch.equal(c[n].cpu(), torch.from_numpy(cache[n])) for n in ("k", "ks", "v", "vs"))


# ----------------------------------------------------------------------------------------------------------------- attention
class Case:
    """A cache of random rows with NaN everywhere behind the sequences' ends, its queries, and the call."""

    def __init__(self, seed, batch, hq, kv, hd, lens, page=0, s_max=None, q_type="bf16", holes=(), q_std=1.5, spread=2):
        r = np.random.default_rng(seed)
        self.batch, self.hq, self.kv, self.hd, self.page, self.q_type = batch, hq, kv, hd, page, q_type
        self.lens = np.asarray(lens, np.int32)
        longest = max(1, int(self.lens.max()))
        if page:
            self.max_pages = -(-longest // page) + 1
            self.pages = batch * self.max_pages + 3
            self.s_max = self.max_pages * page
            self.table = r.permutation(self.pages)[:batch * self.max_pages].reshape(batch, -1).astype(np.int32)
        else:
            self.s_max = s_max or -(-longest // 16) * 16
            self.max_pages, self.pages, page = 1, batch, self.s_max
            self.table = np.arange(batch, dtype=np.int32)[:, None]
        self.cache = empty_cache(self.pages, kv, page, hd, 0.0123, 0.0345)
        live = np.zeros((self.pages, page), bool)
        for b in range(batch):
            n = int(np.clip(self.lens[b], 0, self.s_max))
            for j in range(-(-n // page)):
                live[self.table[b, j], :max(0, min(page, n - j * page))] = True
        x = r.normal(size=(self.pages, kv, page, hd)) * np.exp2(r.uniform(-spread, spread, size=(1, kv, 1, hd)))
        rows = [fp4.quantise((x if n == "k" else r.normal(size=x.shape)).astype(np.float32), self.cache[n + "_scale"]) for n in "kv"]
        stale = np.where(live, 0, 0x7F).astype(np.uint8)[:, None, :, None]
        self.cache.update(k=fp4.pack(rows[0][1]), ks=rows[0][0] | stale, v=fp4.pack(rows[1][1]), vs=fp4.blocks_of_16(rows[1][0] | stale))
        for b, j, name in holes:   # table entries outside the pool
            self.table[b, j] = name
        q = r.normal(size=(batch, hq, hd)).astype(np.float32) * q_std
        self.sq = 1.0
        if q_type == "e4m3":
            self.sq = float(np.float32(np.abs(q).max() / 448))
            self.qd = (torch.from_numpy(q) / self.sq).clamp(-448, 448).to(torch.float8_e4m3fn)
        else:
            self.qd = torch.from_numpy(q).to(torch.bfloat16 if q_type == "bf16" else torch.float16)
        self.scale = 1 / math.sqrt(hd)
        self.load()

    def load(self):
        self.c = on_device(self.cache)
        self.q, self.table_d, self.lens_d = self.qd.cuda().contiguous(), dev(self.table), dev(self.lens)
        self.sqd = torch.tensor([self.sq], device="cuda")
        self.o = torch.full((self.batch, self.hq, self.hd), float("nan"), dtype=torch.float16, device="cuda")
        self.lse = torch.full((self.batch, self.hq), 7.0, device="cuda")

    def call(self, ctx, out=None, lse=True, lens=True, seq_len=0, stream_=None, vds=1.0, **over):
        from goml_b200 import fa_forward as F
        c = self.c
        a = dict(q=self.q.data_ptr(), k_codes=c["k"].data_ptr(), k_scales=c["ks"].data_ptr(), v_codes=c["v"].data_ptr(), v_scales=c["vs"].data_ptr(),
                 o=(self.o if out is None else out).data_ptr(), lOut=self.lse.data_ptr() if lse else 0, seq_lens=self.lens_d.data_ptr() if lens else 0, batch=self.batch, q_heads=self.hq,
                 kv_heads=self.kv, hd=self.hd, s_max=self.s_max, seq_len=seq_len, scale=self.scale, v_descale=vds,
                 q_type=dict(bf16=F.Q_BF16, fp16=F.Q_FP16, e4m3=F.Q_E4M3)[self.q_type], scale_q_dev=self.sqd.data_ptr(), scale_k_dev=c["k_scale"].data_ptr(),
                 scale_v_dev=c["v_scale"].data_ptr(), stream=stream() if stream_ is None else stream_)
        if self.page:
            a.update(block_table=self.table_d.data_ptr(), page_size=self.page, max_pages_per_seq=self.max_pages, num_pages=self.pages)
        ctx.DecodeFP4(**{**a, **over})

    def reference(self, lens=None):
        lens = np.clip(self.lens if lens is None else lens, 0, self.s_max)
        page = self.page or self.s_max
        at = np.clip(self.table, 0, self.pages - 1)
        order = lambda x: np.swapaxes(x[at], 1, 2).reshape(self.batch, self.kv, self.max_pages * page, self.hd)   # noqa: E731
        c = self.cache
        k, v = order(fp4.values(c["k"], c["ks"], c["k_scale"])), order(fp4.values(c["v"], fp4.natural(c["vs"]), c["v_scale"]))
        for b, j in zip(*np.nonzero((self.table < 0) | (self.table >= self.pages))):
            k[b, :, j * page:(j + 1) * page] = v[b, :, j * page:(j + 1) * page] = 0
        return fp4.attention(self.qd.double().numpy() * self.sq, k, v, lens, self.scale)

    def check(self, want, o=None, lse=True, vds=1.0):
        # Weights are rounded to fp16, by 2^-11 at most, and their exponentials are off by what the scores are: hd products of which each addition may lose 2^-23 of
        # the largest partial sum, and twelve more operations (the factors, the maximum's shift, the exponential).  Both sums of the quotient see the latter.  Weights
        # below fp16's normal range (2^-22 of the largest) are off by 2^-33 of it.  O is rounded once more.
        ro, rl, spread, size = want
        o = (self.o if o is None else o).double().cpu().numpy()
        ds = (self.hd + 12) * 2.0 ** -23 * np.maximum(size, 1.0)
        vmax = max(1e-30, float(np.nanmax(np.abs(fp4.values(self.cache["v"], fp4.natural(self.cache["vs"]), self.cache["v_scale"])))))
        tol = (2.0 ** -11 + 2 * ds)[..., None] * spread * abs(vds) + 2.0 ** -11 * np.abs(ro * vds) + self.s_max * 2.0 ** -33 * vmax * abs(vds) + 2.0 ** -24
        assert np.isfinite(o).all() and (np.abs(o - ro * vds) <= tol).all(), float((np.abs(o - ro * vds) / tol).max())
        if lse:
            l = self.lse.double().cpu().numpy()
            assert np.array_equal(np.isneginf(l), np.isneginf(rl))
            f = np.isfinite(rl)
            assert (np.abs(l[f] - rl[f]) <= (2 * ds + 2.0 ** -20 + 2.0 ** -22 * np.abs(rl))[f]).all()


EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 191, 200, 255, 256, 257, 300]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("hq,kv", [(1, 1), (4, 4), (4, 2), (5, 1), (16, 2), (18, 2), (16, 1)])
@pytest.mark.parametrize("page", [0, 64, 192])
def test_decode_at_the_edges_of_lengths(fa_ctx, hd, hq, kv, page):
    c = Case(hq * 100 + kv, len(EDGES), hq, kv, hd, EDGES, page=page)
    c.call(fa_ctx)
    c.check(c.reference())


@pytest.mark.parametrize("hd,hq,kv,page,q_type", [(128, 8, 8, 0, "fp16"), (128, 32, 4, 64, "e4m3"), (64, 32, 2, 128, "e4m3"), (64, 4, 4, 64, "fp16")])
def test_decode_types_of_queries(fa_ctx, hd, hq, kv, page, q_type):
    c = Case(3, 5, hq, kv, hd, [700, 64, 1, 0, 513], page=page, q_type=q_type)
    c.call(fa_ctx)
    c.check(c.reference())


@pytest.mark.parametrize("hd,hq,kv,page,batch,longest", [(128, 4, 4, 0, 1, 9000), (128, 8, 1, 64, 2, 5000), (64, 16, 1, 0, 1, 9000), (64, 4, 4, 64, 150, 90), (128, 2, 2, 64, 300, 40),
                                                         (64, 2, 1, 256, 1100, 50), (128, 8, 8, 64, 70, 300), (64, 16, 2, 64, 170, 200)])
def test_decode_long_many_and_uneven(fa_ctx, hd, hq, kv, page, batch, longest):
    r = np.random.default_rng(batch)
    lens = r.integers(0, longest + 1, batch)
    lens[0] = longest
    c = Case(batch, batch, hq, kv, hd, lens, page=page)
    c.call(fa_ctx)
    first = c.o.clone(), c.lse.clone()
    c.check(c.reference())
    c.call(fa_ctx)
    assert torch.equal(c.o, first[0]) and torch.equal(c.lse, first[1])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("hq,kv,copies", [(1, 1, 1), (4, 2, 1), (16, 2, 1), (16, 1, 1), (18, 2, 1), (2, 1, 120), (4, 4, 30), (16, 1, 260), (18, 2, 130)])
def test_decode_where_the_cache_has_room_for_far_more(fa_ctx, hd, hq, kv, copies):
    # tables of 20000 keys to a sequence: chunks of all pairs are cut into equal pieces, for CTAs, and of many pairs for warps, whatever the lengths turn out to be, if the pool has as much (it is
    # said to have; no entry of a table is behind what it has); with the pool that there is the pairs stay whole
    c = Case(hq * 7 + kv, len(EDGES), hq, kv, hd, EDGES, page=64)
    table = torch.full((len(EDGES), 313), 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, :c.max_pages] = c.table_d
    table, q, lens = table.repeat(copies, 1), c.q.repeat(copies, 1, 1), c.lens_d.repeat(copies)
    o, lse = (torch.full((len(lens), hq, *tail), 7.0, dtype=d, device="cuda") for d, tail in ((torch.float16, (hd,)), (torch.float32, ())))
    want = [np.concatenate([x] * copies) for x in c.reference()]
    c.lse = lse
    for pool in (313 * len(lens), c.pages):
        results = []
        for _ in range(2):
            o.fill_(7.0)
            c.call(fa_ctx, out=o, lOut=lse.data_ptr(), q=q.data_ptr(), seq_lens=lens.data_ptr(), block_table=table.data_ptr(), max_pages_per_seq=313, batch=len(lens), num_pages=pool)
            results.append((o.clone(), lse.clone()))
        assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
        c.check(want, o=o)


def test_decode_sharp_and_flat_weights(fa_ctx):
    for q_std in (0.0, 1e-3, 30.0):
        c = Case(11, 3, 8, 2, 128, [1500, 400, 3], page=64, q_std=q_std)
        c.call(fa_ctx)
        c.check(c.reference())


@pytest.mark.parametrize("hd,hq,kv,n", [(128, 8, 8, 1000), (64, 8, 2, 700), (128, 16, 1, 3000)])
def test_decode_of_rows_that_one_key_dominates(fa_ctx, hd, hq, kv, n):
    # One key's score is 50 above all others', wherever it lies (75 or 107 against 19 or 27 if all of a key's dims are as large as they can be): O is its value, rounded once.
    for place in (0, n // 2, n - 1):
        c = Case(hd + place, 1, hq, kv, hd, [n], page=64, q_type="fp16")
        page, at = c.table[0, place // 64], place % 64
        c.cache["ks"] = np.where(c.cache["ks"] == 0x7F, 0x7F, np.minimum(c.cache["ks"], 0x40)).astype(np.uint8)
        c.cache["k"][page, :, at], c.cache["ks"][page, :, at] = 0x77, 0x70      # every dim 6, 128 and the tensor scale
        c.qd = torch.full_like(c.qd, 1.0)
        c.load()
        c.call(fa_ctx)
        ro, _, _, _ = c.reference()
        v = (fp4.values(c.cache["v"], fp4.natural(c.cache["vs"]), c.cache["v_scale"]))[page, :, at].astype(np.float64)
        assert (np.abs(ro - np.repeat(v, hq // kv, axis=0)[None]) <= 2.0 ** -20 * np.abs(v).max()).all()
        o = c.o.double().cpu().numpy()
        assert (np.abs(o - ro) <= 2.0 ** -11 * np.abs(ro) + 2.0 ** -20 * np.abs(v).max() + 2.0 ** -24).all()


def test_decode_queries_of_any_size(fa_ctx):
    # a power of two per row brings queries into fp16's range: sizes far outside it change nothing but the scores
    c = Case(13, 4, 4, 2, 64, [300, 300, 300, 300], page=0)
    scales = torch.tensor([1e-30, 1e30, 2.0 ** -80, 1.0])[:, None, None]
    c.qd = (c.qd.float() * scales).bfloat16()
    c.load()
    c.scale = 1.0
    c.sqd = torch.tensor([1.0], device="cuda")
    for b, s in enumerate((1e30, 1e-30, 2.0 ** 80, 1.0)):
        c.scale = s / 8
        c.call(fa_ctx)
        ro, rl, spread, size = c.reference()
        o = c.o.double().cpu().numpy()[b]
        assert (np.abs(o - ro[b]) <= (2.0 ** -10 + 2.0 ** -15 * np.maximum(size[b], 1))[:, None] * spread[b] + 2.0 ** -11 * np.abs(ro[b]) + 2.0 ** -24).all()


def test_decode_lengths_outside_their_range_and_one_for_all(fa_ctx):
    c = Case(17, 3, 4, 2, 128, [-5, 2 ** 31 - 1, 70], page=0, s_max=112)
    c.cache = {n: (np.where(x & 0x7F == 0x7F, 1, x).astype(np.uint8) if n in ("ks", "vs") else x) for n, x in c.cache.items()}
    c.load()
    c.call(fa_ctx)
    c.check(c.reference())
    for n in (0, 1, 65, 112):
        c.call(fa_ctx, lens=False, seq_len=n)
        c.check(c.reference(np.full(3, n)))


def test_decode_table_entries_outside_the_pool(fa_ctx):
    c = Case(19, 4, 4, 1, 64, [300, 200, 64, 129], page=64, holes=[(0, 1, -1), (0, 4, 10 ** 6), (2, 0, -2 ** 31), (3, 2, 2 ** 31 - 1)])
    c.call(fa_ctx)
    c.check(c.reference())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("which", ["k", "v"])
def test_decode_nan_stays_with_what_sees_it(fa_ctx, hd, which):
    c = Case(23, 3, 4, 2, hd, [200, 200, 0], page=64)
    name = "ks" if which == "k" else "vs"
    x = fp4.natural(c.cache["vs"]) if which == "v" else c.cache["ks"].copy()
    x[c.table[0, 1], 1, 3, 0] = 0x7F   # key 67 of sequence 0, kv head 1, dims 0 to 15
    c.cache[name] = fp4.blocks_of_16(x) if which == "v" else x
    c.load()
    c.call(fa_ctx)
    o, lse = c.o.cpu(), c.lse.cpu()
    clean = torch.ones_like(o, dtype=torch.bool)
    if which == "k":
        clean[0, 2:] = False
        assert lse[0, 2:].isnan().all() and torch.isfinite(lse[0, :2]).all()
    else:
        clean[0, 2:, :16] = False
        assert torch.isfinite(lse[:2]).all()
    assert o[~clean].isnan().all() and torch.isfinite(o[clean]).all() and not o[2].any() and lse[2].isneginf().all()
    # every key NaN: no quiet zero
    c.cache["ks"][...] = 0x7F
    c.load()
    c.call(fa_ctx)
    assert c.o[:2].isnan().all() and not c.o[2].any()


def test_decode_infinite_queries(fa_ctx):
    c = Case(29, 2, 2, 1, 64, [100, 100], page=64)
    c.qd[0, 0, 5], c.qd[1, 1, 0] = float("inf"), float("nan")
    c.load()
    c.call(fa_ctx)
    assert not torch.isfinite(c.o[0, 0]).all() and c.o[1, 1].isnan().all() and torch.isfinite(c.o[0, 1]).all() and torch.isfinite(c.o[1, 0]).all()


def test_decode_output_alignment_lse_and_descale(fa_ctx):
    c = Case(31, 3, 6, 2, 64, [100, 64, 7], page=64)
    buf = torch.full((c.o.numel() + 8,), 7.0, dtype=torch.float16, device="cuda")
    for off in (1, 2, 3):
        buf.fill_(7.0)
        o = buf[off:off + c.o.numel()].view(c.o.shape)
        c.call(fa_ctx, out=o, lse=False, vds=0.5)
        c.check(c.reference(), o=o, lse=False, vds=0.5)
        assert (buf[:off] == 7).all() and (buf[off + c.o.numel():] == 7).all()
    assert (c.lse == 7).all()
    c.call(fa_ctx, scale_q_dev=0, scale_k_dev=0, scale_v_dev=0, scale=c.scale * 0.0123)
    c.check(c.reference(), o=c.o * np.float32(0.0345), lse=False)


def test_decode_refuses(fa_ctx):
    from goml_b200 import fa_forward as F
    c = Case(37, 2, 4, 2, 64, [10, 20], page=64)
    for over, status in [(dict(q=0), 1), (dict(k_codes=0), 1), (dict(k_scales=0), 1), (dict(v_codes=0), 1), (dict(v_scales=0), 1), (dict(o=0), 1), (dict(batch=0), 1), (dict(q_heads=0), 1),
                         (dict(kv_heads=-1), 1), (dict(hd=96), 3), (dict(q_heads=5), 4), (dict(q_heads=34), 4), (dict(page_size=32), 1), (dict(page_size=0), 1), (dict(num_pages=0), 1),
                         (dict(max_pages_per_seq=0), 1), (dict(max_pages_per_seq=1 << 30), 1), (dict(block_table=0, s_max=24), 1), (dict(block_table=0, s_max=0), 1),
                         (dict(seq_lens=0, seq_len=-1), 1), (dict(seq_lens=0, seq_len=c.s_max + 1), 1), (dict(q_type=3), 1), (dict(q_type=-1), 1), (dict(q=c.q.data_ptr() + 2), 1),
                         (dict(k_codes=c.c["k"].data_ptr() + 8), 1), (dict(v_scales=c.c["vs"].data_ptr() + 4), 1), (dict(o=c.o.data_ptr() + 1), 1), (dict(lOut=c.lse.data_ptr() + 2), 1),
                         (dict(batch=1 << 30, kv_heads=4, q_heads=4), 4)]:
        with pytest.raises(F.FAError, match="fa_decode_fp4") as e:
            c.call(fa_ctx, **over)
        assert e.value.status == status and e.value.msg.startswith("fa_decode_fp4: "), over
    assert F.FALoad().fa_decode_fp4(fa_ctx.ptr, None) == F.FA_ERR_INVALID_ARG
    c.call(fa_ctx)
    c.check(c.reference())


def test_decode_in_graphs_on_streams_and_side_by_side(fa_ctx):
    # two cut pairs' calls at once on two streams, and captured and replayed with other lengths
    cases = [Case(s, 2, 8, 2, 128, [3000 + s, 1777], page=64) for s in (41, 43)]
    for c in cases:
        c.call(fa_ctx)
        torch.cuda.synchronize()
        c.check(c.reference())
    want = [(c.o.clone(), c.lse.clone()) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        for c, s in zip(cases, streams):
            c.call(fa_ctx, stream_=s.cuda_stream)
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.o, w[0]) and torch.equal(c.lse, w[1])
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            c.call(fa_ctx)
        graphs.append(g)
        c.o.fill_(float("nan"))
    for _ in range(3):
        for g, s in zip(graphs, streams):   # both graphs draw scratch; they run side by side
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.o, w[0]) and torch.equal(c.lse, w[1])
    cases[0].lens_d.copy_(torch.tensor([5, 0], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    cases[0].check(cases[0].reference(np.array([5, 0])))


def test_decode_and_append_where_offsets_pass_32_bits(fa_ctx):
    # pools of more than 4 GB of codes, the pages in use at their end
    from goml_b200 import block_glue as BG
    kv, hd, page, pages = 8, 128, 64, 140000
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.fail("this test takes 11 GB of the GPU")
    c = Case(47, 1, 8, kv, hd, [150], page=page)
    big = {n: torch.empty((pages, *c.c[n].shape[1:]), dtype=torch.uint8, device="cuda") for n in ("k", "ks", "v", "vs")}
    for n in big:
        big[n][pages - c.pages:] = c.c[n]
    want = c.reference()
    c.table_d += pages - c.pages
    c.call(fa_ctx, k_codes=big["k"].data_ptr(), k_scales=big["ks"].data_ptr(), v_codes=big["v"].data_ptr(), v_scales=big["vs"].data_ptr(), num_pages=pages)
    c.check(want)
    r = np.random.default_rng(1)
    qkv = tokens_of(r, 20, 8 + 2 * kv, hd, "normal")
    cos, sin = rope_table(32, hd, 10000.0)
    small = empty_cache(2, kv, page, hd, 0.01, 0.02)
    fp4.append(qkv, cos, sin, np.arange(20), np.arange(20) + page, 8, small)
    args = [dev(qkv.reshape(20, -1)).bfloat16(), dev(cos), dev(sin), torch.arange(20, dtype=torch.int32, device="cuda"),
            torch.arange(20, dtype=torch.int32, device="cuda") + page * (pages - 1)]
    scales = torch.tensor([0.01, 0.02], device="cuda")
    out = torch.empty(2, 20, kv, hd, dtype=torch.bfloat16, device="cuda")
    ptr = [big[n].data_ptr() for n in ("k", "ks", "v", "vs")] + [scales.data_ptr(), scales.data_ptr() + 4]
    BG.FP4RopeAppend(*[a.data_ptr() for a in args], 0, *ptr, 20, 8, kv, hd, 32, page, pages, stream())
    BG.FP4CacheRows(args[4].data_ptr(), *ptr, out[0].data_ptr(), out[1].data_ptr(), 20, kv, hd, page, pages, stream())
    torch.cuda.synchronize()
    for n in ("k", "ks", "v", "vs"):
        rows = lambda x: fp4.natural(x) if n == "vs" else x   # noqa: E731
        assert np.array_equal(rows(big[n][-1].cpu().numpy())[:, :20], rows(small[n][1])[:, :20])
    for i, (x, s) in enumerate(((fp4.values(small["k"], small["ks"], 1), np.float32(0.01)), (fp4.values(small["v"], fp4.natural(small["vs"]), 1), np.float32(0.02)))):
        want = torch.from_numpy(np.swapaxes(x[1, :, :20].astype(np.float32) * s, 0, 1).copy()).bfloat16()
        assert torch.equal(out[i].cpu(), want)


# --------------------------------------------------------------------------------------------------------------- the page plan
def run_plan(lens, fresh, table, ring, head, count, page, rows, per_seq=0, in_place=False, state=None, buffers=None):
    from goml_b200 import block_glue as BG
    batch, max_pages = table.shape
    d = dict(lens=dev(np.asarray(lens, np.int32)), fresh=dev(np.asarray(fresh, np.int32)), table=dev(table), ring=dev(ring),
             state=dev(np.array([head, count, 0, 1234], np.int32)))
    new = lambda n: torch.full((n,), -77, dtype=torch.int32, device="cuda")   # noqa: E731
    lens_out, state_out = (d["lens"], d["state"]) if in_place else (new(batch), new(4))
    taken, starts, positions, slots = new(batch + 1), new(batch + 2), new(rows + 1), new(rows + 1)
    BG.KVPagePlan(d["lens"].data_ptr() or 4, d["fresh"].data_ptr() or 4, d["table"].data_ptr() or 4, d["ring"].data_ptr(), d["state"].data_ptr(), lens_out.data_ptr() or 4,
                  state_out.data_ptr(), taken.data_ptr(), starts.data_ptr(), positions.data_ptr(), slots.data_ptr(), batch, max_pages, page, len(ring), rows, per_seq, stream())
    torch.cuda.synchronize()
    assert taken[batch] == starts[batch + 1] == positions[rows] == slots[rows] == -77     # nothing behind the outputs
    assert d["state"][2] == 0 and d["state"][3] == 1234
    get = lambda x, n: x[:n].cpu().numpy()   # noqa: E731
    return dict(lens=get(lens_out, batch), taken=get(taken, batch), starts=get(starts, batch + 1), positions=get(positions, rows), slots=get(slots, rows), table=d["table"].cpu().numpy(),
                ring=d["ring"].cpu().numpy(), state=tuple(state_out[:2].tolist()))


def same_plan(got, want):
    for n in want:
        assert np.array_equal(got[n], want[n]), n


def a_server(r, batch, page, max_pages, spare, longest_new):
    """Lengths, a table of different pages, the ring of the others, and the step's new tokens."""
    lens = r.integers(0, max_pages * page + 1, batch) if batch else np.zeros(0, int)
    held = -(-lens // page)
    pages = int(held.sum()) + spare
    order = r.permutation(pages).astype(np.int32)
    table = np.full((batch, max_pages), -1, np.int32)
    at = 0
    for b in range(batch):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    head = int(r.integers(0, pages))
    ring = np.full(pages, -9, np.int32)
    ring[(head + np.arange(spare)) % pages] = order[at:]
    fresh = r.choice([-1, 0, 1, 1, 1, longest_new], batch)
    fresh = np.where(fresh > 1, r.integers(1, longest_new + 1, batch), fresh)
    return lens, fresh, table, ring, head, spare


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,page,max_pages,spare,longest_new,rows,per_seq", [
    (0, 64, 1, 3, 1, 10, 0), (1, 64, 4, 5, 40, 64, 0), (1, 1, 9, 4, 3, 2, 0), (8, 64, 5, 20, 1, 8, 1), (33, 16, 8, 60, 50, 900, 0), (33, 16, 8, 10, 50, 900, 0), (33, 16, 8, 60, 50, 300, 0),
    (100, 7, 20, 300, 6, 500, 5), (511, 64, 3, 400, 100, 9000, 0), (513, 64, 3, 100, 100, 40000, 0), (1025, 128, 3, 2000, 300, 70000, 0), (5000, 16, 4, 9000, 20, 30000, 0),
    (2000, 64, 3, 1500, 3, 8000, 4), (40, 16, 300, 20000, 4000, 100000, 0), (600, 64, 3, 1, 10, 0, 0),
    (700, 64, 9, 6000, 500, 160000, 0), (3000, 64, 4, 9000, 200, 160001, 0), (4097, 64, 4, 12000, 250, 500003, 0), (3000, 16, 40, 60000, 600, 400001, 0), (200, 64, 40, 9000, 2500, 120001, 0)])
def test_plan(cuda, built_libs, batch, page, max_pages, spare, longest_new, rows, per_seq, in_place):
    r = np.random.default_rng(batch + rows)
    lens, fresh, table, ring, head, count = a_server(r, batch, page, max_pages, spare, longest_new)
    args = lens, fresh, table, ring, head, count, page, rows, per_seq
    same_plan(run_plan(*args, in_place=in_place), fp4.plan(*args))


def test_plan_of_nonsense_touches_nothing_else(cuda, built_libs):
    # any numbers in the lengths, the table, the ring and its state
    r = np.random.default_rng(2)
    any_int = lambda *shape: r.integers(-2 ** 31, 2 ** 31, shape).astype(np.int32)   # noqa: E731
    for batch, max_pages, pages, page, rows, per_seq in ((300, 7, 50, 16, 2000, 0), (50, 3, 9, 64, 100, 2), (700, 40, 13, 1, 5000, 0)):
        lens, fresh = any_int(batch), r.choice([-3, 0, 1, 7, 2 ** 31 - 1, 100], batch).astype(np.int32)
        lens = np.where(r.random(batch) < 0.5, r.integers(0, max_pages * page + 9, batch), lens)
        for head, count in ((2 ** 31 - 1, 2 ** 31 - 1), (-5, -5), (pages - 1, pages), (3, pages // 2)):
            args = lens, fresh, any_int(batch, max_pages), any_int(pages), head, count, page, rows, per_seq
            same_plan(run_plan(*args), fp4.plan(*args))


def test_plans_one_after_another_keep_every_page_once(cuda, built_libs):
    # a server's steps in place, replayed from one graph with new wishes each time: pages are in one place at any time, none is lost
    from goml_b200 import block_glue as BG
    r = np.random.default_rng(9)
    batch, page, max_pages, pages, rows = 60, 16, 12, 400, 700
    d = dict(lens=np.zeros(batch), fresh=np.zeros(batch), table=np.full((batch, max_pages), -1), ring=r.permutation(pages), state=np.array([0, pages, 0, 0]))
    d = {n: dev(x.astype(np.int32)) for n, x in d.items()}
    new = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")   # noqa: E731
    taken, starts, positions, slots = new(batch), new(batch + 1), new(rows), new(rows)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        BG.KVPagePlan(d["lens"].data_ptr(), d["fresh"].data_ptr(), d["table"].data_ptr(), d["ring"].data_ptr(), d["state"].data_ptr(), d["lens"].data_ptr(), d["state"].data_ptr(),
                      taken.data_ptr(), starts.data_ptr(), positions.data_ptr(), slots.data_ptr(), batch, max_pages, page, pages, rows, 0, stream())
    refused = 0
    for step in range(60):
        before = {n: x.cpu().numpy() for n, x in d.items()}
        fresh = np.where(r.random(batch) < 0.08, -1, np.where(before["lens"] == 0, r.integers(0, 80, batch), r.integers(0, 3, batch))).astype(np.int32)
        d["fresh"].copy_(torch.from_numpy(fresh))
        g.replay()
        torch.cuda.synchronize()
        want = fp4.plan(before["lens"], fresh, before["table"], before["ring"], before["state"][0], before["state"][1], page, rows)
        got = {n: x.cpu().numpy() for n, x in d.items()} | dict(taken=taken.cpu().numpy(), starts=starts.cpu().numpy(), positions=positions.cpu().numpy(), slots=slots.cpu().numpy())
        got["state"] = tuple(got["state"][:2].tolist())
        same_plan(got, want)
        refused += int((fresh > 0).sum() - (got["taken"] > 0).sum())
        held = -(-got["lens"] // page)
        everywhere = [p for b in range(batch) for p in got["table"][b, :held[b]]] + [got["ring"][(got["state"][0] + i) % pages] for i in range(got["state"][1])]
        assert sorted(everywhere) == list(range(pages))
    assert refused > 0   # the pool has run out at times
