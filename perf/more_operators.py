"""Operators of a server whose sequences share what they begin with, or attend to a window: what it calls for each step, prompt and change of who is served.

  prompt   `FAContext.ForwardSinks`: prompts where a token sees the `window` tokens up to itself and the first `sinks` ones
  window   `FAContext.DecodeWindow`: the same for one new token of every sequence, against an e4m3 cache
  shared   `FAContext.DecodeShared`: one new token of every sequence, where sequences of a group have their first keys in common, which are read once for all
  fork     `KVPageFork`, `KVPageCopy`: sequences that begin as copies of others: whole pages are shared, a last page that is not full is copied
  release  `KVPageRelease`: sequences end, are cut back, or give back the pages that their window has left behind; a page is free when nobody has it any more
  compact  `KVPageCompact`, `KVPageCopy`: the pages in use move to the front of the pool

Caches hold e4m3 codes with one fp32 scale for all keys and one for all values: [batch, kv heads, keys, hd], or pages [pages, kv heads, page, hd] and a block table.
`shares[p]` counts the sequences that have page p besides one.
"""
import math

import torch

own = False

DEV = "cuda"
BANK = 1 << 14   # different rows that a cache is filled from
NAN = 127        # the e4m3 code of a NaN


def listed():
    gqa = dict(q_heads=32, kv_heads=8, hd=128)
    small = dict(q_heads=64, kv_heads=4, hd=64)
    return [
        # a short prompt of a small model: where the launch counts
        dict(name="prompt_short_hd64", kind="prompt", bh=32, s=1001, hd=64, window=256, sinks=4),
        # two documents of 8192 tokens, 32 heads: the largest prompts
        dict(name="prompt_long", kind="prompt", bh=64, s=8192, hd=128, window=1024, sinks=64),
        # one user's next token, a kv head for every query head, a contiguous cache
        dict(name="window_one", kind="window", batch=1, s=5000, page=0, window=1024, sinks=4, q_heads=32, kv_heads=32, hd=128),
        # 128 users in pages, whose contexts are mostly longer than the window: the largest decode call
        dict(name="window_batch", kind="window", batch=128, s=8000, page=64, window=4096, sinks=4, **gqa),
        # eight answers sampled to one prompt
        dict(name="shared_samples", kind="shared", batch=8, groups=1, prefix=2000, suffix=300, page=64, **gqa),
        # 64 users behind three system prompts, the longest of 12000 tokens
        dict(name="shared_system", kind="shared", batch=64, groups=3, prefix=12000, suffix=600, page=128, **gqa),
        # an answer in progress is split into a few
        dict(name="fork_few", kind="fork", batch=16, share=0.5, s=700, page=64, pools=2, kv_heads=8, hd=128, cut=False, window=0),
        # a server takes new users behind prompts that are in the cache
        dict(name="fork_many", kind="fork", batch=512, share=0.6, s=3000, page=64, pools=8, kv_heads=4, hd=64, cut=True, window=0),
        # drafted tokens that were not accepted, answers that end, of a few users
        dict(name="release_few", kind="release", batch=32, s=2000, page=64, window=0, sinks=0),
        # sequences with windows, the pages behind which go back; some end
        dict(name="release_window", kind="release", batch=2048, s=9000, page=128, window=2048, sinks=4),
        # a small pool, half of it empty
        dict(name="compact_small", kind="compact", batch=24, s=1500, page=64, used=0.5, pools=2, kv_heads=8, hd=128),
        # a pool whose memory is wanted for something else
        dict(name="compact_large", kind="compact", batch=700, s=2500, page=64, used=0.6, pools=4, **{k: small[k] for k in ("kv_heads", "hd")}),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "window", "window", "shared", "shared", "shared", "fork", "release", "compact"])
    hd, kv = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 8, 32])
    if kind == "prompt":
        bh, s = _log(rng, 1, 256), _log(rng, 1, 8192)
        bh = max(1, min(bh, int(64 * 8192 * 128 / (s * hd))))
        return dict(kind=kind, bh=bh, s=s, hd=hd, window=min(s, _log(rng, 1, 2048)), sinks=rng.choice([0, 1, 4, 4, _log(rng, 1, 300)]))
    heads = dict(q_heads=kv * (rng.choice([1, 1, 2]) if kv == 32 else rng.choice([1, 2, 4, 5, 8, 16])), kv_heads=kv, hd=hd)
    page = rng.choice([64, 64, 128, 192, 256])
    if kind == "window":
        s, window, sinks = _log(rng, 1, 60000), _log(rng, 1, 8192), rng.choice([0, 1, 4, 4, _log(rng, 1, 600)])
        most = max(1, min(256, int(2.0e9 / (2 * kv * hd * s)), int(4.0e8 / (heads["q_heads"] * min(s, window + sinks)))))
        return dict(kind=kind, batch=_log(rng, 1, most) if most > 1 else 1, s=s, page=rng.choice([0, page, page]), window=window, sinks=sinks, **heads)
    if kind == "shared":
        prefix, suffix = _log(rng, 1, 30000), _log(rng, 1, 2000)
        most = max(1, min(200, int(8.0e8 / (heads["q_heads"] * (prefix + suffix))), int(2.5e8 / (kv * hd * (prefix + suffix) / 4))))
        batch = _log(rng, 1, most) if most > 1 else 1
        return dict(kind=kind, batch=batch, groups=min(batch, rng.choice([1, 1, 2, 5, 16])), prefix=prefix, suffix=suffix, page=rng.choice([0, page, page, page]), **heads)
    if kind == "release":
        batch = _log(rng, 1, 4096)
        s = min(_log(rng, 10, 20000), 24000000 // batch)
        return dict(kind=kind, batch=batch, s=s, page=rng.choice([16, 64, 128, 256]), window=rng.choice([0, _log(rng, 1, 4096)]), sinks=rng.choice([0, 4, 300]))
    batch, page, pools = _log(rng, 2, 512), rng.choice([64, 64, 128]), rng.choice([1, 2, 4, 8])
    s = max(1, min(_log(rng, 10, 8000), int(2.0e9 / (batch * pools * min(kv, 8) * hd))))
    pool = dict(batch=batch, s=s, page=page, pools=pools, kv_heads=min(kv, 8), hd=hd)
    if kind == "fork":
        return dict(kind=kind, share=rng.uniform(0.1, 0.9), cut=rng.random() < 0.5, window=rng.choice([0, 0, _log(rng, 1, 2000)]), **pool)
    return dict(kind=kind, used=rng.uniform(0.1, 0.95), **pool)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(g, lo, hi, n):
    """n whole numbers in [lo, hi]."""
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV, dtype=torch.int64)


def _codes(x):
    """e4m3 codes of x and what one of them stands for, as a quantiser by the largest value makes them."""
    scale = (x.abs().amax() / 448).reshape(1)
    return (x / scale).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _channels(g, n, hd, std):
    """Rows of a head as projections make them: some channels several times as wide as the others."""
    wide = torch.exp(0.6 * torch.randn(hd, generator=g, device=DEV))
    return torch.randn(n, hd, generator=g, device=DEV) * (wide * (std / wide.square().mean().sqrt()))


def _from_bank(g, shape, std):
    """Codes of rows [*shape] taken from a bank of rows, and their scale."""
    bank, scale = _codes(_channels(g, BANK, shape[-1], std))
    return bank[torch.randint(0, BANK, shape[:-1], generator=g, device=DEV)], scale


def _cache(g, shape, used):
    """Codes of keys and values [pages, kv heads, page, hd]; what no sequence has (used [pages, page] is false) holds what was there before: anything, NaN among it."""
    k, k_scale = _from_bank(g, shape, 1.0)
    v, v_scale = _from_bank(g, shape, 0.7)
    stale = torch.where(used, 0, NAN).to(torch.uint8)[:, None, :, None]
    k |= stale
    v |= stale
    return dict(k=k, v=v, k_scale=k_scale, v_scale=v_scale)


def _queries(g, batch, case):
    q, scale = _codes(_channels(g, batch * case["q_heads"], case["hd"], 1.5))
    return dict(q=q.reshape(batch, case["q_heads"], case["hd"]), q_scale=scale, scale=1.0 / math.sqrt(case["hd"]),
                o=torch.empty(batch, case["q_heads"], case["hd"], dtype=torch.float16, device=DEV), lse=torch.empty(batch, case["q_heads"], device=DEV))


def _lengths(g, batch, s):
    """Contexts between half of s and s; of several sequences one is empty, one has a single key."""
    lens = _ints(g, (s + 1) // 2, s, batch)
    lens[batch // 2] = s
    if batch > 8:
        lens[1], lens[batch - 1] = 0, 1
    return lens


def _spread(g, lo, hi, n):
    """n lengths over [lo, hi] in no order: the same ones whatever the seed, so that a pool has as many pages."""
    at = torch.linspace(lo, hi, n, device=DEV, dtype=torch.float64).round().long()
    return at[torch.randperm(n, generator=g, device=DEV)]


def _paged(g, batch, capacity, spare):
    """A table of different pages in no order, and those that are left over."""
    order = torch.randperm(batch * capacity + spare, generator=g, device=DEV).int()
    return order[:batch * capacity].reshape(batch, capacity).contiguous(), order[batch * capacity:]


def _used(lens, table, pages, page):
    used = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
    key = torch.arange(table.shape[1] * page, device=DEV)
    at = table.long()[:, key // page] * page + key % page
    used.view(-1)[at[key < lens[:, None]]] = True
    return used


def _prepare_prompt(case, g):
    bh, s, hd = case["bh"], case["s"], case["hd"]
    q, q_scale = _from_bank(g, (bh, s, hd), 1.5)
    k, k_scale = _from_bank(g, (bh, s, hd), 1.0)
    v, v_scale = _from_bank(g, (bh, s, hd), 0.7)
    return dict(case=case, q=q, k=k, v=v, q_scale=q_scale, k_scale=k_scale, v_scale=v_scale, scale=1.0 / math.sqrt(hd),
                o=torch.empty(bh, s, hd, dtype=torch.float16, device=DEV), lse=torch.empty(bh, s, device=DEV))


def _prepare_window(case, g):
    batch, s, page = case["batch"], case["s"], case["page"]
    lens = _lengths(g, batch, s)
    if page:
        table, _ = _paged(g, batch, -(-s // page), 5)
        pages = table.numel() + 5
    else:   # a contiguous cache: one page to a sequence
        page, pages = s, batch
        table = torch.arange(batch, dtype=torch.int32, device=DEV)[:, None].contiguous()
    cache = _cache(g, (pages, case["kv_heads"], page, case["hd"]), _used(lens, table, pages, page))
    if case["page"]:
        # the pages between the sinks and the window have gone back to the pool: their entries name none
        j = torch.arange(table.shape[1], device=DEV) * page
        table = torch.where((j >= case["sinks"]) & (j + page <= (lens - case["window"])[:, None]), -1, table).int().contiguous()
    return dict(case=case, lens=lens.int(), table=table, pages=pages, page=page, **cache, **_queries(g, batch, case))


def _prepare_shared(case, g):
    batch, groups, page, kv, hd = case["batch"], case["groups"], case["page"], case["kv_heads"], case["hd"]
    # groups of different sizes, none empty; the last one's prefix is the longest
    cuts = torch.randperm(batch - 1, generator=g, device=DEV)[:groups - 1].sort().values + 1
    starts = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), batch)])
    group = torch.bucketize(torch.arange(batch, device=DEV), starts[1:], right=True)
    first = starts[group]
    prefix = _ints(g, (case["prefix"] + 1) // 2, case["prefix"], groups)
    prefix[groups - 1] = case["prefix"]
    shared = prefix[group]
    # some have only a part of it in common with the group's first sequence
    part = (torch.rand(batch, generator=g, device=DEV) < 0.15) & (torch.arange(batch, device=DEV) != first)
    shared = torch.where(part, (shared * torch.rand(batch, generator=g, device=DEV)).long(), shared)
    lens = shared + _ints(g, (case["suffix"] + 1) // 2, case["suffix"], batch)
    if batch > 8:   # one has nothing of its own yet, one place is vacant
        quiet, vacant = int(starts[groups - 1]) + 1, batch - 1
        if quiet < vacant:
            lens[quiet] = shared[quiet]
            lens[vacant] = shared[vacant] = 0
    s = case["prefix"] + case["suffix"]
    if page:
        table, _ = _paged(g, batch, -(-s // page), 5)
        j = torch.arange(table.shape[1], device=DEV)
        table = torch.where(j < (shared // page)[:, None], table[first], table).contiguous()   # whole pages are the group's
        pages = table.numel() + 5
        # what lies in a page that is not whole is a copy
        tail, where = shared % page, (shared // page).clamp(max=table.shape[1] - 1)
    else:
        page, pages = s, batch
        table = torch.arange(batch, dtype=torch.int32, device=DEV)[:, None].contiguous()
        tail, where = shared, torch.zeros_like(shared)
    cache = _cache(g, (pages, kv, page, hd), _used(lens, table, pages, page))
    for b, (n, j, f) in enumerate(zip(tail.tolist(), where.tolist(), first.tolist())):
        if n and b != f:
            for x in (cache["k"], cache["v"]):
                x[table[b, j].long(), :, :n] = x[table[f, j].long(), :, :n]
    return dict(case=case, lens=lens.int(), shared=shared.int(), starts=starts.int(), table=table, pages=pages, page=page, **cache, **_queries(g, batch, case))


def _ring_of(g, free, pages):
    """A ring with the free pages in it from some place on."""
    head = int(_ints(g, 0, pages - 1, 1))
    ring = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    ring[(head + torch.arange(free.numel(), device=DEV)) % pages] = free.int()
    return ring, torch.tensor([head, free.numel(), 0, 0], dtype=torch.int32, device=DEV)


def _first_kept(lens, window, page, sinks):
    """Pages up to which a window has given back those behind the sinks."""
    return ((lens + 1 - window) // page).clamp(min=0) if window else torch.zeros_like(lens)


def _held_pages(lens, gone, sinks, page, capacity):
    """[batch, capacity]: which pages of its row a sequence has."""
    j = torch.arange(capacity, device=DEV)
    return (j < ((lens + page - 1) // page)[:, None]) & ((j < -(-sinks // page)) | (j >= gone[:, None]))


def _page_state(g, case, lens, capacity, spare, sinks=0, window=0, shared=0.0):
    """Sequences with their pages, of which some are had by two sequences, and the ring of the others."""
    batch, page = case["batch"], case["page"]
    gone = _first_kept(lens, window, page, sinks)
    has = _held_pages(lens, gone, sinks, page, capacity)
    pages = int(has.sum()) + spare
    order = torch.randperm(pages, generator=g, device=DEV)
    table = torch.full((batch, capacity), -1, dtype=torch.int64, device=DEV)
    table[has] = order[:pages - spare]
    shares = torch.zeros(pages, dtype=torch.int64, device=DEV)
    free = [order[pages - spare:]]
    if shared and batch > 1:   # a sequence begins with the pages of its neighbour, as a fork leaves it
        pair = torch.arange(1, batch, 2, device=DEV)
        pair = pair[torch.rand(pair.numel(), generator=g, device=DEV) < shared]
        j = torch.arange(capacity, device=DEV)
        same = has[pair] & has[pair - 1] & (j < (torch.minimum(lens[pair], lens[pair - 1]) // (2 * page))[:, None])
        free.append(table[pair][same])
        shares.index_add_(0, table[pair - 1][same], torch.ones_like(table[pair - 1][same]))
        table[pair] = torch.where(same, table[pair - 1], table[pair])
    free = torch.cat(free)
    ring, state = _ring_of(g, free, pages)
    new = lambda *shape: torch.full(shape, -1, dtype=torch.int32, device=DEV)   # noqa: E731
    return dict(case=case, lens=lens.int(), table=table.int().contiguous(), ring=ring, state=state, shares=shares.int(), gone=gone.int(), pages=pages, page=page,
                sinks=sinks, lens_out=new(batch), state_out=torch.zeros_like(state), shares_out=new(pages), gone_out=new(batch), taken=new(batch))


def _pools(g, case, pages):
    shape = (pages, case["kv_heads"], case["page"], case["hd"])
    return [torch.randint(0, 256, shape, generator=g, device=DEV, dtype=torch.uint8) for _ in range(case["pools"])]


def _prepare_fork(case, g):
    batch, s, page, window = case["batch"], case["s"], case["page"], case["window"]
    sinks = 4 if window else 0
    # so many places are taken by forks of the others
    forks = min(batch - 1, max(1, round(case["share"] * batch)))
    order = torch.randperm(batch, generator=g, device=DEV)
    fork, older = order[:forks], order[forks:]
    lens = torch.zeros(batch, dtype=torch.int64, device=DEV)
    lens[older] = _spread(g, (s + 1) // 2, s, batch - forks)
    parent = torch.full_like(lens, -1)
    parent[fork] = older[_ints(g, 0, batch - forks - 1, forks)]
    keep = torch.where(torch.rand(batch, generator=g, device=DEV) < 0.5, (lens[parent.clamp(min=0)] * torch.rand(batch, generator=g, device=DEV)).long(), s) if case["cut"] else None
    capacity = -(-s // page) + 1
    # nearly all of them find a page
    st = _page_state(g, case, lens, capacity, max(1, int(0.95 * forks)), sinks, window)
    new = lambda n: torch.full((n,), -1, dtype=torch.int32, device=DEV)   # noqa: E731
    return st | dict(parent=parent.int(), keep=None if keep is None else keep.int(), copy_from=new(batch), copy_to=new(batch), copies=new(1), pools=_pools(g, case, st["pages"]))


def _prepare_release(case, g):
    batch, s, window = case["batch"], case["s"], case["window"]
    lens = _spread(g, 0, s, batch)
    what = torch.rand(batch, generator=g, device=DEV)
    keep = torch.where(what < 0.15, 0, torch.where(what < 0.5, (lens - _ints(g, 1, 8, batch)).clamp(min=0), s))   # some end, some are cut back, others go on
    keep[0] = 0
    # the window has moved since the pages behind it were given back the last time
    before = (lens - 3 * case["page"]).clamp(min=0) if window else lens
    st = _page_state(g, case, lens, -(-s // case["page"]) + 1, 7 + batch, case["sinks"], 0, 0.3)
    if window:
        gone = _first_kept(before, window, case["page"], case["sinks"])
        has = _held_pages(lens, gone, case["sinks"], case["page"], st["table"].shape[1])
        # what has gone is in no row and, where nobody else had it, in the ring
        count = torch.zeros(st["pages"], dtype=torch.int64, device=DEV).index_add_(0, st["table"][has].long(), torch.ones_like(st["table"][has].long()))
        st["ring"], st["state"] = _ring_of(g, (count == 0).nonzero()[:, 0], st["pages"])
        st["shares"], st["gone"] = (count - 1).clamp(min=0).int(), gone.int()
    return st | dict(keep=keep.int())


def _prepare_compact(case, g):
    batch, s, page = case["batch"], case["s"], case["page"]
    lens = _spread(g, 0, s, batch)
    held = int(((lens + page - 1) // page).sum())
    st = _page_state(g, case, lens, -(-s // page) + 1, max(1, int(held * (1 / case["used"] - 1))), 0, 0, 0.3)
    pages = st["pages"]
    new = lambda *shape: torch.full(shape, -1, dtype=torch.int32, device=DEV)   # noqa: E731
    return st | dict(table_out=st["table"].clone(), ring_out=new(pages), moved_to=new(pages), copy_from=new(pages // 2 + 1), copy_to=new(pages // 2 + 1), copies=new(1),
                     pools=_pools(g, case, pages))


def prepare(case, seed):
    make = dict(prompt=_prepare_prompt, window=_prepare_window, shared=_prepare_shared, fork=_prepare_fork, release=_prepare_release, compact=_prepare_compact)
    return make[case["kind"]](case, _generator(seed))


# ----------------------------------------------------------------------------------------------------------- plain forms
def _values(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _weigh(score, seen, values):
    """O and LSE of scores [.., keys] of which those not seen are left out."""
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, values) / torch.where(total == 0, 1.0, total)
    return o, torch.where(total == 0, -math.inf, top + torch.log(total))[..., 0]


def _prompt(st):
    case = st["case"]
    s, window, sinks = case["s"], case["window"], case["sinks"]
    factor = st["scale"] * st["q_scale"] * st["k_scale"]
    o, lse = torch.empty_like(st["o"]), torch.empty_like(st["lse"])
    for q0 in range(0, s, 512):
        q1 = min(s, q0 + 512)
        lo = max(0, q0 - window + 1)
        key = torch.cat([torch.arange(min(sinks, lo), device=DEV), torch.arange(lo, q1, device=DEV)])
        query = torch.arange(q0, q1, device=DEV)[:, None]
        seen = (key <= query) & ((key > query - window) | (key < sinks))
        score = torch.matmul(_values(st["q"][:, q0:q1]) * factor, _values(st["k"][:, key]).transpose(1, 2))
        x, lse[:, q0:q1] = _weigh(score, seen, _values(st["v"][:, key]))
        o[:, q0:q1] = (x * st["v_scale"]).half()
    return dict(o=o, lse=lse)


def _rows(st, name, at, seen):
    """Rows [batch, kv heads, keys, hd] of the cache at keys `at` [batch, keys] of every sequence, zeros where not seen."""
    page = st["page"]
    at = torch.where(seen, at, 0)
    entry = torch.gather(st["table"].long(), 1, at // page)
    ok = seen & (entry >= 0) & (entry < st["pages"])
    x = _values(st[name][entry.clamp(0, st["pages"] - 1), :, at % page]).transpose(1, 2)
    return x.masked_fill_(~ok[:, None, :, None], 0.0)


def _attend(st, at, seen):
    batch, hq, hd = st["q"].shape
    kv = st["case"]["kv_heads"]
    q = _values(st["q"]).reshape(batch, kv, hq // kv, hd) * (st["scale"] * st["q_scale"] * st["k_scale"])
    score = torch.matmul(q, _rows(st, "k", at, seen).transpose(2, 3))
    o, lse = _weigh(score, seen[:, None, None], _rows(st, "v", at, seen))
    return dict(o=(o * st["v_scale"]).half().reshape(batch, hq, hd), lse=lse.reshape(batch, hq))


def _window(st):
    case, n = st["case"], st["lens"].long()[:, None]
    window, sinks = min(case["window"], case["s"]), min(case["sinks"], case["s"])
    first = torch.arange(sinks, device=DEV).expand(n.shape[0], -1)
    last = n - window + torch.arange(window, device=DEV)
    return _attend(st, torch.cat([first, last], 1), torch.cat([first < n, (last >= 0) & ((last >= sinks) | (last >= n))], 1) & torch.cat([first < n, last < n], 1))


def _shared(st):
    key = torch.arange(st["case"]["prefix"] + st["case"]["suffix"], device=DEV)
    return _attend(st, key.expand(st["case"]["batch"], -1), key < st["lens"][:, None])


def _copy(st, copy_from, copy_to, n):
    """Pages copy_from[i] to copy_to[i], i < n (on the GPU): a copy from a page to itself stands for none."""
    some = torch.arange(copy_from.numel(), device=DEV) < n
    # those that are none repeat the first one, or leave page 0 as it is
    a = torch.where(some, copy_from, torch.where(n > 0, copy_from[0], 0)).long()
    b = torch.where(some, copy_to, torch.where(n > 0, copy_to[0], 0)).long()
    for pool in st["pools"]:
        pool[b] = pool[a]
    return {f"pool{i}": pool for i, pool in enumerate(st["pools"])}


def _fork(st):
    page, pages, (batch, capacity) = st["page"], st["pages"], st["table"].shape
    lens, parent, gone, table = st["lens"].long(), st["parent"].long(), st["gone"].long(), st["table"]
    head, count = st["state"][0].long(), st["state"][1].long()
    b = torch.arange(batch, device=DEV)
    p = parent.clamp(0, batch - 1)
    ok = (parent >= 0) & (parent < batch) & (parent != b) & (lens == 0)
    n = lens[p] if st["keep"] is None else torch.minimum(lens[p], st["keep"].long().clamp(min=0))
    full, part = n // page, n % page > 0
    sink_pages = -(-st["sinks"] // page)
    ok = ok & ~(part & (full >= sink_pages) & (full < gone[p]))   # its last page is one that the parent has given back
    need = ok & part
    upto = need.cumsum(0)
    ok = ok & (~need | (upto <= count))
    need = need & ok
    n = torch.where(ok, n, 0)
    j = torch.arange(capacity, device=DEV)
    same = ok[:, None] & (j < full[:, None]) & ((j < sink_pages) | (j >= gone[p][:, None]))
    fresh = st["ring"][(head + upto - 1).remainder(pages)]
    table_out = torch.where(same, table[p], torch.where(need[:, None] & (j == full[:, None]), fresh[:, None], table))
    had = torch.where(same, table[p].long().clamp(0, pages - 1), pages).reshape(-1)
    shares = torch.cat([st["shares"].long(), lens.new_zeros(1)]).index_add_(0, had, torch.ones_like(had))[:pages]
    used = need.sum()
    slot = torch.where(need, upto - 1, batch)
    pick = lambda x: torch.full((batch + 1,), -1, dtype=torch.int64, device=DEV).scatter_(0, slot, x.long())[:batch]   # noqa: E731
    copy_from, copy_to = pick(torch.gather(table[p], 1, full.clamp(max=capacity - 1)[:, None])[:, 0]), pick(fresh)
    return dict(lens=torch.where(ok, n, lens).int(), taken=n.int(), table=table_out.int(), shares=shares.int(), state=torch.stack([(head + used).remainder(pages), count - used]).int(),
                gone=torch.where(ok, torch.minimum(gone[p], full), gone).int(), copy_from=copy_from.int(), copy_to=copy_to.int(), copies=used.reshape(1).int()) | _copy(st, copy_from, copy_to, used)


def _release(st):
    case, page, pages, (batch, capacity) = st["case"], st["page"], st["pages"], st["table"].shape
    lens, gone = st["lens"].long(), st["gone"].long()
    head, count = st["state"][0].long(), st["state"][1].long()
    after = torch.minimum(lens, st["keep"].long().clamp(min=0))
    left = torch.minimum(torch.maximum(gone, _first_kept(after, case["window"], page, st["sinks"])), (after + page - 1) // page)
    given = _held_pages(lens, gone, st["sinks"], page, capacity) & ~_held_pages(after, left, st["sinks"], page, capacity)
    given = given & (st["table"] >= 0) & (st["table"] < pages)
    had = torch.where(given, st["table"].long().clamp(0, pages - 1), pages).reshape(-1)
    shares = torch.cat([st["shares"].long(), lens.new_zeros(1)]).index_add_(0, had, -torch.ones_like(had))[:pages]
    free = shares < 0
    rank = free.cumsum(0) - 1
    free_in = free & (count + rank < pages)   # a ring holds all pages
    ring = torch.cat([st["ring"], st["ring"][:1]])
    ring[torch.where(free_in, (head + count + rank).remainder(pages), pages)] = torch.arange(pages, dtype=torch.int32, device=DEV)
    return dict(lens=after.int(), gone=left.int(), shares=shares.clamp(min=0).int(), ring=ring[:pages], state=torch.stack([head, count + free_in.sum()]).int())


def _compact(st):
    page, pages, (batch, capacity) = st["page"], st["pages"], st["table"].shape
    head, count = st["state"][0].long(), st["state"][1].long()
    i = torch.arange(pages, device=DEV)
    in_ring = st["ring"][(head + i).remainder(pages)].long()
    in_ring = torch.where((i < count) & (in_ring >= 0) & (in_ring < pages), in_ring, pages)
    free = torch.zeros(pages + 1, dtype=torch.bool, device=DEV).index_fill_(0, in_ring, True)[:pages]
    used = (~free).sum()
    hole, mover = free & (i < used), ~free & (i >= used)
    moves = hole.sum()
    nth = lambda which: torch.full((pages + 1,), -1, dtype=torch.int64, device=DEV).scatter_(0, torch.where(which, which.cumsum(0) - 1, pages), i)   # noqa: E731
    copy_from, copy_to = nth(mover)[:pages // 2 + 1], nth(hole)[:pages // 2 + 1]
    target = copy_to[(mover.cumsum(0) - 1).clamp(0, pages // 2)]
    moved_to = torch.where(free, -1, torch.where(mover, target, i))
    j = torch.arange(capacity, device=DEV)
    held = (j < ((st["lens"].long() + page - 1) // page)[:, None])
    at = st["table"].long()
    inside = (at >= 0) & (at < pages)
    table = torch.where(held, torch.where(inside, moved_to[at.clamp(0, pages - 1)], -1), at)
    shares = torch.zeros(pages + 1, dtype=torch.int64, device=DEV).scatter_(0, torch.where(free, pages, moved_to), st["shares"].long())[:pages]
    n_free = pages - used
    last = torch.arange(copy_from.numel(), device=DEV) < moves   # behind the last one nothing is written
    copy_from, copy_to = torch.where(last, copy_from, -1), torch.where(last, copy_to, -1)
    return dict(table=table.int(), ring=torch.where(i < n_free, used + i, -1).int(), state=torch.stack([0 * used, n_free]).int(), shares=shares.int(), moved_to=moved_to.int(),
                copy_from=copy_from.int(), copy_to=copy_to.int(), copies=moves.reshape(1).int()) | _copy(st, copy_from, copy_to, moves)


# -------------------------------------------------------------------------------------------------- the framework's calls
_context = []


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _fa():
    from goml_b200 import fa_forward as F
    if not _context:
        _context.append(F.FACreate())
    return _context[0]


def _own_prompt(st):
    case = st["case"]
    _fa().ForwardSinks(st["q"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(), st["o"].data_ptr(), st["lse"].data_ptr(), case["bh"], case["s"], case["hd"], case["window"],
                       case["sinks"], st["scale"], 1.0, st["q_scale"].data_ptr(), st["k_scale"].data_ptr(), st["v_scale"].data_ptr(), _stream())
    return dict(o=st["o"], lse=st["lse"])


def _own_window(st):
    case, (batch, capacity) = st["case"], st["table"].shape
    _fa().DecodeWindow(st["q"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(), st["o"].data_ptr(), st["lse"].data_ptr(), st["lens"].data_ptr(), batch, case["q_heads"],
                       case["kv_heads"], case["hd"], capacity * st["page"], 0, case["window"], case["sinks"], st["scale"], 1.0, st["q_scale"].data_ptr(), st["k_scale"].data_ptr(),
                       st["v_scale"].data_ptr(), _stream(), st["table"].data_ptr() if case["page"] else 0, st["page"], capacity, st["pages"])
    return dict(o=st["o"], lse=st["lse"])


def _own_shared(st):
    case, (batch, capacity) = st["case"], st["table"].shape
    _fa().DecodeShared(st["q"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(), st["o"].data_ptr(), st["lse"].data_ptr(), st["lens"].data_ptr(), st["shared"].data_ptr(),
                       st["starts"].data_ptr(), case["groups"], batch, case["q_heads"], case["kv_heads"], case["hd"], capacity * st["page"], st["scale"], 1.0,
                       st["q_scale"].data_ptr(), st["k_scale"].data_ptr(), st["v_scale"].data_ptr(), _stream(), st["table"].data_ptr() if case["page"] else 0, st["page"], capacity,
                       st["pages"])
    return dict(o=st["o"], lse=st["lse"])


def _own_copy(st):
    from goml_b200 import block_glue as BG
    BG.KVPageCopy([(pool.data_ptr(), pool.stride(0)) for pool in st["pools"]], st["copy_from"].data_ptr(), st["copy_to"].data_ptr(), st["copies"].data_ptr(),
                  st["copy_from"].numel(), st["pages"], _stream())
    return {f"pool{i}": pool for i, pool in enumerate(st["pools"])}


def _own_fork(st):
    from goml_b200 import block_glue as BG
    batch, capacity = st["table"].shape
    BG.KVPageFork(st["lens"].data_ptr(), st["parent"].data_ptr(), 0 if st["keep"] is None else st["keep"].data_ptr(), st["table"].data_ptr(), st["ring"].data_ptr(),
                  st["state"].data_ptr(), st["shares"].data_ptr(), st["gone"].data_ptr(), st["lens_out"].data_ptr(), st["state_out"].data_ptr(), st["shares_out"].data_ptr(),
                  st["gone_out"].data_ptr(), st["taken"].data_ptr(), st["copy_from"].data_ptr(), st["copy_to"].data_ptr(), st["copies"].data_ptr(), batch, capacity, st["page"],
                  st["pages"], st["sinks"], _stream())
    return dict(lens=st["lens_out"], taken=st["taken"], table=st["table"], shares=st["shares_out"], state=st["state_out"][:2], gone=st["gone_out"], copy_from=st["copy_from"],
                copy_to=st["copy_to"], copies=st["copies"])


def _own_release(st):
    from goml_b200 import block_glue as BG
    batch, capacity = st["table"].shape
    BG.KVPageRelease(st["lens"].data_ptr(), st["keep"].data_ptr(), st["table"].data_ptr(), st["ring"].data_ptr(), st["state"].data_ptr(), st["shares"].data_ptr(),
                     st["gone"].data_ptr(), st["lens_out"].data_ptr(), st["state_out"].data_ptr(), st["shares_out"].data_ptr(), st["gone_out"].data_ptr(), batch, capacity,
                     st["page"], st["pages"], st["case"]["window"], st["sinks"], _stream())
    return dict(lens=st["lens_out"], gone=st["gone_out"], shares=st["shares_out"], ring=st["ring"], state=st["state_out"][:2])


def _own_compact(st):
    from goml_b200 import block_glue as BG
    batch, capacity = st["table"].shape
    BG.KVPageCompact(st["lens"].data_ptr(), st["table"].data_ptr(), st["ring"].data_ptr(), st["state"].data_ptr(), st["shares"].data_ptr(), st["table_out"].data_ptr(),
                     st["ring_out"].data_ptr(), st["state_out"].data_ptr(), st["shares_out"].data_ptr(), st["moved_to"].data_ptr(), st["copy_from"].data_ptr(),
                     st["copy_to"].data_ptr(), st["copies"].data_ptr(), batch, capacity, st["page"], st["pages"], _stream())
    return dict(table=st["table_out"], ring=st["ring_out"], state=st["state_out"][:2], shares=st["shares_out"], moved_to=st["moved_to"], copy_from=st["copy_from"],
                copy_to=st["copy_to"], copies=st["copies"])


def run(st):
    kind = st["case"]["kind"]
    if own:
        out = dict(prompt=_own_prompt, window=_own_window, shared=_own_shared, fork=_own_fork, release=_own_release, compact=_own_compact)[kind](st)
        return out | _own_copy(st) if kind in ("fork", "compact") else out
    return dict(prompt=_prompt, window=_window, shared=_shared, fork=_fork, release=_release, compact=_compact)[kind](st)


# ------------------------------------------------------------------------------------------------------------------- work
def _seen(n, window, sinks):
    return min(n, window + sinks)


def work(case):
    kind, batch, page = case["kind"], case.get("batch"), case.get("page")
    if kind == "prompt":
        bh, s, hd, window, sinks = (case[x] for x in ("bh", "s", "hd", "window", "sinks"))
        pairs = sum(_seen(i + 1, window, sinks) for i in range(s))
        return dict(bytes=bh * s * (5 * hd + 4), flops=4 * bh * hd * pairs)
    if kind in ("window", "shared"):
        hq, kv, hd = case["q_heads"], case["kv_heads"], case["hd"]
        others = batch - 1 - (2 if batch > 8 else 0)
        if kind == "window":
            s = case["s"]
            pairs = keys = _seen(s, case["window"], case["sinks"]) + others * _seen(int(0.75 * s), case["window"], case["sinks"])
        else:   # the prefix of each group once, and what every sequence has of its own
            keys = case["prefix"] * (1 + 0.75 * (case["groups"] - 1)) + 0.75 * batch * case["suffix"]
            pairs = batch * 0.8 * case["prefix"] + 0.75 * batch * case["suffix"]
        return dict(bytes=2 * kv * hd * keys + batch * (hq * (3 * hd + 4) + 4), flops=4 * hq * hd * pairs)
    s = case["s"]
    held = -(-s // page)
    if kind == "release":
        return dict(bytes=batch * (5 * 4 + 0.15 * 0.5 * held * 4) + 0.5 * batch * held * 8, flops=0)
    bytes_of_page = case["pools"] * case["kv_heads"] * page * case["hd"]
    if kind == "fork":
        forks = case["share"] * batch
        return dict(bytes=batch * 24 + forks * (0.75 * held * 16 + 2 * bytes_of_page), flops=0)
    pages = 0.5 * batch * held / case["used"]
    return dict(bytes=pages * 24 + batch * held * 4 + 2 * bytes_of_page * pages * case["used"] * (1 - case["used"]), flops=0)


# ------------------------------------------------------------------------------------------------- by definition, in 64 bits
def _e4m3(codes):
    """Values of e4m3 bytes from the bits: sign, four of exponent with a bias of 7, three of mantissa; 127 and 255 are NaN."""
    c = codes.long()
    e, m = (c >> 3) & 15, (c & 7).double()
    x = torch.where(e == 0, torch.ldexp(m, torch.full_like(e, -9)), torch.ldexp(8 + m, e - 10))
    return torch.where(c & 127 == 127, math.nan, torch.where(c >= 128, -x, x))


def _softmax_of(q, k, v, seen, factor, v_scale):
    """O and LSE of q [.., queries, hd] on keys [.., keys, hd] that `seen` [queries, keys] lets through."""
    x = torch.einsum("...qd,...kd->...qk", q, k) * factor
    x = torch.where(seen, x, -math.inf)
    lse = torch.logsumexp(x, -1)
    weight = torch.where(seen, torch.exp(x - lse[..., None]), 0.0)
    return torch.einsum("...qk,...kd->...qd", weight, v) * v_scale, lse


def _exact_prompt(st):
    case = st["case"]
    s, window, sinks = case["s"], case["window"], case["sinks"]
    factor = st["scale"] * float(st["q_scale"]) * float(st["k_scale"])
    o, lse = torch.zeros(st["o"].shape, dtype=torch.float64, device=DEV), torch.zeros(st["lse"].shape, dtype=torch.float64, device=DEV)
    for h in range(case["bh"]):
        q, k, v = (_e4m3(st[x][h]) for x in ("q", "k", "v"))
        for q0 in range(0, s, 1024):
            i = torch.arange(q0, min(s, q0 + 1024), device=DEV)
            lo = max(0, q0 + 1 - window)
            j = torch.arange(lo, int(i[-1]) + 1, device=DEV)
            j = torch.cat([torch.arange(min(sinks, lo), device=DEV), j])
            back = i[:, None] - j
            o[h, i], lse[h, i] = _softmax_of(q[i], k[j], v[j], (back >= 0) & ((back < window) | (j < sinks)), factor, float(st["v_scale"]))
    return dict(o=o, lse=lse)


def _exact_decode(st):
    """A sequence at a time, the keys that it sees one by one from its own row of the table."""
    case, page = st["case"], st["page"]
    batch, hq, hd = st["q"].shape
    kv = case["kv_heads"]
    factor = st["scale"] * float(st["q_scale"]) * float(st["k_scale"])
    o, lse = torch.zeros(batch, hq, hd, dtype=torch.float64, device=DEV), torch.full((batch, hq), -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(st["lens"].tolist()):
        if case["kind"] == "window":
            keys = [i for i in range(min(case["sinks"], n))] + list(range(max(0, case["sinks"], n - case["window"]), n))
        else:
            keys = list(range(n))
        if not keys:
            continue
        at = torch.tensor(keys, device=DEV)
        where = st["table"][b].long()[at // page]
        k, v = (_e4m3(st[x][where, :, at % page]).transpose(0, 1) for x in ("k", "v"))
        x, y = _softmax_of(_e4m3(st["q"][b]).reshape(kv, hq // kv, hd), k, v, torch.ones(1, len(keys), dtype=torch.bool, device=DEV), factor, float(st["v_scale"]))
        o[b], lse[b] = x.reshape(hq, hd), y.reshape(hq)
    return dict(o=o, lse=lse)


def exact(case, seed):
    if case["kind"] in ("fork", "release", "compact"):
        return None   # whole numbers
    st = prepare(case, seed)
    return _exact_prompt(st) if case["kind"] == "prompt" else _exact_decode(st)
