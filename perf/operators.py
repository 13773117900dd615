"""Operators of a decoder that keeps its keys and values in 4 bits: what a serving program calls for each step.

  plan    `KVPagePlan`: from the sequences' lengths and the new tokens of a step, pages out of a ring of free ones, the block table's new entries,
          and every new token's position and place (slot) in the cache; pages of sequences that end go back into the ring
  append  `FP4RopeAppend`: rows of the QKV projection -> RoPE -> queries in bf16, keys and values in 4 bits at their slots; behind it
          `FP4CacheRows`, which reads the rows at these slots back as bf16 values
  attend  `FAContext.DecodeFP4`: one query token of every sequence against the 4-bit cache, contiguous or in pages
  step    plan, append and attend as one step of a server

A value of the cache is code * block scale * tensor scale: e2m1 codes, two to a byte (the even dim in the low half), an e4m3 scale for 16
consecutive dims, one fp32 scale for all keys and one for all values.  Codes lie as [pages, kv heads, page, hd / 2], scales of keys as
[pages, kv heads, page, hd / 16], scales of values as [pages, kv heads, page / 16, hd / 16, 16] (the 16 keys of a block side by side).  A
contiguous cache is one page to a sequence.
"""
import math

import torch

own = False

DEV = "cuda"
THETA = 10000.0
#: magnitudes of the eight e2m1 codes, and the values halfway between neighbours with whether a tie takes the upper one (to even)
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
HALFWAY = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))
BANK = 1 << 14   # different rows of keys and values that a large cache is filled from


def listed():
    gqa = dict(q_heads=32, kv_heads=8, hd=128)
    full = dict(q_heads=32, kv_heads=32, hd=128)
    return [
        # the next token of eight users: the smallest plan, where the launch counts
        dict(name="plan_few", kind="plan", batch=8, page=64, s=2000, prompt=0, rows=8, per_seq=1),
        # a busy server's step: most sequences go on by a token, some begin with a prompt, some end; the step's rows are packed into a padded batch
        dict(name="plan_mixed", kind="plan", batch=192, page=128, s=6000, prompt=2000, rows=16384, per_seq=0),
        # many short requests that arrive together, as an evaluation run sends them
        dict(name="plan_large", kind="plan", batch=4096, page=64, s=300, prompt=1000, rows=300000, per_seq=0),
        # new tokens of a decode step, grouped-query heads
        dict(name="append_step", kind="append", tokens=24, page=128, **gqa),
        # a ragged batch of prompts in head dim 64, some rows of it padding
        dict(name="append_ragged_hd64", kind="append", tokens=3001, page=64, q_heads=32, kv_heads=8, hd=64),
        # eight prompts of 2048 tokens, a kv head for every query head
        dict(name="append_prompts", kind="append", tokens=16384, page=256, **full),
        # one user's next token
        dict(name="attend_one", kind="attend", batch=1, s=1000, page=0, q="bf16", **full),
        # 24 users with contexts of up to 6000 tokens in pages, four query heads per kv head
        dict(name="attend_gqa_paged", kind="attend", batch=24, s=6000, page=128, q="bf16", **gqa),
        # a single long document
        dict(name="attend_long", kind="attend", batch=1, s=200000, page=0, q="bf16", **gqa),
        # sixteen query heads per kv head of 64, e4m3 queries
        dict(name="attend_wide_hd64", kind="attend", batch=48, s=3001, page=64, q="e4m3", q_heads=64, kv_heads=4, hd=64),
        # 64 users, a kv head for every query head: the largest call
        dict(name="attend_batch", kind="attend", batch=64, s=4096, page=64, q="bf16", **full),
        # a whole step of a server in one layer: plan, append, attend; a few of its places are vacant
        dict(name="step", kind="step", batch=40, s=2500, page=64, **gqa),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "append", "attend", "attend", "attend", "step"])
    if kind == "plan":
        batch, page = _log(rng, 1, 4096), rng.choice([16, 64, 64, 128, 256])
        if rng.random() < 0.4:
            per_seq = rng.choice([1, 1, 2, 5])
            return dict(kind=kind, batch=batch, page=page, s=_log(rng, 10, 8000), prompt=0, rows=batch * per_seq, per_seq=per_seq)
        prompt = min(_log(rng, 2, 8000), 1200000 // batch)
        return dict(kind=kind, batch=batch, page=page, s=_log(rng, 10, 8000), prompt=prompt, rows=max(1, int(batch * prompt * rng.uniform(0.05, 0.35))) + batch,
                    per_seq=0)
    hd, kv = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 8, 32])
    heads = dict(q_heads=kv * (rng.choice([1, 1, 2]) if kv == 32 else rng.choice([1, 2, 4, 5, 8, 16])), kv_heads=kv, hd=hd)
    if kind == "append":
        most = min(16384, int(16384 * 96 * 128 / ((heads["q_heads"] + 2 * kv) * hd)))
        return dict(kind=kind, tokens=_log(rng, 1, most), page=rng.choice([16, 64, 128, 256]), **heads)
    s = _log(rng, 1, 100000 if kind == "attend" else 8000)
    most = max(1, min(256, int(1.1e9 / (2.25 * kv * hd / 2 * s)), int(4.0e8 / (heads["q_heads"] * s))))
    batch = _log(rng, 1, most) if most > 1 else 1
    page = rng.choice([64, 64, 128, 192, 256])
    if kind == "step":
        return dict(kind=kind, batch=batch, s=s, page=page, **heads)
    return dict(kind=kind, batch=batch, s=s, page=rng.choice([0, page, page]), q=rng.choice(["bf16", "bf16", "fp16", "e4m3"]), **heads)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(g, lo, hi, n):
    """n whole numbers in [lo, hi]."""
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV, dtype=torch.int64)


def _rope_tables(rows, hd):
    angle = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * THETA ** (-2.0 * torch.arange(hd // 2, device=DEV, dtype=torch.float64) / hd)
    return angle.cos().float(), angle.sin().float()


def _channels(g, n, hd, std):
    """Rows of a head as projections make them: some channels several times as wide as the others."""
    wide = torch.exp(0.6 * torch.randn(hd, generator=g, device=DEV))
    return torch.randn(n, hd, generator=g, device=DEV) * (wide * (std / wide.square().mean().sqrt()))


def _filled(g, pages, kv, page, hd, std):
    """Codes and scales of a cache that holds rows of the bank everywhere, and their tensor scale."""
    rows = _channels(g, BANK, hd, std)
    scale = (rows.abs().amax() / (6 * 448)).reshape(1)
    sb, codes = _quantise(rows.reshape(BANK, hd // 16, 16), scale)
    codes = codes.reshape(BANK, hd // 2, 2)
    packed = (codes[..., 0] | codes[..., 1] << 4).to(torch.uint8)
    at = torch.randint(0, BANK, (pages * kv * page,), generator=g, device=DEV)
    return packed[at].reshape(pages, kv, page, hd // 2), sb.view(torch.uint8)[at].reshape(pages, kv, page, hd // 16), scale


def _blocks_of_16(scales):
    """[pages, kv, page, groups] -> [pages, kv, page / 16, groups, 16]."""
    pages, kv, page, groups = scales.shape
    return scales.reshape(pages, kv, page // 16, 16, groups).transpose(3, 4).contiguous()


def _cache(g, case, lens, table, pages, page):
    """A cache whose places behind the sequences' ends hold what was there before: anything, NaN among it."""
    kv, hd = case["kv_heads"], case["hd"]
    k, ks, k_scale = _filled(g, pages, kv, page, hd, 1.0)
    v, vs, v_scale = _filled(g, pages, kv, page, hd, 0.7)
    used = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
    key = torch.arange(table.shape[1] * page, device=DEV)
    live = key < lens[:, None]
    at = (table.long()[:, key // page] * page + key % page)
    used.view(-1)[at[live]] = True
    stale = torch.where(used, 0, 127).to(torch.uint8)[:, None, :, None]
    return dict(k=k, v=v, ks=ks | stale, vs=_blocks_of_16(vs | stale), k_scale=k_scale, v_scale=v_scale)


def _paged(g, batch, capacity, spare):
    """A table of different pages in no order, and those that are left over."""
    order = torch.randperm(batch * capacity + spare, generator=g, device=DEV).int()
    return order[:batch * capacity].reshape(batch, capacity).contiguous(), order[batch * capacity:]


def _lengths(g, batch, s):
    """Contexts between half of s and s; of several sequences one is empty, one has a single key."""
    lens = _ints(g, (s + 1) // 2, s, batch)
    lens[batch // 2] = s
    if batch > 8:
        lens[1], lens[batch - 1] = 0, 1
    return lens.int()


def _rows_of_qkv(g, tokens, case):
    hq, kv, hd = case["q_heads"], case["kv_heads"], case["hd"]
    x = _channels(g, tokens * (hq + 2 * kv), hd, 1.0).reshape(tokens, hq + 2 * kv, hd)
    return x.bfloat16().reshape(tokens, -1)


def _prepare_plan(case, g):
    batch, page, per_seq = case["batch"], case["page"], case["per_seq"]
    lens = _ints(g, 0, case["s"], batch)
    fresh = torch.ones_like(lens)
    what = torch.rand(batch, generator=g, device=DEV)
    if case["prompt"] > 1:   # a quarter begins with a prompt
        lens = torch.where(what < 0.25, 0, lens)
        fresh = torch.where(what < 0.25, _ints(g, 1, case["prompt"], batch), fresh)
    if per_seq > 1:
        fresh = _ints(g, 1, per_seq, batch)
    fresh = torch.where(what > 0.95, -1, torch.where(what > 0.9, 0, fresh))   # some end, some wait
    fresh[batch // 2] = max(1, min(case["prompt"], per_seq or case["rows"]))
    capacity = -(-(case["s"] + max(case["prompt"], per_seq, 1)) // page)
    held = (lens + page - 1) // page
    # the server has pages for nearly all of the step's tokens
    wanted = int(((lens + fresh.clamp(min=0) + page - 1) // page - held).sum() * 0.97) + 1
    pages = batch * -(-case["s"] // page) + batch * -(-max(case["prompt"], per_seq, 1) // page) + 8   # the others are somebody else's
    order = torch.randperm(pages, generator=g, device=DEV).int()
    first = held.cumsum(0) - held
    j = torch.arange(capacity, device=DEV)
    table = torch.where(j < held[:, None], order[(first[:, None] + j).clamp(max=pages - 1)], -1).int().contiguous()
    free = order[int(held.sum()):int(held.sum()) + wanted]
    head = int(_ints(g, 0, pages - 1, 1))
    ring = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    ring[(head + torch.arange(wanted, device=DEV)) % pages] = free
    return _plan_state(case, lens.int(), fresh.int(), table, ring, head, wanted, case["rows"], per_seq)


def _plan_state(case, lens, fresh, table, ring, head, count, rows, per_seq):
    new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=DEV)   # noqa: E731
    batch = lens.numel()
    state = torch.tensor([head, count, 0, 0], dtype=torch.int32, device=DEV)
    return dict(case=case, lens=lens, fresh=fresh, table=table, ring=ring, state=state, rows=rows, per_seq=per_seq, page=case["page"], lens_out=new(batch),
                state_out=torch.zeros_like(state), taken=new(batch), starts=new(batch + 1), positions=new(rows), slots=new(rows))


def _prepare_append(case, g):
    tokens, page, hd, kv = case["tokens"], case["page"], case["hd"], case["kv_heads"]
    rope = 8192
    pages = -(-tokens // page) + 3
    # sequences one behind another, each from some position on, every token at a place of its own
    positions = (_ints(g, 0, rope // 2, 1) + torch.arange(tokens, device=DEV)) % rope
    slots = torch.randperm(pages, generator=g, device=DEV)[torch.arange(tokens, device=DEV) // page] * page + torch.arange(tokens, device=DEV) % page
    padding = torch.rand(tokens, generator=g, device=DEV) < (0.05 if tokens > 64 else 0.0)
    qkv = _rows_of_qkv(g, tokens, case)
    cos, sin = _rope_tables(rope, hd)
    scale = lambda x: (x.float().abs().amax() / (6 * 448)).reshape(1)   # noqa: E731
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device=DEV)   # noqa: E731
    out = lambda heads: torch.empty(tokens, heads, hd, dtype=torch.bfloat16, device=DEV)   # noqa: E731
    return dict(case=case, qkv=qkv, positions=torch.where(padding, -1, positions).int(), slots=torch.where(padding, -1, slots).int(), cos=cos, sin=sin, pages=pages,
                page=page, k_scale=1.1 * scale(qkv), v_scale=scale(qkv[:, -kv * hd:]), k=zeros(pages, kv, page, hd // 2), v=zeros(pages, kv, page, hd // 2),
                ks=zeros(pages, kv, page, hd // 16), vs=zeros(pages, kv, page // 16, hd // 16, 16), q_out=out(case["q_heads"]), k_out=out(kv), v_out=out(kv))


def _prepare_attend(case, g):
    batch, s, page, hq, hd = case["batch"], case["s"], case["page"], case["q_heads"], case["hd"]
    lens = _lengths(g, batch, s)
    if page:
        table, _ = _paged(g, batch, -(-s // page), 5)
        pages = table.numel() + 5
    else:   # a contiguous cache: one page to a sequence
        page = -(-s // 16) * 16
        table, pages = torch.arange(batch, dtype=torch.int32, device=DEV)[:, None].contiguous(), batch
    q = _channels(g, batch * hq, hd, 1.5).reshape(batch, hq, hd)
    q_scale = torch.ones(1, device=DEV)
    if case["q"] == "e4m3":
        q_scale = (q.abs().amax() / 448).reshape(1)
        q = (q / q_scale).clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        q = q.to(torch.bfloat16 if case["q"] == "bf16" else torch.float16)
    return dict(case=case, q=q, q_scale=q_scale, lens=lens, table=table, pages=pages, page=page, scale=1.0 / math.sqrt(hd), **_cache(g, case, lens, table, pages, page),
                o=torch.empty(batch, hq, hd, dtype=torch.float16, device=DEV), lse=torch.empty(batch, hq, device=DEV))


def _prepare_step(case, g):
    batch, s, page, hq, hd = case["batch"], case["s"], case["page"], case["q_heads"], case["hd"]
    capacity = -(-(s + 1) // page)
    table, spare = _paged(g, batch, capacity, 3)
    lens = _lengths(g, batch, s)
    fresh = torch.ones_like(lens)
    if batch > 4:   # vacant places, and one that its user has left
        vacant = torch.rand(batch, generator=g, device=DEV) < 0.1
        vacant[0], vacant[batch // 2] = False, False
        lens, fresh = torch.where(vacant, 0, lens), torch.where(vacant, 0, fresh)
        fresh[2] = -1
    held = (lens.long() + page - 1) // page
    pages = table.numel() + spare.numel()
    # what the sequences do not hold is free
    free = torch.cat([table[torch.arange(capacity, device=DEV) >= held[:, None]], spare])
    head = int(_ints(g, 0, pages - 1, 1))
    ring = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    ring[(head + torch.arange(free.numel(), device=DEV)) % pages] = free
    cache = _cache(g, case, lens, table, pages, page)
    table = torch.where(torch.arange(capacity, device=DEV) < held[:, None], table, -1).int().contiguous()
    cos, sin = _rope_tables(capacity * page, hd)
    new = lambda dtype, *shape: torch.empty(shape, dtype=dtype, device=DEV)   # noqa: E731
    return _plan_state(case, lens, fresh, table, ring, head, free.numel(), batch, 1) | cache | dict(
        qkv=_rows_of_qkv(g, batch, case), cos=cos, sin=sin, pages=pages, scale=1.0 / math.sqrt(hd), q_scale=torch.ones(1, device=DEV),
        q_out=new(torch.bfloat16, batch, hq, hd), o=new(torch.float16, batch, hq, hd), lse=new(torch.float32, batch, hq))


def prepare(case, seed):
    make = dict(plan=_prepare_plan, append=_prepare_append, attend=_prepare_attend, step=_prepare_step)[case["kind"]]
    return make(case, _generator(seed))


# ----------------------------------------------------------------------------------------------------------- plain forms
def _plan(st):
    lens, fresh, table, ring = st["lens"].long(), st["fresh"].long(), st["table"], st["ring"]
    page, rows, per_seq, (batch, capacity) = st["page"], st["rows"], st["per_seq"], st["table"].shape
    head, count, pages = st["state"][0].long(), st["state"][1].long(), ring.numel()
    lens = lens.clamp(0, capacity * page)
    n, ends = fresh.clamp(min=0), fresh < 0
    held, past = (lens + page - 1) // page, lens + n
    upto = n.cumsum(0)
    first = torch.arange(batch, device=DEV) * per_seq if per_seq else upto - n
    fits = (n > 0) & (past <= capacity * page) & ((n <= per_seq) if per_seq else (upto <= rows))
    need = torch.where(fits, (past + page - 1) // page - held, 0)
    need_upto = need.cumsum(0)
    served = fits & ((need == 0) | (need_upto <= count))
    taken = torch.where(served, n, 0)
    i = torch.arange(rows, device=DEV)
    b = i // per_seq if per_seq else torch.searchsorted(upto, i, right=True)
    owned = b < batch
    b = b.clamp(max=batch - 1)
    k = i - first[b]
    owned = owned & (k < n[b]) & served[b]
    position = torch.where(owned, lens[b] + k, 0)
    j = position // page
    fresh_page = ring[(head + (need_upto - need)[b] + j - held[b]).remainder(pages)]
    got = torch.where(j < held[b], table[b, j.clamp(max=capacity - 1)], fresh_page)
    table_out = torch.cat([table, table[:, :1]], 1)   # a column more takes what is no new page
    table_out[b, torch.where(owned & (j >= held[b]) & (position % page == 0), j, capacity)] = got
    good = owned & (got >= 0) & (got < pages)
    back = torch.where(ends, held, 0)
    at = count + (back.cumsum(0) - back)[:, None] + torch.arange(capacity, device=DEV)
    given = (torch.arange(capacity, device=DEV) < back[:, None]) & (at < pages)
    ring_out = torch.cat([ring, ring[:1]])
    ring_out[torch.where(given, (head + at).remainder(pages), pages)] = table
    used = torch.where(served, need, 0).sum()
    starts = torch.cat([first, per_seq * batch * torch.ones_like(first[:1]) if per_seq else upto[-1:]]).clamp(max=rows)
    return dict(lens=torch.where(ends, 0, lens + taken).int(), taken=taken.int(), starts=starts.int(), positions=torch.where(owned, position, -1).int(),
                slots=torch.where(good, got * page + position % page, -1).int(), table=table_out[:, :capacity].contiguous(), ring=ring_out[:pages],
                state=torch.stack([(head + used).remainder(pages), count - used + given.sum()]).int())


def _quantise(y, scale):
    """(block scales in e4m3, codes 0 to 15) of y [..., 16]; which of two neighbours is nearer is decided in 64 bits (values of few bits often lie halfway)."""
    t = (y.abs().amax(-1).double() / (6.0 * scale.double())).clamp(max=448.0)
    step = torch.ldexp(torch.ones_like(t), (torch.frexp(t).exponent - 4).clamp(min=-9))   # between e4m3 numbers near t
    sb = (torch.round(t / step) * step).to(torch.float8_e4m3fn)
    d = sb.float() * scale
    ratio = (y.double() / d[..., None].double()).abs()
    code = sum((ratio >= h if up else ratio > h).to(torch.int32) for h, up in HALFWAY)
    return sb, torch.where(d[..., None] == 0, 0, code | torch.signbit(y).int() << 3)


def _values(sb, codes, scale):
    """What codes [..., 16] stand for, in 32 bits."""
    m = torch.tensor(MAGNITUDES + tuple(-x for x in MAGNITUDES), device=DEV)
    return m[codes.long()] * sb.float()[..., None] * scale


def _rotate(x, c, s):
    half = x.shape[-1] // 2
    x0, x1 = x[..., :half], x[..., half:]
    return torch.cat([x0 * c - x1 * s, x0 * s + x1 * c], -1)


def _append(st, positions, slots):
    """Queries, and for keys and values (block scales, codes) of every token."""
    case = st["case"]
    hq, kv, hd = case["q_heads"], case["kv_heads"], case["hd"]
    x = st["qkv"].float().reshape(-1, hq + 2 * kv, hd)
    active = (positions >= 0) & (positions < st["cos"].shape[0])
    at = torch.where(active, positions, 0).long()
    c, s = st["cos"][at][:, None], st["sin"][at][:, None]
    q = torch.where(active[:, None, None], _rotate(x[:, :hq], c, s), 0.0).bfloat16()
    k = _quantise(_rotate(x[:, hq:hq + kv], c, s).reshape(-1, kv, hd // 16, 16), st["k_scale"])
    v = _quantise(x[:, hq + kv:].reshape(-1, kv, hd // 16, 16), st["v_scale"])
    return q, k, v, active & (slots >= 0) & (slots < st["pages"] * st["page"])


def _append_and_read(st):
    q, k, v, stored = _append(st, st["positions"], st["slots"])
    read = lambda x, scale: torch.where(stored[:, None, None], _values(*x, scale).flatten(-2), 0.0).bfloat16()   # noqa: E731
    return dict(q=q, k=read(k, st["k_scale"]), v=read(v, st["v_scale"]))


def _of_sequences(st, codes, scales, scale, lens, table):
    """Keys or values [batch, kv heads, keys, hd] of all sequences in 32 bits, zeros behind a sequence's end."""
    batch, capacity = table.shape
    kv, page, half = codes.shape[1:]
    at = table.long().clamp(0, st["pages"] - 1)
    pairs = torch.tensor(MAGNITUDES + tuple(-x for x in MAGNITUDES), device=DEV)
    pairs = torch.stack([pairs.repeat(16), pairs.repeat_interleave(16)], -1)   # [byte, (low, high)]
    x = pairs[codes[at].transpose(1, 2).reshape(batch, kv, capacity * page, half).long()].reshape(batch, kv, capacity * page, half // 8, 16)
    x *= scales[at].transpose(1, 2).reshape(batch, kv, capacity * page, half // 8).view(torch.float8_e4m3fn).float()[..., None] * scale
    live = torch.arange(capacity * page, device=DEV) < lens[:, None]
    return x.masked_fill_(~live[:, None, :, None, None], 0.0).flatten(-2), live


def _attend(st, q, lens, table, k, ks, v, vs):
    batch, hq, hd = q.shape
    kv = k.shape[1]
    keys, live = _of_sequences(st, k, ks, st["k_scale"], lens, table)
    score = torch.matmul(q.float().reshape(batch, kv, hq // kv, hd) * (st["scale"] * st["q_scale"]), keys.transpose(2, 3))
    del keys
    score = score.masked_fill_(~live[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    values, _ = _of_sequences(st, v, vs.transpose(3, 4).reshape(ks.shape), st["v_scale"], lens, table)
    o = torch.matmul(p, values) / torch.where(total == 0, 1.0, total)
    lse = torch.where(total == 0, -math.inf, top + torch.log(total))
    return dict(o=o.reshape(batch, hq, hd).half(), lse=lse.reshape(batch, hq))


def _put(st, name, scales, x, slots, stored):
    """The cache's codes and scales with the tokens' rows in their places."""
    sb, codes = x
    pages, kv, page, half = st[name].shape
    codes = codes.reshape(*codes.shape[:2], half, 2)
    packed = (codes[..., 0] | codes[..., 1] << 4).to(torch.uint8)
    at = torch.where(stored, slots, 0).long()
    page_at, key_at = at // page, at % page
    keep = stored[:, None, None]
    out, scales = st[name].clone(), scales.clone()
    out[page_at, :, key_at] = torch.where(keep, packed, out[page_at, :, key_at])
    scales[page_at, :, key_at] = torch.where(keep, sb.view(torch.uint8), scales[page_at, :, key_at])
    return out, scales


def _step(st):
    plan = _plan(st)
    q, k, v, stored = _append(st, plan["positions"], plan["slots"])
    # a token that is not stored takes the place of the first that is, with the same row
    one = torch.argmax(stored.int())
    slots = torch.where(stored, plan["slots"], plan["slots"][one])
    pick = lambda x: tuple(torch.where(stored.reshape(-1, *[1] * (t.dim() - 1)), t.float(), t[one].float()).to(t.dtype) for t in x)   # noqa: E731
    any_stored = stored.any().expand_as(stored)
    kc, ks = _put(st, "k", st["ks"], pick(k), slots, any_stored)
    natural = st["vs"].transpose(3, 4).reshape(st["ks"].shape)
    vc, vs = _put(st, "v", natural, pick(v), slots, any_stored)
    return plan | dict(q=q) | _attend(st, q, plan["lens"], plan["table"], kc, ks, vc, _blocks_of_16(vs))


# -------------------------------------------------------------------------------------------------- the framework's calls
_context = []


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_plan(st):
    from goml_b200 import block_glue as BG
    batch, capacity = st["table"].shape
    BG.KVPagePlan(st["lens"].data_ptr(), st["fresh"].data_ptr(), st["table"].data_ptr(), st["ring"].data_ptr(), st["state"].data_ptr(), st["lens_out"].data_ptr(),
                  st["state_out"].data_ptr(), st["taken"].data_ptr(), st["starts"].data_ptr(), st["positions"].data_ptr(), st["slots"].data_ptr(), batch,
                  capacity, st["page"], st["ring"].numel(), st["rows"], st["per_seq"], _stream())
    return dict(lens=st["lens_out"], taken=st["taken"], starts=st["starts"], positions=st["positions"], slots=st["slots"], table=st["table"], ring=st["ring"],
                state=st["state_out"][:2])


def _own_append(st):
    from goml_b200 import block_glue as BG
    case = st["case"]
    BG.FP4RopeAppend(st["qkv"].data_ptr(), st["cos"].data_ptr(), st["sin"].data_ptr(), st["positions"].data_ptr(), st["slots"].data_ptr(), st["q_out"].data_ptr(),
                     st["k"].data_ptr(), st["ks"].data_ptr(), st["v"].data_ptr(), st["vs"].data_ptr(), st["k_scale"].data_ptr(), st["v_scale"].data_ptr(),
                     st["positions"].numel(), case["q_heads"], case["kv_heads"], case["hd"], st["cos"].shape[0], st["page"], st["pages"], _stream())
    return dict(q=st["q_out"])


def _own_rows(st):
    from goml_b200 import block_glue as BG
    case = st["case"]
    BG.FP4CacheRows(st["slots"].data_ptr(), st["k"].data_ptr(), st["ks"].data_ptr(), st["v"].data_ptr(), st["vs"].data_ptr(), st["k_scale"].data_ptr(),
                    st["v_scale"].data_ptr(), st["k_out"].data_ptr(), st["v_out"].data_ptr(), st["slots"].numel(), case["kv_heads"], case["hd"], st["page"],
                    st["pages"], _stream())
    return dict(k=st["k_out"], v=st["v_out"])


def _own_attend(st, q, q_type, lens, paged):
    from goml_b200 import fa_forward as F
    if not _context:
        _context.append(F.FACreate())
    case, (batch, capacity) = st["case"], st["table"].shape
    _context[0].DecodeFP4(q.data_ptr(), st["k"].data_ptr(), st["ks"].data_ptr(), st["v"].data_ptr(), st["vs"].data_ptr(), st["o"].data_ptr(), st["lse"].data_ptr(),
                          lens.data_ptr(), batch, case["q_heads"], case["kv_heads"], case["hd"], capacity * st["page"], 0, st["scale"], 1.0, q_type,
                          st["q_scale"].data_ptr(), st["k_scale"].data_ptr(), st["v_scale"].data_ptr(), _stream(),
                          st["table"].data_ptr() if paged else 0, st["page"], capacity, st["pages"])
    return dict(o=st["o"], lse=st["lse"])


def run(st):
    case = st["case"]
    if case["kind"] == "plan":
        return _own_plan(st) if own else _plan(st)
    if case["kind"] == "append":
        return _own_append(st) | _own_rows(st) if own else _append_and_read(st)
    if case["kind"] == "attend":
        if own:
            return _own_attend(st, st["q"], ("bf16", "fp16", "e4m3").index(case["q"]), st["lens"], case["page"] > 0)
        return _attend(st, st["q"], st["lens"], st["table"], st["k"], st["ks"], st["v"], st["vs"])
    if own:
        return _own_plan(st) | _own_append(st) | _own_attend(st, st["q_out"], 0, st["lens_out"], True)
    return _step(st)


# ------------------------------------------------------------------------------------------------------------------- work
def _keys(case):
    """Keys that the sequences of a case have on average (as _lengths makes them)."""
    others = case["batch"] - 1 - (2 if case["batch"] > 8 else 0)
    return case["s"] * (1 + 0.75 * others * (0.9 if case["kind"] == "step" else 1.0))


def work(case):
    if case["kind"] == "plan":
        new = case["batch"] if not case["prompt"] else min(case["rows"], case["batch"] * (0.7 + 0.125 * case["prompt"]))
        return dict(bytes=case["batch"] * 20 + case["rows"] * 8 + 8 * new / case["page"], flops=0)
    hq, kv, hd = case["q_heads"], case["kv_heads"], case["hd"]
    cached = 2 * kv * (hd // 2 + hd // 16)   # bytes of a token in the cache
    if case["kind"] == "append":
        t = case["tokens"]
        return dict(bytes=t * (8 + 2 * (hq + 2 * kv) * hd + 2 * hq * hd + 2 * cached + 4 * kv * hd + 4 * hd), flops=t * hd * (3 * hq + 8 * kv))
    attend = dict(bytes=_keys(case) * cached + case["batch"] * hq * (hd * (3 if case.get("q") == "e4m3" else 4) + 4), flops=4 * hq * hd * _keys(case))
    if case["kind"] == "step":
        attend["bytes"] += case["batch"] * (28 + 2 * (hq + 2 * kv) * hd + cached)
    return attend


# ------------------------------------------------------------------------------------------------- by definition, in 64 bits
def _nearest_code_value(x):
    """x [...] rounded to the e2m1 grid in 64 bits, ties to the code with an even number."""
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device=DEV)
    a = x.abs().clamp(max=6.0)
    hi = torch.searchsorted(grid, a.contiguous()).clamp(1, 7)
    below, above = a - grid[hi - 1], grid[hi] - a
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return torch.where(up, grid[hi], grid[hi - 1]) * torch.sign(x)


def _nearest_e4m3(x):
    """x >= 0 rounded to e4m3 in 64 bits (three bits behind the leading one, quanta of 2^-9 at least), at most 448."""
    quantum = torch.exp2(torch.floor(torch.log2(x.clamp(min=2.0 ** -30))) - 3).clamp(min=2.0 ** -9)
    return (torch.round(x / quantum) * quantum).clamp(max=448.0)


def _exact_rows(x, c, s, scale):
    """Values in the cache of rows x [tokens, heads, hd], rotated where c is given."""
    if c is not None:
        half = x.shape[-1] // 2
        x = torch.stack([x[..., :half] * c - x[..., half:] * s, x[..., :half] * s + x[..., half:] * c], -2).flatten(-2)
    groups = x.reshape(*x.shape[:-1], -1, 16)
    s32 = scale.double()
    d = (_nearest_e4m3(groups.abs().amax(-1) / (6 * s32)).float() * scale).double()[..., None]   # a scale is a number of 32 bits
    return x, (torch.where(d == 0, 0.0, _nearest_code_value(groups / torch.where(d == 0, 1.0, d))) * d).flatten(-2)


def _exact_append(st, positions, slots):
    case = st["case"]
    hq, kv, hd = case["q_heads"], case["kv_heads"], case["hd"]
    x = st["qkv"].double().reshape(-1, hq + 2 * kv, hd)
    keep = (positions >= 0)[:, None, None]
    at = positions.clamp(min=0).long()
    c, s = st["cos"].double()[at][:, None], st["sin"].double()[at][:, None]
    q, _ = _exact_rows(x[:, :hq], c, s, st["k_scale"])
    _, k = _exact_rows(x[:, hq:hq + kv], c, s, st["k_scale"])
    _, v = _exact_rows(x[:, hq + kv:], None, None, st["v_scale"])
    stored = keep & (slots >= 0)[:, None, None]
    return torch.where(keep, q, 0.0), torch.where(stored, k, 0.0), torch.where(stored, v, 0.0)


def _e2m1(codes):
    """[..., n] bytes -> [..., 2n] values, from the bits: sign, two of exponent, one of mantissa."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    sign, c = torch.where(c >= 8, -1.0, 1.0), c % 8
    e, m = torch.floor(c / 2), c % 2
    return sign * torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e - 1))


def _exact_attend(st, q, lens, table, last=None):
    """O and LSE a sequence at a time; `last`: the keys and values [batch, kv heads, hd] of every sequence's last place, where its cache has them not yet."""
    hd, page = q.shape[-1], st["page"]
    kv = st["k"].shape[1]
    o, lse = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens.tolist()):
        if not n:
            continue
        cached = n if last is None or last[2][b] is False else n - 1
        at = table[b, :-(-n // page)].long()
        value = lambda codes, scales, scale: (_e2m1(codes).reshape(*codes.shape[:-1], -1, 16) * scales.view(torch.float8_e4m3fn).double()[..., None]   # noqa: E731
                                              * scale.double()).flatten(-2)
        k = value(st["k"][at], st["ks"][at], st["k_scale"]).transpose(0, 1).reshape(kv, -1, hd)[:, :cached]
        v = value(st["v"][at], st["vs"][at].transpose(3, 4).reshape(-1, kv, page, hd // 16), st["v_scale"]).transpose(0, 1).reshape(kv, -1, hd)[:, :cached]
        if cached < n:
            k, v = torch.cat([k, last[0][b][:, None]], 1), torch.cat([v, last[1][b][:, None]], 1)
        x = torch.einsum("gid,gkd->gik", q[b].double().reshape(kv, -1, hd), k) * (float(st["scale"]) * st["q_scale"].double())
        lse[b] = torch.logsumexp(x, -1).reshape(-1)
        o[b] = torch.einsum("gik,gkd->gid", torch.softmax(x, -1), v).reshape(-1, hd)
    return o, lse


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "plan":
        return None   # whole numbers
    if case["kind"] == "append":
        q, k, v = _exact_append(st, st["positions"], st["slots"])
        return dict(q=q, k=k, v=v)
    if case["kind"] == "attend":
        o, lse = _exact_attend(st, st["q"], st["lens"], st["table"])
        return dict(o=o, lse=lse)
    # a step: every sequence with a new token has pages enough, so what it takes up is known from its length
    fresh, lens = st["fresh"].tolist(), st["lens"].tolist()
    go = [f > 0 for f in fresh]
    after = torch.tensor([0 if f < 0 else n + (f > 0) for f, n in zip(fresh, lens)], device=DEV)
    positions = torch.tensor([n if t else -1 for t, n in zip(go, lens)], device=DEV)
    q, k, v = _exact_append(st, positions, positions)
    table = st["table"].clamp(min=0)
    rounded = q.bfloat16()   # the queries are handed on in bf16
    o, lse = _exact_attend(st, rounded, after, table, (k, v, go))
    return dict(q=q, o=o, lse=lse)
