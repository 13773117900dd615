"""Restatement of the 4-bit KV cache on the CPU (numpy): the format, RoPE + append, reading rows back, decode attention, and the plan of a step's pages.

A value is code * block scale * tensor scale: e2m1 codes, two to a byte (even dim in the low half), an e4m3 scale for 16 dims, one fp32 scale for all keys and one
for all values.  Everything is decided in 64 bits, apart from what the format fixes in 32: RoPE with each product rounded, and block scale * tensor scale."""
import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127])   # numbers of codes 0 to 126


def _nearest(x, grid):
    """Index of the number of `grid` (ascending, codes in order) nearest to x >= 0; ties to the even code; past the end the last."""
    hi = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
    below, above = x - grid[hi - 1], grid[hi] - x
    return np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, hi - 1)


def quantise(y, scale):
    """(block scale bytes [..., groups], codes 0..15 [..., groups, 16]) of y [..., hd] fp32 for the tensor scale `scale` (fp32).  A NaN in a group makes its
    scale 0x7f (its codes say nothing)."""
    y = np.asarray(y, np.float32).reshape(*y.shape[:-1], -1, 16)
    s = np.float32(scale)
    top = np.abs(y).max(-1).astype(np.float64)
    nan = np.isnan(top)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        b = _nearest(np.minimum(np.where(nan, 0, top) / (6 * np.float64(s)), 448.0), E4M3)
        d = (E4M3[b].astype(np.float32) * s).astype(np.float64)
        none = d < 2.0 ** -126
        ratio = np.abs(y).astype(np.float64) / np.where(none, 1, d)[..., None]
    codes = _nearest(np.where(np.isnan(ratio), 0, np.minimum(ratio, 6.0)), MAGNITUDES) + 8 * np.signbit(y)
    return np.where(nan, 0x7F, b).astype(np.uint8), np.where(none[..., None], 0, codes).astype(np.uint8)


def pack(codes):
    """[..., groups, 16] codes -> [..., hd / 2] bytes."""
    c = codes.reshape(*codes.shape[:-2], -1, 2)
    return (c[..., 0] | c[..., 1] << 4).astype(np.uint8)


def values(packed, scales, scale):
    """[..., hd] fp64 values of [..., hd / 2] bytes and [..., hd / 16] block scale bytes (natural order)."""
    c = np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1, 16)
    v = MAGNITUDES[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.append(E4M3, np.nan)[scales & 0x7F] * np.where(scales & 0x80, -1.0, 1.0)
    return (v * s[..., None] * np.float64(np.float32(scale))).reshape(*packed.shape[:-1], -1)


def blocks_of_16(scales):
    """Block scales [..., keys, groups] in the order the cache holds those of values: [..., keys / 16, groups, 16]."""
    *lead, keys, groups = scales.shape
    return np.ascontiguousarray(np.swapaxes(scales.reshape(*lead, keys // 16, 16, groups), -1, -2))


def natural(v_scales):
    """The inverse of blocks_of_16."""
    x = np.swapaxes(v_scales, -1, -2)
    return np.ascontiguousarray(x.reshape(*x.shape[:-3], -1, x.shape[-1]))


def rope(x, cos, sin):
    """x [..., hd] fp32, cos and sin [..., hd / 2] fp32: half-split RoPE, each product rounded to fp32."""
    half = x.shape[-1] // 2
    x0, x1 = x[..., :half], x[..., half:]
    return np.concatenate([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1).astype(np.float32)


def append(qkv, cos, sin, positions, slots, q_heads, cache):
    """qkv [tokens, q_heads + 2 kv, hd] fp32 (bf16 values).  Writes K and V into `cache` (a dict k, ks, v, vs, k_scale, v_scale with the arrays' shapes) and returns
    Q [tokens, q_heads, hd] in fp32, not yet rounded to bf16."""
    pages, kv, page, _ = cache["k"].shape
    q = np.zeros((len(qkv), q_heads, qkv.shape[-1]), np.float32)
    vs = natural(cache["vs"])
    for i, (pos, slot) in enumerate(zip(positions, slots)):
        if not 0 <= pos < len(cos):
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            q[i] = rope(qkv[i, :q_heads], cos[pos], sin[pos])
            k = rope(qkv[i, q_heads:q_heads + kv], cos[pos], sin[pos])
        if 0 <= slot < pages * page:
            pg, at = divmod(int(slot), page)
            for name, scales, rows, scale in (("k", cache["ks"], k, cache["k_scale"]), ("v", vs, qkv[i, q_heads + kv:], cache["v_scale"])):
                b, codes = quantise(rows, scale)
                cache[name][pg, :, at] = pack(codes)
                scales[pg, :, at] = b
    cache["vs"][...] = blocks_of_16(vs)
    return q


def attention(q, k, v, lens, scale):
    """q [batch, q_heads, hd]; k, v [batch, kv, keys, hd] fp64, keys at or past lens[b] unused.  Returns O, LSE, and for bounds: sum p|v| / sum p and the largest
    sum |q_d k_d| * scale of a query."""
    batch, hq, hd = q.shape
    kv = k.shape[1]
    o, lse = np.zeros((batch, hq, hd)), np.full((batch, hq), -np.inf)
    spread, size = np.zeros((batch, hq, hd)), np.zeros((batch, hq))
    for b in range(batch):
        n = int(lens[b])
        if n == 0:
            continue
        for h in range(hq):
            kk, vv = k[b, h * kv // hq, :n], v[b, h * kv // hq, :n]
            s = kk @ q[b, h] * scale
            top = s.max()
            p = np.exp(s - top)
            o[b, h], spread[b, h] = p @ vv / p.sum(), p @ np.abs(vv) / p.sum()
            lse[b, h] = top + np.log(p.sum())
            size[b, h] = (np.abs(kk) @ np.abs(q[b, h])).max() * abs(scale)
    return o, lse, spread, size


def plan(lens, fresh, table, ring, head, count, page, rows, per_seq=0):
    """kv_page_plan one sequence after another.  Returns a dict of its outputs."""
    batch, max_pages = table.shape
    pages = len(ring)
    table, ring, capacity = table.copy(), ring.copy(), max_pages * page
    head, count = max(head, 0) % pages, min(max(count, 0), pages)
    out = dict(lens=np.zeros(batch, np.int32), taken=np.zeros(batch, np.int32), starts=np.zeros(batch + 1, np.int32),
               positions=np.full(rows, -1, np.int32), slots=np.full(rows, -1, np.int32))
    wanted = used = back = start = 0
    old_ring = ring.copy()
    for b in range(batch):
        n, f = min(max(int(lens[b]), 0), capacity), int(fresh[b])
        held = -(-n // page)
        if per_seq:
            start = b * per_seq
        out["starts"][b] = min(start, rows)
        out["lens"][b] = n
        if f < 0:
            for j in range(held):
                if count + back < pages:
                    ring[(head + count + back) % pages] = table[b, j]
                    back += 1
            out["lens"][b] = 0
        elif f > 0 and n + f <= capacity and (f <= per_seq if per_seq else start + f <= rows):
            need = -(-(n + f) // page) - held
            wanted += need
            if need == 0 or wanted <= count:
                for j in range(need):
                    table[b, held + j] = old_ring[(head + wanted - need + j) % pages]
                used += need
                out["taken"][b] = f
                out["lens"][b] = n + f
                for i in range(f):
                    pg = int(table[b, (n + i) // page])
                    out["positions"][start + i] = n + i
                    if 0 <= pg < pages:
                        out["slots"][start + i] = pg * page + (n + i) % page
        start += max(f, 0)
    out["starts"][batch] = min(batch * per_seq if per_seq else start, rows)
    return dict(out, table=table, ring=ring, state=((head + used) % pages, count - used + back))
