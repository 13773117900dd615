"""Calls of fa_decode_fp4 that reach every form of its kernel: whole pairs and a line, teams of CTAs and of warps, one and two column tiles, pieces longer than 32 steps (whose table entries
are asked for 32 steps at a time), and pairs cut into so many pieces that their sums are formed on two levels.  Many sequences share the pages of a few (`order`), so that the caches are
small; tables are `table` pages wide and the pool is said to have `pool` of them, by which the form is chosen."""


def _pages(lens):
    return len(lens) * (-(-max(lens) // 64) + 1) + 3     # of tests.test_fp4_gpu.Case with pages of 64


_LONG = [17000, 8256, 16385, 129]      # CTAs take 256 keys a step
_MIDDLE = [4200, 2049, 4097, 65]       # warps take 64
_SHORT = [10000, 64, 1, 100, 0, 3]
_MIXED = [0] + [1, 2, 3, 4, 5, 2] * 150 + [0] + [3, 2, 5, 1] * 150 + [0]


def _form(plan, teams, hq, kv, hd, lens, order, table, pool, **what):
    return dict(plan=plan, teams=teams, hq=hq, kv=kv, hd=hd, lens=[lens[i] for i in order], distinct=lens, order=order, table=table, pool=pool, **what)


FORMS = {
    "pairs, CTAs, 128": _form("pair", "ctas", 4, 1, 128, _LONG, [0, 1, 2, 3] * 40, 300, _pages(_LONG), steps=64),
    "pairs, CTAs, 64, 16 heads": _form("pair", "ctas", 16, 1, 64, _LONG, [0, 1, 2, 3] * 40, 300, _pages(_LONG), steps=64),
    "pairs, warps, 128": _form("pair", "warps", 4, 1, 128, _MIDDLE, [0, 1, 2, 3] * 444, 100, _pages(_MIDDLE), steps=64),
    "pairs, warps, 64": _form("pair", "warps", 1, 1, 64, _MIDDLE, [0, 1, 2, 3] * 444, 100, _pages(_MIDDLE), steps=64),
    "pairs, warps, 128, 16 heads": _form("pair", "warps", 16, 1, 128, _MIDDLE, [0, 1, 2, 3] * 444, 100, _pages(_MIDDLE), steps=64),
    "line, CTAs, 128, long pieces": _form("line", "ctas", 4, 1, 128, _LONG[:1] + _LONG[2:3], [0, 1] * 150, 266, 266 * 300, steps=32, cuts=0),
    "line, CTAs, 64, 16 heads, long pieces": _form("line", "ctas", 16, 1, 64, _LONG[:1] + _LONG[2:3], [0, 1] * 120, 266, 266 * 240, steps=32, cuts=0),
    "line, warps, 128, long pieces": _form("line", "warps", 4, 1, 128, [8500, 8449], [0, 1] * 280, 133, 133 * 560, steps=32, cuts=0),
    "line, CTAs, 128, two levels": _form("line", "ctas", 4, 1, 128, [17000, 200], [1, 0, 1], 300, 900, cuts=17),
    "line, warps, 128, two levels": _form("line", "warps", 4, 1, 128, _SHORT, _MIXED, 157, 31250, cuts=17),
    "line, warps, 64, two levels": _form("line", "warps", 2, 2, 64, _SHORT, _MIXED, 157, 31250, cuts=17),
    "line, warps, 64, 16 heads, two levels": _form("line", "warps", 16, 1, 64, _SHORT, _MIXED * 2, 157, 50000, cuts=17),
    "line, warps, 128, 16 heads, two levels": _form("line", "warps", 32, 2, 128, _SHORT, _MIXED, 157, 50000, cuts=17),
}


def form_of(f):
    """Arguments of the layout's choice: sequences, query and kv heads, keys that a table has room for, keys that the pool has."""
    return len(f["order"]), f["hq"], f["kv"], f["table"] * 64, f["pool"] * 64
