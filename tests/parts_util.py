"""What the tests of decode attention over parts of the keys share: caches with anything behind the sequences' ends, and the comparison with the restatement."""
import numpy as np
import torch

from oracle import parts

NAN = 127


def codes(r, shape, std=60.0):
    """e4m3 codes of normal data, without NaN."""
    from oracle import e4m3_encode
    return e4m3_encode(np.clip(r.normal(size=shape) * std, -448, 448).astype(np.float32)).reshape(shape)


class Cache:
    """Sequences of a contiguous or paged cache; places that no sequence has hold NaN codes."""

    def __init__(self, seed, lens, kv, hd, page=0, s_max=None, spare=3, std=60.0, room=0):
        """room: keys that a sequence can have at least, whatever the lengths are."""
        r = self.r = np.random.default_rng(seed)
        self.lens, self.kv, self.hd, self.page = np.array(lens, np.int32), kv, hd, page
        batch, most = len(lens), max(1, max(lens))
        self.rows = [(codes(r, (kv, n, hd), std), codes(r, (kv, n, hd), 50.0)) for n in lens]
        if page:
            self.width = max(-(-most // page) + 1, -(-room // page))
            self.pages = sum(-(-n // page) for n in lens) + spare
            order, at = r.permutation(self.pages), 0
            self.table = r.integers(-4, self.pages + 4, (batch, self.width)).astype(np.int32)   # behind a sequence's end: anything
            for b, n in enumerate(lens):
                c = -(-n // page)
                self.table[b, :c] = order[at:at + c]
                at += c
            self.s_max = self.width * page
        else:
            self.s_max = s_max or max(most + 7, room)
            self.pages, self.width, page = batch, 1, self.s_max
            self.table = np.arange(batch, dtype=np.int32)[:, None]
        self.k = np.full((self.pages, kv, page, hd), NAN, np.uint8)
        self.v = np.full((self.pages, kv, page, hd), NAN + 128, np.uint8)
        for b in range(batch):
            self.put(b)

    def put(self, b, first=0, last=None):
        """The rows [first, last) of a sequence to their places."""
        page = self.k.shape[2]
        for x, rows in zip((self.k, self.v), self.rows[b]):
            n = rows.shape[1] if last is None else last
            for j in range(first // page, -(-n // page)):
                p, lo, hi = self.table[b, j], max(first, j * page), min(n, (j + 1) * page)
                if lo < hi and 0 <= p < self.pages:
                    x[p, :, lo - j * page:hi - j * page] = rows[:, lo:hi]

    def share(self, starts, shared):
        """Sequences begin like the first of their group: whole pages are its own ones, the rest is copied."""
        for i in range(len(starts) - 1):
            for b in range(starts[i] + 1, starts[i + 1]):
                n, a = min(shared[b], int(self.lens[b])), starts[i]
                for x, y in zip(self.rows[b], self.rows[a]):
                    x[:, :n] = y[:, :n]
                whole = n // self.page if self.page else 0
                self.table[b, :whole] = self.table[a, :whole]
                self.put(b, whole * self.page)

    def to_gpu(self, q_group):
        hq = self.kv * q_group
        self.q = codes(self.r, (len(self.lens), hq, self.hd), 60.0)
        dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()   # noqa: E731
        self.d = dict(k=dev(self.k), v=dev(self.v), q=dev(self.q), lens=dev(self.lens), table=dev(self.table))
        # O and LSE with room behind them that must stay
        n = len(self.lens) * hq
        self.o = torch.full((n * self.hd + 64,), 5.0, dtype=torch.float16, device="cuda")
        self.lse = torch.full((n + 16,), 5.0, device="cuda")
        return hq

    def results(self, hq):
        torch.cuda.synchronize()
        n = len(self.lens) * hq
        assert (self.o[n * self.hd:] == 5).all() and (self.lse[n:] == 5).all()
        return self.o[:n * self.hd].double().cpu().numpy().reshape(-1, hq, self.hd), self.lse[:n].double().cpu().numpy().reshape(-1, hq)

    def check(self, o, lse, seen, scale, v_scale):
        """seen(b): keys that sequence b sees.  Keys of pages that the table does not have in the pool count as zeros."""
        hq = self.q.shape[1]
        group = hq // self.kv
        for b in range(len(self.lens)):
            keys = np.asarray(sorted(seen(b)), np.int64)
            for h in range(self.kv):
                k, v = self.rows[b][0][h][keys].copy(), self.rows[b][1][h][keys].copy()
                if self.page and len(keys):
                    out = ~((self.table[b, keys // self.page] >= 0) & (self.table[b, keys // self.page] < self.pages))
                    k[out], v[out] = 0, 0
                want, want_l, tol, tol_l = parts.attend(self.q[b, h * group:(h + 1) * group], k, v, np.ones((group, len(keys)), bool), scale, v_scale)
                got, got_l = o[b, h * group:(h + 1) * group], lse[b, h * group:(h + 1) * group]
                assert (np.abs(got - want) <= tol).all(), (b, h, np.abs(got - want).max(), (np.abs(got - want) / tol).max())
                assert np.array_equal(np.isneginf(got_l), np.isneginf(want_l))
                fine = ~np.isneginf(want_l)
                off = np.abs(got_l[fine] - want_l[fine])
                assert (off <= tol_l[fine]).all(), (b, h, off.max(), tol_l[fine].min())
