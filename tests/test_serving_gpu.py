"""Page and attention calls together, as a server's steps are: prompts, forks, appended tokens, attention over common prefixes and over windows, sequences that end, pools made dense."""
import numpy as np
import pytest
import torch

import oracle as O
from oracle import parts
from tests.parts_util import codes
from tests.test_decode_append_gpu import rope_tables
from tests.test_decoder_block_gpu import _make_block

pytestmark = pytest.mark.gpu
PAGE, SCALE, K_SCALE, V_SCALE = 64, 0.09, 0.011, 0.013


def ints(x):
    return torch.tensor([int(i) for i in x], dtype=torch.int32, device="cuda")


class Server:
    """An e4m3 cache in pages, the calls on it, and on the CPU what each sequence's keys and values have been."""

    def __init__(self, fa, batch, kv, group, hd, pages, width, seed, sinks=0, window=0):
        self.fa, self.B, self.kv, self.hq, self.hd, self.n, self.width = fa, batch, kv, kv * group, hd, pages, width
        self.window, self.sinks, self.r = window, sinks, np.random.default_rng(seed)
        new = lambda *shape, value=0: torch.full(shape, value, dtype=torch.int32, device="cuda")   # noqa: E731
        self.table, self.lens, self.ring, self.state = new(batch, width, value=-1), new(batch), torch.arange(pages, dtype=torch.int32, device="cuda"), ints([0, pages, 0, 0])
        self.shares, self.gone, self.taken, self.starts = new(pages), new(batch), new(batch), new(batch + 1)
        self.copy_from, self.copy_to, self.copies, self.moved = new(max(batch, pages)), new(max(batch, pages)), new(1), new(pages)
        self.positions, self.slots = new(4096), new(4096)
        self.k = torch.full((pages, kv, PAGE, hd), 127, dtype=torch.uint8, device="cuda")   # NaN where nobody has written
        self.v = torch.full_like(self.k, 255)
        self.scales = torch.tensor([0.0, 0.0, K_SCALE, V_SCALE], device="cuda")    # of Q and its amax, written by the append; of K and V
        self.q = torch.zeros((batch, self.hq, hd), dtype=torch.uint8, device="cuda")
        self.o, self.lse = torch.zeros((batch, self.hq, hd), dtype=torch.float16, device="cuda"), torch.zeros((batch, self.hq), device="cuda")
        self.qkv = torch.zeros((batch, (self.hq + 2 * kv) * hd), dtype=torch.bfloat16, device="cuda")
        self.cos, self.sin = rope_tables(1024, hd)
        self.rows = [(np.zeros((kv, 0, hd), np.uint8),) * 2 for _ in range(batch)]

    @property
    def stream(self):
        return torch.cuda.current_stream().cuda_stream

    def plan(self, fresh, rows, tokens_per_seq=0):
        from goml_b200 import block_glue as BG
        p = lambda x: x.data_ptr()   # noqa: E731
        BG.KVPagePlan(p(self.lens), p(fresh), p(self.table), p(self.ring), p(self.state), p(self.lens), p(self.state), p(self.taken), p(self.starts), p(self.positions), p(self.slots),
                      self.B, self.width, PAGE, self.n, rows, tokens_per_seq, self.stream)

    def prompts(self, lengths):
        self.plan(ints(lengths), sum(lengths))
        starts, slots = self.starts.tolist(), self.slots.long()
        for b, n in enumerate(lengths):
            if n:
                self.rows[b] = tuple(codes(self.r, (self.kv, n, self.hd)) for _ in range(2))
                at = slots[starts[b]:starts[b] + n]
                for x, y in zip((self.k, self.v), self.rows[b]):
                    x[at // PAGE, :, at % PAGE] = torch.from_numpy(y).cuda().transpose(0, 1)

    def fork(self, parent, keep=None):
        from goml_b200 import block_glue as BG
        p = lambda x: 0 if x is None else x.data_ptr()   # noqa: E731
        keep_d = None if keep is None else ints(keep)
        parent_d = ints(parent)
        gone = self.gone if self.window else None
        BG.KVPageFork(p(self.lens), p(parent_d), p(keep_d), p(self.table), p(self.ring), p(self.state), p(self.shares), p(gone), p(self.lens), p(self.state), p(self.shares),
                      p(gone), p(self.taken), p(self.copy_from), p(self.copy_to), p(self.copies), self.B, self.width, PAGE, self.n, self.sinks, self.stream)
        self.copy(self.B)
        before = list(self.rows)
        for b, (a, n) in enumerate(zip(parent, self.taken.tolist())):
            if n:
                self.rows[b] = tuple(x[:, :n].copy() for x in before[a])

    def copy(self, most):
        from goml_b200 import block_glue as BG
        BG.KVPageCopy([(self.k.data_ptr(), self.k.stride(0)), (self.v.data_ptr(), self.v.stride(0))], self.copy_from.data_ptr(), self.copy_to.data_ptr(), self.copies.data_ptr(), most,
                      self.n, self.stream)

    def release(self, keep=None):
        from goml_b200 import block_glue as BG
        p = lambda x: 0 if x is None else x.data_ptr()   # noqa: E731
        gone = self.gone if self.window else None
        BG.KVPageRelease(p(self.lens), p(keep), p(self.table), p(self.ring), p(self.state), p(self.shares), p(gone), p(self.lens), p(self.state), p(self.shares), p(gone), self.B,
                         self.width, PAGE, self.n, self.window, self.sinks, self.stream)

    def cut(self, keep):
        self.release(ints(keep))
        self.rows = [tuple(x[:, :max(n, 0)] for x in rows) for rows, n in zip(self.rows, keep)]

    def compact(self):
        from goml_b200 import block_glue as BG
        p = lambda x: x.data_ptr()   # noqa: E731
        BG.KVPageCompact(p(self.lens), p(self.table), p(self.ring), p(self.state), p(self.shares), p(self.table), p(self.ring), p(self.state), p(self.shares), p(self.moved),
                         p(self.copy_from), p(self.copy_to), p(self.copies), self.B, self.width, PAGE, self.n, self.stream)
        self.copy(self.copy_from.numel())

    def append(self, fresh):
        from goml_b200 import block_glue as BG
        p = lambda x: x.data_ptr()   # noqa: E731
        self.plan(fresh, self.B, 1)
        s = p(self.scales)
        BG.DecodeRopeAppend(p(self.qkv), p(self.cos), p(self.sin), p(self.positions), p(self.q), s, s + 4, p(self.k), p(self.v), s + 8, s + 12, self.B, self.hq, self.kv, self.hd, 0,
                            self.cos.shape[0], block_table=p(self.table), page_size=PAGE, max_pages_per_seq=self.width, num_pages=self.n, stream=self.stream)

    def token(self):
        """The next tokens' projections, and behind the append what they have become in the cache."""
        self.qkv.copy_(torch.from_numpy(self.r.normal(size=self.qkv.shape)).cuda())

    def appended(self):
        for b, slot in enumerate(self.slots[:self.B].tolist()):
            if slot >= 0:
                self.rows[b] = tuple(np.concatenate([x, c[slot // PAGE, :, slot % PAGE].cpu().numpy()[:, None]], 1) for x, c in zip(self.rows[b], (self.k, self.v)))

    def attend(self, how="all", shared=None, starts=None):
        s, pool = self.scales.data_ptr(), (self.stream, self.table.data_ptr(), PAGE, self.width, self.n)
        heads = (self.B, self.hq, self.kv, self.hd, 0)
        to = (self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.o.data_ptr(), self.lse.data_ptr(), self.lens.data_ptr())
        if how == "shared":
            self.fa.DecodeShared(*to, shared.data_ptr(), starts.data_ptr(), starts.numel() - 1, *heads, SCALE, 1.0, s, s + 8, s + 12, *pool)
        elif how == "window":
            self.fa.DecodeWindow(*to, *heads, 0, self.window, self.sinks, SCALE, 1.0, s, s + 8, s + 12, *pool)
        else:
            self.fa.Decode(*to, *heads, 0, SCALE, 1.0, s, s + 8, s + 12, *pool)

    def check(self):
        assert self.lens.tolist() == [x[0].shape[1] for x in self.rows]
        q, o, lse, scale = self.q.cpu().numpy(), self.o.double().cpu().numpy(), self.lse.double().cpu().numpy(), SCALE * float(self.scales[0]) * K_SCALE
        group = self.hq // self.kv
        for b, (k, v) in enumerate(self.rows):
            n = k.shape[1]
            seen = np.array([not self.window or j < self.sinks or j >= n - self.window for j in range(n)], bool)
            for h in range(self.kv):
                at = slice(h * group, (h + 1) * group)
                want, want_l, tol, tol_l = parts.attend(q[b, at], k[h], v[h], np.repeat(seen[None], group, 0), scale, V_SCALE)
                assert (np.abs(o[b, at] - want) <= tol).all(), (b, h, np.abs(o[b, at] - want).max())
                fine = ~np.isneginf(want_l)
                assert np.array_equal(np.isneginf(lse[b, at]), ~fine) and (np.abs(lse[b, at][fine] - want_l[fine]) <= tol_l[fine]).all()


@pytest.mark.parametrize("hd,kv,group", [(128, 2, 4), (64, 1, 8)])
@pytest.mark.parametrize("together", [False, True])
@pytest.mark.parametrize("graphed", [False, True])
def test_samples_of_prompts(fa_ctx, hd, kv, group, together, graphed):
    # two prompts, three answers to one and two to the other, of which one is cut back, one ends, and others go on in a pool made dense
    B, pages = 6, 24
    width = int((1.91e8 if hd == 128 else 1.01e8) / (3 * kv * hd * 2)) // PAGE + 2 if together else 8   # room for which common keys are read together, or each sequence its own
    s = Server(fa_ctx, B, kv, group, hd, pages, width, hd + kv)
    s.prompts([150, 0, 0, 128, 0, 0])
    s.fork([-1, 0, 0, -1, 3, -1])
    assert s.taken.tolist() == [0, 150, 150, 0, 128, 0] and s.shares.sum() == 6
    starts, shared = ints([0, 3, 5, 6]), ints([150, 150, 150, 128, 128, 0])
    fresh = ints([1, 1, 1, 1, 1, 0])

    def step():
        s.append(fresh)
        s.attend("shared", shared, starts)

    run = step
    if graphed:
        saved = [x.clone() for x in (s.table, s.lens, s.ring, s.state, s.k, s.v)]
        step()
        torch.cuda.synchronize()
        for x, y in zip((s.table, s.lens, s.ring, s.state, s.k, s.v), saved):
            x.copy_(y)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            step()
        run = g.replay

    def steps(n):
        for _ in range(n):
            s.token()
            run()
            s.appended()
            s.check()

    steps(3)
    s.cut([152, 153, 151, 0, 131, 0])     # drafted tokens go, and an answer ends whose first pages another one has
    starts.copy_(ints([0, 3, 3, 6]))
    shared.copy_(ints([150, 150, 150, 0, 0, 0]))
    fresh.copy_(ints([1, 1, 1, 0, 1, 0]))
    steps(2)
    s.attend()
    before = s.o.clone(), s.lse.clone()
    s.compact()
    used = s.n - int(s.state[1])
    assert used == len({p for b, n in enumerate(s.lens.tolist()) for p in s.table[b, :-(-n // PAGE)].tolist()}) and s.table.max() < used
    s.attend()
    assert torch.equal(s.o, before[0]) and torch.equal(s.lse, before[1])    # the same keys in other places
    s.fork([-1, -1, -1, 2, -1, 4], [0, 0, 0, 100, 0, 1000])     # answers that begin anew from others' middle
    shared.copy_(ints([150, 150, 150, 0, 0, 0]))
    fresh.copy_(ints([1] * 6))
    steps(70)                            # over the end of pages
    s.cut([0] * 6)
    assert int(s.state[1]) == s.n and not s.shares.any()
    s.fa.DeviceStatus()


@pytest.mark.parametrize("window,sinks", [(100, 4), (64, 0), (1, 70)])
def test_windows_that_move_on(fa_ctx, window, sinks):
    # a prompt's last row is what the decode call gives; pages that a window has passed go back and are written over by others
    B, kv, hd, n = 3, 2, 128, 333
    s = Server(fa_ctx, B, kv, 1, hd, 26, 16, 9, sinks, window)
    s.prompts([n] * B)
    q = torch.from_numpy(codes(s.r, (B * kv, n, hd), 60.0)).cuda()
    k, v = (torch.from_numpy(np.stack([rows[i] for rows in s.rows]).reshape(B * kv, n, hd)).cuda() for i in range(2))
    o, lse = torch.zeros((B * kv, n, hd), dtype=torch.float16, device="cuda"), torch.zeros((B * kv, n), device="cuda")
    s.scales[0] = 0.012
    p = s.scales.data_ptr()
    fa_ctx.ForwardSinks(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), B * kv, n, hd, window, sinks, SCALE, 1.0, p, p + 8, p + 12, s.stream)
    s.release()
    s.q.copy_(q[:, -1].reshape(s.q.shape))
    s.attend("window")
    s.check()
    s.o.copy_(o[:, -1].reshape(s.o.shape))
    s.lse.copy_(lse[:, -1].reshape(s.lse.shape))
    s.check()
    fresh = ints([1, 0, 1])
    held = -(-sinks // PAGE) + -(-window // PAGE) + 1
    for step in range(150):
        if step == 20:
            s.cut([s.rows[0][0].shape[1] - 3, 0, s.rows[2][0].shape[1]])
            s.fork([-1, 2, -1])
            assert s.taken.tolist()[1] == s.rows[2][0].shape[1]
            fresh = ints([1, 1, 1])
        s.token()
        s.append(fresh)
        s.appended()
        s.attend("window")
        if step % 10 == 0 or 18 < step < 23:
            s.check()
        s.release()
        free = s.ring[(torch.arange(int(s.state[1]), device="cuda") + s.state[0]) % s.n].long()
        s.k[free], s.v[free] = 127, 127     # anything may be there
        assert s.n - len(free) <= B * held
    s.check()
    s.cut([0] * B)
    assert int(s.state[1]) == s.n and not s.shares.any()
    s.fa.DeviceStatus()


def test_forked_sequences_of_a_block(cuda, built_libs):
    # the block's steps on pages that sequences have in common give what they give where each has had the prompt itself
    from goml_b200 import nn
    B, d, H, Fh, S = 3, 256, 4, 704, 100
    blk, _, _, _, t = _make_block("fp4fork", d, H, Fh)
    x = t(O.seeded_normal("x", (S, d), config="fp4fork")).repeat(B, 1)
    outs, free = [], []
    for forked in (False, True):
        pages = nn.KVPages(B, 9, 64, 3, shared=True)
        pools = [nn.FP4KVPool(pages, H, d // H) for _ in range(2)]
        pages.plan(ints([S, 0, 0]) if forked else S, tokens_per_seq=S)
        for pool in pools:
            blk(x, B, S, pool)
        if forked:
            pages.fork(ints([-1, 0, 0]), pools)
            assert pages.forked.tolist() == [0, S, S] and int(pages.state[1]) == 5
        got = []

        def step(fresh, seed):
            pages.plan(ints(fresh), tokens_per_seq=1)
            y = t(O.seeded_normal(f"t{seed}", (B, d), config="fp4fork"))
            for pool in pools:
                y = blk.decode_step(y, pool)
            got.append(y.clone())

        for i in range(4):
            step([1, 1, 1], i)
        pages.release(ints([S + 4, S + 1, S + 4]))
        step([-1, 1, 1], 4)                 # the parent ends
        assert pages.lens.tolist() == [0, S + 2, S + 5]
        pages.compact(pools)
        free.append(int(pages.state[1]))
        for i in range(30):                 # over a page's end
            step([0, 1, 1], 5 + i)
        assert pages.lens.tolist() == [0, S + 32, S + 35]
        outs.append(got)
        if forked:
            pages.release(ints([0, 30, 10 ** 6]))    # into the page that both have: no token may go there
            pages.plan(1, tokens_per_seq=1)
            assert pages.taken.tolist() == [1, 0, 1] and pages.lens.tolist() == [1, 30, S + 36]
            pages.plan(ints([-1, 0, 0]), tokens_per_seq=1)
            pages.fork(ints([1, -1, -1]), pools)
            pages.plan(1, tokens_per_seq=1)
            assert pages.taken.tolist() == [1, 0, 1] and pages.lens.tolist() == [31, 30, S + 37]
            pages.plan(-1, tokens_per_seq=1)
            assert int(pages.state[1]) == 9 and not pages.shares.any()
    for a, b in zip(*outs):
        assert torch.equal(a[1:], b[1:])
    assert free == [5, 6]
    blk.fa.DeviceStatus()
    blk.close()


class WindowServer(Server):
    """A server that tells a fork of the window which its sequences have."""

    def fork(self, parent, keep=None):
        from goml_b200 import block_glue as BG
        whole = BG.KVPageFork
        BG.KVPageFork = lambda *a: whole(*a, window=self.window)
        try:
            super().fork(parent, keep)
        finally:
            BG.KVPageFork = whole


def test_copies_of_windowed_sequences_have_what_they_see(fa_ctx):
    # a parent of 1000 keys has pages 0 and from 12 on; copies of its first keys are attended to, with anything in the pages that are free
    window, sinks, keeps = 200, 4, [0, 1000, 968, 967, 966, 800, 768, 200, 65, 64, 30]
    s = WindowServer(fa_ctx, len(keeps), 2, 2, 128, 40, 16, 21, sinks, window)
    s.prompts([1000] + [0] * 10)
    s.release()
    assert s.gone.tolist()[0] == 12
    s.fork([-1] + [0] * 10, keeps)
    assert s.taken.tolist() == [0, 1000, 968, 967, 0, 0, 0, 0, 0, 64, 30]
    for _ in range(3):
        free = s.ring[(torch.arange(int(s.state[1]), device="cuda") + s.state[0]) % s.n].long()
        s.k[free], s.v[free] = 127, 127
        s.token()
        s.append(ints([1] * 4 + [0] * 5 + [1] * 2))
        s.appended()
        s.attend("window")
        s.check()
        s.release()
    s.fork([-1] * 4 + [1] * 5 + [-1] * 2, [0] * 4 + [1003, 1002, 900, 967, 64] + [0] * 2)    # places that were not taken are empty still
    assert s.taken.tolist() == [0, 0, 0, 0, 1003, 1002, 0, 967, 64, 0, 0]
    s.token()
    s.append(ints([1] * 6 + [0] + [1] * 4))
    s.appended()
    s.attend("window")
    s.check()
    s.cut([0] * 11)
    assert int(s.state[1]) == s.n and not s.shares.any()
    s.fa.DeviceStatus()
