"""Page calls of 2^31 - 1 pages and of as many sequences, the most that they take: steps and sums go past the last one."""
import pytest
import torch

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def room(words):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 4 * words + (4 << 30):
        pytest.skip("not enough memory free")


def stream():
    return torch.cuda.current_stream().cuda_stream


def at(*tensors):
    return [0 if x is None else x.data_ptr() for x in tensors]


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def test_the_most_pages(cuda, built_libs):
    from goml_b200 import block_glue as BG
    room(5 * MOST)
    n = MOST
    # pages 0, 5, n - 2 and n - 1 are in use, all others in the ring
    lens, table, state = ints([2, 2, 0]), ints([[n - 1, 5, -1], [0, n - 2, -1], [-1, -1, -1]]), ints([0, n - 4, 0, 0])
    ring = torch.empty(n, dtype=torch.int32, device="cuda")
    ring[:4] = ints([1, 2, 3, 4])
    torch.arange(6, n - 2, dtype=torch.int32, device="cuda", out=ring[4:n - 4])
    ring[n - 4:] = -1
    shares, other = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
    # a copy of the first, with the new shares elsewhere
    taken, frm, to, copies = ints([0] * 3), torch.full((n // 2 + 9,), -7, dtype=torch.int32, device="cuda"), torch.full((n // 2 + 9,), -7, dtype=torch.int32, device="cuda"), ints([9])
    shares[n - 3] = 4
    other.fill_(-5)
    BG.KVPageFork(*at(lens, ints([-1, -1, 0]), None, table, ring, state, shares, None, lens, state, other, None, taken, frm, to, copies), 3, 3, 1, n, 0, stream())
    assert taken.tolist() == [0, 0, 2] and table.tolist()[2] == [n - 1, 5, -1] and copies.item() == 0 and state.tolist()[:2] == [0, n - 4]
    assert other[5] == 1 and other[n - 1] == 1 and other[n - 3] == 4 and torch.count_nonzero(other) == 3
    shares[n - 3] = 0
    shares[5] = shares[n - 1] = 1
    moved = other.fill_(-9)
    BG.KVPageCompact(*at(lens, table, ring, state, shares, table, ring, state, shares, moved, frm, to, copies), 3, 3, 1, n, stream())
    assert copies.item() == 3 and frm[:4].tolist() == [5, n - 2, n - 1, -7] and to[:4].tolist() == [1, 2, 3, -7]
    assert table.tolist() == [[3, 1, -1], [0, 2, -1], [3, 1, -1]] and state.tolist()[:2] == [0, n - 4]
    assert moved[ints([0, 5, n - 2, n - 1]).long()].tolist() == [0, 1, 2, 3] and torch.count_nonzero(moved.add_(1)) == 4
    assert shares[:4].tolist() == [0, 1, 0, 1] and torch.count_nonzero(shares) == 2
    assert ring[n - 5:].tolist() == [n - 1, -1, -1, -1, -1]
    assert torch.equal(ring[:n - 4], torch.arange(4, n, dtype=torch.int32, device="cuda", out=moved[:n - 4]))
    del moved
    BG.KVPageRelease(*at(lens, ints([0, 0, 0]), table, ring, state, shares, None, lens, state, shares, None), 3, 3, 1, n, 0, 0, stream())
    assert lens.tolist() == [0, 0, 0] and state.tolist()[:2] == [0, n] and not shares.any()
    assert ring[n - 5:].tolist() == [n - 1, 0, 1, 2, 3] and torch.equal(ring[:n - 4], torch.arange(4, n, dtype=torch.int32, device="cuda", out=other[:n - 4]))
    # a full ring, and shares that say of every page that nobody has it any more: there is no room for any
    shares.fill_(-1)
    BG.KVPageRelease(*at(lens, None, table, ring, state, shares, None, lens, state, shares, None), 3, 3, 1, n, 0, 0, stream())
    assert state.tolist()[:2] == [0, n] and not shares.any() and torch.equal(ring[:n - 4], other[:n - 4]) and ring[n - 4:].tolist() == [0, 1, 2, 3]


def test_the_most_sequences(cuda, built_libs):
    from goml_b200 import block_glue as BG
    room(7 * MOST)
    n, pages = MOST, 8
    lens, taken, frm, to = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(4))
    parent, table = (torch.full((n,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    ring, state, shares, copies = ints(list(range(pages))), ints([1, 6, 0, 0]), ints([0] * pages), ints([9])   # pages 0 and 7 are in use
    # the first has a full page and the second one that is not; the last two become their copies
    lens[:2], table[:2] = ints([2, 1]), ints([7, 0])
    parent[n - 2:] = ints([0, 1])
    frm.fill_(-7)
    to.fill_(-7)
    BG.KVPageFork(*at(lens, parent, None, table, ring, state, shares, None, lens, state, shares, None, taken, frm, to, copies), n, 1, 2, pages, 0, stream())
    assert lens[n - 3:].tolist() == [0, 2, 1] and taken[n - 3:].tolist() == [0, 2, 1] and torch.count_nonzero(taken) == 2 and torch.count_nonzero(lens) == 4
    assert table[n - 3:].tolist() == [-1, 7, 1] and shares.tolist() == [0] * 7 + [1] and state.tolist()[:2] == [2, 5]
    assert copies.item() == 1 and frm[:2].tolist() == [0, -7] and to[:2].tolist() == [1, -7]
    keep = taken.fill_(MOST)
    keep[0] = 0
    keep[n - 1] = 0
    BG.KVPageRelease(*at(lens, keep, table, ring, state, shares, None, lens, state, shares, None), n, 1, 2, pages, 0, 0, stream())
    assert lens[n - 3:].tolist() == [0, 2, 0] and lens[:2].tolist() == [0, 1] and torch.count_nonzero(lens) == 2
    assert shares.tolist() == [0] * 8 and state.tolist()[:2] == [2, 6] and ring.tolist() == [0, 1, 2, 3, 4, 5, 6, 1]
