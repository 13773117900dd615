"""Pages that change hands, without a GPU: the restatement that the GPU tests compare with, and what the entry points refuse."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

from oracle import pages as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rows(*entries):
    return np.array(entries, np.int32)


def test_a_fork_shares_whole_pages_and_asks_for_a_copy_of_the_last():
    table = rows([5, 6, 7], [-1, -1, -1], [-1, -1, -1], [-1, -1, -1])
    ring = rows(*range(10))
    shares = np.zeros(10, np.int32)
    got = P.fork([40, 0, 0, 0], [-1, 0, 0, 0], [99, 32, 99, 99], table, ring, 8, 1, shares, None, 16)
    # the first is cut at a page's end and needs none; the second takes page 8; there is none for the third
    assert got["taken"] == [0, 32, 40, 0] and got["lens"] == [40, 32, 40, 0] and got["moves"] == [(7, 8)] and got["state"] == (9, 0)
    assert list(got["table"][1]) == [5, 6, -1] and list(got["table"][2]) == [5, 6, 8] and list(got["table"][3]) == [-1, -1, -1]
    assert list(got["shares"]) == [0, 0, 0, 0, 0, 2, 2, 0, 0, 0]


def test_a_page_is_free_when_nobody_has_it():
    table = rows([5, 6, 7], [5, 6, 8])
    shares = np.zeros(10, np.int32)
    shares[5] = shares[6] = 1
    got = P.release([40, 40], [0, 20], table, rows(*[-1] * 10), 9, 0, shares, None, 16)
    # the first ends, the second keeps two pages: 5 and 6 have one holder left
    assert got["lens"] == [0, 20] and got["state"] == (9, 2) and list(got["shares"]) == [0] * 10
    assert [got["ring"][9], got["ring"][0]] == [7, 8]


def test_a_window_gives_back_what_no_later_token_sees():
    table = rows([0, 1, 2, 3, 4])
    shares = np.zeros(5, np.int32)
    # 67 keys: token 67 sees 36 to 67 with a window of 32, pages of 16 from 32 on; page 0 holds the sinks
    got = P.release([67], None, table, rows(*[-1] * 5), 0, 0, shares, [0], 16, window=32, sinks=4)
    assert got["gone"] == [2] and got["state"] == (0, 1) and got["ring"][0] == 1
    again = P.release([67], None, table, got["ring"], 0, 1, got["shares"], got["gone"], 16, window=32, sinks=4)
    assert again["gone"] == [2] and again["state"] == (0, 1)
    ended = P.release([67], [0], table, again["ring"], 0, 1, again["shares"], again["gone"], 16, window=32, sinks=4)
    assert ended["gone"] == [0] and sorted(ended["ring"]) == [0, 1, 2, 3, 4]


def test_used_pages_become_the_first():
    table = rows([6, 1], [4, -1])
    got = P.compact([20, 16], table, rows(0, 2, 3, 5, -1, -1, -1), 0, 4, rows(0, 3, 0, 0, 1, 0, 2), 16)
    assert got["moves"] == [(4, 0), (6, 2)] and got["table"].tolist() == [[2, 1], [0, -1]] and got["state"] == (0, 4)
    assert got["ring"] == [3, 4, 5, 6, -1, -1, -1] and list(got["shares"]) == [1, 3, 2, 0, 0, 0, 0] and got["moved_to"] == [-1, 1, -1, -1, 0, -1, 2]


def structures():
    from goml_b200 import block_glue as BG
    return {"kv_page_fork_args_t": BG.KVPageForkArgs, "kv_page_release_args_t": BG.KVPageReleaseArgs, "kv_page_compact_args_t": BG.KVPageCompactArgs,
            "kv_page_pool_t": BG.KVPagePool, "kv_page_copy_args_t": BG.KVPageCopyArgs}


def test_structures_match_the_header(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("gcc not available")
    lines = [f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f}));' for f, _ in s._fields_) for n, s in structures().items()]
    src = tmp_path / "s.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "fp8_block.h"\nint main(void) {' + "\n".join(lines) + "return 0; }")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "s"), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [x for s in structures().values() for x in (C.sizeof(s), *(getattr(s, f).offset for f, _ in s._fields_))]


A = 1 << 20   # an address that no refused call looks at
FORK = dict(lens=A, parent=A, keep=A, block_table=A, ring=A, ring_state=A, shares=A, gone=A, lens_out=A, ring_state_out=A, shares_out=A, gone_out=A, taken=A, copy_from=A, copy_to=A,
            copies=A, batch=4, max_pages_per_seq=8, page_size=16, num_pages=32, sinks=0)
RELEASE = dict(lens=A, keep=A, block_table=A, ring=A, ring_state=A, shares=A, gone=A, lens_out=A, ring_state_out=A, shares_out=A, gone_out=A, batch=4, max_pages_per_seq=8, page_size=16,
               num_pages=32, window=0, sinks=0)
COMPACT = dict(lens=A, block_table=A, ring=A, ring_state=A, shares=A, block_table_out=A, ring_out=A, ring_state_out=A, shares_out=A, moved_to=A, copy_from=A, copy_to=A, copies=A, batch=4,
               max_pages_per_seq=8, page_size=16, num_pages=32)
COPY = dict(pools=[(A, 1024)], copy_from=A, copy_to=A, copies=A, most=3, num_pages=32)
SIZES = [dict(batch=-1), dict(max_pages_per_seq=0), dict(page_size=0), dict(num_pages=0), dict(page_size=1 << 28), dict(num_pages=1 << 28)]
OPTIONAL = {"keep", "gone", "gone_out"}


def bad_pointers(good):
    for name, value in good.items():
        if value == A:
            yield {name: A + 2}
            if name not in OPTIONAL:
                yield {name: 0}


def refusals():
    for entry, good in (("KVPageFork", FORK), ("KVPageRelease", RELEASE), ("KVPageCompact", COMPACT)):
        for bad in [*bad_pointers(good), *SIZES]:
            yield entry, good | bad
    for entry, good in (("KVPageFork", FORK), ("KVPageRelease", RELEASE)):
        yield entry, good | dict(gone=0)
        yield entry, good | dict(gone_out=0)
        yield entry, good | dict(sinks=-1)
    yield "KVPageRelease", RELEASE | dict(window=-1)
    yield "KVPageRelease", RELEASE | dict(window=5, gone=0, gone_out=0)
    for bad in [*bad_pointers(COPY), dict(most=-1), dict(num_pages=0), dict(pools=[(0, 1024)]), dict(pools=[(A + 8, 1024)]), dict(pools=[(A, 1032)]), dict(pools=[(A, 0)]),
                dict(pools=[(A, -16)]), dict(pools=[(A, 1 << 31)]), dict(pools=[(A, 1024)] * 70 + [(A + 4, 1024)])]:
        yield "KVPageCopy", COPY | bad


@pytest.mark.parametrize("entry,args", list(refusals()))
def test_refused(built_libs, entry, args):
    from goml_b200 import block_glue as BG
    with pytest.raises(BG.BlockGlueError, match="CUDA error 1$"):
        getattr(BG, entry)(**args)


def test_null_argument_blocks_are_refused(built_libs):
    lib = C.CDLL(os.path.join(built_libs, "libfp8block.so"))
    for name in ("kv_page_fork", "kv_page_release", "kv_page_compact", "kv_page_copy"):
        assert getattr(lib, name)(None) == 1


def test_nothing_to_copy_needs_no_gpu(built_libs):
    from goml_b200 import block_glue as BG
    BG.KVPageCopy(**COPY | dict(most=0))
    BG.KVPageCopy(**COPY | dict(pools=[]))


def test_a_copy_whose_window_sees_what_has_gone_is_not_taken():
    # every length that a windowed parent can be cut to: taken where the copy has each page of the keys that the next token sees, which are gone through one by one
    page, width = 4, 10
    for window in (1, 3, 4, 9, 12, 40):
        for sinks in (0, 1, 5):
            for n in range(0, 41, 3):
                table, ring, shares = rows(range(width), [-1] * width), rows(*range(20)), np.zeros(20, np.int32)
                free = P.release([n], None, table[:1], ring, 10, 10, shares, [0], page, window, sinks)
                gone = free["gone"][0]
                for keep in range(n + 1):
                    got = P.fork([n, 0], [-1, 0], [0, keep], table, free["ring"], *free["state"], free["shares"], [gone, 0], page, sinks, window)
                    seen = [j for j in range(keep) if j < sinks or j >= keep + 1 - window]
                    if keep % page:
                        seen.append(keep - 1)      # the page that the next token goes to
                    taken = all(j // page < -(-sinks // page) or j // page >= gone for j in seen)
                    assert got["taken"] == [0, keep if taken else 0] and (taken or got["lens"] == [n, 0]), (window, sinks, n, keep)
                    if taken:
                        assert all(got["table"][1, j // page] >= 0 for j in seen) and len(got["moves"]) == (keep % page > 0)


@pytest.mark.parametrize("window", [-1, -2 ** 31])
def test_a_fork_refuses_windows_below_zero(built_libs, window):
    from goml_b200 import block_glue as BG
    with pytest.raises(BG.BlockGlueError, match="CUDA error 1$"):
        BG.KVPageFork(**FORK, window=window)


def test_cut_sequences_that_lack_what_their_window_sees_are_told_by_gone():
    # the header's rule, for every length that a windowed sequence can be cut back to
    page, width = 4, 10
    lacking = 0
    for window in (1, 3, 4, 9, 12, 40):
        for sinks in (0, 1, 5):
            for n in range(0, 41, 3):
                table, ring, shares = rows(range(width)), rows(*range(20)), np.zeros(20, np.int32)
                once = P.release([n], None, table, ring, 10, 10, shares, [0], page, window, sinks)
                for keep in range(n + 1):
                    cut = P.release([n], [keep], table, once["ring"], *once["state"], once["shares"], once["gone"], page, window, sinks)
                    m, gone, first = cut["lens"][0], cut["gone"][0], -(-sinks // page)
                    seen = [j for j in range(m) if j < sinks or j >= m + 1 - window] + ([m] if m % page else [])
                    has = all(j // page < first or j // page >= gone for j in seen)
                    assert m == keep and has == (not (gone > first and gone > max(m + 1 - window, 0) // page)), (window, sinks, n, keep)
                    lacking += not has
    assert lacking > 100
