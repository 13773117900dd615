"""fa_decode_window, fa_decode_shared, fa_forward_sinks and the pages' sharing of nn, without a GPU: refusals, what is launched where, and the restatement against the formula."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from goml_b200 import fa_forward as F, nn
from oracle import e4m3_decode, parts
from tests.parts_util import codes
from tests.test_fp4_pool_cpu import CPU, current, ints, planned   # noqa: F401


def test_entries_refuse_what_has_no_context(built_libs):
    lib = F.FALoad()
    block = C.create_string_buffer(256)
    assert lib.fa_decode_window(None, block, 1, 1) == F.FA_ERR_INVALID_ARG
    assert lib.fa_decode_shared(None, block, None, None, 1) == F.FA_ERR_INVALID_ARG
    assert lib.fa_forward_sinks(None, block, 1) == F.FA_ERR_INVALID_ARG
    ctx = F.FAContext(0)
    with pytest.raises(F.FAError, match="DecodeWindow"):
        ctx.DecodeWindow(1, 1, 1, 1, 0, 1, 1, 1, 1, 64, 64, 0, 1, 0, 1.0)
    with pytest.raises(F.FAError, match="DecodeShared"):
        ctx.DecodeShared(1, 1, 1, 1, 0, 1, 1, 1, 1, 1, 1, 1, 64, 64, 1.0)
    with pytest.raises(F.FAError, match="ForwardSinks"):
        ctx.ForwardSinks(1, 1, 1, 1, 0, 1, 64, 64, 16, 4, 1.0)


@pytest.mark.parametrize("rows,keys,hd", [(1, 1, 64), (3, 200, 128), (2, 0, 64)])
def test_the_restatement_is_the_softmax(rows, keys, hd):
    r = np.random.default_rng(rows + keys)
    q, k, v = codes(r, (rows, hd)), codes(r, (keys, hd)), codes(r, (keys, hd))
    seen = r.random((rows, keys)) < 0.6
    if rows > 1:
        seen[1] = False
    o, lse, tol, tol_l = parts.attend(q, k, v, seen, 0.001, 0.5)
    x = np.where(seen, 0.001 * (e4m3_decode(q).astype(float) @ e4m3_decode(k).astype(float).T), -np.inf)
    for i in range(rows):
        if not seen[i].any():
            assert not o[i].any() and np.isneginf(lse[i])
            continue
        w = np.exp(x[i] - np.log(np.exp(x[i][seen[i]]).sum()))
        assert np.allclose(o[i], 0.5 * w @ e4m3_decode(v).astype(float), rtol=1e-12, atol=1e-12) and np.isclose(lse[i], np.log(np.exp(x[i][seen[i]]).sum()), rtol=1e-12)
        # the sum of magnitudes of a score is at most hd times the largest factors
        size = 0.001 * hd * float(np.abs(e4m3_decode(q[i])).max()) * float(np.abs(e4m3_decode(k)).max())
        e = 2 * (2.0 ** -22 + (hd * 2.0 ** -23 + 2.0 ** -22) * size) + 2.0 ** -17
        largest = 0.5 * float(np.abs(e4m3_decode(v)).max())
        assert (tol[i] > 0).all() and (tol[i] <= largest * (2.0 ** -10 + 2 * e + keys * 2.0 ** -25) + 2.0 ** -25).all() and 0 < tol_l[i] <= 2 * e + 2.0 ** -22 * (1 + abs(lse[i]))


@pytest.fixture
def changes(planned, monkeypatch):   # noqa: F811
    """What KVPages hands to the calls that share, free and move pages, with the device that is current."""
    calls = []
    for name, numbers in (("KVPageFork", slice(16, None)), ("KVPageRelease", slice(11, None)), ("KVPageCompact", slice(13, None)), ("KVPageCopy", slice(0, None))):
        monkeypatch.setattr(nn.BG, name, lambda *a, name=name, numbers=numbers: calls.append((name, current[-1], a[numbers], a)))
    return calls


def test_pages_that_are_not_shared_do_not_fork(changes):
    pages = nn.KVPages(2, 8, 64, 3, device="cpu")
    with pytest.raises(ValueError, match="fork: .*shared=False"):
        pages.fork(torch.zeros(2, dtype=torch.int32), [])
    with pytest.raises(ValueError, match="release: .*shared=False"):
        pages.release(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="compact: .*shared=False"):
        pages.compact([])
    pages.plan(1)
    assert not changes


def test_sharing_calls(changes):
    stream = ("stream of", CPU)
    pages = nn.KVPages(2, 9, 64, 3, device="cpu", shared=True)
    pools = [nn.FP4KVPool(pages, 2, hd) for hd in (64, 128)]
    parent = torch.tensor([-1, 0], dtype=torch.int32)
    for bad in (parent.long(), parent[:1], torch.zeros(4, dtype=torch.int32)[::2], parent.to("meta")):
        with pytest.raises(ValueError, match="KVPages.fork: needs 2 int32"):
            pages.fork(bad, pools)
        with pytest.raises(ValueError, match="KVPages.fork: needs 2 int32"):
            pages.fork(parent, pools, keep=bad)
        with pytest.raises(ValueError, match="KVPages.release: needs 2 int32"):
            pages.release(bad)
    other = nn.FP4KVPool(nn.KVPages(2, 9, 64, 3, device="cpu", shared=True), 2, 64)
    for call in (lambda: pages.fork(parent, [other]), lambda: pages.compact([*pools, other])):
        with pytest.raises(ValueError, match="the pools must be of these pages"):
            call()
    assert not changes
    pages.fork(parent, iter(pools))
    pages.compact(pools)
    pages.release(parent)
    pages.fork(parent, [])       # no pool, no copy
    names = [c[0] for c in changes]
    assert names == ["KVPageFork", "KVPageCopy", "KVPageCompact", "KVPageCopy", "KVPageRelease", "KVPageFork"]
    assert all(c[1] == CPU for c in changes) and current == ["another device"]
    assert changes[0][2] == (2, 3, 64, 9, 0, stream) and changes[2][2] == (2, 3, 64, 9, stream) and changes[4][2] == (2, 3, 64, 9, 0, 0, stream)
    bytes_of = lambda pool, hd: [(t.data_ptr(), 2 * 64 * n) for t, n in ((pool.k, hd // 2), (pool.v, hd // 2), (pool.ks, hd // 16), (pool.vs, hd // 16))]   # noqa: E731
    for i, most in ((1, 2), (3, pages._from.numel())):
        assert changes[i][3][0] == bytes_of(pools[0], 64) + bytes_of(pools[1], 128) and changes[i][3][4:] == (most, 9, stream)
    assert pages._from.numel() >= 9 // 2


def test_ends_go_through_release_and_cut_sequences_wait(changes, planned):   # noqa: F811
    pages = nn.KVPages(5, 16, 64, 3, device="cpu", shared=True)
    keeps = []
    release = nn.BG.KVPageRelease
    nn.BG.KVPageRelease = lambda *a: (keeps.append(ints(a[1], 5)), release(*a))
    pages.lens.copy_(torch.tensor([30, 64, 70, 192, 0]))
    pages.table.copy_(torch.tensor([[7, -1, -1], [7, -1, -1], [7, 3, -1], [7, 8, 9], [-1, -1, -1]]))
    pages.shares[7] = 3
    pages.plan(torch.tensor([1, 1, 1, -1, 1], dtype=torch.int32), tokens_per_seq=1)
    assert keeps == [[0x7fffffff] * 3 + [0, 0x7fffffff]]
    assert planned[-1]["fresh"] == [0, 1, 1, -1, 1]     # the first was cut back into page 7; the last is empty


CPP = r"""
#include <cstdio>
#include "../../goml_b200/host/goml_cuda.hpp"
using namespace goml::cuda;
template <class F> static std::string thrown(F f) { try { f(); return ""; } catch (const std::exception& e) { return e.what(); } }
int main() {
    std::puts(thrown([] { kv_page_fork_args_t a{}; a.batch = 1; KVPageFork(a); }).c_str());
    std::puts(thrown([] { kv_page_release_args_t a{}; a.batch = 1; KVPageRelease(a); }).c_str());
    std::puts(thrown([] { kv_page_compact_args_t a{}; a.batch = 1; KVPageCompact(a); }).c_str());
    std::puts(thrown([] { kv_page_copy_args_t a{}; a.num_pools = 1; a.most = 1; KVPageCopy(a); }).c_str());
    void (FAContext::*window)(const fa_decode_args_t&, int, int) = &FAContext::DecodeWindow;
    void (FAContext::*shared)(const fa_decode_args_t&, uintptr_t, uintptr_t, int) = &FAContext::DecodeShared;
    void (FAContext::*sinks)(const fa_forward_args_t&, int) = &FAContext::ForwardSinks;
    return window == nullptr || shared == nullptr || sinks == nullptr;
}
"""


def test_cpp_host_layer(tmp_path, built_libs):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    host = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_cpp")
    exe = str(tmp_path / "parts_host")
    r = subprocess.run(["g++", "-std=c++17", "-I", os.path.join(cuda, "include"), "-iquote", host, "-x", "c++", "-", "-o", exe, "-L", os.path.join(cuda, "lib64"), "-lcudart", "-ldl",
                        "-lpthread"], input=CPP, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, env=dict(os.environ, GOML_LIBS_DIR=built_libs))
    lines = r.stdout.splitlines()
    assert r.returncode == 0 and len(lines) == 4, (r.returncode, r.stdout, r.stderr)
    assert all(name in line for name, line in zip(("kv_page_fork", "kv_page_release", "kv_page_compact", "kv_page_copy"), lines)), lines


def test_go_layer_names_every_entry():
    # no Go here: what its files load is what the libraries' headers declare
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = "".join(open(os.path.join(root, "go", "backend", "cuda", f)).read() for f in ("fa_forward_b200.go", "fp8_block.go"))
    for name in ("fa_decode_window", "fa_decode_shared", "fa_forward_sinks", "kv_page_fork", "kv_page_release", "kv_page_compact", "kv_page_copy"):
        assert f', "{name}")' in text, name
