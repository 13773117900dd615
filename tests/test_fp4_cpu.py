"""The 4-bit KV cache and the page plan without a GPU: what their entry points refuse, and the restatement that the GPU tests compare with."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

from oracle import fp4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_grid_of_codes():
    # to nearest, halfway to the even code, saturating; signs kept
    y = np.zeros((1, 16), np.float32)
    y[0] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, 0.26, 5.01, -6, 0.2, -5, 2.49]
    b, c = fp4.quantise(y, 1.0)
    assert fp4.E4M3[b[0, 0]] == 1.0
    assert list(c[0, 0]) == [7, 0, 2, 2, 4, 4, 6, 6, 8, 10, 1, 7, 15, 0, 14, 4]
    assert list(fp4.values(fp4.pack(c), b, 1.0)[0]) == [6, 0, 1, 1, 2, 2, 4, 4, -0.0, -1, 0.5, 6, -6, 0, -4, 2]


def test_block_scales():
    assert len(fp4.E4M3) == 127 and fp4.E4M3[126] == 448 and fp4.E4M3[1] == 2.0 ** -9 and fp4.E4M3[0x38] == 1
    y = np.zeros((4, 16), np.float32)
    y[:, 3] = [6 * 448 * 2, 6 * 1.0625, 6 * 1.1875, 6 * 2.0 ** -10]   # saturates; halfway between 1 and 1.125 (even: 1), and 1.125 and 1.25 (1.25); half the least one
    b, c = fp4.quantise(y, 1.0)
    assert [fp4.E4M3[x] for x in b[:, 0]] == [448, 1, 1.25, 0]
    assert c[0, 0, 3] == 7 and not c[3].any()
    y[1, 5], y[2, 5] = np.nan, np.inf
    b, c = fp4.quantise(y, 1.0)
    assert b[1, 0] == 0x7F and fp4.E4M3[b[2, 0]] == 448 and c[2, 0, 5] == 7
    assert np.isnan(fp4.values(fp4.pack(c), b, 1.0)[1]).all()


def test_a_value_is_off_by_at_most_half_a_code():
    # nearest code: half of the widest step (2 of 6) of the block scale, which itself lies within 2^-4 of max / 6 (or at 448)
    r = np.random.default_rng(3)
    y = r.normal(size=(500, 128)).astype(np.float32)
    s = np.float32(np.abs(y).max() / (6 * 448))
    b, c = fp4.quantise(y, s)
    top = np.abs(y).reshape(500, 8, 16).max(-1)
    err = np.abs(fp4.values(fp4.pack(c), b, s) - y).reshape(500, 8, 16).max(-1)
    assert (err <= top / 6 * (1 + 2.0 ** -4) + top * 2.0 ** -4).all()


def test_scale_orders():
    x = np.arange(2 * 48 * 4, dtype=np.uint8).reshape(2, 48, 4)
    y = fp4.blocks_of_16(x)
    assert y.shape == (2, 3, 4, 16) and y[1, 2, 3, 5] == x[1, 37, 3] and np.array_equal(fp4.natural(y), x)


def test_the_plan_one_sequence_at_a_time():
    table = np.full((4, 3), -1, np.int32)
    table[0, 0], table[1, :2] = 9, (5, 6)
    ring = np.array([-7, -7, -7, -7, -7, -7, -7, -7, 3, 4], np.int32)
    got = fp4.plan([16, 20, 0, 0], [1, -1, 40, 5], table, ring, 8, 2, 16, 60)
    # the first takes page 3; the third needs three pages and there is one: it waits, and so does all behind it that needs a page
    assert list(got["taken"]) == [1, 0, 0, 0] and list(got["lens"]) == [17, 0, 0, 0] and list(got["starts"]) == [0, 1, 1, 41, 46]
    assert got["table"][0, 1] == 3 and got["slots"][0] == 48 and got["positions"][0] == 16 and (got["slots"][1:] == -1).all()
    assert got["state"] == (9, 3) and list(got["ring"][:2]) == [5, 6]


def _lib(built_libs):
    return C.CDLL(os.path.join(built_libs, "libfp8block.so"))


def test_structures_match_the_header(tmp_path):
    from goml_b200 import block_glue as BG, fa_forward as F
    if not shutil.which("gcc"):
        pytest.skip("gcc not available")
    structs = {"fp4_append_args_t": BG.FP4AppendArgs, "fp4_rows_args_t": BG.FP4RowsArgs, "kv_page_plan_args_t": BG.KVPagePlanArgs, "fa_decode_fp4_args_t": F.DecodeFP4Args}
    lines = [f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f}));' for f, _ in s._fields_) for n, s in structs.items()]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "fp8_block.h"\nint main(void) {' + "\n".join(lines) + "return 0; }")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "s"), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [x for s in structs.values() for x in (C.sizeof(s), *(getattr(s, f).offset for f, _ in s._fields_))]


APPEND = dict(qkv_bf16=4096, cos_tab=4096, sin_tab=4096, positions=4096, slots=4096, q_out=4096, k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096, k_scale=4096,
              v_scale=4096, tokens=4, q_heads=8, kv_heads=2, head_dim=128, rope_rows=64, page_size=64, num_pages=10)


@pytest.mark.parametrize("bad", [dict(qkv_bf16=0), dict(qkv_bf16=4104), dict(q_out=4104), dict(cos_tab=0), dict(sin_tab=4098), dict(positions=0), dict(slots=4097), dict(k_codes=0),
                                 dict(k_scales=4100), dict(v_codes=4104), dict(v_scales=0), dict(k_scale=0), dict(v_scale=4097), dict(tokens=-1), dict(q_heads=0), dict(kv_heads=0),
                                 dict(head_dim=96), dict(rope_rows=0), dict(page_size=0), dict(page_size=24), dict(num_pages=0), dict(page_size=1 << 20, num_pages=1 << 12),
                                 dict(tokens=1 << 30), dict(q_heads=1 << 30)])
def test_append_refuses(built_libs, bad):
    from goml_b200 import block_glue as BG
    with pytest.raises(BG.BlockGlueError, match="fp4_rope_append: CUDA error 1$"):
        BG.FP4RopeAppend(**{**APPEND, **bad})


def test_nothing_to_append(built_libs):
    from goml_b200 import block_glue as BG
    BG.FP4RopeAppend(**{**APPEND, "tokens": 0, "q_out": 0})
    assert _lib(built_libs).fp4_rope_append(None) == 1


ROWS = dict(slots=4096, k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096, k_scale=4096, v_scale=4096, k_out=4096, v_out=4096, tokens=4, kv_heads=2, head_dim=64,
            page_size=16, num_pages=10)


@pytest.mark.parametrize("bad", [dict(slots=0), dict(slots=4098), dict(k_codes=0), dict(k_scales=4104), dict(v_codes=0), dict(v_scales=0), dict(k_scale=0), dict(v_scale=0), dict(k_out=0),
                                 dict(v_out=4104), dict(tokens=-1), dict(kv_heads=0), dict(head_dim=32), dict(page_size=8), dict(num_pages=-1), dict(tokens=1 << 30)])
def test_rows_refuse(built_libs, bad):
    from goml_b200 import block_glue as BG
    with pytest.raises(BG.BlockGlueError, match="fp4_cache_rows: CUDA error 1$"):
        BG.FP4CacheRows(**{**ROWS, **bad})
    BG.FP4CacheRows(**{**ROWS, "tokens": 0})


PLAN = dict(lens=4096, fresh=4096, block_table=4096, ring=4096, ring_state=4096, lens_out=4096, ring_state_out=4096, taken=4096, starts=4096, positions=4096, slots=4096,
            batch=4, max_pages_per_seq=3, page_size=64, num_pages=20, rows=8)


@pytest.mark.parametrize("bad", [{n: 0} for n in ("lens", "fresh", "block_table", "ring", "ring_state", "lens_out", "ring_state_out", "taken", "starts", "positions", "slots")]
                         + [dict(lens=4098), dict(slots=4097), dict(batch=-1), dict(max_pages_per_seq=0), dict(page_size=0), dict(num_pages=0), dict(rows=-1), dict(tokens_per_seq=-1),
                            dict(tokens_per_seq=3), dict(page_size=1 << 20, max_pages_per_seq=1 << 12), dict(page_size=1 << 20, num_pages=1 << 12)])
def test_plan_refuses(built_libs, bad):
    from goml_b200 import block_glue as BG
    with pytest.raises(BG.BlockGlueError, match="kv_page_plan: CUDA error 1$"):
        BG.KVPagePlan(**{**PLAN, **bad})


def test_decode_without_a_context(built_libs):
    from goml_b200 import fa_forward as F
    assert F.FALoad().fa_decode_fp4(None, None) == F.FA_ERR_INVALID_ARG
    with pytest.raises(F.FAError, match="FAContext.DecodeFP4: nil ctx"):
        F.FAContext(0).DecodeFP4(16, 16, 16, 16, 16, 16, 0, 0, 1, 1, 1, 64, 64, 64, 1.0)


DECODE = dict(q=4096, k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096, o=4096, lOut=0, seq_lens=4096, batch=2, q_heads=4, kv_heads=2, hd=64, s_max=48, seq_len=0, scale=1.0)
PAGED = dict(block_table=4096, page_size=64, max_pages_per_seq=3, num_pages=9)


@pytest.mark.parametrize("bad,status", [
    (dict(q=0), 1), (dict(k_codes=0), 1), (dict(k_scales=0), 1), (dict(v_codes=0), 1), (dict(v_scales=0), 1), (dict(o=0), 1), (dict(batch=0), 1), (dict(q_heads=0), 1), (dict(kv_heads=-1), 1),
    (dict(hd=96), 3), (dict(q_heads=5), 4), (dict(q_heads=34), 4), (dict(PAGED, page_size=32), 1), (dict(PAGED, page_size=0), 1), (dict(PAGED, num_pages=0), 1),
    (dict(PAGED, max_pages_per_seq=0), 1), (dict(PAGED, max_pages_per_seq=1 << 30), 1), (dict(s_max=24), 1), (dict(s_max=0), 1), (dict(seq_lens=0, seq_len=-1), 1),
    (dict(seq_lens=0, seq_len=49), 1), (dict(s_max=0x7fffffe0), 1), (dict(s_max=0x7fffffd0), 1),
    (dict(q_type=3), 1), (dict(q_type=-1), 1), (dict(q=4098), 1), (dict(k_codes=4104), 1), (dict(v_scales=4100), 1), (dict(o=4097), 1), (dict(lOut=4098), 1),
    (dict(seq_lens=4098), 1), (dict(PAGED, block_table=4097), 1), (dict(batch=1 << 30, kv_heads=4), 4)])
def test_decode_refuses(built_libs, bad, status):
    # a context of zeros serves no GPU: arguments are refused before that is looked at
    from goml_b200 import fa_forward as F
    F.FALoad()
    zeros = C.create_string_buffer(4096)
    with pytest.raises(F.FAError, match="fa_decode_fp4") as e:
        F.FAContext(C.addressof(zeros)).DecodeFP4(**{**DECODE, **bad})
    assert e.value.status == status and e.value.msg.startswith("fa_decode_fp4: ")
    for fine in (DECODE, dict(DECODE, **PAGED)):
        with pytest.raises(F.FAError) as e:
            F.FAContext(C.addressof(zeros)).DecodeFP4(**fine)
        assert e.value.status == F.FA_ERR_UNSUPPORTED_ARCH


def test_kernels_that_overlap_their_predecessors_are_seen():
    from tests.test_kernel_sources import other_uses, plain_launches, sources
    for name, kernels in {"fa_decode_fp4_sm100.cu": {"fa_decode_fp4_kernel"}, "fp4_cache_sm100.cu": {"fp4_append_kernel", "fp4_rows_kernel"},
                          "kv_pages_sm100.cu": {"kv_page_plan_kernel"}}.items():
        assert other_uses(sources()[name]) == kernels and not plain_launches(sources()[name])


def test_pages_and_pools_refuse():
    import torch
    from goml_b200 import nn
    for bad in (dict(batch=0), dict(num_pages=0), dict(page_size=96), dict(page_size=0), dict(max_pages_per_seq=0), dict(max_pages_per_seq=1 << 26)):
        with pytest.raises(ValueError, match="KVPages"):
            nn.KVPages(**{**dict(batch=2, num_pages=8, page_size=64, device="cpu"), **bad})
    pages = nn.KVPages(2, 8, 64, 3, device="cpu")
    assert pages.capacity == 192 and pages.table.shape == (2, 3) and pages.state.tolist() == [0, 8, 0, 0] and sorted(pages.ring.tolist()) == list(range(8))
    for bad in (dict(heads=0), dict(hd=96), dict(k_scale=0.0), dict(v_scale=float("nan"))):
        with pytest.raises(ValueError, match="FP4KVPool"):
            nn.FP4KVPool(pages, **{**dict(heads=2, hd=64), **bad})
    pool = nn.FP4KVPool(pages, 2, 128)
    assert pool.k.shape == (8, 2, 64, 64) and pool.ks.shape == (8, 2, 64, 8) and pool.vs.shape == (8, 2, 4, 8, 16)
    for fresh, more in ((torch.zeros(3, dtype=torch.int32), dict(rows=1)), (torch.zeros(2, dtype=torch.int64), dict(rows=1)), (torch.zeros(2, dtype=torch.int32), {}),
                        (1, dict(rows=1, tokens_per_seq=1)), (1, dict(rows=-1))):
        with pytest.raises(ValueError, match="KVPages.plan"):
            pages.plan(fresh, **more)


CPP = r"""
#include <cstddef>
#include <cstdio>
#include "../../goml_b200/host/goml_cuda.hpp"
using namespace goml::cuda;
template <class F> static std::string thrown(F f) { try { f(); return ""; } catch (const std::exception& e) { return e.what(); } }
int main() {
    std::puts(thrown([] { fp4_append_args_t a{}; a.tokens = 1; FP4RopeAppend(a); }).c_str());
    std::puts(thrown([] { fp4_rows_args_t a{}; a.tokens = 1; FP4CacheRows(a); }).c_str());
    std::puts(thrown([] { kv_page_plan_args_t a{}; a.batch = 1; KVPagePlan(a); }).c_str());
    std::printf("%zu %zu %zu %zu\n", sizeof(fa_decode_fp4_args_t), sizeof(fp4_append_args_t), sizeof(fp4_rows_args_t), sizeof(kv_page_plan_args_t));
    void (FAContext::*decode)(const fa_decode_fp4_args_t&) = &FAContext::DecodeFP4;
    return decode == nullptr;
}
"""


def test_cpp_host_layer(tmp_path, built_libs):
    from goml_b200 import block_glue as BG, fa_forward as F
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    host = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_cpp")
    exe = str(tmp_path / "fp4_host")
    r = subprocess.run(["g++", "-std=c++17", "-I", os.path.join(cuda, "include"), "-iquote", host, "-x", "c++", "-", "-o", exe, "-L", os.path.join(cuda, "lib64"), "-lcudart", "-ldl",
                        "-lpthread"], input=CPP, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, env=dict(os.environ, GOML_LIBS_DIR=built_libs))
    sizes = " ".join(str(C.sizeof(c)) for c in (F.DecodeFP4Args, BG.FP4AppendArgs, BG.FP4RowsArgs, BG.KVPagePlanArgs))
    assert r.returncode == 0 and r.stdout.splitlines() == ["fp4_rope_append: CUDA error 1", "fp4_cache_rows: CUDA error 1", "kv_page_plan: CUDA error 1", sizes], r.stdout + r.stderr
