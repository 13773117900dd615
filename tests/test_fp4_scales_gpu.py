"""fp4_rope_append over the whole range of tensor scales: bytes equal to those of the restatement in 64 bits (oracle/fp4.py)."""
import numpy as np
import pytest

from oracle import fp4
from oracle.glue import rope_table
from tests.test_fp4_gpu import bf16, empty_cache, run_append, same_cache

pytestmark = pytest.mark.gpu

# Largest value of a group as a multiple of 6 * scale: nothing at all, below and at the borders of the least block scales, ordinary ones, the largest, beyond it
TOPS = np.array([0.0, 2.0 ** -11, 2.0 ** -10, 1.5 * 2.0 ** -9, 2.0 ** -7, 0.11, 1.0, 1.0625, 37.0, 448.0, 1e5])
# of a group's values, as multiples of its d: every code, halfway between two, beside it, and past the last
PARTS = np.array([0.0, 0.25, 0.5, 0.75, 0.251, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -1.25, -5.0, -0.0, 4.99])


def rows(r, tokens, heads, hd, scale):
    """bf16 values of groups whose largest lies all over the range of block scales; some groups are zeros throughout, some have nothing but their sixteen PARTS."""
    groups = (tokens, heads, hd // 16)
    top = r.choice(TOPS, groups) * 6 * float(scale)
    parts = np.broadcast_to(PARTS, (*groups, 16)).copy()
    drawn = r.random(groups) < 0.5
    parts[drawn] = r.normal(size=(int(drawn.sum()), 16)) * 3
    parts[..., 10] = np.where(r.random(groups) < 0.5, 6.0, -6.0)
    with np.errstate(over="ignore"):
        x = (top[..., None] / 6 * parts).astype(np.float32)
    return bf16(np.clip(x, -3.3e38, 3.3e38).reshape(tokens, heads, hd))


@pytest.mark.parametrize("hd,tokens", [(64, 70), (128, 2100)])   # one round of threads, and several
@pytest.mark.parametrize("k_scale,v_scale", [(2.0 ** -110, 2.0 ** -115), (2.0 ** -118, 1e-36), (2.0 ** -127, 2.0 ** -132), (2.0 ** -136, 2.0 ** -149), (3e-39, 1.2e-38), (5e-36, 2e-37),
                                             (2.0 ** 97, 1e31), (2.0 ** 115, 7.5e35), (1e34, 2.0 ** 118)])
def test_append_at_every_scale(cuda, built_libs, k_scale, v_scale, hd, tokens):
    r = np.random.default_rng(hd)
    hq, kv = 1, 2
    qkv = np.concatenate([bf16(r.normal(size=(tokens, hq, hd))), rows(r, tokens, kv, hd, np.float32(k_scale)), rows(r, tokens, kv, hd, np.float32(v_scale))], 1)
    cos, sin = rope_table(64, hd, 10000.0)
    positions = np.where(r.random(tokens) < 0.7, 0, r.integers(0, 64, tokens))   # position 0 turns nothing: halfway stays halfway
    pages = -(-tokens // 16)
    cache = empty_cache(pages, kv, 16, hd, k_scale, v_scale)
    _, c = run_append(qkv, cos, sin, positions, np.arange(tokens), hq, cache)
    fp4.append(qkv, cos, sin, positions, np.arange(tokens), hq, cache)
    same_cache(c, cache)
