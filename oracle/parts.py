"""Attention over parts of the keys in 64 bits, with how far the kernels' arithmetic may be off (fa_decode_window, fa_decode_shared, fa_forward_sinks of include/fa_sm120.h)."""
import numpy as np

from . import e4m3_decode


def attend(q, k, v, seen, scale, v_scale=1.0):
    """O [rows, hd], LSE [rows] and their tolerances of code rows q [rows, hd] on code rows k, v [keys, hd]; seen [rows, keys].

    Where the kernels round: scores are sums of hd exact products in 32 bits (each addition within 2^-23 of the sum of magnitudes: truncating adders count twice the half step) times a
    factor of 32 bits, and 2^x is good to 2^-22, so a weight is off by e = 2 (2^-22 + hd 2^-23 scale sum|q k|) of itself at most, with what the running maximum's differences add (2^-23 of
    the largest score in log2 units, twice).  Weights are rounded to fp16 for the product with V: 2^-11 of themselves, or 2^-25 of the largest one where they are that small.
    Sums over keys are in 32 bits (2^-23 of the sum of magnitudes for each of the log2 levels and pieces: 64 of them are allowed for).  O is rounded to fp16: 2^-11, or 2^-25 near zero."""
    q, k, v = (e4m3_decode(x).astype(np.float64) for x in (q, k, v))
    rows, hd = q.shape
    o, lse = np.zeros((rows, hd)), np.full(rows, -np.inf)
    tol_o, tol_l = np.full((rows, hd), 2.0 ** -25), np.zeros(rows)
    for r in range(rows):
        at = np.flatnonzero(seen[r])
        if not len(at):
            continue
        x = k[at] @ q[r] * scale
        top = x.max()
        w = np.exp(x - top)
        total = w.sum()
        o[r], lse[r] = (w @ v[at]) / total * v_scale, top + np.log(total)
        size = (np.abs(k[at]) @ np.abs(q[r])).max() * abs(scale)
        e = 2 * (2.0 ** -22 + (hd * 2.0 ** -23 + 2.0 ** -22) * size) + 64 * 2.0 ** -23
        mag = (w @ np.abs(v[at])) / total * abs(v_scale)
        small = len(at) * 2.0 ** -25 * np.abs(v[at]).max() / total * abs(v_scale)
        tol_o[r] += mag * (2.0 ** -11 + 2 * e) + small + np.abs(o[r]) * 2.0 ** -11
        tol_l[r] = 2 * e + 2.0 ** -22 * (1 + abs(lse[r]))
    return o, lse, tol_o, tol_l
