"""Bounds of attention over the 4-bit cache for each row and channel, from the tokens that the row sees alone."""
import numpy as np

from oracle import kv_oracle as kvo
from tests.kv_helpers import HALF_STEP

# Few rows, float32: three bfloat16 terms, each off by 2^-8 of itself. Two-byte types: a weight is two terms w + u (off by
# 2^-16), and times a scale s the first is x = w s rounded, the second w s - x + u s rounded, of at most 2^-8 + 2^-8 of
# the product: off by 2^-15 of it.
WEIGHT = {"bf16": 1.5 * 2.0 ** -15, "f16": 1.5 * 2.0 ** -15, "f32": 2.0 ** -24}


def attention_and_bound(q, setup, dtype, scale, causal=True, window=0, many=False):
    """The oracle's output and logarithms, and how far the kernel's may be off, [rows, q_heads, d] and [rows, q_heads].

    To first order an output is off by sum_t p_t (|v_t| + |o|) e_t, where e_t is what the weight of token t is off by:
    * its score. For two-byte queries sums of products with codes of up to 15 are rounded d / 16 + 5 times to no less than 22
      bits of the largest, 16 scale sum |q| s. Each product is cut off at 2^-25 of the largest of its step, for which the tensor cores
      take a subnormal code n 2^-24 as 2^-14 (measured: beside n 2^-24 times 2^13, products of 2^-26 are kept, of 2^-27 not). The
      query is scaled to [2^13, 2^14), so that is 2^-26 of 2^-1 2^24 = 1/4 where the largest |q| stands as 2^13 or more: off by
      2^-15 scale max |q| s for each channel. A float32 query is held in 23 bits of its largest magnitude, met by codes of up
      to 8, and three sums are rounded to 24 bits;
    * the exponential and its argument, 2^-21 (1 + |score|);
    * its own rounding: WEIGHT, or with many rows 2^-11 and, relative to the row's largest weight, 2^-32 (the smallest float16 is
      2^-24, and the reference weight 2^7). Weights below 2^-126 of the reference, which is 2^8 of the
      largest weight at most, are zeros.
    Sums over the tokens take a step for 16 of them and each term, each off by 2^-22 of what was added up."""
    want, lse = kvo.attention(q, setup.cache, setup.table, setup.lens, setup.cu, scale, causal, window)
    off, lse_off = np.zeros(want.shape), np.zeros(lse.shape)
    d, group, page = q.shape[2], setup.cache.group, setup.cache.page_size
    terms = 3 if dtype == "f32" else 1 if many else 2
    for b, n in enumerate(setup.lens):
        if n == 0:
            continue
        k, v = setup.cache.rows(b, setup.table, n)
        ratio = q.shape[1] // k.shape[1]
        t = np.arange(n)
        steps = np.repeat(setup.cache.scales[0][setup.table[b][t // page], :, t % page], group, -1)
        new = setup.cu[b + 1] - setup.cu[b]
        for i in range(new):
            pos, row = n - new + i, setup.cu[b] + i
            seen = np.ones(n, bool)
            if causal:
                seen &= t <= pos
            if window:
                seen &= t > pos - window
            if pos < 0 or not seen.any():
                continue
            for h in range(q.shape[1]):
                x, ks, vs, s = q[row, h], k[seen, h // ratio], v[seen, h // ratio], steps[seen, h // ratio]
                score = ks @ x * scale
                p = np.exp(score - lse[row, h])
                if dtype == "f32":
                    e = 8 * abs(scale) * (s @ (np.abs(x).max() * 2.0 ** -23 + np.abs(x) * 3 * 2.0 ** -24))
                else:
                    e = 16 * abs(scale) * (s @ np.abs(x)) * (d / 16 + 5) * 2.0 ** -22
                    e = e + 2.0 ** -15 * abs(scale) * np.abs(x).max() * s.sum(-1)
                e = e + 2.0 ** -21 * (1 + np.abs(score))
                lse_off[row, h] = (p * e).sum() + 2.0 ** -21 * (1 + abs(lse[row, h]))
                e = e + (2.0 ** -11 if many else WEIGHT[dtype]) + (seen.sum() / 16 + 4) * terms * 2.0 ** -22
                least = (2.0 ** -32 if many else 2.0 ** -118) * p.max()
                off[row, h] = (p * e + least) @ np.abs(vs) + (p * e).sum() * np.abs(want[row, h])
    return want, lse, off, lse_off


def check(q, out, lse, setup, dtype, scale, causal=True, window=0, many=False):
    want, want_lse, off, lse_off = attention_and_bound(q, setup, dtype, scale, causal, window, many)
    got = out.double().cpu().numpy()
    # Rounded once to the output's type, whose smallest steps are 2^-24 (float16), 2^-133 and 2^-149.
    tol = off + HALF_STEP[dtype] * (np.abs(want) + off) + {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -150}[dtype]
    err = np.abs(got - want)
    assert np.all(err <= tol), f"{(err > tol).mean():.3g} of the outputs are off by up to {(err / tol).max():.3g} times the bound"
    if lse is not None:
        l = lse.double().cpu().numpy()
        some = np.isfinite(want_lse)
        assert np.array_equal(np.isfinite(l), some)
        assert np.all(np.abs(l[some] - want_lse[some]) <= lse_off[some])
