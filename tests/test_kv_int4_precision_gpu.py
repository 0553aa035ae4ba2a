"""How exact attention over the 4-bit cache is, against bounds of each row's own tokens (kv_bounds)."""
import numpy as np
import pytest
import torch

import int4_int8_ext as ext
from tests import kv_bounds
from tests.kv_helpers import Setup, typed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d,group,q_heads,heads,lens,news", [
    (64, 32, 4, 2, [40, 300, 3], [1, 2, 1]), (128, 64, 16, 1, [200, 17], [1, 1]), (96, 32, 8, 8, [130], [3]),
    (256, 128, 2, 1, [90, 5], [1, 2]), (192, 64, 12, 1, [77], [1]), (128, 32, 4, 4, [1, 2, 5, 9], [1, 1, 1, 1]),
])
def test_few_rows_keep_the_bits_of_their_weights(cuda, dtype, d, group, q_heads, heads, lens, news):
    """Sixteen bits of a weight (24 for float32): outputs that nearly cancel show them."""
    s = Setup(d + len(lens), lens, news, heads, d, group, 16, cuda)
    idx, cu = s.index()
    q, qt = typed(s.g.standard_normal((s.cu[-1], q_heads, d)), dtype)
    scale = 0.02
    out, lse = ext.attention_int4_kv(qt.to(cuda), *s.tensors, *idx, cu_q=cu, max_q=max(news), max_len=max(lens), scale=scale,
                                     return_lse=True)
    kv_bounds.check(q, out, lse, s, dtype, scale)


@pytest.mark.parametrize("n", [1, 3])
def test_float32_weights_have_a_third_term(cuda, n):
    """Two or three tokens: nothing averages out what the third bfloat16 term of a weight brings."""
    lens = [2, 3, 3, 2]
    s = Setup(31, lens, [min(n, x) for x in lens], 4, 128, 32, 16, cuda)
    idx, cu = s.index()
    q, qt = typed(s.g.standard_normal((s.cu[-1], 8, 128)), "f32")
    out, lse = ext.attention_int4_kv(qt.to(cuda), *s.tensors, *idx, cu_q=cu, max_q=n, scale=0.001, return_lse=True)
    kv_bounds.check(q, out, lse, s, "f32", 0.001)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d,group,lens,news,causal,window", [
    (64, 32, [300, 40], [100, 40], True, 0), (128, 64, [200], [150], True, 30), (96, 32, [260], [64], False, 0),
])
def test_many_rows_round_weights_to_eleven_bits(cuda, dtype, d, group, lens, news, causal, window):
    s = Setup(d + 7, lens, news, 2, d, group, 32, cuda)
    idx, cu = s.index()
    q, qt = typed(s.g.standard_normal((s.cu[-1], 4, d)), dtype)
    out, lse = ext.attention_int4_kv(qt.to(cuda), *s.tensors, *idx, cu_q=cu, max_q=max(news), max_len=max(lens), scale=0.02,
                                     causal=causal, window=window, return_lse=True)
    kv_bounds.check(q, out, lse, s, dtype, 0.02, causal, window, many=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_many_rows_in_few_row_tiles_joined_from_splits(cuda, dtype):
    """1024 rows of tiles and more, each sequence split: a block of the join takes several rows."""
    lens, news = [1500 + 37 * i for i in range(3)], [5, 4, 5]
    s = Setup(33, lens, news, 8, 64, 64, 32, cuda)
    idx, cu = s.index()
    q, qt = typed(s.g.standard_normal((s.cu[-1], 64, 64)), dtype)
    out, lse = ext.attention_int4_kv(qt.to(cuda), *s.tensors, *idx, cu_q=cu, max_q=5, max_len=max(lens), scale=0.02,
                                     return_lse=True)
    kv_bounds.check(q, out, lse, s, dtype, 0.02)


@pytest.mark.parametrize("d,group", [(64, 64), (128, 32), (256, 128)])
def test_float32_scores_are_sums_without_rounding_but_the_querys_own(cuda, d, group):
    """One token a sequence: the logarithm is its score. In units of 2^-14 to 2^-13 of the largest |q|, times the scales, a channel is
    off by its query's second term, rounded by 2^-10 at most, times a code of up to 8. Such errors are independent: the root
    of their mean square is sqrt(d) 8 2^-10 / sqrt(3) = 0.07 for 256 channels. Scores of up to 2^19 units are rounded four times
    to 24 bits, each off by 2^-6 / sqrt(3) at most: 0.02 together. (Products cut off at 1/4 would show as sqrt(d) / 14, 0.6 and more.)"""
    batch = 512
    s = Setup(37, [1] * batch, [1] * batch, 1, d, group, 16, cuda)
    idx, _ = s.index()
    q, qt = typed(s.g.standard_normal((batch, 8, d)), "f32")
    scale = d ** -0.5
    _, lse = ext.attention_int4_kv(qt.to(cuda), *s.tensors, *idx, scale=scale, return_lse=True)
    keys = np.stack([s.cache.rows(b, s.table, 1)[0][0, 0] for b in range(batch)])
    want = np.einsum("bhd,bd->bh", q, keys) * scale
    steps = s.cache.scales[0][s.table[:, 0], 0, 0].max(-1)
    unit = np.exp2(np.frexp(np.abs(q).max(-1))[1] - 14.0) * steps[:, None] * scale
    assert np.abs(want / unit).max() < 2 ** 19
    off = (lse.double().cpu().numpy() - want) / unit
    assert np.sqrt((off ** 2).mean()) <= 0.1 and np.abs(off).max() <= 8 * d * 2.0 ** -10 + 4 * 2.0 ** -6
