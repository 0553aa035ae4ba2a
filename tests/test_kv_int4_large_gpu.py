"""Rows, queries and outputs of more than 2^31 elements."""
import pytest
import torch

import int4_int8_ext as ext
from quant_pipeline.ops import Int4KVCache

pytestmark = pytest.mark.gpu


def test_more_than_2_31_elements(cuda):
    """One call each on [270000, 64, 128] rows: every part of a sequence against what small calls give."""
    rows, heads, d, window, page = 270000, 64, 128, 9, 64
    assert rows * heads * d > 2 ** 31
    g = torch.Generator(device=cuda).manual_seed(0)
    piece = torch.randn((1000, heads, d), generator=g, device=cuda, dtype=torch.float16)
    x = torch.empty((rows, heads, d), dtype=torch.float16, device=cuda)
    for i in range(0, rows, 1000):  # another order of the heads in each piece
        x[i:i + 1000] = piece.roll(i // 1000, dims=1)
    pages = -(-rows // page)
    cache = Int4KVCache(pages, page, heads, d, 64, device=cuda)
    table = torch.randperm(pages, generator=g, device=cuda).to(torch.int32).view(1, pages)
    lens = torch.tensor([rows], dtype=torch.int32, device=cuda)
    cache.write(x, x, table, lens)
    k, v = cache.read(rows, table, lens, dtype=torch.float16)
    for at in (0, 131071, 262143, rows - 50):
        part = x[at:at + 50].float().unflatten(-1, (-1, 64))
        half = part.abs().amax(-1, keepdim=True) / 7 * (1 + 2.0 ** -7) / 2  # of the scale, the next bfloat16
        for got in (k, v):
            assert ((got[at:at + 50].float().unflatten(-1, (-1, 64)) - part).abs() <= half * (1 + 2.0 ** -10)).all()
    del v
    out, lse = cache.attend(x, table, lens, window=window, max_len=rows, return_lse=True)
    for at in (window, 131071, 262143, rows - 50):  # the same tokens in float64, from what was read back
        q, keys = x[at:at + 50].double(), k[at - window:at + 50].double()
        scores = torch.einsum("ihd,thd->hit", q, keys) * d ** -0.5
        i, t = torch.arange(50, device=cuda)[:, None], torch.arange(50 + window, device=cuda)
        scores.masked_fill_((t > i + window) | (t <= i), -torch.inf)
        want = torch.einsum("hit,thd->ihd", scores.softmax(-1), keys)
        # Weights of 11 bits and an output of 11: values of at most 8 scales; scores of at most 60, off by 60 (8 + 5) 2^-22.
        size = keys.abs().max()
        assert (out[at:at + 50].double() - want).abs().max() <= size * (2 * 2.0 ** -11 + 2 * 60 * 13 * 2.0 ** -22)
        assert (lse[at:at + 50].double() - scores.logsumexp(-1).t()).abs().max() <= 60 * 13 * 2.0 ** -22 + 2.0 ** -16
    assert ext.device_error() == 0
