"""Calls on a 4-bit cache right behind each other, each reading what the one before has just written."""
import numpy as np
import pytest
import torch

import int4_int8_ext as ext
from quant_pipeline.ops import Int4KVCache

pytestmark = pytest.mark.gpu


def _layers(cuda, n):
    caches = [Int4KVCache(40, 16, 2, 64, 32, device=cuda) for _ in range(n)]
    table = torch.arange(40, dtype=torch.int32, device=cuda).flip(0).view(1, 40)
    return caches, table


@pytest.mark.parametrize("news", [[1] * 60, [90, 1, 70, 1, 1, 100, 3, 80, 1]])
def test_each_call_sees_what_the_one_before_wrote(cuda, news):
    """Tokens and prompts through four caches, the next one's rows made from the last one's output: without a wait between
    the calls as with one behind each. Lengths are written on the way too."""
    g = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn((sum(news), 4, 64), generator=g, device=cuda, dtype=torch.float32).half()

    def run(wait):
        caches, table = _layers(cuda, 4)
        lens = torch.zeros(1, dtype=torch.int32, device=cuda)
        outs, at = [], 0
        for n in news:
            h = x[at:at + n].clone()
            at += n
            lens.fill_(at)
            for cache in caches:
                cache.write(h[:, :2], h[:, 2:], table, lens)
                if wait:
                    torch.cuda.synchronize()
                k, v = cache.read(n, table, lens, dtype=torch.float16)
                if wait:
                    torch.cuda.synchronize()
                out = cache.attend(h, table, lens)
                if wait:
                    torch.cuda.synchronize()
                h = out + torch.cat([k, v], dim=1)
                if wait:
                    torch.cuda.synchronize()
            outs.append(h)
        return torch.cat(outs)

    want = run(True)
    for _ in range(3):
        assert torch.equal(run(False), want)
    assert ext.device_error() == 0


def test_two_streams_at_once(cuda):
    """Two caches, each used on a stream of its own at the same time, prompts and tokens: as one after the other."""
    def rows(seed, n):
        return torch.randn((n, 4, 64), generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).half()

    def run(seed, lens_list):
        caches, table = _layers(cuda, 1)
        out, at = [], 0
        for i, n in enumerate(lens_list):
            h = rows(seed + i, n)
            at += n
            lens = torch.full((1,), at, dtype=torch.int32, device=cuda)
            caches[0].write(h[:, :2], h[:, 2:], table, lens)
            out.append(caches[0].attend(h, table, lens))
        return torch.cat(out)

    plans = [[200, 1, 1, 150, 1], [1, 120, 1, 1, 230]]
    want = [run(10 * i, p) for i, p in enumerate(plans)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in plans]
    for _ in range(5):
        got = []
        for i, p in enumerate(plans):
            with torch.cuda.stream(streams[i]):
                got.append(run(10 * i, p))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
