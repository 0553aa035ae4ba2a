"""Attention over a 4-bit cache whose scales are far apart: what a row does not see, or gives no weight, takes nothing from
what it does see."""
import numpy as np
import pytest
import torch

import int4_int8_ext as ext
from tests import kv_bounds
from tests.kv_helpers import Setup, offsets, typed

pytestmark = pytest.mark.gpu


def _filled(s, k, v):
    s.cache.write(k, v, s.table, s.lens, offsets(s.lens))
    s.tensors = s.upload()


def _run(cuda, s, dtype, scale, q_heads=2, **options):
    idx, cu = s.index()
    q, qt = typed(s.g.standard_normal((s.cu[-1], q_heads, s.tensors[0].shape[3] * 2)), dtype)
    return q, ext.attention_int4_kv(qt.to(cuda), *s.tensors, *idx, cu_q=cu, max_q=max(s.news), scale=scale, return_lse=True,
                                    **options)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [12, 150])  # few rows, and many
@pytest.mark.parametrize("exp", [14, 20, 30, 60])
@pytest.mark.parametrize("which", ["keys", "values"])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (96, 32)])
def test_hidden_tokens_of_any_size_take_nothing(cuda, dtype, n, exp, which, d, group):
    """Tokens 2^exp times as large as the others, hidden from rows before them (causality) and behind them (the window)."""
    length, bad, window = 300, 200, 40
    s = Setup(exp + n, [length], [n], 1, d, group, 16, cuda)
    k, v = (typed(s.g.standard_normal((length, 1, d)), "bf16")[0] for _ in range(2))
    (k if which == "keys" else v)[bad - 3:bad] *= 2.0 ** exp
    _filled(s, k, v)
    pos = np.arange(length - n, length)
    hidden = (pos < bad - 3) | (pos >= bad - 1 + window)
    assert hidden.any()
    q, (out, lse) = _run(cuda, s, dtype, 0.05, window=window)
    want, want_lse, off, lse_off = kv_bounds.attention_and_bound(q, s, dtype, 0.05, True, window, many=n > 32)
    got = out.double().cpu().numpy()
    half = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    err, tol = np.abs(got - want)[hidden], (off + half * (np.abs(want) + off) + 2.0 ** -25)[hidden]
    assert np.all(err <= tol), (err / tol).max()
    assert np.all(np.abs(lse.double().cpu().numpy() - want_lse)[hidden] <= lse_off[hidden])


@pytest.mark.parametrize("n", [12, 150])
@pytest.mark.parametrize("exp", [13, 24, 50])
def test_seen_tokens_without_weight_take_nothing(cuda, n, exp):
    """Large values whose tokens' scores are far below the others'."""
    s = Setup(exp, [300], [n], 1, 64, 32, 16, cuda)
    k, v = (s.g.standard_normal((300, 1, 64)) for _ in range(2))
    large = np.arange(300) % 50 == 7
    k[:, 0, 0] = np.where(large, -7.0, 0.5)
    v = v * np.where(large, 2.0 ** exp, 1)[:, None, None]
    k, v = (typed(x, "bf16")[0] for x in (k, v))
    _filled(s, k, v)
    idx, cu = s.index()
    q, qt = s.g.standard_normal((n, 2, 64)) * 0.1, None
    q[..., 0] = 30.0  # a large token's score is 225 below the others'
    q, qt = typed(q, "bf16")
    out, lse = ext.attention_int4_kv(qt.to(cuda), *s.tensors, *idx, scale=1.0, return_lse=True)
    kv_bounds.check(q, out, lse, s, "bf16", 1.0, many=n > 32)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [12, 150])
@pytest.mark.parametrize("window", [0, 64])
@pytest.mark.parametrize("ratio", [0.1, 10.0])
def test_values_that_shrink_or_grow(cuda, dtype, n, window, ratio):
    """Values ten times smaller, or larger, every 60 tokens; with a window only the last ones are seen."""
    s = Setup(41, [600], [n], 2, 64, 32, 16, cuda)
    size = ratio ** (np.arange(600) // 60 - (9 if ratio > 1 else 0))
    k, v = (s.g.standard_normal((600, 2, 64)) for _ in range(2))
    k, v = typed(k, "bf16")[0], typed(v * 1e4 * size[:, None, None], "bf16")[0]
    _filled(s, k, v)
    q, (out, lse) = _run(cuda, s, dtype, 0.05, q_heads=4, window=window)
    kv_bounds.check(q, out, lse, s, dtype, 0.05, True, window, many=n > 32)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("exp", [-40, -22, -14, -9, 8, 14])
def test_caches_of_any_size_that_is_even(cuda, dtype, exp):
    """All scales near 2^exp, some of them on either side of a power of two."""
    s = Setup(43, [300], [150], 1, 128, 64, 16, cuda)
    k, v = (typed(s.g.standard_normal((300, 1, 128)) * np.exp2(s.g.integers(-1, 2, (300, 1, 1)) + float(exp)), "bf16")[0]
            for _ in range(2))
    if dtype == "f16":
        v = typed(v * 2.0 ** (-exp), "bf16")[0]  # outputs that the type can hold
    _filled(s, k, v)
    scale = 0.05 * 2.0 ** -exp
    q, (out, lse) = _run(cuda, s, dtype, scale)
    kv_bounds.check(q, out, lse, s, dtype, scale, many=True)


@pytest.mark.parametrize("batch,lens", [(1, [5000]), (3, [3000, 100, 1500])])
def test_large_hidden_values_in_calls_that_are_split(cuda, batch, lens):
    """A long cache, few row tiles: the pieces of a sequence meet large values in some places only."""
    news = [min(n, 70) for n in lens]
    s = Setup(47, lens, news, 1, 64, 32, 16, cuda)
    total = sum(lens)
    k, v = (typed(s.g.standard_normal((total, 1, 64)), "bf16")[0] for _ in range(2))
    for b, at in enumerate(offsets(lens)[1:]):
        v[at - 3] *= 2.0 ** 40  # hidden from all rows but the last three
    _filled(s, k, v)
    q, (out, lse) = _run(cuda, s, "f16", 0.05, max_len=max(lens))
    want, want_lse, off, lse_off = kv_bounds.attention_and_bound(q, s, "f16", 0.05, many=True)
    ok = np.ones(len(q), bool)
    for at in s.cu[1:]:
        ok[at - 3:at] = False
    got = out.double().cpu().numpy()
    err, tol = np.abs(got - want)[ok], (off + 2.0 ** -11 * (np.abs(want) + off) + 2.0 ** -25)[ok]
    assert np.all(err <= tol), (err / tol).max()
    assert np.all(np.abs(lse.double().cpu().numpy() - want_lse)[ok] <= lse_off[ok])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [12, 150])
def test_a_sink_with_small_values_and_a_long_tail(cuda, dtype, n):
    """One token takes nearly all of the weight and has zeros for values: what is left comes from equal small weights, of
    2^-20 to 2^-24 of the largest."""
    s = Setup(53, [2000], [n], 1, 64, 32, 16, cuda)
    k, v = np.zeros((2000, 1, 64)), 1 + 0.1 * s.g.standard_normal((2000, 1, 64))
    k[0, 0, 0] = 7.0
    v[0] = 0
    k, v = (typed(x, "bf16")[0] for x in (k, v))
    _filled(s, k, v)
    idx, cu = s.index()
    q = np.zeros((n, 2, 64))
    q[:, 0, 0], q[:, 1, 0] = np.linspace(13.9, 16.6, n), np.linspace(14.3, 16.1, n)  # scores of the sink, in nats
    q, qt = typed(q, dtype)
    out, lse = ext.attention_int4_kv(qt.to(cuda), *s.tensors, *idx, scale=1.0 / 7, return_lse=True)
    kv_bounds.check(q, out, lse, s, dtype, 1.0 / 7, many=n > 32)


def test_a_captured_call_decides_at_each_replay(cuda):
    """A captured prompt over a cache whose scales are even, then far apart, then even again: as eager calls give it."""
    s = Setup(59, [300], [150], 2, 64, 32, 16, cuda)
    idx, _ = s.index()
    _, qt = typed(s.g.standard_normal((150, 4, 64)), "bf16")
    qt, even = qt.to(cuda), s.tensors[2].clone()
    far = even.clone()
    far[int(s.table[0][5])] *= 2.0 ** 40

    def call():
        return ext.attention_int4_kv(qt, *s.tensors, *idx, scale=0.05)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for scales in (even, far, even, far):
        s.tensors[2].copy_(scales)
        graph.replay()
        assert torch.equal(out, call()) and not out.isnan().any()
    del graph


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_nan_values_beside_scales_far_apart(cuda, dtype):
    """The rows that see the NaN give NaN in its group, the others what they gave without it."""
    length, n, bad = 300, 150, 220
    s = Setup(61, [length], [n], 1, 64, 32, 16, cuda)
    k, v = (typed(s.g.standard_normal((length, 1, 64)), "bf16")[0] for _ in range(2))
    v[180] *= 2.0 ** 40
    _filled(s, k, v)
    idx, _ = s.index()
    _, qt = typed(s.g.standard_normal((n, 2, 64)), dtype)
    run = lambda: ext.attention_int4_kv(qt.to(cuda), *s.tensors, *idx, scale=0.05, window=30)  # noqa: E731
    want = run()
    s.tensors[2][int(s.table[0][bad // 16]), 0, bad % 16, 1, 1] = float("nan")  # the second group's values
    got = run()
    pos = torch.arange(length - n, length, device=cuda)
    sees = (pos >= bad) & (pos < bad + 30)
    assert got[sees][..., 32:].isnan().all()
    assert torch.equal(got[sees][..., :32], want[sees][..., :32]) and torch.equal(got[~sees], want[~sees])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [12, 150])
@pytest.mark.parametrize("exp", [12, 20, 25, 30, 60])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("d", [64, 128])
def test_scores_of_any_size(cuda, dtype, n, exp, sign, d):
    """Scores from 7 2^exp to 56 2^exp, or their opposites, 2^-8 apart or more: the largest takes all of the weight, and the
    output is its value. Keys of one channel, code 7 times a bfloat16 of each token's own: every product is exact."""
    s = Setup(67 + exp, [300], [n], 1, d, 64, 16, cuda)
    i = s.g.permutation(300)
    k, v = np.zeros((300, 1, d)), s.g.standard_normal((300, 1, d))
    k[:, 0, 0] = sign * 7 * (1 + i % 128 / 128) * 2.0 ** (i // 128 + exp - 3)
    v = typed(v, "bf16")[0]
    _filled(s, k, v)
    idx, _ = s.index()
    q = np.zeros((n, 2, d))
    q[..., 0] = 8
    out, lse = ext.attention_int4_kv(typed(q, dtype)[1].to(cuda), *s.tensors, *idx, scale=1.0, return_lse=True)
    keys, values = s.cache.rows(0, s.table, 300)
    scores = 8 * keys[:, 0, 0]
    top = [np.argmax(scores[:p + 1]) for p in range(300 - n, 300)]
    # One weight, off by its rounding and that of the sums; the output is rounded once.
    half, weight = kv_bounds.HALF_STEP[dtype], 2.0 ** -20 + (2.0 ** -11 if n > 32 and dtype != "f32" else kv_bounds.WEIGHT[dtype])
    for h in range(2):
        err = np.abs(out[:, h].double().cpu().numpy() - values[top, 0])
        assert np.all(err <= (half + weight + half * weight) * np.abs(values[top, 0]))
        assert np.all(np.abs(lse[:, h].double().cpu().numpy() - scores[top]) <= 2.0 ** -21 * np.abs(scores[top]))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [12, 150])
@pytest.mark.parametrize("length,most", [(300, None), (3000, 3000)])  # the second is split
def test_values_near_the_largest_numbers(cuda, dtype, n, length, most):
    """Sums of up to 3000 weights of at most 1 with values below 2^116 do not overflow."""
    s = Setup(71, [length], [n], 1, 64, 32, 16, cuda)
    k, v = (s.g.standard_normal((length, 1, 64)) for _ in range(2))
    v = np.clip(v, -3, 3) * 2.0 ** 114
    k, v = (typed(x, "bf16")[0] for x in (k, v))
    _filled(s, k, v)
    q, (out, lse) = _run(cuda, s, dtype, 0.5, max_len=most)
    assert out.isfinite().all()
    kv_bounds.check(q, out, lse, s, dtype, 0.5, many=n > 32 and dtype != "f32")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [4, 150])
def test_values_near_the_largest_numbers_behind_a_rising_score(cuda, dtype, n):
    """A token whose score is 5 above those before it, and values of 2^123: no weight goes beyond the largest's 1."""
    s = Setup(73, [160], [n], 1, 64, 32, 16, cuda)
    k, v = np.zeros((160, 1, 64)), s.g.choice([-1.0, 1.0], (160, 1, 64)) * 2.0 ** 123
    k[140, 0, 0] = 7
    _filled(s, k, typed(v, "bf16")[0])
    idx, _ = s.index()
    q = np.zeros((n, 2, 64))
    q[..., 0] = 5
    q, qt = typed(q, dtype)
    out, lse = ext.attention_int4_kv(qt.to(cuda), *s.tensors, *idx, scale=1 / 7, return_lse=True)
    assert out.isfinite().all()
    kv_bounds.check(q, out, lse, s, dtype, 1 / 7, many=n > 32 and dtype != "f32")
