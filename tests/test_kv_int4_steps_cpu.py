"""Learned steps of the 4-bit cache, and derivatives that it does not have, without a GPU."""
import pytest
import torch

import int4_int8_ext as ext


def _cache():
    k, v = (torch.zeros((3, 2, 4, 32), dtype=torch.uint8) for _ in range(2))
    return dict(k_codes=k, v_codes=v, scales=torch.zeros((3, 2, 4, 2, 2), dtype=torch.bfloat16),
                block_table=torch.zeros((2, 2), dtype=torch.int32), seq_lens=torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("name", ["k_step", "v_step"])
def test_refuses_steps_that_require_a_gradient(name):
    x, step = torch.zeros(4, 2, 64), torch.nn.Parameter(torch.ones(2, 2))
    with pytest.raises(RuntimeError, match=name + " requires a gradient.*no_grad"):
        ext.kv_cache_write_int4(x, x, **_cache(), **{name: step})
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):  # what is refused next here
        ext.kv_cache_write_int4(x, x, **_cache(), **{name: step})


def test_refuses_scales_that_require_a_gradient():
    x, c = torch.zeros(4, 2, 64), _cache()
    c["scales"].requires_grad_()
    for call in (lambda: ext.kv_cache_write_int4(x, x, **c), lambda: ext.kv_cache_read_int4(**c, rows=4),
                 lambda: ext.attention_int4_kv(x, **c)):
        with pytest.raises(RuntimeError, match="scales requires a gradient"):
            call()


def test_refuses_forward_mode_tangents():
    """They would be dropped, also under no_grad."""
    import torch.autograd.forward_ad as fwd

    x, c = torch.zeros(4, 2, 64), _cache()
    with fwd.dual_level(), torch.no_grad():
        dual = fwd.make_dual(x, torch.ones_like(x))
        step = fwd.make_dual(torch.ones(2, 2), torch.ones(2, 2))
        for call, name in ((lambda: ext.kv_cache_write_int4(dual, x, **c), "k"),
                           (lambda: ext.kv_cache_write_int4(x, dual, **c), "v"),
                           (lambda: ext.kv_cache_write_int4(x, x, **c, k_step=step), "k_step"),
                           (lambda: ext.attention_int4_kv(dual, **c), "q")):
            with pytest.raises(RuntimeError, match=name + " has a forward-mode tangent"):
                call()
