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


def _class(**o):
    from quant_pipeline.ops import Int4KVCache

    return Int4KVCache(2, 16, 3, 128, 64, **o)


@pytest.mark.parametrize("name", ["k_step", "v_step"])
@pytest.mark.parametrize("step", [torch.ones(3, 3), torch.ones(3), torch.ones(2, 3, 2), torch.ones(3, 2).half(),
                                  torch.ones((3, 2), dtype=torch.int32), 0.1], ids=str)
def test_the_cache_class_refuses_bad_steps(name, step):
    with pytest.raises(ValueError, match=name + " must be float32 \\[kv_heads, head_dim / group_size\\]"):
        _class(**{name: step})


def test_the_cache_class_takes_steps_as_constants_on_its_device():
    param = torch.nn.Parameter(torch.arange(6.0).view(2, 3).t() + 1)  # not contiguous
    cache = _class(k_step=param)
    assert not cache.k_step.requires_grad and cache.k_step.is_contiguous() and cache.v_step is None
    assert torch.equal(cache.k_step, param) and "k_step" in cache.state_dict() and not list(cache.parameters())
    with torch.no_grad():
        param.mul_(2)
    assert torch.equal(cache.k_step * 2, param)
    moved = _class(device=torch.device("meta"), k_step=param, v_step=torch.ones(3, 2))
    assert moved.k_step.device.type == moved.v_step.device.type == moved.k_codes.device.type == "meta"
