"""Paged key/value cache in 4 bits: the state an attention layer keeps between steps.

No reference counterpart (the reference has no attention); it completes the
W4A8 linear layers for models that decode. Codes use int4_pack's nibble
order, so ``unpack_int4_weights(cache.k_codes)`` gives them as int8."""
from typing import Optional, Tuple

import torch
import torch.nn as nn

import int4_int8_ext as ext


class Int4KVCache(nn.Module):
    """``num_pages`` pages of ``page_size`` tokens for ``kv_heads`` heads of ``head_dim`` channels, one
    bfloat16 scale for ``group_size`` channels: 4 + 16 / group_size bits a value.

    Which pages a sequence has is the caller's: each call takes ``block_table`` int32 [batch, pages a
    sequence], ``seq_lens`` int32 [batch] and, for sequences with different numbers of rows,
    ``cu_q`` int32 [batch + 1]; the rows given are the last tokens of their sequences
    (``int4_int8_ext.kv_cache_write_int4``). Buffers move and are saved with the module. ``k_step`` and
    ``v_step`` (float32 [kv_heads, head_dim / group_size]), if given, are learned LSQ steps that take
    the place of each row's own scales; the cache keeps a copy of them on its device, without gradients. ``half()``, ``to(dtype)`` and the like on a model that holds the cache
    leave its types as they are. Inference only."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, group_size: int = 64,
                 device: Optional[torch.device] = None, k_step: Optional[torch.Tensor] = None,
                 v_step: Optional[torch.Tensor] = None) -> None:
        super().__init__()
        if head_dim not in ext.KV_HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {ext.KV_HEAD_DIMS}")
        if group_size not in ext.KV_GROUPS or head_dim % group_size:
            raise ValueError(f"group_size must be one of {ext.KV_GROUPS} and divide head_dim")
        if min(num_pages, page_size, kv_heads) < 1:
            raise ValueError("num_pages, page_size and kv_heads must be positive")
        self.group_size = group_size
        codes = (num_pages, kv_heads, page_size, head_dim // 2)
        self.register_buffer("k_codes", torch.zeros(codes, dtype=torch.uint8, device=device))
        self.register_buffer("v_codes", torch.zeros(codes, dtype=torch.uint8, device=device))
        self.register_buffer("scales", torch.zeros((num_pages, kv_heads, page_size, 2, head_dim // group_size),
                                                   dtype=torch.bfloat16, device=device))
        shape = (kv_heads, head_dim // group_size)
        for name, step in (("k_step", k_step), ("v_step", v_step)):
            if step is not None:
                if not isinstance(step, torch.Tensor) or step.dtype != torch.float32 or tuple(step.shape) != shape:
                    raise ValueError(f"{name} must be float32 [kv_heads, head_dim / group_size]")
                step = step.detach().to(self.scales.device, copy=True).contiguous()
            self.register_buffer(name, step)

    def _apply(self, fn, *args, **kwargs):
        def moved(t: torch.Tensor) -> torch.Tensor:
            u = fn(t)
            return u if u.dtype == t.dtype else t.to(u.device)
        return super()._apply(moved, *args, **kwargs)

    def write(self, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
              cu_q: Optional[torch.Tensor] = None) -> None:
        ext.kv_cache_write_int4(k, v, self.k_codes, self.v_codes, self.scales, block_table, seq_lens, cu_q=cu_q,
                                k_step=self.k_step, v_step=self.v_step)

    def read(self, rows: int, block_table: torch.Tensor, seq_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None,
             dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        return ext.kv_cache_read_int4(self.k_codes, self.v_codes, self.scales, block_table, seq_lens, rows=rows,
                                      dtype=dtype, cu_q=cu_q)

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
               cu_q: Optional[torch.Tensor] = None, **options):
        """``options``: causal, window, scale, max_q, max_len, return_lse (``int4_int8_ext.attention_int4_kv``)."""
        return ext.attention_int4_kv(q, self.k_codes, self.v_codes, self.scales, block_table, seq_lens, cu_q=cu_q,
                                     **options)
