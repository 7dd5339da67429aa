"""The 8-bit KV cache of one layer: its tensors and the calls over them.

Half the bytes of the bf16 cache that the reference's decoder benches keep
(npu_ops/python/bench_decode_layer.py:70-73).  Positions are held in blocks of 64: a
complete block in 8 bits (int8 or fp8 e4m3) with one fp32 scale for its keys and one for
its values per sequence and head, the open last block in bf16.  A block is quantised once,
when its last position is written, so what is held does not depend on the calls that
wrote it, prompt chunks or single tokens.

A sequence's positions are appended in order.  It may be taken back (rejected drafts) to
any position of its open block by writing from there again; behind a block's end the bf16
values of that block are gone.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops  # noqa: F401  (registers torch.ops.npu.*)

BLOCK = 64
DTYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


class KV8Cache:
    """Keys and values of ``batch`` sequences of up to ``max_len`` positions in one layer.

    ``pos`` of the calls below is an int64 tensor on the device, the position of the call's
    first token: one for every sequence, or one each.  Tokens at positions outside
    [0, max_len) write nothing and give zeros, so prompts of several lengths share a batch
    padded on the left (pos = length - T)."""

    def __init__(self, batch: int, kv_heads: int, max_len: int, head_dim: int, dtype="int8", device="cuda"):
        dtype = DTYPES.get(dtype, dtype)
        if dtype not in DTYPES.values():
            raise ValueError(f"KV8Cache: dtype must be 'int8', 'fp8' or their torch types, not {dtype!r}")
        if head_dim not in (64, 128):
            raise ValueError(f"KV8Cache: head_dim must be 64 or 128, not {head_dim}")
        if min(batch, kv_heads, max_len) <= 0:
            raise ValueError(f"KV8Cache: batch={batch}, kv_heads={kv_heads} and max_len={max_len} must be > 0")
        self.kv_heads, self.max_len, self.dtype = kv_heads, max_len, dtype
        nb = -(-max_len // BLOCK)
        z = lambda shape, dt: torch.zeros(shape, dtype=dt, device=device)  # noqa: E731
        self.k_codes = z((batch, kv_heads, nb, BLOCK, head_dim), dtype)
        self.vt_codes = z((batch, kv_heads, nb, head_dim, BLOCK), dtype)
        self.kv_scale = z((batch, kv_heads, nb, 2), torch.float32)
        self.k_tail = z((batch, kv_heads, BLOCK, head_dim), torch.bfloat16)
        self.vt_tail = z((batch, kv_heads, head_dim, BLOCK), torch.bfloat16)

    @property
    def tensors(self) -> Tuple[torch.Tensor, ...]:
        """The five tensors in the order in which the ops take them."""
        return self.k_codes, self.vt_codes, self.kv_scale, self.k_tail, self.vt_tail

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.tensors)

    def append(self, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, heads: int,
               bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        """qkv [B, T, (heads + 2 kv_heads) * head_dim]: bias, rotary embedding, the keys and values
        appended; returns q [B, T, heads, head_dim]."""
        return torch.ops.npu.w4a8_rope_kv8(qkv, cos, sin, pos, *self.tensors, heads, self.kv_heads, self.max_len, bias)

    def attend(self, q: torch.Tensor, pos: torch.Tensor, window: int = 0, sinks: int = 0,
               scale: Optional[float] = None) -> torch.Tensor:
        """Causal attention of append's q (same pos); window > 0: only the last ``window`` positions
        up to a token's own and the first ``sinks``."""
        return torch.ops.npu.w4a8_attention_kv8(q, *self.tensors, pos, self.max_len, window, sinks, scale)

    def step(self, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, heads: int,
             bias: Optional[torch.Tensor] = None, window: int = 0, sinks: int = 0,
             scale: Optional[float] = None) -> torch.Tensor:
        """append and attend of one token a sequence, qkv [B, W], in one call; returns [B, 1, heads, head_dim]."""
        return torch.ops.npu.w4a8_attention_kv8_rope(qkv, cos, sin, pos, *self.tensors, heads, self.kv_heads,
                                                     self.max_len, bias, window, sinks, scale)

    def read(self, length: torch.Tensor, first: int = 0, n: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Positions first .. first + n - 1 as bf16 k, v [B, kv_heads, n, head_dim] (all from `first` on without
        n), zeros from length (one, or one per sequence: the positions held, max_len where it is larger) on."""
        if n is None:
            n = self.max_len - first
        if self.max_len % BLOCK:       # the op holds lengths to whole blocks: the last one would count as complete
            length = length.clamp(max=self.max_len)
        return torch.ops.npu.w4a8_kv8_read(*self.tensors, length, first, n)
