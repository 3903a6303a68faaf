"""Attention with a sliding window, and a few first tokens that stay visible,
over uncompressed keys and values.

The reference leaves sliding-window layers to the model (patch.py:270-321) and
its caches refuse a window (cache.py:708-724). Here the same kernels as those of
the 8-bit cache attend over 16-bit keys and values in place: only the tiles
that a query sees are read.
"""

from __future__ import annotations

import torch

from . import _lib
from .kv8 import _NO_ROWS, HEAD_DIMS, _attention_desc, _lengths, _on, _ready, _rows4


def window_attention(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, window: int | None = None,
                     sinks: int = 0, lens=None, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of each sequence's last T_q tokens, each seeing the
    last ``window`` tokens up to its own and the first ``sinks`` (``window``
    None: every token up to its own).

    ``queries`` (B, Hq, T_q, D), or (B, Hq, D) for T_q = 1; ``keys`` /
    ``values`` (B, Hkv, T, D), all fp16 or all bf16, D 64, 96, 128 or 256, of
    any strides with contiguous rows (others, and rows that are not 16-byte
    aligned, are copied); Hq a multiple of Hkv. ``lens``: tokens per sequence,
    None (T), an int, or an int32 device tensor (B,) (cut to [0, T]); keys and
    values past a sequence's length are not read. Query i sits at position
    lens - T_q + i; before position 0 it sees nothing and gives 0. Default
    scale D**-0.5.

    Returns (B, Hq, T_q, D) of the queries' type, or ``out`` (that type or
    float32). Scores, softmax and sums are float32; the softmax's weights are
    rounded to 16 bits (bf16 with few query rows: to two parts). For inference:
    no gradients."""
    if keys.dim() != 4 or values.shape != keys.shape or values.dtype != keys.dtype or values.device != keys.device:
        raise ValueError("keys and values must have one shape (B, Hkv, T, D), dtype and device")
    B, H, T, D = keys.shape
    if D not in HEAD_DIMS:
        raise ValueError(f"head_dim {D} not supported: use one of {HEAD_DIMS}")
    if keys.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"keys and values of {keys.dtype} not supported: fp16 or bf16")
    if H == 0:
        raise ValueError("no kv heads")
    len_b, length = _lengths(T if lens is None else lens, B, T, keys.device, "lens")
    if len_b:
        length = T
    k = v = _NO_ROWS
    if length:
        (k, keys), (v, values) = _rows4(keys), _rows4(values)
    device = keys.device
    desc, out, q = _attention_desc(queries, B, H, D, keys.dtype, device, len_b, length, scale, window, sinks, out, k, v)
    if out.numel() == 0:
        return out
    _ready(device)
    lib = _lib.load()
    with _on(device):
        need = lib.tq_window_attention_workspace_bytes(desc)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _lib.check(lib.tq_window_attention(desc, _lib.ptr(ws), need, _lib.stream_ptr(device)), "tq_window_attention")
    return out
