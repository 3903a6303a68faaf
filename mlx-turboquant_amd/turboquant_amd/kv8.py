"""8-bit KV cache: between the 2 to 4 bits of ``TurboQuantKVCache`` and the 16
of ``FP16KVCache``, for layers whose keys the low widths do not serve (the
outlier and skipped layers, which the reference keeps in 16 bits,
patch.py:337-338).

Tokens of complete blocks (``block`` tokens) are held in 8 bits with one
float32 scale for each block and kv head, keys and values apart; the tokens of
the last, incomplete block in 16 bits until it is complete, so every block is
quantised once, from its 16-bit values. For a block of elements x with largest
magnitude a, QMAX = 127 (``"int8"``) or 448 (``"fp8"``: e4m3):

    scale = a / QMAX        code = round(x * (QMAX / a))

in float32, codes to the nearest with ties to even. A block with a < 2**-110 is
stored as zeros (scale 0); one that holds an infinity or NaN reads back as NaN
throughout (scale NaN).

- ``KV8Store``: the arrays of one layer. ``kv8_write``, ``kv8_read`` and
  ``kv8_attention`` are the operators over it; they take one length for the
  whole batch or a device array of one per sequence, and keep no state, so they
  can be captured in a HIP graph (with ``max_len`` the largest length that the
  replays reach).
- ``KV8Cache``: the cache protocol of ``TurboQuantKVCache`` (``update``,
  ``update_and_fetch``, ``attend``, ``state``, ...) for sequences of one length.
- ``KV8Batch``: sequences of different lengths, as ``RaggedKVBatch``.

Head dims 64, 96, 128 and 256, fp16 and bf16. No gradients: caches are written
by inference.
"""

from __future__ import annotations

import contextlib
import struct

import numpy as np
import torch

from . import _codec, _lib

TILE = 64  # tokens per transposed tile of value codes
HEAD_DIMS = (64, 96, 128, 256)
BLOCKS = (16, 32, 64)
FORMATS = {"int8": (_lib.TQ_KV8_INT8, torch.int8), "fp8": (_lib.TQ_KV8_E4M3, torch.float8_e4m3fn)}


# The C structs as bytes: packing them takes a fraction of the time that filling
# ctypes structures does, which a decode step's host path would wait for.
_STORE = struct.Struct("@6Pq6i")
_ROWS = struct.Struct("@Pqqq")
_DESC = struct.Struct("@10iPf4x" + "Pqqq" * 4)
_NO_ROWS = (0, 0, 0, 0)

_NULL = contextlib.nullcontext()
_current_device = torch.cuda.current_device


def _on(device: torch.device):
    """Launches go to the tensors' own device, whichever is current."""
    return _NULL if device.index is None or device.index == _current_device() else torch.cuda.device(device)


def _rows4(t: torch.Tensor) -> tuple[tuple[int, int, int, int], torch.Tensor]:
    """The fields of a ``tq_rows4`` of (B, H, T, D), and the tensor it points
    into (a copy where the kernels cannot take its strides or address)."""
    nb, nh, nt, _ = t.shape
    sb, sh, st, sd = t.stride()
    p = t.data_ptr()
    if nb == 1:
        sb = 0
    if nh == 1:
        sh = 0
    if nt == 1:
        st = 0
    if sd != 1 or (sb | sh | st) & 7 or p & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        sb, sh, st, _ = t.stride()
        p = t.data_ptr()
    return (p, sb, sh, st), t


def _overlaps(t: torch.Tensor) -> bool:
    """Whether elements of ``t`` may share memory (dims that do not nest)."""
    span = 1
    for stride, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride < span:
            return True
        span = stride * n
    return False


def _lengths(lens, batch: int, cap: int, device, what: str) -> tuple[int, int]:
    """(device array or 0, the length where there is one for all)."""
    if isinstance(lens, torch.Tensor):
        if lens.dtype != torch.int32 or lens.shape != (batch,) or lens.device != device or not lens.is_contiguous():
            raise ValueError(f"{what}: an int, or a contiguous int32 tensor of shape ({batch},) on {device}")
        return lens.data_ptr(), 0
    n = int(lens)
    if not 0 <= n <= cap:
        raise ValueError(f"{what} {n} outside [0, {cap}]")
    return 0, n


class KV8Store:
    """The arrays of one layer's cache: ``batch`` sequences of ``heads`` kv
    heads with room for ``capacity`` tokens (rounded up to 64).

    k_codes (B, H, cap, D) and v_codes (B, H, cap / 64, D, 64) int8 or
    float8_e4m3fn, k_scales and v_scales (B, H, cap / block) float32, k_tail
    and v_tail (B, H, block, D) of the 16-bit type. The values' codes are held
    transposed in tiles of 64 tokens."""

    def __init__(self, batch: int, heads: int, head_dim: int, capacity: int, fmt: str = "int8", block: int = 32,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if batch < 0 or heads < 1 or capacity < 0:
            raise ValueError(f"batch {batch}, heads {heads}, capacity {capacity}")
        _check(fmt, head_dim, block, dtype)
        cap = (capacity + TILE - 1) // TILE * TILE
        code = FORMATS[fmt][1]
        z = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=dev).view(code)
        s = lambda: torch.zeros(batch, heads, cap // block, dtype=torch.float32, device=dev)
        t = lambda: torch.zeros(batch, heads, block, head_dim, dtype=dtype, device=dev)
        self._set(fmt, z(batch, heads, cap, head_dim), z(batch, heads, cap // TILE, head_dim, TILE), s(), s(), t(), t())

    @classmethod
    def from_tensors(cls, fmt: str, k_codes, v_codes, k_scales, v_scales, k_tail, v_tail) -> "KV8Store":
        """A store over existing arrays (not copied), contiguous and on one
        device. Code bytes that no write has reached may hold anything."""
        self = object.__new__(cls)
        _check(fmt, k_codes.shape[-1], k_tail.shape[2] if k_tail.dim() == 4 else 0, k_tail.dtype)
        self._set(fmt, k_codes, v_codes, k_scales, v_scales, k_tail, v_tail)
        return self

    def _set(self, fmt, k_codes, v_codes, k_scales, v_scales, k_tail, v_tail) -> None:
        B, H, cap, D = k_codes.shape
        if H == 0:
            raise ValueError("no kv heads")
        block = k_tail.shape[2]
        code, dev, dtype = FORMATS[fmt][1], k_codes.device, k_tail.dtype
        if cap % TILE:
            raise ValueError(f"k_codes: room for {cap} tokens, not a multiple of {TILE}")
        tensors = (k_codes, v_codes, k_scales, v_scales, k_tail, v_tail)
        scales, tail = (B, H, cap // block), (B, H, block, D)
        shapes = [(B, H, cap, D), (B, H, cap // TILE, D, TILE), scales, scales, tail, tail]
        kinds = [code, code, torch.float32, torch.float32, dtype, dtype]
        if ([t.shape for t in tensors] != shapes or [t.dtype for t in tensors] != kinds or
                not all([t.is_contiguous() for t in tensors]) or any([t.device != dev for t in tensors])):
            for name, t, shape, kind in zip(("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail"), tensors, shapes, kinds):
                if t.shape != shape or t.dtype != kind or t.device != dev or not t.is_contiguous():
                    raise ValueError(f"{name}: expected a contiguous {kind} tensor of shape {shape} on {dev}, got "
                                     f"{t.dtype} {tuple(t.shape)} on {t.device}")
        self.fmt, self.block, self.batch, self.heads, self.cap, self.head_dim = fmt, block, B, H, cap, D
        self.dtype, self.device = dtype, dev
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.k_tail, self.v_tail = k_tail, v_tail
        self.desc = _STORE.pack(k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                                k_tail.data_ptr(), v_tail.data_ptr(), cap, FORMATS[fmt][0], D, block, _lib.dtype_code(dtype),
                                B, H)

    def tensors(self) -> dict:
        """The arrays by the names that ``from_tensors`` takes."""
        return {n: getattr(self, n) for n in ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail")}

    def sequence(self, b: int) -> "KV8Store":
        """The store of sequence ``b`` alone (the same memory)."""
        return KV8Store.from_tensors(self.fmt, **{n: t[b:b + 1] for n, t in self.tensors().items()})

    def grown(self, capacity: int) -> "KV8Store":
        """A store with room for ``capacity`` tokens that holds this one's."""
        new = KV8Store(self.batch, self.heads, self.head_dim, capacity, self.fmt, self.block, self.dtype, self.device)
        if new.cap < self.cap:
            raise ValueError(f"{capacity} tokens < the {self.cap} there is room for")
        for name, t in self.tensors().items():
            d = getattr(new, name)
            if t.element_size() == 1:
                t, d = t.view(torch.uint8), d.view(torch.uint8)
            d[:, :, :t.shape[2]].copy_(t)
        return new

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.tensors().values())


def _check(fmt: str, head_dim: int, block: int, dtype) -> None:
    if fmt not in FORMATS:
        raise ValueError(f"format {fmt!r}: use one of {sorted(FORMATS)}")
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim {head_dim} not supported: use one of {HEAD_DIMS}")
    if block not in BLOCKS:
        raise ValueError(f"blocks of {block} tokens not supported: use one of {BLOCKS}")
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"keys and values of {dtype} not supported: fp16 or bf16")


_devices: set[torch.device] = set()


def _ready(device: torch.device) -> None:
    """Refuse what is not a gfx950 device (looked up once per device)."""
    if device not in _devices:
        if device.type != "cuda":
            raise RuntimeError("turboquant_amd runs on the GPU only; got a CPU tensor")
        _codec._require_gfx950(device)
        _devices.add(device)


def kv8_write(store: KV8Store, keys: torch.Tensor, values: torch.Tensor, start, n_new: torch.Tensor | None = None) -> None:
    """Write keys / values (B, H, T, D) as tokens start .. start + T - 1 of
    their sequences, which hold ``start`` tokens: blocks that become complete
    are quantised, the rest of the tokens goes to the tail, in one launch.

    ``start``: an int, or an int32 device tensor (B,). ``n_new``: None (T for
    all), or an int32 device tensor (B,): sequence b takes its first n_new[b]
    tokens (0 to T); the others are not read. Device values are not checked on
    the host: a sequence whose tokens would not fit, or whose start or count is
    negative (or n_new > T), is left as it is."""
    B, H, D = store.batch, store.heads, store.head_dim
    T = keys.shape[2] if keys.dim() == 4 else 0
    for name, t in (("keys", keys), ("values", values)):
        if t.shape != (B, H, T, D):
            raise ValueError(f"{name}: expected ({B}, {H}, T, {D}) like the store, one T for both, got {tuple(t.shape)}")
        if t.dtype != store.dtype or t.device != store.device:
            raise ValueError(f"{name}: expected {store.dtype} on {store.device}, got {t.dtype} on {t.device}")
    if T > store.cap:
        raise ValueError(f"{T} tokens > the {store.cap} there is room for")
    start_b, s0 = _lengths(start, B, store.cap - T, store.device, "start")
    if n_new is not None and not isinstance(n_new, torch.Tensor):
        raise ValueError("n_new: None, or an int32 tensor of one count per sequence")
    count_b = 0 if n_new is None else _lengths(n_new, B, T, store.device, "n_new")[0]
    if T == 0 or B == 0:
        return
    _ready(store.device)
    (k, keys), (v, values) = _rows4(keys), _rows4(values)
    lib = _lib.load()
    with _on(store.device):
        _lib.check(lib.tq_kv8_write(store.desc, _ROWS.pack(*k), _ROWS.pack(*v), start_b, s0, count_b, T,
                                    _lib.stream_ptr(store.device)), "tq_kv8_write")


def kv8_read(store: KV8Store, lens, start: int = 0, n: int | None = None,
             dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of tokens start .. start + n - 1 as dense (B, H, n, D)
    tensors of ``dtype`` (fp16, bf16 or float32; the store's by default): code
    * scale in float32, rounded once.

    ``lens``: the tokens held, an int or an int32 device tensor (B,); ``n``
    defaults to what is held from ``start`` on (a tensor's ``lens``: to the
    store's end). Tokens at or past a sequence's length are 0."""
    B, H, D = store.batch, store.heads, store.head_dim
    len_b, length = _lengths(lens, B, store.cap, store.device, "lens")
    if n is None:
        n = max(0, (store.cap if len_b else length) - start)
    if start < 0 or n < 0 or start + n > store.cap:
        raise ValueError(f"tokens {start} .. {start + n - 1} outside the store's {store.cap}")
    dtype = store.dtype if dtype is None else dtype
    code = _lib.dtype_code(dtype)
    k = torch.empty(B, H, n, D, dtype=dtype, device=store.device)
    v = torch.empty_like(k)
    if n == 0 or B == 0:
        return k, v
    _ready(store.device)
    lib = _lib.load()
    with _on(store.device):
        _lib.check(lib.tq_kv8_read(store.desc, len_b, length, start, n, code, k.data_ptr(), v.data_ptr(),
                                   _lib.stream_ptr(store.device)), "tq_kv8_read")
    return k, v


def _attention_desc(queries, B, hkv, D, dtype, device, len_b, max_len, scale, window, sinks, out, k=_NO_ROWS, v=_NO_ROWS):
    """(``tq_kv_attn_desc`` as bytes, output, tensor to keep until the launch) of an attention call."""
    q = queries[:, :, None] if queries.dim() == 3 else queries
    shape = q.shape
    if len(shape) != 4 or shape[0] != B or shape[3] != D or shape[1] % hkv or shape[1] == 0:
        raise ValueError(f"query shape {tuple(queries.shape)} does not match {B} sequences of {hkv} kv heads, head_dim {D}")
    if q.dtype != dtype or q.device != device:
        raise ValueError(f"queries: expected {dtype} on {device}, got {q.dtype} on {q.device}")
    if window is not None and window < 1:
        raise ValueError(f"window {window}: at least 1, or None")
    if sinks < 0:
        raise ValueError(f"sinks {sinks}")
    code = out_code = _lib.dtype_code(dtype)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(shape, dtype=dtype, device=device)
        o = (out.data_ptr(), *out.stride()[:3])
    else:
        if out.shape != shape or out.dtype not in (dtype, torch.float32) or out.device != device:
            raise ValueError(f"out: expected {tuple(shape)} of {dtype} or float32 on {device}")
        o, same = _rows4(out)
        if same is not out or _overlaps(out):
            raise ValueError("out: rows must be contiguous, 16-byte aligned and apart, strides multiples of 8")
        out_code = _lib.dtype_code(out.dtype)
    rows, q = _rows4(q)
    desc = _DESC.pack(B, shape[1], hkv, D, shape[2], code, out_code, 0 if window is None else min(window, _MOST),
                      min(sinks, _MOST), max_len, len_b, D ** -0.5 if scale is None else scale, *rows, *o, *k, *v)
    return desc, out, q


_MOST = 2 ** 31 - 1


def kv8_attention(queries: torch.Tensor, store: KV8Store, lens, max_len: int | None = None, scale: float | None = None,
                  window: int | None = None, sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each sequence's last T_q tokens over its cache, scoring the
    8-bit codes directly.

    ``queries`` (B, Hq, T_q, D), or (B, Hq, D) for T_q = 1, of the store's
    type; Hq a multiple of the kv heads, query head h reads kv head
    h // (Hq / Hkv). ``lens``: tokens in the cache, an int or an int32 device
    tensor (B,), then with ``max_len`` its bound (default: the store's room;
    larger lengths are cut to it). Query i sits at position lens - T_q + i and
    sees the tokens up to its own; with ``window``, of those the last
    ``window`` and the first ``sinks``. A query before position 0 (an empty
    sequence, or one shorter than T_q) gives 0. Default scale D**-0.5.

    Returns (B, Hq, T_q, D) of the queries' type, or ``out`` (that type or
    float32, any strides that are multiples of 8; the queries
    themselves may be given). Scores, softmax and sums are
    float32; the softmax's weights are rounded to 16 bits. (Sums of query times
    code must stay in float32's range: with more than 16 query rows per kv head,
    bf16 queries below 2**112.)"""
    D, B, H = store.head_dim, store.batch, store.heads
    len_b, length = _lengths(lens, B, store.cap, store.device, "lens")
    if len_b:
        length = store.cap if max_len is None else int(max_len)
        if not 0 <= length <= store.cap:
            raise ValueError(f"max_len {length} outside [0, {store.cap}]")
    desc, out, q = _attention_desc(queries, B, H, D, store.dtype, store.device, len_b, length, scale, window, sinks, out)
    if out.numel() == 0:
        return out
    _ready(store.device)
    lib = _lib.load()
    with _on(store.device):
        need = lib.tq_kv8_attention_workspace_bytes(store.desc, desc)
        # its own block per call: calls on other streams and captured graphs share nothing
        ws = torch.empty(need, dtype=torch.uint8, device=store.device) if need else None
        _lib.check(lib.tq_kv8_attention(store.desc, desc, _lib.ptr(ws), need,
                                        _lib.stream_ptr(store.device)), "tq_kv8_attention")
    return out


class KV8Cache:
    """8-bit KV cache of one layer with the protocol of ``TurboQuantKVCache``
    (cache.py:19-724): sequences of one length, storage that grows in steps of
    4096 tokens. ``window`` / ``sinks``: what ``attend`` sees by default (a
    sliding-window layer); every token is kept."""

    GROW = 4096

    def __init__(self, head_dim: int = 128, num_kv_heads: int = 1, fmt: str = "int8", block: int = 32,
                 window: int | None = None, sinks: int = 0, device=None):
        _check(fmt, head_dim, block, torch.float16)
        if window is not None and window < 1:
            raise ValueError(f"window {window}: at least 1, or None")
        if sinks < 0:
            raise ValueError(f"sinks {sinks}")
        self.head_dim, self.num_kv_heads = head_dim, num_kv_heads
        self.fmt, self.block = fmt, block
        self.window, self.sinks = window, sinks
        self._device = torch.device(device) if device is not None else None
        self._store: KV8Store | None = None
        self._pending: dict | None = None  # meta_state set before state
        self.offset = 0

    @property
    def store(self) -> KV8Store | None:
        return self._store

    def _reserve(self, keys: torch.Tensor, n: int) -> None:
        if self._store is None:
            B, H, _, D = keys.shape
            if D != self.head_dim:
                raise ValueError(f"head_dim {D} != cache head_dim {self.head_dim}")
            _lib.require_device(keys)
            self._store = KV8Store(B, H, D, (n + self.GROW - 1) // self.GROW * self.GROW, self.fmt, self.block, keys.dtype,
                                   keys.device)
        elif n > self._store.cap:
            cap = max(n, self._store.cap + self._store.cap // 2)
            self._store = self._store.grown((cap + self.GROW - 1) // self.GROW * self.GROW)

    def update(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Append keys / values (B, H, T, D), fp16 or bf16."""
        if keys.shape != values.shape or keys.dim() != 4:
            raise ValueError("keys and values must have the same shape (B, H, T, D)")
        T = keys.shape[2]
        if T == 0:
            return
        if self._store is not None and keys.dtype != self._store.dtype:
            keys, values = keys.to(self._store.dtype), values.to(self._store.dtype)
        self._reserve(keys, self.offset + T)
        kv8_write(self._store, keys, values, self.offset)
        self.offset += T

    def fetch(self, dtype: torch.dtype | None = None) -> tuple[torch.Tensor | None, torch.Tensor | None]:
        """Every key and value (B, H, offset, D), in the cache's 16-bit type by default."""
        if self._store is None:
            return None, None
        return kv8_read(self._store, self.offset, dtype=dtype)

    def update_and_fetch(self, keys: torch.Tensor, values: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Append and return all keys / values for attention, in 16 bits."""
        self.update(keys, values)
        if self._store is None:
            return keys[:, :, :0], values[:, :, :0]
        return self.fetch()

    def attend(self, queries: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None,
               window: int | None = None, sinks: int | None = None) -> torch.Tensor:
        """Causal attention of the cache's last T_q tokens over it
        (``kv8_attention``): queries (B, Hq, T_q, D) or (B, Hq, D), the result
        (B, Hq, T_q, D) in the queries' type. ``window`` and ``sinks`` default
        to the cache's."""
        if self._store is None or self.offset == 0:
            raise ValueError("attend() on an empty cache")
        q = queries if queries.dim() == 4 else queries[:, :, None]
        if q.shape[2] > self.offset:
            raise ValueError(f"{q.shape[2]} query tokens > the {self.offset} cached tokens")
        return kv8_attention(q, self._store, self.offset, scale=scale, window=self.window if window is None else window,
                             sinks=self.sinks if sinks is None else sinks, out=out)

    # ------------------------------------------------------------- protocol
    @property
    def keys(self):
        return self.fetch()[0]

    @property
    def values(self):
        return self.fetch()[1]

    @property
    def state(self) -> tuple:
        """(k_codes, v_codes, k_scales, v_scales, k_tail, v_tail), copies of
        what the cached tokens take, or six None for an empty cache."""
        if self._store is None:
            return (None,) * 6
        tiles, blocks = -(-self.offset // TILE), -(-self.offset // self.block)
        s = self._store
        cut = lambda t, n: t[:, :, :n].clone()
        return (cut(s.k_codes, tiles * TILE), cut(s.v_codes, tiles), cut(s.k_scales, blocks), cut(s.v_scales, blocks),
                s.k_tail.clone(), s.v_tail.clone())

    @state.setter
    def state(self, v) -> None:
        """Load a saved tuple. The length comes from a meta_state set before or
        after; without one, it is the whole blocks saved."""
        if len(v) != 6:
            raise ValueError(f"state tuple of {len(v)} entries; expected 6")
        if all(x is None for x in v):
            self._store, self.offset = None, 0
            return
        kc, vc, ks, vs, kt, vt = v
        B, H, cap, D = kc.shape
        if D != self.head_dim or kt.shape[2] != self.block or kc.dtype != FORMATS[self.fmt][1]:
            raise ValueError(f"saved state of head_dim {D}, blocks of {kt.shape[2]}, {kc.dtype} does not match this cache")
        dev = self._device if self._device is not None else kc.device
        new = KV8Store(B, H, D, cap, self.fmt, self.block, kt.dtype, dev)
        blocks = ks.shape[2]
        if vc.shape != new.v_codes.shape or vs.shape != ks.shape or not 0 <= blocks <= new.k_scales.shape[2]:
            raise ValueError("saved state: shapes do not belong together")
        new.k_codes.view(torch.uint8).copy_(kc.view(torch.uint8))
        new.v_codes.view(torch.uint8).copy_(vc.view(torch.uint8))
        new.k_scales[:, :, :blocks].copy_(ks)
        new.v_scales[:, :, :blocks].copy_(vs)
        new.k_tail.copy_(kt)
        new.v_tail.copy_(vt)
        self._store = new
        self.offset = blocks * self.block
        if self._pending is not None:
            meta, self._pending = self._pending, None
            self.meta_state = meta

    @property
    def meta_state(self) -> dict:
        return {"offset": str(self.offset), "head_dim": str(self.head_dim), "fmt": self.fmt, "block": str(self.block)}

    @meta_state.setter
    def meta_state(self, v) -> None:
        if v.get("fmt", self.fmt) != self.fmt or int(v.get("block", self.block)) != self.block:
            raise ValueError("meta_state of another format or block size")
        n = int(v["offset"])
        if self._store is None:
            self._pending = dict(v)
            return
        held = self.offset
        if not 0 <= n <= held or (n + self.block - 1) // self.block * self.block != held:
            raise ValueError(f"meta_state offset {n} does not belong to a state of {held} tokens in whole blocks")
        self.offset = n

    def make_mask(self, N: int, offset: int = 0, return_array: bool = False, window_size: int | None = None):
        """None for single-token decode, "causal" otherwise; the window of a
        windowed cache is ``attend``'s."""
        return None if N == 1 and not return_array else "causal"

    def empty(self) -> bool:
        return self.offset == 0

    def is_trimmable(self) -> bool:
        return False

    def size(self) -> int:
        return self.offset

    @property
    def nbytes(self) -> int:
        """Bytes that the cached tokens take: codes and scales of the complete
        blocks, and the tail."""
        if self._store is None:
            return 0
        s, full = self._store, self.offset // self.block
        rows = s.batch * s.heads
        return 2 * rows * (full * (self.block * self.head_dim + 4) + (self.offset - full * self.block) * self.head_dim * 2)


class KV8Batch:
    """``batch`` sequences of different lengths of one layer, held in 8 bits:
    ``load`` fills a sequence, ``step`` appends one token to each,
    ``attend`` is the step's attention. ``offset`` (numpy) and ``lens`` (device
    int32) are the lengths; other code only reads them."""

    def __init__(self, batch: int, num_kv_heads: int, head_dim: int = 128, fmt: str = "int8", block: int = 32,
                 capacity: int = 4096, dtype: torch.dtype = torch.float16, window: int | None = None, sinks: int = 0,
                 device=None):
        if window is not None and window < 1:
            raise ValueError(f"window {window}: at least 1, or None")
        if sinks < 0:
            raise ValueError(f"sinks {sinks}")
        self.store = KV8Store(batch, num_kv_heads, head_dim, capacity, fmt, block, dtype, device)
        self.window, self.sinks = window, sinks
        self.offset = np.zeros(batch, dtype=np.int64)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=self.store.device)

    def reserve(self, tokens: int) -> None:
        """Room for ``tokens`` tokens per sequence."""
        if tokens > self.store.cap:
            cap = max(tokens, self.store.cap + self.store.cap // 2)
            self.store = self.store.grown((cap + KV8Cache.GROW - 1) // KV8Cache.GROW * KV8Cache.GROW)

    def load(self, b: int, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Append (H, T, D) keys / values to sequence ``b`` (a prompt, or a
        chunk of one)."""
        if keys.dim() != 3 or keys.shape != values.shape:
            raise ValueError("keys / values must be (num_kv_heads, T, head_dim)")
        if not 0 <= b < self.store.batch:
            raise ValueError(f"sequence {b} of {self.store.batch}")
        T, at = keys.shape[1], int(self.offset[b])
        self.reserve(at + T)
        s = self.store
        kv8_write(s.sequence(b), keys[None].to(s.device, s.dtype), values[None].to(s.device, s.dtype), at)
        self.offset[b] += T
        self.lens[b:b + 1].fill_(int(self.offset[b]))

    def step(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Append one token per sequence ((B, H, D) keys / values)."""
        s = self.store
        if keys.shape != (s.batch, s.heads, s.head_dim) or values.shape != keys.shape:
            raise ValueError("keys / values must be (batch, num_kv_heads, head_dim)")
        self.reserve(int(self.offset.max(initial=0)) + 1)
        s = self.store
        kv8_write(s, keys[:, :, None].to(s.device, s.dtype), values[:, :, None].to(s.device, s.dtype), self.lens)
        self.lens += 1
        self.offset += 1

    def attend(self, q: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of each sequence's last token(s) over its own tokens: q
        (B, Hq, D), the result (B, Hq, D), or (B, Hq, T_q, D) for both. An
        empty sequence gives 0."""
        o = out[:, :, None] if out is not None and q.dim() == 3 else out
        o = kv8_attention(q, self.store, self.lens, int(self.offset.max(initial=0)), scale, self.window, self.sinks, o)
        return o[:, :, 0] if q.dim() == 3 else o
