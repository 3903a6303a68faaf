"""The operators of the 8-bit KV cache and of windowed attention, as cases that can be timed and compared.

A case is a dict of plain values. Its "kind" names the call:

- store   a prompt's keys and values quantised into an 8-bit cache as they are written, and read back in 16 bits for the
          prompt's own attention (what update_and_fetch does);
- read    a filled cache read back;
- step    one decode step of a batch: each sequence's new token is written (a block of tokens that it completes is
          quantised), then one query token per head attends over the cache;
- chunk   causal attention of several query tokens per sequence over a filled cache (`window` > 0: each sees the last
          `window` tokens and the first `sinks`);
- window  attention over uncompressed keys and values, each query seeing the last `window` tokens and the first `sinks`
          (`window` 0: every earlier token).

The cache: tokens of complete blocks in 8 bits (int8, or e4m3) with one float32 scale for each block of tokens and head,
those of the last, incomplete block in 16 bits. Key codes are (batch, heads, tokens, d); value codes are held transposed
in tiles of 64 tokens, (batch, heads, tokens / 64, d, 64).

Keys are N(0, 1) times a per-channel LogNormal(0, 0.5) factor (key channels differ in scale in trained models), values
N(0, 1), queries N(0, 1) times 1.5 (scores then spread over several units, as attention scores do).
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
QMAX = {"int8": 127.0, "fp8": 448.0}
CODE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TILE = 64
TINY = 2.0 ** -110


def listed():
    return [
        # a long prompt of an 8B-class layer into a new cache
        dict(name="store_prompt_8k", kind="store", dtype="bf16", fmt="int8", block=32, d=128, hkv=8, batch=1, tokens=8192,
             start=0, ragged=False),
        # prompts of different lengths, appended to cached prefixes; odd sizes
        dict(name="store_ragged_odd", kind="store", dtype="fp16", fmt="fp8", block=16, d=96, hkv=3, batch=5, tokens=777,
             start=48, ragged=True),
        # a whole 32K context read back
        dict(name="read_32k", kind="read", dtype="bf16", fmt="int8", block=32, d=128, hkv=8, batch=1, tokens=32768,
             ragged=False),
        # sequences of different lengths with incomplete blocks, head_dim 64
        dict(name="read_ragged_odd", kind="read", dtype="fp16", fmt="fp8", block=64, d=64, hkv=4, batch=6, tokens=2011,
             ragged=True),
        # the smallest decode step: a short request on a small grouped-query layer, latency only
        dict(name="step_small", kind="step", dtype="bf16", fmt="int8", block=32, d=64, hkv=2, hq=8, batch=1, tokens=401,
             ragged=False),
        # a serving step: 32 sequences of different lengths on an 8B-class layer
        dict(name="step_batch32", kind="step", dtype="bf16", fmt="int8", block=32, d=128, hkv=8, hq=32, batch=32,
             tokens=16384, ragged=True),
        # one sequence's step over a 128K context
        dict(name="step_fp8_128k", kind="step", dtype="fp16", fmt="fp8", block=64, d=128, hkv=8, hq=32, batch=1,
             tokens=131071, ragged=False),
        # a few drafted tokens verified at once, head_dim 256
        dict(name="verify_d256", kind="chunk", dtype="bf16", fmt="int8", block=16, d=256, hkv=4, hq=8, batch=8, n_q=4,
             tokens=4097, window=0, sinks=0, ragged=True),
        # a prompt chunk over a long cached context: the largest work
        dict(name="chunk_2k_32k", kind="chunk", dtype="bf16", fmt="int8", block=32, d=128, hkv=8, hq=32, batch=1, n_q=2048,
             tokens=32768, window=0, sinks=0, ragged=False),
        # a windowed layer's prompt chunk over an 8-bit cache; 14 heads on 2, odd sizes
        dict(name="chunk_window_odd", kind="chunk", dtype="fp16", fmt="fp8", block=32, d=64, hkv=2, hq=14, batch=3, n_q=999,
             tokens=5003, window=512, sinks=4, ragged=True),
        # a windowed layer's whole prompt, uncompressed
        dict(name="window_prompt_8k", kind="window", dtype="bf16", d=128, hkv=8, hq=32, batch=1, n_q=8192, tokens=8192,
             window=1024, sinks=4, ragged=False),
        # a windowed layer's decode step, uncompressed, 16 sequences
        dict(name="window_decode", kind="window", dtype="fp16", d=128, hkv=8, hq=32, batch=16, n_q=1, tokens=16384,
             window=4096, sinks=16, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "read", "step", "step", "chunk", "chunk", "window", "window"])
    c = dict(kind=kind, dtype=rng.choice(["fp16", "bf16"]), d=rng.choice([64, 96, 128, 128, 256]),
             hkv=rng.choice([1, 2, 3, 4, 8]), batch=_log(rng, 1, 24))
    if kind != "window":
        c.update(fmt=rng.choice(["int8", "fp8"]), block=rng.choice([16, 32, 64]))
    most = 4e8 if kind in ("step", "window") else 2e8  # elements of the keys
    fits = lambda n: max(1, min(n, int(most / (c["batch"] * c["hkv"] * c["d"]))))  # noqa: E731
    if kind in ("store", "read"):
        c["tokens"] = fits(_log(rng, 1, 20000))
        if kind == "store":
            c["start"] = c["block"] * rng.randrange(9)
    else:
        c["hq"] = c["hkv"] * rng.choice([1, 2, 3, 4, 7, 8])
        c["tokens"] = fits(_log(rng, 1, 60000))
        if kind != "step":
            c["n_q"] = 1 if kind == "window" and rng.random() < 0.4 else min(c["tokens"], _log(rng, 2, 2048))
            c["window"] = rng.choice([0, 0, _log(rng, 1, 4096)]) if kind == "chunk" else _log(rng, 1, 8192)
            c["sinks"] = rng.choice([0, 1, 4, 16, 100]) if c["window"] else 0
            pairs = c["batch"] * c["hq"] * c["n_q"] * c["tokens"]
            if pairs > 2.0e9:  # the scores of the largest listed case
                c["tokens"] = max(1, int(c["tokens"] * 2.0e9 / pairs))
                c["n_q"] = min(c["n_q"], c["tokens"])
    c["ragged"] = c["batch"] > 1 and rng.random() < 0.6
    return c


# ------------------------------------------------------------------ inputs
def _lens(case, gen):
    """One length per sequence: `tokens` in the first, and between 1 and `tokens` in the others of a ragged batch."""
    n = torch.full((case["batch"],), case["tokens"], dtype=torch.int32)
    if case["ragged"]:
        u = torch.rand(case["batch"], generator=gen)
        n[1:] = (1 + u * (case["tokens"] - 1)).to(torch.int32)[1:]
    return n


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _kv(case, gen, T):
    B, H, D, dt = case["batch"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    chan = torch.exp(0.5 * _randn(gen, 1, H, 1, D))
    return (_randn(gen, B, H, T, D) * chan).to(dt), _randn(gen, B, H, T, D).to(dt)


def _round_up(n, m):
    return (n + m - 1) // m * m


def _quantise(x, fmt, block):
    """(codes, scales) of (B, H, T, D), T a multiple of block."""
    B, H, T, D = x.shape
    x = x.float().view(B, H, T // block, block * D)
    a = x.abs().amax(-1, keepdim=True)
    dead = ~(a >= TINY) | ~torch.isfinite(a)  # too small to divide by, or infinite or NaN: codes of 0
    top = torch.full_like(a, QMAX[fmt])  # a tensor: torch divides by, and takes the inverse of, a number in two roundings
    s = torch.where(dead, torch.where(a < TINY, 0.0, torch.nan), a / top)
    y = torch.where(dead, 0.0, x * (top / torch.where(dead, 1.0, a)))
    y = torch.round(y).to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)
    return y.view(B, H, T, D), s.squeeze(-1)


def _moved(t, f):
    """f of an 8-bit tensor's bytes."""
    return f(t.view(torch.uint8)).contiguous().view(t.dtype)


def _tiled(codes):
    """Value codes (B, H, T, D) as (B, H, T / 64, D, 64)."""
    B, H, T, D = codes.shape
    return _moved(codes, lambda u: u.view(B, H, T // TILE, TILE, D).transpose(-1, -2))


def _untiled(codes):
    B, H, N, D, _ = codes.shape
    return _moved(codes, lambda u: u.transpose(-1, -2).reshape(B, H, N * TILE, D))


def _rows(x, pos):
    """x (B, H, T, D) at token positions pos (B, n)."""
    B, H, T, D = x.shape
    return x.gather(2, pos.clamp(0, T - 1).view(B, 1, -1, 1).expand(B, H, pos.shape[1], D))


def _filled(case, gen, lens, room):
    """A cache that holds the first lens tokens of drawn keys and values, with room for `room` in all."""
    block, cap = case["block"], _round_up(room, TILE)
    k, v = _kv(case, gen, cap)
    kq, ks = _quantise(k, case["fmt"], block)
    vq, vs = _quantise(v, case["fmt"], block)
    tail = (lens // block * block).view(-1, 1) + torch.arange(block, device=DEV)
    return dict(k_codes=kq, v_codes=_tiled(vq), k_scales=ks, v_scales=vs, k_tail=_rows(k, tail), v_tail=_rows(v, tail))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    kind, B, H, D = case["kind"], case["batch"], case["hkv"], case["d"]
    dt = DTYPES[case["dtype"]]
    n = _lens(case, host)
    lens = n.to(DEV)
    s = dict(case=case, lens=lens, max_len=int(n.max()))
    if kind == "store":
        # the prompts begin at a block's first token: a pass can then be repeated on the same cache
        room, block = case["start"] + case["tokens"], case["block"]
        cap = _round_up(room, TILE)
        s["keys"], s["values"] = _kv(case, gen, case["tokens"])
        s["start"] = torch.full((B,), case["start"], dtype=torch.int32, device=DEV)
        s["after"] = s["start"] + lens
        s["max_len"] = room
        if case["start"]:
            s["store"] = _filled(case, gen, s["start"], room)
        else:
            s["store"] = dict(
                k_codes=torch.zeros(B, H, cap, D, dtype=torch.uint8, device=DEV).view(CODE[case["fmt"]]),
                v_codes=torch.zeros(B, H, cap // TILE, D, TILE, dtype=torch.uint8, device=DEV).view(CODE[case["fmt"]]),
                k_scales=torch.zeros(B, H, cap // block, device=DEV), v_scales=torch.zeros(B, H, cap // block, device=DEV),
                k_tail=torch.zeros(B, H, block, D, dtype=dt, device=DEV),
                v_tail=torch.zeros(B, H, block, D, dtype=dt, device=DEV))
    elif kind == "read":
        s["store"] = _filled(case, gen, lens, case["tokens"])
    elif kind == "step":
        # the cache holds lens tokens; the step's token is the one after them
        s["store"] = _filled(case, gen, lens, case["tokens"] + 1)
        s["keys"], s["values"] = _kv(case, gen, 1)
        s["q"] = (1.5 * _randn(gen, B, case["hq"], 1, D)).to(dt)
        s["after"] = lens + 1
        s["max_len"] += 1
    elif kind == "chunk":
        s["store"] = _filled(case, gen, lens, case["tokens"])
        s["q"] = (1.5 * _randn(gen, B, case["hq"], case["n_q"], D)).to(dt)
    else:
        s["keys"], s["values"] = _kv(case, gen, case["tokens"])
        s["q"] = (1.5 * _randn(gen, B, case["hq"], case["n_q"], D)).to(dt)
    return s


# ------------------------------------------------------------- plain forms
def _write(store, fmt, block, keys, values, start, n_new):
    """Tokens start .. start + n_new - 1 of each sequence into the cache, in place."""
    B, H, T, D = keys.shape
    cap = store["k_codes"].shape[2]
    start, end = start.long().view(B, 1), (start + n_new).long().view(B, 1)
    pos = torch.arange(cap, device=keys.device).view(1, cap)
    held = start // block * block  # the incomplete block's first position before, and after
    kept = end // block * block
    first = torch.arange(cap // block, device=keys.device).view(1, -1) * block
    done = ((first >= held) & (first + block <= end)).view(B, 1, -1, 1)
    for_tail = kept + torch.arange(block, device=keys.device).view(1, block)
    in_tail = ((for_tail >= start) & (for_tail < end)).view(B, 1, block, 1)

    def side(new, codes, scales, tail, tiled):
        at = lambda p: torch.where((p >= start).view(B, 1, -1, 1), _rows(new, p - start), _rows(tail, p - held))  # noqa: E731
        q, s = _quantise(at(pos), fmt, block)
        old = _untiled(codes) if tiled else codes
        q = torch.where(done, q.view(torch.uint8).view(B, H, -1, block * D), old.view(torch.uint8).reshape(B, H, -1, block * D))
        q = q.view(B, H, cap, D).view(codes.dtype)
        tail_now = torch.where(in_tail, at(for_tail), tail)
        codes.view(torch.uint8).copy_((_tiled(q) if tiled else q).view(torch.uint8))
        scales.copy_(torch.where(done.squeeze(-1), s, scales))
        tail.copy_(tail_now)

    side(keys, store["k_codes"], store["k_scales"], store["k_tail"], False)
    side(values, store["v_codes"], store["v_scales"], store["v_tail"], True)


def _read(store, block, lens):
    """Every token's key and value in float32, and 0 past each sequence's length."""
    B, H, cap, D = store["k_codes"].shape
    lens = lens.long().view(B, 1)
    pos = torch.arange(cap, device=lens.device).view(1, cap)
    held = lens // block * block

    def side(codes, scales, tail):
        x = codes.float().view(B, H, cap // block, block, D) * scales.view(B, H, -1, 1, 1)
        x = torch.where((pos < held).view(B, 1, cap, 1), x.view(B, H, cap, D), _rows(tail, pos - held).float())
        return torch.where((pos < lens).view(B, 1, cap, 1), x, 0.0)

    return (side(store["k_codes"], store["k_scales"], store["k_tail"]),
            side(_untiled(store["v_codes"]), store["v_scales"], store["v_tail"]))


def _attend(q, k, v, lens, window, sinks):
    """Causal attention of the last n of each sequence's tokens, k and v in float32; rows that see nothing give 0."""
    B, hq, n, D = q.shape
    H, T = k.shape[1], k.shape[2]
    at = lens.long().view(B, 1, 1) - n + torch.arange(n, device=q.device).view(1, n, 1)
    t = torch.arange(T, device=q.device).view(1, 1, T)
    sees = t <= at
    if window:
        sees = sees & ((t > at - window) | (t < sinks))
    s = torch.matmul(q.float().reshape(B, H, hq // H * n, D), k.transpose(-1, -2).contiguous()) * D ** -0.5
    s = s.view(B, H, hq // H, n, T)
    sees = sees.view(B, 1, 1, n, T)
    s = s.masked_fill(~sees, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    o = torch.matmul(p.view(B, H, hq // H * n, T), v) / p.sum(-1).view(B, H, -1, 1)
    o = o.view(B, hq, n, D)
    return torch.where((at >= 0).view(B, 1, n, 1), o, 0.0).to(q.dtype)


def run(state):
    c, st = state["case"], state.get("store")
    kind, dt = c["kind"], DTYPES[c["dtype"]]
    if own:
        at = os.path.abspath("mlx-turboquant_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        from turboquant_amd import KV8Store, kv8_attention, kv8_read, kv8_write, window_attention
        if kind == "window":
            return window_attention(state["q"], state["keys"], state["values"], window=c["window"] or None, sinks=c["sinks"],
                                    lens=state["lens"])
        store = KV8Store.from_tensors(c["fmt"], **st)
        if kind == "store":
            kv8_write(store, state["keys"], state["values"], state["start"], state["lens"])
            k, v = kv8_read(store, state["after"], n=state["max_len"])
            return dict(k=k, v=v, k_scales=st["k_scales"], v_scales=st["v_scales"], k_tail=st["k_tail"], v_tail=st["v_tail"])
        if kind == "read":
            return kv8_read(store, state["lens"], n=state["max_len"])
        if kind == "step":
            kv8_write(store, state["keys"], state["values"], state["lens"])
            o = kv8_attention(state["q"], store, state["after"], max_len=state["max_len"])
            return dict(o=o, k_scales=st["k_scales"], v_scales=st["v_scales"], k_tail=st["k_tail"], v_tail=st["v_tail"])
        return kv8_attention(state["q"], store, state["lens"], max_len=state["max_len"], window=c["window"] or None,
                             sinks=c["sinks"])
    if kind == "window":
        return _attend(state["q"], state["keys"].float(), state["values"].float(), state["lens"], c["window"], c["sinks"])
    m = state["max_len"]
    if kind in ("store", "step"):
        _write(st, c["fmt"], c["block"], state["keys"], state["values"], state["start"] if kind == "store" else state["lens"],
               state["lens"] if kind == "store" else torch.ones_like(state["lens"]))
        k, v = _read(st, c["block"], state["after"])
        new = dict(k_scales=st["k_scales"], v_scales=st["v_scales"], k_tail=st["k_tail"], v_tail=st["v_tail"])
        if kind == "store":
            return dict(k=k[:, :, :m].to(dt), v=v[:, :, :m].to(dt), **new)
        return dict(o=_attend(state["q"], k[:, :, :m], v[:, :, :m], state["after"], 0, 0), **new)
    k, v = _read(st, c["block"], state["lens"])
    if kind == "read":
        return k[:, :, :m].to(dt), v[:, :, :m].to(dt)
    return _attend(state["q"], k[:, :, :m], v[:, :, :m], state["lens"], c["window"], c["sinks"])


def work(case):
    """Lengths of a ragged batch are uniform over their range: half the longest on average."""
    B, H, D, T = case["batch"], case["hkv"], case["d"], case["tokens"]
    T = T if not case["ragged"] else (T + (B - 1) * T / 2) / B
    kind = case["kind"]
    cached = D + 4.0 / case["block"] if kind != "window" else 2.0 * D  # bytes of a token's key (or value) of one head
    if kind == "store":  # 16 bits in, 8 out, and back
        return {"bytes": 2 * B * H * (T * (2 * D + cached) + (T + case["start"]) * (cached + 2 * D)), "flops": 4.0 * B * H * T * D}
    if kind == "read":
        return {"bytes": 2 * B * H * T * (cached + 2 * D), "flops": 2.0 * B * H * T * D}
    n, hq = case.get("n_q", 1), case["hq"]
    w = case.get("window", 0)
    i = torch.arange(max(0, int(T) - n), max(1, int(T)), dtype=torch.float64) + 1  # tokens up to each query's own
    sees = torch.minimum(i, w + torch.clamp(i - w, 0, case["sinks"])) if w else i
    read = min(T, n + w + case["sinks"]) if w else T
    return {"bytes": 2.0 * B * H * read * cached + 4.0 * B * hq * n * D, "flops": 4.0 * D * B * hq * float(sees.sum())}


# ------------------------------------------------------------------- exact
def _e4m3(y):
    """float64 rounded to the nearest e4m3 value, ties to even."""
    e = torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 1
    step = torch.pow(2.0, (e - 3).double())
    return (torch.round(y / step) * step).clamp(-448, 448)


def _exact_block(x, fmt):
    """(values that a block of tokens (H, block, D) reads back as, scales (H,)) in float64."""
    scale = x.abs().amax((-1, -2), keepdim=True) / QMAX[fmt]
    y = x / torch.where(scale > 0, scale, 1.0)
    y = torch.round(y) if fmt == "int8" else _e4m3(y)
    return y * scale, scale[:, 0, 0]


def _exact_cached(store, b, n, block):
    """Keys and values (H, n, D) in float64 of the first n tokens of sequence b."""
    D = store["k_codes"].shape[-1]
    full = n // block * block
    vt = store["v_codes"][b].view(torch.uint8).permute(0, 1, 3, 2).reshape(store["v_codes"].shape[1], -1, D)
    out = []
    for codes, scales, tail in ((store["k_codes"][b], store["k_scales"][b], store["k_tail"][b]),
                                (vt.view(store["v_codes"].dtype), store["v_scales"][b], store["v_tail"][b])):
        x = codes[:, :full].to(torch.float32).double() * scales[:, :full // block].double().repeat_interleave(block, 1)[..., None]
        out.append(torch.cat([x, tail[:, :n - full].double()], 1))
    return out


def _exact_rows(q, k, v, first, window, sinks):
    """One kv head: q (G, n, D) at positions first, first + 1, ..., k and v (T, D), all float64."""
    G, n, D = q.shape
    out = torch.zeros_like(q)
    T = k.shape[0]
    for lo in range(max(0, -first), n, 256):  # queries before position 0 see nothing
        p = first + torch.arange(lo, min(n, lo + 256), device=q.device)
        t = torch.arange(T, device=q.device)
        hidden = t[None] > p[:, None]
        if window:
            hidden |= (t[None] <= p[:, None] - window) & (t[None] >= sinks)
        s = (q[:, lo:lo + 256] @ k.T.contiguous()) / math.sqrt(D)
        out[:, lo:lo + 256] = torch.softmax(s.masked_fill(hidden[None], -math.inf), -1) @ v
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kind, B, H, D = c["kind"], c["batch"], c["hkv"], c["d"]
    st = s.get("store")
    n_of = s["lens"].tolist()
    if kind in ("store", "step"):
        block = c["block"]
        start = s["start"].tolist() if kind == "store" else n_of
        count = n_of if kind == "store" else [1] * B
        ks, vs, kt, vt = (st[x].double() for x in ("k_scales", "v_scales", "k_tail", "v_tail"))
        ks, vs, kt, vt = ks.clone(), vs.clone(), kt.clone(), vt.clone()
        m = s["max_len"]
        both = [torch.zeros(B, H, m, D, dtype=torch.float64, device=DEV) for _ in range(2)] if kind == "store" else []
        o = torch.zeros(B, c["hq"], 1, D, dtype=torch.float64, device=DEV) if kind == "step" else None
        for b in range(B):
            held, end = start[b] // block * block, start[b] + count[b]
            before = _exact_cached(st, b, start[b], block)
            after = []
            for x, new, scales, tail in zip(before, (s["keys"], s["values"]), (ks, vs), (kt, vt)):
                line = torch.cat([x, new[b, :, :count[b]].double()], 1)
                for p in range(held, end - block + 1, block):
                    line[:, p:p + block], scales[b, :, p // block] = _exact_block(line[:, p:p + block], c["fmt"])
                p = max(end // block * block, start[b])
                tail[b, :, p % block:p % block + end - p] = line[:, p:end]
                after.append(line)
            if kind == "store":
                both[0][b, :, :end], both[1][b, :, :end] = after
            else:
                for h in range(H):
                    G = c["hq"] // H
                    o[b, h * G:(h + 1) * G] = _exact_rows(s["q"][b, h * G:(h + 1) * G].double(), after[0][h], after[1][h], end - 1, 0, 0)
        rest = dict(k_scales=ks, v_scales=vs, k_tail=kt, v_tail=vt)
        return dict(k=both[0], v=both[1], **rest) if kind == "store" else dict(o=o, **rest)
    if kind == "read":
        k = torch.zeros(B, H, s["max_len"], D, dtype=torch.float64, device=DEV)
        v = torch.zeros_like(k)
        for b in range(B):
            k[b, :, :n_of[b]], v[b, :, :n_of[b]] = _exact_cached(st, b, n_of[b], c["block"])
        return k, v
    o = torch.zeros(B, c["hq"], c["n_q"], D, dtype=torch.float64, device=DEV)
    G = c["hq"] // H
    for b in range(B):
        if kind == "chunk":
            k, v = _exact_cached(st, b, n_of[b], c["block"])
        else:
            k, v = s["keys"][b, :, :n_of[b]].double(), s["values"][b, :, :n_of[b]].double()
        for h in range(H):
            o[b, h * G:(h + 1) * G] = _exact_rows(s["q"][b, h * G:(h + 1) * G].double(), k[h], v[h], n_of[b] - c["n_q"],
                                                  c["window"], c["sinks"])
    return o
