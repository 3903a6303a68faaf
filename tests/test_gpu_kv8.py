"""8-bit KV cache and windowed attention against plain implementations in 64
bits: codes and read-back bit for bit, attention within the roundings that the
kernels are documented to make.

Attention's bound, per output element: half a step of the output's type on the
result, and on A = sum p |v| (what an error in each weight is multiplied by):
half a step of the type that the weights are rounded to, twice the scores'
absolute error (numerator and denominator) of float32 sums of D products, and
2**-20 for the exponentials and float32 sums of the rest."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
QMAX = {"int8": 127.0, "fp8": 448.0}
# Weights too small for a relative error: fp16 ones are at most 2^14 and 2^-24 apart where they are subnormal, so off by
# 2^-25 / 2^14 of the largest; bf16 ones have float32's range, which ends at 2^-126. Each multiplies its |v|.
SMALLEST = {torch.float16: 2.0 ** -39, torch.bfloat16: 2.0 ** -126}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(seed, *shape, dtype=torch.float16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


# ------------------------------------------------------------------ oracles
def quantise(x, fmt, block):
    """(codes (B, H, n, block, D) as float32, scales (B, H, n)) of whole blocks, by the float32 definition, on the CPU."""
    B, H, T, D = x.shape
    x = x.cpu().float().view(B, H, T // block, block, D)
    a = x.abs().flatten(-2).amax(-1)
    finite = torch.isfinite(x).all(-1).all(-1)
    live = finite & (a >= 2.0 ** -110)
    top = torch.full_like(a, QMAX[fmt])  # a tensor: one rounding (a number over a tensor is two)
    scale = torch.where(live, a / top, torch.where(finite, 0.0, math.nan))
    y = x * torch.where(live, top / torch.where(live, a, 1.0), 0.0)[..., None, None]
    y = torch.where(live[..., None, None], y, 0.0)
    codes = torch.round(y) if fmt == "int8" else y.to(torch.float8_e4m3fn).float()
    return codes, scale


def exact_tokens(x, n, fmt, block):
    """The (H, n, D) float64 values that n cached tokens x (H, >= n, D) stand for."""
    full = n // block * block
    codes, scale = quantise(x[None, :, :full], fmt, block)
    v = (codes.double() * scale.double()[..., None, None]).view(x.shape[0], full, x.shape[2])
    return torch.cat([v, x[:, full:n].cpu().double()], 1)


def attend(q, k, v, n, window, sinks, scale=None, weights=None):
    """(out, bound without the output's rounding) in float64 of q (Hq, nq, D) over k, v (H, n, D)."""
    hq, nq, D = q.shape
    H = k.shape[0]
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    scale = D ** -0.5 if scale is None else scale
    out, tol = torch.zeros(hq, nq, D, dtype=torch.float64), torch.zeros(hq, nq, D, dtype=torch.float64)
    t = torch.arange(n)
    for i in range(nq):
        pos = n - nq + i
        if pos < 0:
            continue
        sees = (t <= pos) & ((t > pos - window) | (t < sinks)) if window else t <= pos
        for h in range(hq):
            kk, vv = k[h // (hq // H)][sees], v[h // (hq // H)][sees]
            s = kk @ q[h, i] * scale
            p = torch.softmax(s, 0)
            out[h, i] = p @ vv
            err = (D + 8) * 2.0 ** -24 * float((kk.abs() @ q[h, i].abs()).max()) * abs(scale)
            tol[h, i] = (half_step(weights) + 2 * err + 2.0 ** -20) * (p @ vv.abs()) + SMALLEST[weights] * vv.abs().sum(0)
    return out, tol


def check(got, want, tol, dtype, what=""):
    got = got.cpu().double()
    bound = tol + half_step(dtype) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)  # half the smallest
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / bound.clamp(min=1e-300)).max():.3g} times the bound"


def store_of(x, fmt, block, cap, v=None):
    from turboquant_amd import KV8Store, kv8_write
    B, H, T, D = x.shape
    s = KV8Store(B, H, D, cap, fmt, block, x.dtype, DEV)
    kv8_write(s, x, x if v is None else v, 0)
    return s


def codes_of(store):
    """(key codes, value codes) (B, H, cap, D) float32."""
    B, H, cap, D = store.k_codes.shape
    k = store.k_codes.float()
    v = store.v_codes.float().transpose(-1, -2).reshape(B, H, cap, D)
    return k.cpu(), v.cpu()


# -------------------------------------------------------------------- write
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,block,T", [(64, 16, 1), (64, 64, 200), (96, 16, 333), (96, 32, 65), (128, 32, 64), (128, 64, 63), (128, 16, 500),
                                       (256, 64, 257), (256, 32, 31)])
def test_write_codes_scales_tails(fmt, dtype, D, block, T):
    from turboquant_amd import KV8Store, kv8_write
    k, v = rand(T, 2, 3, T, D, dtype=dtype), rand(T + 1, 2, 3, T, D, dtype=dtype, scale=3.0)
    store = KV8Store(2, 3, D, T, fmt, block, dtype, DEV)
    kv8_write(store, k, v, 0)
    full = T // block * block
    kc, vc = codes_of(store)
    for x, codes, scales, tail in ((k, kc, store.k_scales, store.k_tail), (v, vc, store.v_scales, store.v_tail)):
        want, scale = quantise(x[:, :, :full], fmt, block)
        assert torch.equal(codes[:, :, :full], want.view(2, 3, full, D))
        assert (codes[:, :, full:] == 0).all()
        assert torch.equal(scales[:, :, :full // block].cpu(), scale)
        assert (scales[:, :, full // block:] == 0).all()
        assert torch.equal(tail[:, :, :T - full], x[:, :, full:])
        assert (tail[:, :, T - full:] == 0).all()


@pytest.mark.parametrize("fmt,block,D", [("int8", 32, 128), ("fp8", 16, 96), ("int8", 64, 64)])
def test_write_in_pieces_equals_one_write(fmt, block, D):
    """Tokens in pieces of every alignment, single tokens among them: the same bytes as one write."""
    from turboquant_amd import KV8Store, kv8_write
    T = 300
    k, v = rand(1, 1, 2, T, D), rand(2, 1, 2, T, D)
    one, two = KV8Store(1, 2, D, T, fmt, block, k.dtype, DEV), KV8Store(1, 2, D, T, fmt, block, k.dtype, DEV)
    kv8_write(one, k, v, 0)
    at = 0
    for n in [1, 1, 13, 1, 15, 1, 16, 17, 32, 33, 64, 1, 65, 2, 38]:
        kv8_write(two, k[:, :, at:at + n], v[:, :, at:at + n], at)
        at += n
    assert at == T
    full = T // block * block
    for name, t in one.tensors().items():
        u = getattr(two, name)
        if name.endswith("tail"):
            t, u = t[:, :, :T - full], u[:, :, :T - full]
        assert torch.equal(t.float(), u.float()), name


def test_write_ragged_and_strided():
    """Per-sequence starts and counts (0 and refused ones among them), from a (B, T, H, D) layout."""
    from turboquant_amd import KV8Store, kv8_write
    B, H, D, block, T = 6, 2, 128, 32, 70
    store = KV8Store(B, H, D, 256, "int8", block, torch.bfloat16, DEV)
    base = rand(3, B, 100, H, D, dtype=torch.bfloat16).transpose(1, 2)
    kv8_write(store, base, base, 0)
    before = {n: t.clone() for n, t in store.tensors().items()}
    start = torch.tensor([100, 100, 100, 250, -1, 100], dtype=torch.int32, device=DEV)
    count = torch.tensor([70, 0, 28, 70, 5, 71], dtype=torch.int32, device=DEV)
    new = rand(4, B, T, H, D, dtype=torch.bfloat16).transpose(1, 2)
    kv8_write(store, new, new, start, count)
    for b, n in ((0, 70), (2, 28)):
        x = torch.cat([base[b], new[b, :, :n]], 1)[None]
        full = (100 + n) // block * block
        codes, scale = quantise(x[:, :, :full], "int8", block)
        assert torch.equal(store.k_codes[b:b + 1, :, :full].cpu().float(), codes.view(1, H, full, D))
        assert torch.equal(store.v_scales[b:b + 1, :, :full // block].cpu(), scale)
        assert torch.equal(store.v_tail[b, :, :100 + n - full], x[0, :, full:])
    for b in (1, 3, 4, 5):  # no tokens, past the end, before the start, more than were given
        for n, t in store.tensors().items():
            assert torch.equal(t[b].float(), before[n][b].float()), (b, n)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_write_special_blocks(fmt):
    """Blocks of zeros, of the smallest and largest numbers, with infinities and NaN."""
    from turboquant_amd import kv8_read
    for dtype in (torch.float16, torch.bfloat16):
        x = rand(5, 1, 1, 7 * 16, 64, dtype=dtype)
        big = torch.finfo(dtype).max
        x[:, :, 0:16] = 0
        x[:, :, 16:32] = torch.finfo(dtype).tiny if dtype == torch.bfloat16 else 2.0 ** -24
        x[:, :, 32:48] = big
        x[0, 0, 50, 3] = math.inf
        x[0, 0, 70, 4] = math.nan
        x[:, :, 80:96] = -0.0
        store = store_of(x, fmt, 16, 128)
        k, v = kv8_read(store, 112, dtype=torch.float32)
        codes, scale = quantise(x, fmt, 16)
        want = (codes * scale[..., None, None]).view(x.shape)
        for got in (k.cpu(), v.cpu()):
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
        assert torch.isnan(k[0, 0, 48:80]).all()
        assert (k[0, 0, 0:16] == 0).all()


# --------------------------------------------------------------------- read
@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt,D,block,lens", [("int8", 128, 32, [200, 1, 0, 77]), ("fp8", 96, 16, [63, 64, 65, 200]), ("int8", 256, 64, [130, 200, 5, 64]),
                                              ("fp8", 64, 32, [31, 32, 33, 100])])
def test_read_is_code_times_scale(out, fmt, D, block, lens):
    from turboquant_amd import kv8_read
    B, H, T = len(lens), 2, 200
    dtype = torch.bfloat16 if out == torch.bfloat16 else torch.float16
    k, v = rand(6, B, H, T, D, dtype=dtype), rand(7, B, H, T, D, dtype=dtype)
    store = store_of(k, fmt, block, T, v)
    for b, n in enumerate(lens):  # the tail of a sequence of n tokens
        full = n // block * block
        store.k_tail[b, :, :n - full] = k[b, :, full:n]
        store.v_tail[b, :, :n - full] = v[b, :, full:n]
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for start, n in ((0, 200), (33, 100), (64, 1), (199, 1)):
        got = kv8_read(store, lt, start, n, out)
        for x, g in zip((k, v), got):
            codes, scale = quantise(x[:, :, :T // block * block], fmt, block)
            val = (codes * scale[..., None, None]).view(B, H, -1, D)
            for b, ln in enumerate(lens):
                full = ln // block * block
                want = torch.zeros(H, T, D)
                want[:, :full] = val[b, :, :full]
                want[:, full:ln] = x[b, :, full:ln].cpu().float()
                assert torch.equal(g[b].cpu(), want[:, start:start + n].to(out)), (start, n, b)


# ---------------------------------------------------------------- attention
CASES = [
    # D, Hq, Hkv, tokens, n_q, window, sinks, fmt, block
    (128, 8, 2, 1, 1, 0, 0, "int8", 32), (128, 8, 2, 31, 1, 0, 0, "int8", 32), (128, 8, 2, 32, 1, 0, 0, "fp8", 32),
    (128, 4, 4, 65, 1, 0, 0, "int8", 16), (128, 32, 2, 300, 1, 0, 0, "fp8", 16), (64, 7, 1, 257, 1, 0, 0, "int8", 64),
    (96, 6, 2, 333, 1, 0, 0, "fp8", 16), (256, 8, 4, 129, 1, 0, 0, "int8", 32), (256, 2, 1, 700, 3, 0, 0, "fp8", 64),
    (128, 8, 2, 1000, 4, 0, 0, "int8", 32), (128, 8, 2, 1000, 1, 100, 4, "int8", 32), (128, 8, 2, 1000, 1, 1, 0, "fp8", 32),
    (64, 4, 2, 777, 2, 64, 70, "int8", 16), (96, 3, 3, 500, 5, 130, 1, "fp8", 32), (128, 2, 2, 4000, 1, 0, 0, "int8", 64),
    (128, 8, 2, 100, 5, 0, 0, "int8", 32), (128, 8, 2, 200, 200, 0, 0, "fp8", 32), (64, 14, 2, 150, 150, 0, 0, "int8", 16),
    (96, 6, 2, 333, 77, 50, 3, "fp8", 16), (256, 4, 2, 190, 100, 0, 0, "int8", 64), (128, 8, 2, 600, 70, 65, 100, "int8", 32),
    (128, 4, 4, 700, 129, 1, 0, "fp8", 64), (64, 2, 1, 900, 40, 64, 64, "int8", 32), (256, 20, 1, 500, 1, 0, 0, "fp8", 32),
    (96, 8, 2, 40, 33, 0, 0, "int8", 64), (128, 24, 1, 3000, 1, 200, 10, "int8", 16),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_kv8_attention(case, dtype):
    from turboquant_amd import kv8_attention
    D, hq, H, T, nq, window, sinks, fmt, block = case
    k, v = rand(8, 1, H, T, D, dtype=dtype), rand(9, 1, H, T, D, dtype=dtype, scale=2.0)
    q = rand(10, 1, hq, nq, D, dtype=dtype, scale=1.5)
    store = store_of(k, fmt, block, T + 70, v)
    for t in (store.k_codes, store.v_codes):  # what no token has reached may hold anything
        t.view(torch.uint8)[:, :, -1:].fill_(0x7f)
    got = kv8_attention(q, store, T, window=window or None, sinks=sinks)
    rows = hq // H * nq
    want, tol = attend(q[0], exact_tokens(k[0], T, fmt, block), exact_tokens(v[0], T, fmt, block), T, window, sinks,
                       weights=torch.float16 if rows <= 16 else dtype)
    check(got[0], want, tol, dtype)
    wide = torch.empty(got.shape, dtype=torch.float32, device=DEV)
    kv8_attention(q, store, T, window=window or None, sinks=sinks, out=wide)
    assert torch.equal(wide.to(dtype), got)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", [c for c in CASES if c[7] == "int8"], ids=lambda c: "-".join(map(str, c[:7])))
def test_window_attention(case, dtype):
    from turboquant_amd import window_attention
    D, hq, H, T, nq, window, sinks, _, _ = case
    k, v = rand(11, 1, H, T, D, dtype=dtype), rand(12, 1, H, T, D, dtype=dtype, scale=2.0)
    q = rand(13, 1, hq, nq, D, dtype=dtype, scale=1.5)
    got = window_attention(q, k, v, window or None, sinks)
    want, tol = attend(q[0], k[0], v[0], T, window, sinks, weights=dtype)
    check(got[0], want, tol, dtype)


@pytest.mark.parametrize("nq", [1, 3, 50])
def test_ragged_lengths_and_rows_before_the_start(nq):
    """Sequences of 0 and 1 tokens, and shorter than the chunk: rows that see nothing are 0; bytes past a length do not matter."""
    from turboquant_amd import kv8_attention, window_attention
    lens, D, hq, H, block, cap = [0, 1, 40, 500, 64, 63], 128, 8, 2, 32, 512
    B = len(lens)
    k, v, q = rand(14, B, H, cap, D), rand(15, B, H, cap, D), rand(16, B, hq, nq, D)
    store = store_of(k, "int8", block, cap, v)
    for b, n in enumerate(lens):
        full = n // block * block
        store.k_tail[b, :, :n - full], store.v_tail[b, :, :n - full] = k[b, :, full:n], v[b, :, full:n]
        store.k_tail[b, :, n - full:], store.v_tail[b, :, n - full:] = math.nan, math.nan
        store.k_scales[b, :, full // block:], store.v_scales[b, :, full // block:] = math.nan, math.inf
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kn, vn = k.clone(), v.clone()
    for b, n in enumerate(lens):
        kn[b, :, n:], vn[b, :, n:] = math.nan, math.inf
    for window, sinks in ((None, 0), (20, 3)):
        got = kv8_attention(q, store, lt, window=window, sinks=sinks)
        dense = window_attention(q, kn, vn, window, sinks, lens=lt)
        for b, n in enumerate(lens):
            want, tol = attend(q[b], exact_tokens(k[b], n, "int8", block), exact_tokens(v[b], n, "int8", block), n, window or 0, sinks,
                               weights=torch.float16)
            check(got[b], want, tol, q.dtype, f"8-bit, sequence {b}")
            want, tol = attend(q[b], k[b, :, :n], v[b, :, :n], n, window or 0, sinks, weights=torch.float16)
            check(dense[b], want, tol, q.dtype, f"16-bit, sequence {b}")
            assert (got[b, :, :max(0, nq - n)] == 0).all() and (dense[b, :, :max(0, nq - n)] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq", [4, 60])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_infinite_and_nan_values_reach_only_rows_that_see_them(dtype, nq, bad):
    from turboquant_amd import kv8_attention, window_attention
    D, hq, H, T, window, sinks = 64, 4, 2, 200, 30, 2
    k, v, q = rand(17, 1, H, T, D, dtype=dtype), rand(18, 1, H, T, D, dtype=dtype), rand(19, 1, hq, nq, D, dtype=dtype)
    clean = v.clone()
    at = [40, T - nq - 28, T - 1]  # outside every window; inside some rows'; seen by the last row alone
    v[0, 0, at, 7] = bad
    k2 = k.clone()
    k2[0, 1, at, 9] = bad  # a key: its token's scores only
    got = window_attention(q, k, v, window, sinks)
    base = window_attention(q, k, clean, window, sinks)
    keys = window_attention(q, k2, clean, window, sinks)

    def same(a, b):
        # The rows of a tile with such a value are added one by one: other float32 sums of the same weights and values (|v| < 8),
        # 2^-20 of them apart, which a rounding to 16 bits may make one step.
        return bool(((a.float() - b.float()).abs() <= torch.finfo(dtype).eps * b.float().abs() + 2.0 ** -17).all())

    pos = torch.arange(T - nq, T)
    hit = torch.stack([(pos >= t) & (t > pos - window) for t in at]).any(0)
    assert hit.any() and not hit.all()
    for h in range(hq):
        for i in range(nq):
            if h < hq // H and hit[i]:
                assert not torch.isfinite(got[0, h, i, 7])
                assert same(got[0, h, i, [d for d in range(D) if d != 7]], base[0, h, i, [d for d in range(D) if d != 7]])
            else:
                assert same(got[0, h, i], base[0, h, i]), (h, i)
            if h < hq // H or not hit[i]:
                assert same(keys[0, h, i], base[0, h, i]), (h, i)
    # the same tokens in the 16-bit tail and in blocks of a cache (a block that holds one is NaN)
    block = 16
    store, ref = store_of(k, "int8", block, T, v), store_of(k, "int8", block, T, clean)
    got, base = kv8_attention(q, store, T, window=window, sinks=sinks), kv8_attention(q, ref, T, window=window, sinks=sinks)
    full = T // block * block
    seen = torch.zeros(nq, dtype=torch.bool)
    for t in at:
        lo, hi = (t // block * block, t // block * block + block) if t < full else (t, t + 1)
        seen |= torch.stack([(pos >= x) & ((x > pos - window) | (x < sinks)) for x in range(lo, hi)]).any(0)
    for h in range(hq):
        for i in range(nq):
            if h < hq // H and seen[i]:
                assert not torch.isfinite(got[0, h, i, 7])
            else:
                assert same(got[0, h, i], base[0, h, i]), (h, i)


@pytest.mark.parametrize("nq", [1, 40])
def test_strides_and_copies(nq):
    """(B, T, H, D) views, an odd slice (copied), broadcast heads, and a strided output."""
    from turboquant_amd import kv8_attention, window_attention
    B, hq, H, T, D = 2, 4, 2, 130, 64
    k, v, q = rand(20, B, T, H, D), rand(21, B, T, H, D), rand(22, B, nq, hq, D)
    plain = window_attention(q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous(), 50, 1)
    out = torch.full((B, nq, hq, D), 7.0, dtype=q.dtype, device=DEV)
    r = window_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), 50, 1, out=out.transpose(1, 2))
    assert r.data_ptr() == out.data_ptr() and torch.equal(out.transpose(1, 2), plain)
    odd = torch.zeros(B, H, T, D + 3, dtype=k.dtype, device=DEV)
    odd[..., 3:] = k.transpose(1, 2)
    assert torch.equal(window_attention(q.transpose(1, 2), odd[..., 3:], v.transpose(1, 2), 50, 1), plain)
    flat = torch.zeros(B * H * T * D + 1, dtype=k.dtype, device=DEV)
    flat[1:] = k.transpose(1, 2).reshape(-1)
    assert torch.equal(window_attention(q.transpose(1, 2), flat[1:].view(B, H, T, D), v.transpose(1, 2), 50, 1), plain)
    one = k[:, :, :1].transpose(1, 2).expand(B, H, T, D)  # a stride of 0
    assert torch.equal(window_attention(q.transpose(1, 2), one, v.transpose(1, 2), 50, 1),
                       window_attention(q.transpose(1, 2), one.contiguous(), v.transpose(1, 2), 50, 1))
    store = store_of(k.transpose(1, 2), "fp8", 16, T, v.transpose(1, 2))
    plain = kv8_attention(q.transpose(1, 2).contiguous(), store, T)
    kv8_attention(q.transpose(1, 2), store, T, out=out.transpose(1, 2))
    assert torch.equal(out.transpose(1, 2), plain)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("nq", [1, 30])
def test_scales_far_apart(fmt, nq):
    """Blocks whose value scales differ by 2^60 (bf16) or 2^20 (fp16), the large ones with hardly any weight, and queries of large
    and tiny rows: weights must not underflow."""
    from turboquant_amd import kv8_attention
    D, hq, H, T, block = 128, 4, 1, 256, 32
    for dtype, up in ((torch.bfloat16, 60), (torch.float16, 14)):
        k, v, q = rand(23, 1, H, T, D, dtype=dtype), rand(24, 1, H, T, D, dtype=dtype), rand(25, 1, hq, nq, D, dtype=dtype)
        v = v * 2.0 ** -8
        k[:, :, 32:64], v[:, :, 32:64] = 0.25 * k[:, :, 32:64], v[:, :, 32:64] * 2.0 ** up
        v[:, :, 64:96] = 0
        q[:, 1] *= 2.0 ** 7
        q[:, 2] *= 2.0 ** -10
        store = store_of(k, fmt, block, T, v)
        want, tol = attend(q[0], exact_tokens(k[0], T, fmt, block), exact_tokens(v[0], T, fmt, block), T, 0, 0,
                           weights=torch.float16 if nq == 1 else dtype)
        check(kv8_attention(q, store, T)[0], want, tol, dtype)


def test_bf16_queries_of_any_size():
    """bf16 queries past fp16's range, and keys that bring the scores back."""
    from turboquant_amd import kv8_attention
    D, T = 128, 100
    for e in (100, -100):
        k = (rand(26, 1, 1, T, D).float() * 2.0 ** -e).bfloat16()
        q = (rand(27, 1, 2, 1, D).float() * 2.0 ** e).bfloat16()
        v = rand(28, 1, 1, T, D, dtype=torch.bfloat16)
        if e == 100:
            k = k.float().clamp(min=-1e38).bfloat16()
        store = store_of(k, "int8", 32, T, v)
        want, tol = attend(q[0], exact_tokens(k[0], T, "int8", 32), exact_tokens(v[0], T, "int8", 32), T, 0, 0, weights=torch.float16)
        check(kv8_attention(q, store, T)[0], want, tol, torch.bfloat16)


@pytest.mark.parametrize("e", [-128, 112])
def test_bf16_queries_at_the_ends_of_their_range(e):
    """Queries down to subnormal numbers, and up, with keys that bring the scores back to a few units."""
    from turboquant_amd import kv8_attention
    D, T = 64, 70
    k = (rand(120, 1, 1, T, D).float() * 2.0 ** min(-e, 124)).bfloat16()
    q = (rand(121, 1, 2, 1, D).float() * 2.0 ** e).bfloat16()
    v = rand(122, 1, 1, T, D, dtype=torch.bfloat16)
    store = store_of(k, "fp8", 32, T, v)
    want, tol = attend(q[0], exact_tokens(k[0], T, "fp8", 32), exact_tokens(v[0], T, "fp8", 32), T, 0, 0, weights=torch.float16)
    check(kv8_attention(q, store, T)[0], want, tol, torch.bfloat16)


@pytest.mark.parametrize("B", [65, 200])
def test_many_sequences(B):
    """More sequences than a wave has lanes, empty ones among them, over enough tiles that they are shared out."""
    from turboquant_amd import kv8_attention, window_attention
    D, hq, H, cap = 64, 2, 1, 4096
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, cap + 1, (B,), generator=g)
    lens[[0, 3, 63, 64, B - 1]] = torch.tensor([0, 0, 5, 4096, 0])
    lens[10:60] = 0
    k, v, q = rand(123, B, H, cap, D), rand(124, B, H, cap, D), rand(125, B, hq, 1, D)
    store = store_of(k, "int8", 64, cap, v)
    for b, n in enumerate(lens.tolist()):
        full = n // 64 * 64
        store.k_tail[b, :, :n - full], store.v_tail[b, :, :n - full] = k[b, :, full:n], v[b, :, full:n]
    lt = lens.to(torch.int32).to(DEV)
    got, dense = kv8_attention(q, store, lt), window_attention(q, k, v, lens=lt)
    windowed = window_attention(q, k, v, 3000, 70, lens=lt)
    for b in sorted({0, 1, 3, 9, 60, 62, 63, 64, B // 2, B - 2, B - 1}):
        n = int(lens[b])
        if n == 0:
            assert (got[b] == 0).all() and (dense[b] == 0).all() and (windowed[b] == 0).all()
            continue
        want, tol = attend(q[b], exact_tokens(k[b], n, "int8", 64), exact_tokens(v[b], n, "int8", 64), n, 0, 0, weights=torch.float16)
        check(got[b], want, tol, q.dtype, f"8-bit, {b}")
        want, tol = attend(q[b], k[b, :, :n], v[b, :, :n], n, 0, 0, weights=torch.float16)
        check(dense[b], want, tol, q.dtype, f"16-bit, {b}")
        want, tol = attend(q[b], k[b, :, :n], v[b, :, :n], n, 3000, 70, weights=torch.float16)
        check(windowed[b], want, tol, q.dtype, f"windowed, {b}")


@pytest.mark.parametrize("nq", [1, 40])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinite_values_that_are_seen(nq, dtype):
    """+inf gives +inf, -inf gives -inf, both or NaN give NaN, in tiles that all rows see and in those that some do."""
    from turboquant_amd import window_attention
    D, T = 64, 300
    k, v, q = rand(126, 1, 1, T, D, dtype=dtype, scale=0.2), rand(127, 1, 1, T, D, dtype=dtype), rand(128, 1, 2, nq, D, dtype=dtype)
    v[0, 0, 10, 0] = v[0, 0, T - 1, 1] = math.inf
    v[0, 0, 70, 2] = v[0, 0, T - 1, 3] = -math.inf
    v[0, 0, 5, 4], v[0, 0, 200, 4], v[0, 0, 6, 5] = math.inf, -math.inf, math.nan
    got = window_attention(q, k, v).float().cpu()
    assert (got[..., 0] == math.inf).all() and (got[..., 2] == -math.inf).all() and torch.isnan(got[..., 4:6]).all()
    assert (got[:, :, -1, 1] == math.inf).all() and (got[:, :, -1, 3] == -math.inf).all()
    assert torch.isfinite(got[:, :, :-1, [1, 3]]).all() and torch.isfinite(got[..., 6:]).all()


def test_captured_chunk_replays():
    """A chunk's attention in a HIP graph (more LDS than a launch has by default), split and not, replayed with eager work between."""
    from turboquant_amd import kv8_attention, window_attention
    for D, T, nq in ((128, 3000, 60), (256, 500, 200)):
        k, v, q = rand(129, 1, 2, T, D), rand(130, 1, 2, T, D), rand(131, 1, 4, nq, D)
        store, lens = store_of(k, "fp8", 32, T, v), torch.full((1,), T, dtype=torch.int32, device=DEV)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            a, b = kv8_attention(q, store, lens), window_attention(q, k, v, 100, 4, lens=lens)
        for i in range(4):
            q.copy_(rand(140 + i, 1, 4, nq, D))
            n = T - 37 * i // 32 * 32  # whole blocks: the tail of another length is not there
            n = n // 32 * 32 if i else T
            lens.fill_(n)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(a, kv8_attention(q, store, lens)) and torch.equal(b, window_attention(q, k, v, 100, 4, lens=lens)), (D, i)


def test_offsets_past_31_bits():
    """Tokens whose codes lie past 2^31 bytes: written, read back and attended to in place."""
    from turboquant_amd import KV8Store, kv8_attention, kv8_read, kv8_write, window_attention
    D, T = 256, 100
    far = 2 ** 31 // D + 40
    store = KV8Store(1, 1, D, far + T, "int8", 32, torch.float16, DEV)
    k, v = rand(29, 1, 1, T + 40, D), rand(30, 1, 1, T + 40, D)
    base = far - 40  # a block's first token
    kv8_write(store, k, v, base)
    small = store_of(k, "int8", 32, T + 40, v)
    kr, vr = kv8_read(store, far + T, base, T + 40)
    ks, vs = kv8_read(small, T + 40)
    assert torch.equal(kr, ks) and torch.equal(vr, vs)
    for nq in (1, 20):
        q = rand(31, 1, 2, nq, D)
        want, tol = attend(q[0], exact_tokens(k[0], T + 40, "int8", 32), exact_tokens(v[0], T + 40, "int8", 32), T + 40, 64, 0,
                           weights=torch.float16)
        check(kv8_attention(q, store, far + T, window=64)[0], want, tol, q.dtype)
    del store
    big = torch.zeros(1, 1, 2 ** 30 // D + 200, D, dtype=torch.float16, device=DEV)  # 16-bit: past 2^31 bytes
    big[:, :, -140:] = k
    for nq in (1, 20):
        q = rand(32, 1, 2, nq, D)
        want, tol = attend(q[0], k[0], k[0], 140, 64, 0, weights=torch.float16)
        check(window_attention(q, big, big, 64)[0], want, tol, q.dtype)


def test_steps_of_a_batch_equal_single_sequences():
    """The operators together, as a serving loop runs them: prompts of different lengths, then steps over block borders."""
    from turboquant_amd import KV8Batch, KV8Cache
    B, H, hq, D, steps = 4, 2, 8, 128, 40
    prompts = [1, 30, 200, 77]
    batch = KV8Batch(B, H, D, "int8", 32, capacity=128, dtype=torch.bfloat16)
    caches = []
    for b, n in enumerate(prompts):
        k, v = rand(40 + b, H, n, D, dtype=torch.bfloat16), rand(50 + b, H, n, D, dtype=torch.bfloat16)
        batch.load(b, k[:, :n // 2], v[:, :n // 2])
        batch.load(b, k[:, n // 2:], v[:, n // 2:])
        caches.append(KV8Cache(D, H))
        caches[b].update(k[None], v[None])
    for i in range(steps):
        k, v, q = (rand(100 + 3 * i + j, B, h, D, dtype=torch.bfloat16) for j, h in enumerate((H, H, hq)))
        batch.step(k, v)
        out = batch.attend(q)
        for b in range(B):
            caches[b].update(k[b:b + 1, :, None], v[b:b + 1, :, None])
            want = caches[b].attend(q[b:b + 1, :, None])
            # another split of the tiles: the merges' float32 sums differ in their last bits
            assert torch.allclose(out[b].float(), want[0, :, 0].float(), rtol=2 ** -7, atol=2 ** -12), (i, b)
    assert batch.offset.tolist() == [n + steps for n in prompts] == batch.lens.tolist()


def test_batch_with_windows_drafts_and_outputs():
    from turboquant_amd import KV8Batch, kv8_attention
    B, H, hq, D = 3, 2, 6, 64
    batch = KV8Batch(B, H, D, "fp8", 16, capacity=64, window=20, sinks=3)
    assert (batch.attend(rand(150, B, hq, D)) == 0).all()  # nothing in it yet
    for b, n in enumerate((5, 130, 0)):
        if n:
            batch.load(b, rand(151 + b, H, n, D), rand(161 + b, H, n, D))
    for i in range(4):
        batch.step(rand(170 + i, B, H, D), rand(180 + i, B, H, D))
    assert batch.lens.tolist() == [9, 134, 4] and batch.store.cap >= 134
    q = rand(190, B, hq, 4, D)
    want = kv8_attention(q, batch.store, batch.lens, 134, None, 20, 3)
    assert torch.equal(batch.attend(q), want)
    last = batch.attend(q[:, :, -1])
    assert last.shape == (B, hq, D) and torch.allclose(last.float(), want[:, :, -1].float(), rtol=2 ** -9, atol=2 ** -12)
    out = torch.empty(B, hq, D, dtype=torch.float32, device=DEV)
    assert batch.attend(q[:, :, -1], out=out).data_ptr() == out.data_ptr() and torch.equal(out.half(), last)


def test_captured_step_replays():
    """A decode step (write, length, attention) in a HIP graph, replayed over block borders with eager work between, two graphs
    on their own streams at once: every replay as the eager step."""
    from turboquant_amd import KV8Store, kv8_attention, kv8_write
    B, H, hq, D, cap = 2, 2, 8, 128, 512
    dt = torch.float16
    k0, v0 = rand(60, B, H, 100, D), rand(61, B, H, 100, D)

    def fresh():
        s = KV8Store(B, H, D, cap, "int8", 32, dt, DEV)
        kv8_write(s, k0, v0, 0)
        return s, torch.full((B,), 100, dtype=torch.int32, device=DEV)

    def step(s, lens, k, v, q):
        kv8_write(s, k, v, lens)
        lens += 1
        return kv8_attention(q, s, lens, max_len=cap)

    def make(seed):
        s, lens = fresh()
        k, v, q = rand(seed, B, H, 1, D), rand(seed + 1, B, H, 1, D), rand(seed + 2, B, hq, 1, D)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            step(s, lens, k, v, q)
            torch.cuda.synchronize()
            lens.fill_(100)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            out = step(s, lens, k, v, q)
        return g, stream, s, lens, k, v, q, out

    graphs = [make(70), make(80)]
    eager = [fresh() for _ in graphs]
    for i in range(70):
        news = [(rand(1000 + i, B, H, 1, D), rand(2000 + i, B, H, 1, D), rand(3000 + i, B, hq, 1, D)) for _ in graphs]
        for (g, stream, s, lens, k, v, q, out), (a, b, c) in zip(graphs, news):
            k.copy_(a), v.copy_(b), q.copy_(c)
        torch.cuda.synchronize()
        for g, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for (g, stream, s, lens, k, v, q, out), (es, el), (a, b, c) in zip(graphs, eager, news):
            assert torch.equal(out, step(es, el, a, b, c)), i


def test_streams():
    """Calls on a side stream, with the current stream busy: in order with that stream's work."""
    from turboquant_amd import kv8_attention, kv8_read
    k, q = rand(90, 1, 2, 300, 128), rand(91, 1, 8, 1, 128)
    store = store_of(k, "fp8", 32, 300)
    want, wr = kv8_attention(q, store, 300), kv8_read(store, 300)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q2 = q.clone()
        for _ in range(3):
            got, r = kv8_attention(q2, store, 300), kv8_read(store, 300)[0]
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(r, wr)


@pytest.mark.parametrize("lens", [(40000,), (20011, 0, 12000)], ids=str)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_one_head_over_many_workgroups(D, lens):
    """A row whose parts are more than the join takes at once, in whole caches and ragged ones."""
    from turboquant_amd import kv8_attention, window_attention
    B, T, block = len(lens), max(lens), 32
    k, v, q = rand(94, B, 1, T, D), rand(95, B, 1, T, D, scale=2.0), rand(96, B, 3, 1, D, scale=1.5)
    v[:, :, :T // 2] *= 1e-3  # parts of unlike scales
    store = store_of(k, "int8", block, T, v)
    for b, n in enumerate(lens):
        full = n // block * block
        store.k_tail[b, :, :n - full], store.v_tail[b, :, :n - full] = k[b, :, full:n], v[b, :, full:n]
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    calls = [lt] if B > 1 else [lt, lens[0]]
    for n_arg in calls:
        got = kv8_attention(q, store, n_arg)
        dense = window_attention(q, k, v, lens=n_arg)
        for b, n in enumerate(lens):
            want, tol = attend(q[b], exact_tokens(k[b], n, "int8", block), exact_tokens(v[b], n, "int8", block), n, 0, 0,
                               weights=torch.float16) if n else (torch.zeros(3, 1, D), torch.zeros(3, 1, D))
            check(got[b], want.double(), tol.double(), q.dtype, f"8-bit, sequence {b}")
            want, tol = attend(q[b], k[b, :, :n], v[b, :, :n], n, 0, 0, weights=torch.float16) if n else (want, tol)
            check(dense[b], want.double(), tol.double(), q.dtype, f"16-bit, sequence {b}")


@pytest.mark.parametrize("D,nq,T,window", [(64, 512, 4100, 0), (96, 512, 4100, 0), (128, 512, 4100, 0), (128, 300, 9000, 0),
                                           (128, 770, 3000, 0), (256, 300, 3000, 0), (128, 1030, 4100, 2500), (64, 40, 9000, 0)])
def test_chunks_in_parts(D, nq, T, window):
    """Prompt chunks whose tiles go to several workgroups, in tall and low row tiles: some queries of each against float64."""
    from turboquant_amd import kv8_attention, window_attention
    H, hq, block, dtype = 8, 32, 32, torch.bfloat16
    k, v = rand(99, 1, H, T, D, dtype=dtype), rand(100, 1, H, T, D, dtype=dtype, scale=2.0)
    q = rand(101, 1, hq, nq, D, dtype=dtype, scale=1.5)
    got = kv8_attention(q, store_of(k, "int8", block, T, v), T, window=window or None, sinks=5)
    dense = window_attention(q, k, v, window or None, 5)
    ke, ve = exact_tokens(k[0], T, "int8", block), exact_tokens(v[0], T, "int8", block)
    for i in (0, 31, nq // 2, nq - 1):
        n = T - nq + i + 1
        for name, x, kk, vv in (("8-bit", got, ke, ve), ("16-bit", dense, k[0], v[0])):
            want, tol = attend(q[0, :, i:i + 1], kk[:, :n], vv[:, :n], n, window, 5, weights=dtype)
            check(x[0, :, i:i + 1], want, tol, dtype, f"{name}, query {i}")


@pytest.mark.parametrize("B,H,T,nq", [(1, 2, 300, 1), (1, 2, 6000, 1), (2, 2, 6000, 3), (1, 2, 900, 70), (32, 8, 200, 20)])
def test_output_over_the_queries(B, H, T, nq):
    """``out`` may be the queries themselves."""
    from turboquant_amd import kv8_attention, window_attention
    k, q = rand(97, B, H, T, 64), rand(98, B, 2 * H, nq, 64)
    store = store_of(k, "fp8", 16, T)
    for call in (lambda x, **a: kv8_attention(x, store, T, **a), lambda x, **a: window_attention(x, k, k, **a)):
        want, mine = call(q), q.clone()
        assert call(mine, out=mine) is mine and torch.equal(mine, want)


def test_repeatable():
    """The same call gives the same bits (no atomics)."""
    from turboquant_amd import kv8_attention
    k = rand(92, 2, 2, 5000, 128)
    store = store_of(k, "int8", 32, 5000)
    for nq in (1, 33):
        q = rand(93, 2, 8, nq, 128)
        want = kv8_attention(q, store, 5000)
        for _ in range(5):
            assert torch.equal(kv8_attention(q, store, 5000), want)


# ------------------------------------------------------------------- caches
def test_cache_protocol_and_state():
    from turboquant_amd import KV8Cache
    c = KV8Cache(96, 2, "fp8", 16)
    assert c.empty() and c.size() == 0 and not c.is_trimmable() and c.nbytes == 0
    k, v = rand(94, 1, 2, 77, 96), rand(95, 1, 2, 77, 96)
    a, b = c.update_and_fetch(k[:, :, :50], v[:, :, :50])
    assert a.shape == (1, 2, 50, 96) and a.dtype == k.dtype
    a, b = c.update_and_fetch(k[:, :, 50:], v[:, :, 50:])
    assert torch.equal(a[:, :, 64:], k[:, :, 64:]) and torch.equal(b[:, :, 64:], v[:, :, 64:])
    assert c.offset == 77 and c.nbytes == 2 * 2 * (4 * (16 * 96 + 4) + 13 * 96 * 2)
    for first in ("state", "meta_state"):
        d = KV8Cache(96, 2, "fp8", 16)
        for name in (first, {"state": "meta_state", "meta_state": "state"}[first]):
            setattr(d, name, getattr(c, name))
        assert d.offset == 77
        q = rand(96, 1, 4, 1, 96)
        assert torch.equal(c.attend(q), d.attend(q))
        x = rand(97, 1, 2, 30, 96)
        e = KV8Cache(96, 2, "fp8", 16)
        e.update(torch.cat([k, x], 2), torch.cat([v, x], 2))
        d.update(x, x)
        assert torch.equal(d.attend(q), e.attend(q))
    with pytest.raises(ValueError, match="query tokens"):
        c.attend(rand(98, 1, 4, 78, 96))


def test_cache_grows_past_its_step():
    from turboquant_amd import KV8Cache
    c = KV8Cache(64, 1, "int8", 32)
    k, v = rand(110, 1, 1, 9000, 64), rand(111, 1, 1, 9000, 64)
    for lo, hi in ((0, 4000), (4000, 4097), (4097, 9000)):
        c.update(k[:, :, lo:hi], v[:, :, lo:hi])
    one = store_of(k, "int8", 32, 9000, v)
    from turboquant_amd import kv8_read
    a, b = c.fetch()
    ra, rb = kv8_read(one, 9000)
    assert torch.equal(a, ra) and torch.equal(b, rb)


def test_windowed_cache_reads_its_window():
    from turboquant_amd import KV8Cache, kv8_attention
    k, v, q = rand(112, 1, 2, 500, 128), rand(113, 1, 2, 500, 128), rand(114, 1, 4, 20, 128)
    c = KV8Cache(128, 2, window=64, sinks=4)
    c.update(k, v)
    assert torch.equal(c.attend(q), kv8_attention(q, c.store, 500, window=64, sinks=4))
    assert torch.equal(c.attend(q, window=30, sinks=0), kv8_attention(q, c.store, 500, window=30))


def test_numpy_lengths_and_empty_batches():
    from turboquant_amd import KV8Store, kv8_attention, kv8_read, kv8_write, window_attention
    s = KV8Store(0, 2, 64, 64, "int8", 32, torch.float16, DEV)
    e = torch.empty(0, 2, 3, 64, dtype=torch.float16, device=DEV)
    kv8_write(s, e, e, 0)
    assert kv8_read(s, 0, 0, 5)[0].shape == (0, 2, 5, 64)
    assert kv8_attention(torch.empty(0, 4, 1, 64, dtype=torch.float16, device=DEV), s, 0).shape == (0, 4, 1, 64)
    s = KV8Store(1, 2, 64, 0, "int8", 32, torch.float16, DEV)
    q = rand(115, 1, 4, 2, 64)
    assert (kv8_attention(q, s, np.int64(0)) == 0).all()
    assert (window_attention(q, e[:0].new_empty(1, 2, 0, 64), e[:0].new_empty(1, 2, 0, 64)) == 0).all()
    assert kv8_attention(q[:, :, :0], s, 0).shape == (1, 4, 0, 64)
