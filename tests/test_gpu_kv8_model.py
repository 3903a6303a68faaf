"""The 8-bit cache and windowed attention where the package's own paths call them: skipped layers held in 8 bits, inside a
``transformers`` model, and FP16KVCache's several query tokens and windows."""

import pytest
import torch

from test_gpu_kv8 import DEV, attend, check, exact_tokens, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,hq,H,nq,window,sinks", [(128, 8, 2, 1, 100, 4), (128, 8, 2, 50, None, 0), (64, 4, 4, 1, 7, 0), (96, 6, 2, 300, 64, 2)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_fp16_cache_windows_and_chunks(D, hq, H, nq, window, sinks, dtype):
    from turboquant_amd.patch import FP16KVCache
    c = FP16KVCache()
    k, v, q = rand(1, 1, H, 300, D, dtype=dtype), rand(2, 1, H, 300, D, dtype=dtype), rand(3, 1, hq, nq, D, dtype=dtype)
    for lo, hi in ((0, 200), (200, 201), (201, 300)):
        c.update(k[:, :, lo:hi], v[:, :, lo:hi])
    got = c.attend(q, window=window, sinks=sinks)
    assert got.dtype == torch.float32 and got.shape == q.shape
    want, tol = attend(q[0], k[0], v[0], 300, window or 0, sinks, weights=dtype)
    # float32 out: its own half step, and nothing of a 16-bit one
    assert bool(((got[0].cpu().double() - want).abs() <= tol + 2.0 ** -24 * want.abs()).all())
    with pytest.raises(ValueError, match="query tokens"):
        c.attend(rand(4, 1, hq, 301, D, dtype=dtype))


def test_fp16_cache_one_token_keeps_its_kernel():
    from turboquant_amd.cache import dense_attention
    from turboquant_amd.patch import FP16KVCache
    c = FP16KVCache()
    k, v, q = rand(5, 1, 2, 300, 128), rand(6, 1, 2, 300, 128), rand(7, 1, 8, 1, 128)
    c.update(k, v)
    assert torch.equal(c.attend(q), dense_attention(q, c.keys, c.values))
    assert torch.equal(c.attend(q[:, :, 0]), dense_attention(q, c.keys, c.values))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_skipped_layer_in_8_bits_inside_a_model(fmt):
    pytest.importorskip("transformers")
    from test_gpu_hf import _tokens, run, tiny_llama
    from turboquant_amd import KV8Cache, apply_turboquant
    from turboquant_amd.hf import TurboQuantCache
    m = tiny_llama(seed=9)
    apply_turboquant(m, key_bits=4, value_bits=2, residual_window=512, auto_detect_outliers=False, skip_layers=[1],
                     skip_layer_format=fmt)
    prompt, steps = _tokens(300, 10), _tokens(40, 11)
    m.set_attn_implementation("sdpa")
    dense = run(m, TurboQuantCache(m, fused=False), prompt, steps)
    m.set_attn_implementation("turboquant")
    cache = TurboQuantCache(m)
    fused = run(m, cache, prompt, steps)
    c = cache.layers[1].cache
    assert isinstance(c, KV8Cache) and c.fmt == fmt and c.offset == 340 and cache.layers[1].fused
    e = ((fused - dense).norm(dim=-1) / dense.norm(dim=-1)).max().item()
    print(f"{fmt}: fused vs dense path rel {e:.2e}")
    assert torch.isfinite(fused).all()
    # The same codes on both sides; the dense path rounds each key and value to fp16 (2^-11) before SDPA, and a score of a few units
    # moves by a few 2^-11: at most 1 percent through two layers.
    assert e < 1e-2


def test_sliding_window_of_an_8_bit_layer():
    pytest.importorskip("transformers")
    from turboquant_amd import KV8Cache
    from turboquant_amd.hf import TurboQuantLayer, turboquant_attention
    D, hq, H, T, window = 128, 8, 2, 200, 50
    layer = TurboQuantLayer(KV8Cache(D, H))
    k, v, q = rand(20, 1, H, T, D), rand(21, 1, H, T, D), rand(22, 1, hq, 1, D)
    layer.update(k[:, :, :-1], v[:, :, :-1])
    ks, vs = layer.update(k[:, :, -1:], v[:, :, -1:])
    for w in (None, window, 4 * T):
        out, _ = turboquant_attention(None, q, ks, vs, None, scaling=D ** -0.5, sliding_window=w)
        assert out.shape == (1, 1, hq, D)
        want, tol = attend(q[0], exact_tokens(k[0], T, "int8", 32), exact_tokens(v[0], T, "int8", 32), T, w or 0, 0, weights=torch.float16)
        check(out[0].transpose(0, 1), want, tol, q.dtype, str(w))
    # a step that carries a mask attends over the dense keys and values
    mask = torch.ones(1, 1, 1, T, dtype=torch.bool, device=DEV)
    mask[..., :3] = False
    module = torch.nn.Module()
    module.num_key_value_groups = hq // H
    out, _ = turboquant_attention(module, q, ks, vs, mask, scaling=D ** -0.5)
    kk, vv = layer.dense_kv()
    want, tol = attend(q[0], kk[0, :, 3:], vv[0, :, 3:], T - 3, 0, 0, weights=torch.float16)
    check(out[0].transpose(0, 1), want, 4 * tol, q.dtype)  # SDPA's own roundings
