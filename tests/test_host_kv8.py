"""8-bit KV cache and windowed attention: what is refused before any device work, and the structs' layouts (CPU only)."""

import ctypes
import math
import os
import shutil
import subprocess
import tempfile

import pytest
import torch

from turboquant_amd import KV8Batch, KV8Cache, KV8Store, kv8_attention, kv8_read, kv8_write, window_attention
from turboquant_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
H16 = torch.float16


def store(B=2, H=2, D=64, cap=128, fmt="int8", block=32, dtype=H16):
    return KV8Store(B, H, D, cap, fmt, block, dtype, "cpu")


def test_struct_layouts_match_header():
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = {"tq_kv8_store": _lib.KV8StoreDesc, "tq_rows4": _lib.Rows4, "tq_kv_attn_desc": _lib.KVAttnDesc}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "tq_abi.h"', "int main(void){"]
    for cname, cls in fields.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for f, _ in cls._fields_:
            lines.append(f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));')
    lines.append("return 0;}")
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "l.c")
        open(src, "w").write("\n".join(lines))
        subprocess.run([cc, "-I", os.path.join(ROOT, "include"), src, "-o", os.path.join(d, "l")], check=True)
        out = subprocess.run([os.path.join(d, "l")], capture_output=True, text=True, check=True).stdout.split("\n")
    got = dict(line.rsplit(" ", 1) for line in out if line)
    for cname, cls in fields.items():
        assert int(got[f"{cname} size"]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, f"{cname}.{f}"


def test_packed_structs_match():
    """The bytes that the Python layer packs, read as the structs."""
    from turboquant_amd import kv8
    s = store(1, 2, 96, 192, "fp8", 16, torch.bfloat16)
    d = _lib.KV8StoreDesc.from_buffer_copy(s.desc)
    assert len(s.desc) == ctypes.sizeof(d) and (d.cap, d.fmt, d.d, d.block, d.kv_dtype, d.batch, d.heads) == (192, 1, 96, 16, 1, 1, 2)
    assert [getattr(d, n) for n in s.tensors()] == [t.data_ptr() for t in s.tensors().values()]
    q, out = x(1, 4, 3, 96), x(1, 3, 4, 96).float().transpose(1, 2)
    b, o, _ = kv8._attention_desc(q, 1, 2, 96, H16, q.device, 16, 100, 0.5, 7, 3, out, (32, 1, 2, 3), (48, 4, 5, 6))
    d = _lib.KVAttnDesc.from_buffer_copy(b)
    assert len(b) == ctypes.sizeof(d) and o is out
    assert [getattr(d, n) for n, _ in d._fields_[:12]] == [1, 4, 2, 96, 3, 0, 2, 7, 3, 100, 16, 0.5]
    assert [[getattr(r, n) for n, _ in r._fields_] for r in (d.q, d.out, d.k, d.v)] == [
        [q.data_ptr(), 0, 3 * 96, 96], [out.data_ptr(), 0, 96, 4 * 96], [32, 1, 2, 3], [48, 4, 5, 6]]
    assert bytes(_lib.Rows4(1, 2, 3, 4)) == kv8._ROWS.pack(1, 2, 3, 4)


@pytest.mark.parametrize("kw,what", [
    (dict(D=80), "head_dim 80"), (dict(D=512), "head_dim 512"), (dict(block=48), "blocks of 48"), (dict(fmt="int4"), "format"),
    (dict(dtype=torch.float32), "float32"), (dict(cap=-1), "capacity"),
])
def test_store_refuses(kw, what):
    with pytest.raises(ValueError, match=what):
        store(**kw)


def test_store_shapes():
    s = store(cap=65)
    assert s.cap == 128 and s.v_codes.shape == (2, 2, 2, 64, 64) and s.k_scales.shape == (2, 2, 4) and s.k_tail.shape == (2, 2, 32, 64)
    assert s.sequence(1).k_codes.data_ptr() == s.k_codes[1].data_ptr()
    g = s.grown(200)
    assert g.cap == 256 and g.block == 32
    with pytest.raises(ValueError, match="room"):
        s.grown(64)
    t = s.tensors()
    for name, bad in (("k_codes", t["k_codes"].float()), ("v_codes", t["v_codes"][:, :, :1]), ("k_scales", t["k_scales"].double()),
                      ("v_tail", t["v_tail"].bfloat16()), ("k_tail", t["k_tail"].transpose(0, 1))):
        with pytest.raises(ValueError):
            KV8Store.from_tensors("int8", **{**t, name: bad})
    with pytest.raises(ValueError):
        KV8Store.from_tensors("fp8", **t)


def x(*shape, dtype=H16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,what", [
    (lambda s: kv8_write(s, x(2, 2, 3, 96), x(2, 2, 3, 96), 0), "keys"),
    (lambda s: kv8_write(s, x(1, 2, 3, 64), x(1, 2, 3, 64), 0), "keys"),
    (lambda s: kv8_write(s, x(2, 2, 3, 64), x(2, 2, 4, 64), 0), "values"),
    (lambda s: kv8_write(s, x(2, 2, 3, 64, dtype=torch.bfloat16), x(2, 2, 3, 64), 0), "keys"),
    (lambda s: kv8_write(s, x(2, 2, 3, 64), x(2, 2, 3, 64), -1), "start"),
    (lambda s: kv8_write(s, x(2, 2, 3, 64), x(2, 2, 3, 64), 126), "start"),
    (lambda s: kv8_write(s, x(2, 2, 129, 64), x(2, 2, 129, 64), 0), "129 tokens"),
    (lambda s: kv8_write(s, x(2, 2, 3, 64), x(2, 2, 3, 64), torch.zeros(2, dtype=torch.int64)), "int32"),
    (lambda s: kv8_write(s, x(2, 2, 3, 64), x(2, 2, 3, 64), torch.zeros(3, dtype=torch.int32)), "int32"),
    (lambda s: kv8_write(s, x(2, 2, 3, 64), x(2, 2, 3, 64), 0, 2), "n_new"),
    (lambda s: kv8_read(s, 129), "lens"),
    (lambda s: kv8_read(s, 100, 100, 29), "outside"),
    (lambda s: kv8_read(s, 100, -1, 2), "outside"),
    (lambda s: kv8_read(s, 100, dtype=torch.float64), "unsupported"),
    (lambda s: kv8_attention(x(2, 3, 1, 64), s, 10), "query shape"),
    (lambda s: kv8_attention(x(2, 4, 1, 128), s, 10), "query shape"),
    (lambda s: kv8_attention(x(4, 64), s, 10), "query shape"),
    (lambda s: kv8_attention(x(2, 4, 1, 64, dtype=torch.float32), s, 10), "queries"),
    (lambda s: kv8_attention(x(2, 4, 1, 64), s, -1), "lens"),
    (lambda s: kv8_attention(x(2, 4, 1, 64), s, 129), "lens"),
    (lambda s: kv8_attention(x(2, 4, 1, 64), s, torch.zeros(2, dtype=torch.int32), max_len=129), "max_len"),
    (lambda s: kv8_attention(x(2, 4, 1, 64), s, 10, window=0), "window"),
    (lambda s: kv8_attention(x(2, 4, 1, 64), s, 10, window=3, sinks=-1), "sinks"),
    (lambda s: kv8_attention(x(2, 4, 1, 64), s, 10, out=x(2, 4, 2, 64)), "out"),
    (lambda s: kv8_attention(x(2, 4, 1, 64), s, 10, out=x(2, 4, 1, 64, dtype=torch.bfloat16)), "out"),
    (lambda s: kv8_attention(x(2, 4, 3, 64), s, 10, out=x(2, 4, 64, 3).transpose(2, 3)), "out"),
    (lambda s: kv8_attention(x(2, 4, 3, 64), s, 10, out=x(2, 4, 1, 64).expand(2, 4, 3, 64)), "out"),
    (lambda s: kv8_attention(x(2, 4, 3, 64), s, 10, out=x(2000).as_strided((2, 4, 3, 64), (256, 64, 32, 1))), "out"),
    (lambda s: KV8Store(1, 0, 64, 64, device="cpu"), "heads 0"),
    (lambda s: window_attention(x(2, 4, 1, 64), x(2, 2, 9, 64), x(2, 2, 8, 64)), "keys and values"),
    (lambda s: window_attention(x(2, 4, 1, 80), x(2, 2, 9, 80), x(2, 2, 9, 80)), "head_dim 80"),
    (lambda s: window_attention(x(2, 4, 1, 64).float(), x(2, 2, 9, 64).float(), x(2, 2, 9, 64).float()), "fp16 or bf16"),
    (lambda s: window_attention(x(2, 4, 1, 64), x(2, 2, 9, 64), x(2, 2, 9, 64), window=-1), "window"),
    (lambda s: window_attention(x(2, 4, 1, 64), x(2, 2, 9, 64), x(2, 2, 9, 64), lens=10), "lens"),
    (lambda s: window_attention(x(2, 4, 1, 64), x(2, 0, 9, 64), x(2, 0, 9, 64)), "kv heads"),
])
def test_calls_refused(call, what):
    with pytest.raises(ValueError, match=what):
        call(store())


def test_cpu_tensors_are_refused():
    s = store()
    with pytest.raises(RuntimeError, match="GPU only"):
        kv8_write(s, x(2, 2, 3, 64), x(2, 2, 3, 64), 0)
    with pytest.raises(RuntimeError, match="GPU only"):
        kv8_read(s, 5)
    with pytest.raises(RuntimeError, match="GPU only"):
        kv8_attention(x(2, 4, 1, 64), s, 5)
    with pytest.raises(RuntimeError, match="GPU only"):
        window_attention(x(2, 4, 1, 64), x(2, 2, 9, 64), x(2, 2, 9, 64))
    with pytest.raises(RuntimeError, match="GPU only"):
        KV8Cache(64, 2).update(x(1, 2, 3, 64), x(1, 2, 3, 64))


def test_cache_refuses():
    for kw, what in ((dict(head_dim=80), "head_dim"), (dict(fmt="e5m2"), "format"), (dict(window=0), "window"), (dict(sinks=-1), "sinks")):
        with pytest.raises(ValueError, match=what):
            KV8Cache(**kw)
    with pytest.raises(ValueError, match="window"):
        KV8Batch(1, 1, 64, window=0, device="cpu")
    c = KV8Cache(64, 2)
    with pytest.raises(ValueError, match="empty"):
        c.attend(x(1, 2, 1, 64))
    with pytest.raises(ValueError, match="same shape"):
        c.update(x(1, 2, 3, 64), x(1, 2, 4, 64))
    c.update(x(1, 2, 0, 64), x(1, 2, 0, 64))
    assert c.empty() and c.state == (None,) * 6 and c.fetch() == (None, None)
    with pytest.raises(ValueError, match="state"):
        c.state = (None,) * 5
    with pytest.raises(ValueError, match="format"):
        c.meta_state = {"offset": "3", "fmt": "fp8"}


def test_state_round_trip_on_the_host():
    c = KV8Cache(64, 2, "int8", 32, device="cpu")
    s = store(1, 2, 64, 128)
    s.k_codes.random_(-127, 128)
    s.k_scales.uniform_()
    c.state = (s.k_codes[:, :, :64].clone(), s.v_codes[:, :, :1].clone(), s.k_scales[:, :, :2].clone(), s.v_scales[:, :, :2].clone(),
               s.k_tail.clone(), s.v_tail.clone())
    assert c.offset == 64
    for bad in ("20", "65", "-1", "32"):
        with pytest.raises(ValueError, match="does not belong"):
            c.meta_state = {"offset": bad}
    c.meta_state = {"offset": "50", "fmt": "int8", "block": "32"}
    assert c.offset == 50
    assert torch.equal(c.state[0], s.k_codes[:, :, :64]) and torch.equal(c.state[2], s.k_scales[:, :, :2])
    with pytest.raises(ValueError, match="does not match"):
        KV8Cache(64, 2, "fp8", 32, device="cpu").state = c.state


def _aligned(n):
    buf = ctypes.create_string_buffer(n + 16)
    return buf, (ctypes.addressof(buf) + 15) // 16 * 16


def test_c_entry_points_refuse_before_device_work():
    lib = _lib.load()
    keep, a = _aligned(64)
    good = dict(k_codes=a, v_codes=a, k_scales=a, v_scales=a, k_tail=a, v_tail=a, cap=128, fmt=0, d=64, block=32, kv_dtype=0,
                batch=1, heads=1)
    rows = _lib.Rows4(a, 0, 64, 64)
    R = ctypes.byref

    def st(**kw):
        return R(_lib.KV8StoreDesc(**{**good, **kw}))

    U, I = _lib.TQ_ERR_UNSUPPORTED, _lib.TQ_ERR_INVALID
    for kw, rc in ((dict(d=80), U), (dict(d=0), U), (dict(block=8), U), (dict(block=128), U), (dict(fmt=2), U), (dict(kv_dtype=2), U),
                   (dict(cap=100), I), (dict(cap=-64), I), (dict(cap=2 ** 31), I), (dict(heads=0), I), (dict(batch=-1), I),
                   (dict(k_codes=None), I), (dict(v_tail=a + 2), I)):
        assert lib.tq_kv8_write(st(**kw), R(rows), R(rows), None, 0, None, 1, None) == rc, kw
        assert lib.tq_kv8_read(st(**kw), None, 0, 0, 1, 0, a, a, None) == rc, kw
    assert lib.tq_kv8_write(None, R(rows), R(rows), None, 0, None, 1, None) == I
    assert lib.tq_kv8_write(st(), None, R(rows), None, 0, None, 1, None) == I
    assert lib.tq_kv8_write(st(), R(rows), R(rows), None, 0, None, -1, None) == I
    assert lib.tq_kv8_write(st(), R(rows), R(rows), None, 128, None, 1, None) == I
    assert lib.tq_kv8_write(st(), R(rows), R(rows), None, -1, None, 1, None) == I
    assert lib.tq_kv8_write(st(), R(rows), R(rows), None, 2 ** 31 - 1, None, 1, None) == I
    for bad in (_lib.Rows4(None, 0, 64, 64), _lib.Rows4(a + 2, 0, 64, 64), _lib.Rows4(a, 0, 64, 65)):
        assert lib.tq_kv8_write(st(), R(bad), R(rows), None, 0, None, 1, None) == I
        assert lib.tq_kv8_write(st(), R(rows), R(bad), None, 0, None, 1, None) == I
    assert lib.tq_kv8_write(st(), R(rows), R(rows), None, 0, None, 0, None) == 0
    assert lib.tq_kv8_read(st(), None, 129, 0, 1, 0, a, a, None) == I
    assert lib.tq_kv8_read(st(), None, 5, 100, 29, 0, a, a, None) == I
    assert lib.tq_kv8_read(st(), None, 5, 0, 1, 3, a, a, None) == U
    assert lib.tq_kv8_read(st(), None, 5, 0, 1, 0, None, a, None) == I

    base = dict(batch=1, hq=2, hkv=1, d=64, n_q=1, dtype=0, out_dtype=0, window=0, sinks=0, max_len=100, len_b=None, scale=1.0,
                q=rows, out=rows, k=rows, v=rows)

    def de(**kw):
        return R(_lib.KVAttnDesc(**{**base, **kw}))

    for kw, rc in ((dict(d=80), U), (dict(dtype=2), U), (dict(out_dtype=1), U), (dict(hq=0), I), (dict(hkv=0), I), (dict(hq=3, hkv=2), I),
                   (dict(n_q=-1), I), (dict(window=-1), I), (dict(sinks=-1), I), (dict(max_len=-1), I), (dict(batch=-1), I),
                   (dict(max_len=2 ** 31 - 1), U), (dict(n_q=2 ** 30, hq=64), U), (dict(q=_lib.Rows4(None, 0, 0, 0)), I),
                   (dict(out=_lib.Rows4(a + 8, 0, 0, 0)), I)):
        assert lib.tq_window_attention(de(**kw), a, 1 << 40, None) == rc, kw
        assert lib.tq_kv8_attention(st(), de(**kw), a, 1 << 40, None) == rc, kw
    assert lib.tq_window_attention(de(k=_lib.Rows4(a, 0, 0, 4)), a, 1 << 40, None) == I
    assert lib.tq_kv8_attention(st(), de(max_len=129), a, 1 << 40, None) == I
    assert lib.tq_kv8_attention(st(), de(batch=2), a, 1 << 40, None) == I
    assert lib.tq_kv8_attention(st(kv_dtype=1), de(), a, 1 << 40, None) == I
    assert lib.tq_kv8_attention(None, de(), a, 1 << 40, None) == I
    assert lib.tq_kv8_attention(st(), None, a, 1 << 40, None) == I
    # a call whose work is split needs its workspace
    long = dict(max_len=100000)
    need = lib.tq_window_attention_workspace_bytes(de(**long))
    assert need > 0
    assert lib.tq_window_attention(de(**long), a, need - 1, None) == _lib.TQ_ERR_WORKSPACE
    assert lib.tq_window_attention(de(**long), None, need, None) == _lib.TQ_ERR_WORKSPACE
    assert lib.tq_window_attention_workspace_bytes(de(d=80)) == 0
    # nothing to do
    assert lib.tq_window_attention(de(batch=0), None, 0, None) == 0 and lib.tq_window_attention(de(n_q=0), None, 0, None) == 0


def test_batches_whose_products_wrap_are_refused():
    """2^30 sequences of 2^30 heads: products with rows and tiles come to 2^64, which must not pass for 0."""
    lib = _lib.load()
    keep, a = _aligned(64)
    rows, n = _lib.Rows4(a, 0, 0, 0), 2 ** 30
    d = ctypes.byref(_lib.KVAttnDesc(batch=n, hq=n, hkv=n, d=64, n_q=2048, dtype=0, out_dtype=0, window=0, sinks=0, max_len=1024,
                                     len_b=None, scale=1.0, q=rows, out=rows, k=rows, v=rows))
    s = ctypes.byref(_lib.KV8StoreDesc(k_codes=a, v_codes=a, k_scales=a, v_scales=a, k_tail=a, v_tail=a, cap=1024, fmt=0, d=64, block=32,
                                       kv_dtype=0, batch=n, heads=n))
    U = _lib.TQ_ERR_UNSUPPORTED
    assert lib.tq_window_attention(d, a, 1 << 62, None) == U and lib.tq_window_attention_workspace_bytes(d) == 0
    assert lib.tq_kv8_attention(s, d, a, 1 << 62, None) == U
    assert lib.tq_kv8_write(s, ctypes.byref(rows), ctypes.byref(rows), None, 0, None, 512, None) == U
    assert lib.tq_kv8_read(s, None, 512, 0, 512, 0, a, a, None) == U


def test_workspace_is_bounded_by_what_a_window_reads():
    lib = _lib.load()
    keep, a = _aligned(64)
    rows = _lib.Rows4(a, 0, 0, 0)

    def need(**kw):
        d = dict(batch=1, hq=8, hkv=8, d=128, n_q=1, dtype=0, out_dtype=0, window=0, sinks=0, max_len=1 << 20, len_b=None, scale=1.0,
                 q=rows, out=rows, k=rows, v=rows)
        return lib.tq_window_attention_workspace_bytes(ctypes.byref(_lib.KVAttnDesc(**{**d, **kw})))

    assert need(window=1024, sinks=4) < need() and need(window=1024, max_len=2000) <= need(window=1024)
    assert need(window=1 << 20) == need() and math.isfinite(need(batch=1000))


def _model(head_dim=128, layers=4):
    import types
    return types.SimpleNamespace(config=types.SimpleNamespace(
        num_hidden_layers=layers, num_key_value_heads=8, num_attention_heads=8, hidden_size=8 * head_dim, head_dim=head_dim))


def test_skipped_layers_in_8_bits():
    from turboquant_amd import TurboQuantKVCache, apply_turboquant
    from turboquant_amd.patch import FP16KVCache
    for fmt in ("int8", "fp8"):
        m = apply_turboquant(_model(), skip_layers=[1, 3], auto_detect_outliers=False, skip_layer_format=fmt)
        assert [type(c) for c in m.make_cache()] == [TurboQuantKVCache, KV8Cache, TurboQuantKVCache, KV8Cache]
        assert m.make_cache()[1].fmt == fmt and m._turboquant_config["skip_layer_format"] == fmt
    m = apply_turboquant(_model(), skip_layers=[1], auto_detect_outliers=False)
    assert type(m.make_cache()[1]) is FP16KVCache
    with pytest.raises(ValueError, match="skip_layer_format"):
        apply_turboquant(_model(), skip_layer_format="int4")
    with pytest.raises(ValueError, match="head_dim 80"):
        apply_turboquant(_model(80), skip_layer_format="int8")


def test_8_bit_layer_in_transformers_refuses_float32():
    pytest.importorskip("transformers")
    from turboquant_amd.hf import TurboQuantLayer, fused_supported
    with pytest.raises(ValueError, match="fp16 or bf16"):
        TurboQuantLayer(KV8Cache(64, 2)).update(x(1, 2, 3, 64).float(), x(1, 2, 3, 64).float())
    assert fused_supported(KV8Cache(96, 2), 6, 2, 96) and not fused_supported(KV8Cache(64, 2), 3, 2, 64)
