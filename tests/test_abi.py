"""The shared library loads on a machine without a GPU and exports every symbol that
include/b200gptq.h declares (no kernel is launched here)."""
import ctypes
import os
import re

from conftest import ROOT


def _declared_symbols():
    text = open(os.path.join(ROOT, "include", "b200gptq.h")).read()
    return sorted(set(re.findall(r"B200GPTQ_API\s+[\w\s\*]+?\b(b200gptq_\w+)\s*\(", text)))


def test_header_declares_the_expected_entry_points():
    names = _declared_symbols()
    for must in ("b200gptq_gemv", "b200gptq_gemm", "b200gptq_dequant", "b200gptq_sort_rows",
                 "b200gptq_workspace_bytes", "b200gptq_strerror"):
        assert must in names


def test_library_exports_every_declared_symbol():
    from autogptq.tvm_b200 import build
    path = build.build()  # no-op when the library is newer than its sources
    lib = ctypes.CDLL(path)
    for name in _declared_symbols():
        assert hasattr(lib, name), f"{name} is declared in the header but not exported"


def test_status_strings_and_host_side_queries():
    from autogptq.tvm_b200 import _lib
    lib = _lib.lib
    assert lib.b200gptq_abi_version() >= 1
    assert lib.b200gptq_strerror(0) == b"ok"
    for code in range(-8, 0):
        assert lib.b200gptq_strerror(code) not in (b"", b"unknown status")
    assert lib.b200gptq_strerror(-99) == b"unknown status"
    # argument validation happens on the host before anything touches the device
    assert lib.b200gptq_gemv(None, None, None, None, None, None, None, None, 1, 4096, 4096, 4, 128, None, 0, None) == -1
    assert lib.b200gptq_dequant(None, None, None, None, 4096, 4096, 4, 128, None, None, None) == -1


def test_quantlinear_refuses_cpu_tensors_and_bad_bits():
    import pytest
    import torch
    from autogptq.tvm_b200 import QuantLinear
    with pytest.raises(NotImplementedError):
        QuantLinear(5, 128, 256, 64, False)
    with pytest.raises(ValueError):
        QuantLinear(4, 128, 100, 64, False)
    layer = QuantLinear(4, 128, 256, 64, True)
    assert layer.qweight.shape == (32, 64) and layer.qzeros.shape == (2, 8) and layer.scales.shape == (2, 64)
    assert layer.g_idx.tolist()[:3] == [0, 0, 0] and int(layer.g_idx[-1]) == 1
    with pytest.raises(RuntimeError):
        layer(torch.zeros(1, 256))


def test_a_prepared_module_can_be_copied_and_saved():
    """The native call object and the plans stay behind (they hold addresses); everything else travels."""
    import copy
    import io
    import torch
    from autogptq.tvm_b200 import QuantLinear, _lib
    m = QuantLinear(4, 128, 256, 64, True)
    m.bias.normal_()
    m._native = _lib._host.Layer(256, 64, 4, 128, 0, m.__dict__, True, 16, m.qweight, None, None)
    m._native_state, m._native_tuning = m._constants(), None
    m._plans = {(1, None, 0): (ctypes.c_void_p(1), m._constants())}
    m._ready_for = m._stored()
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    for c in (copy.deepcopy(m), torch.load(f, weights_only=False)):
        assert c._native is None and c._plans == {} and not c._ready()
        assert torch.equal(c.bias, m.bias) and torch.equal(c.g_idx, m.g_idx) and c.groupsize == 128
    assert m._native is not None and m._ready()


def test_attention_refuses_caches_that_are_not_aligned():
    """Keys and values are read 16 bytes at a time; the check comes before anything is launched (the addresses are made up)."""
    from autogptq.tvm_b200 import _lib
    a, off = 0x100000, 0x100008
    for k, v in ((off, a), (a, off)):
        for hd in (64, 128):
            assert _lib.lib.b200gptq_attn_decode(a, k, v, a, a, 1, 8, hd, 256, 1.0, None) == -4
            assert _lib.lib.b200gptq_attn_step(a, a, a, a, k, v, a, 1, 8, hd, 256, 1, 1.0, None) == -4


def test_attention_with_a_window_or_a_prefix_refuses_on_the_host():
    """Every check comes before anything is launched (the addresses are made up)."""
    import ctypes
    from autogptq.tvm_b200 import _lib
    A = 0x100000
    good = dict(q=A, k_cache=A, v_cache=A, out=A, pos=A, dtype=0, batch=2, tokens=1, heads=8, kv_heads=2, hd=64, max_seq=40, window=4, scale=1.0)

    def call(fn=_lib.lib.b200gptq_attn, ws=None, ws_bytes=0, **change):
        a = _lib.AttnArgs(**{k: v for k, v in dict(good, **change).items() if "stride" not in k})
        for n in ("q_stride", "out_stride", "k_stride", "v_stride"):
            setattr(a, n, (ctypes.c_int64 * 3)(*change.get(n, (512, 64, 64))))
        for n in ("k_prefix_stride", "v_prefix_stride"):
            setattr(a, n, (ctypes.c_int64 * 2)(*change.get(n, (512, 64))))
        return fn(ctypes.byref(a), ws, ws_bytes, None) if fn is _lib.lib.b200gptq_attn else fn(ctypes.byref(a))

    assert _lib.lib.b200gptq_attn(None, None, 0, None) == -1 and _lib.lib.b200gptq_attn_workspace_bytes(None) == -1
    for change, status in [
        (dict(q=None), -1), (dict(k_cache=None), -1), (dict(v_cache=None), -1), (dict(out=None), -1), (dict(pos=None), -1),
        (dict(window=0, prefix=5), -1), (dict(window=0, prefix=5, k_prefix=A), -1),
        (dict(dtype=2), -3), (dict(dtype=-1), -3), (dict(batch=0), -3), (dict(tokens=0), -3), (dict(heads=0), -3), (dict(kv_heads=3), -3), (dict(kv_heads=0), -3),
        (dict(hd=80), -3), (dict(max_seq=0), -3), (dict(window=-1), -3), (dict(sinks=-1), -3), (dict(prefix=-1), -3), (dict(prefix=5), -3),
        (dict(window=0, sinks=3), -3), (dict(batch=1 << 20, tokens=1 << 20), -8), (dict(max_seq=(1 << 29) + 1), -8), (dict(window=(1 << 29) + 1), -8),
        (dict(q=A + 8), -4), (dict(k_cache=A + 2), -4), (dict(v_cache=A + 8), -4), (dict(out=A + 8), -4), (dict(pos=A + 4), -4), (dict(counts=A + 4), -4),
        (dict(q_stride=(512, 64, 68)), -4), (dict(k_stride=(4, 64, 64)), -4), (dict(v_stride=(512, 4, 64)), -4), (dict(out_stride=(512, 64, 1)), -4),
        (dict(window=0, prefix=5, k_prefix=A, v_prefix=A + 8), -4), (dict(window=0, prefix=5, k_prefix=A, v_prefix=A, v_prefix_stride=(512, 4)), -4),
        (dict(window=0, prefix=200000, k_prefix=A, v_prefix=A), -5),
    ]:
        assert call(**change) == status, change
    assert call(fn=_lib.lib.b200gptq_attn_workspace_bytes) == 0
    need = call(fn=_lib.lib.b200gptq_attn_workspace_bytes, window=0, prefix=200000)
    assert need > 0 and need % (2 * 8 * 66 * 4) == 0
    assert call(window=0, prefix=200000, k_prefix=A, v_prefix=A, ws=A, ws_bytes=need - 1) == -5
    assert call(window=0, prefix=200000, k_prefix=A, v_prefix=A, ws=A + 8, ws_bytes=need) == -4
    assert call(fn=_lib.lib.b200gptq_attn_workspace_bytes, hd=96) == -3


def test_logit_rules_refuse_on_the_host():
    import ctypes
    from autogptq.tvm_b200 import _lib
    A = 0x100000
    good = dict(logits=A, out=A, history=A, lengths=A, bias_tokens=A, bias_values=A, dtype=0, rows=2, vocab=100, history_len=5, biases=2, logits_stride=100, out_stride=100)
    assert _lib.lib.b200gptq_adjust_logits(None, None) == -1
    for change, status in [(dict(logits=None), -1), (dict(out=None), -1), (dict(lengths=None), -1), (dict(bias_tokens=None), -1), (dict(bias_values=None), -1),
                           (dict(rows=0), -3), (dict(vocab=0), -3), (dict(history_len=-1), -3), (dict(biases=-1), -3), (dict(dtype=3), -3), (dict(logits_stride=-1), -3),
                           (dict(logits=A + 1), -4), (dict(out=A + 2, dtype=2), -4), (dict(history=A + 4), -4), (dict(lengths=A + 4), -4),
                           (dict(repetition=A + 2), -4), (dict(presence=A + 1), -4), (dict(bias_values=A + 2), -4), (dict(mask=A + 2), -4)]:
        assert _lib.lib.b200gptq_adjust_logits(ctypes.byref(_lib.LogitArgs(**dict(good, **change))), None) == status, change


def test_attention_and_logit_rules_refuse_cpu_tensors():
    import pytest
    import torch
    from autogptq.tvm_b200 import ops
    q, k, p = torch.zeros(1, 1, 2, 64).half(), torch.zeros(1, 2, 8, 64).half(), torch.zeros(1).long()
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_window(q, k, k, p, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_prefix(q, k[0], k[0], k, k, p)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.adjust_logits(torch.zeros(1, 8))
    with pytest.raises(TypeError):
        ops.attn_window(None, k, k, p, 4)
    with pytest.raises(TypeError):
        ops.attn_prefix(q, None, None, k, k, p)
