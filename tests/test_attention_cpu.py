"""CPU: rotary positions and attention refuse what they cannot take before anything is launched, in Python and at the C entry."""
import ctypes

import pytest
import torch

from htgs_b200 import _native, sequence as seq

BAD, SMALL = _native.HTGS_ERR_INVALID_ARGUMENT, _native.HTGS_ERR_WORKSPACE_TOO_SMALL


@pytest.mark.parametrize("compiled", [True, False])
def test_cpu_tensors_are_refused(compiled, monkeypatch):
    if not compiled:
        monkeypatch.setattr(_native, "_pybind_modules", False)
    x, n = torch.zeros(4, 2, 8), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: seq.rotary(x, x, torch.zeros(4, 3)), lambda: seq.attention(x, x, x), lambda: seq.attention_step(x, x, x, x[:, None], x[:, None].clone(), n)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        seq.attention([1.0], x, x)


def refused(rc, code=BAD):
    assert rc == code and _native.last_error()


def test_rotary_checks_its_arguments():
    def rotary(**k):
        r = _native.HtgsRotary()
        values = {"x": 64, "y": 64, "positions": 64, "stride": 16, "head_stride": 8, "positions_stride": 1, "rows": 4, "base": 1e4, "heads": 2, "sections": (4, 0), "axes": 1,
                  "positions_type": 0, "width": 8, "type": 0} | k
        r.x[0], r.y[0], r.x_stride[0], r.x_head_stride[0], r.heads[0] = (values[n] for n in ("x", "y", "stride", "head_stride", "heads"))
        for i, n in enumerate(values["sections"]):
            r.sections[i] = n
        for name in ("positions", "positions_stride", "rows", "base", "axes", "positions_type", "width", "type"):
            setattr(r, name, values[name])
        return _native.lib().htgs_rotary(ctypes.byref(r), None)
    for k in ({"x": None}, {"y": None}, {"positions": None}, {"stride": -1}, {"rows": -1}, {"rows": 1 << 31}, {"base": 0.0}, {"base": -1.0}, {"base": float("inf")}, {"base": float("nan")},
              {"heads": 0}, {"heads": 1 << 20}, {"sections": (3, 0)}, {"sections": (5, 0)}, {"sections": (5, -1), "axes": 2}, {"axes": 0}, {"axes": 5}, {"positions_type": 2}, {"width": 7},
              {"width": 0}, {"width": 258}, {"type": 3}, {"positions_stride": -1}):
        refused(rotary(**k))
    refused(_native.lib().htgs_rotary(None, None))
    assert rotary(rows=0) == 0


def attention(**k):
    values = {"q": 64, "k": 64, "v": 64, "offsets": None, "qs": 32, "ks": 16, "vs": 16, "qh": 16, "kh": 16, "vh": 16, "rows": 40, "heads": 2, "key_heads": 1, "width": 16, "n": 1,
              "type": 2, "causal": 0, "window": -1, "scale": 0.25} | k
    return _native.HtgsAttention(*values.values())


def test_attention_checks_its_arguments():
    lib = _native.lib()
    for k in ({"q": None}, {"k": None}, {"v": None}, {"qs": -1}, {"kh": -1}, {"rows": -1}, {"rows": 1 << 31}, {"heads": 0}, {"heads": 3, "key_heads": 2}, {"key_heads": 0}, {"width": 0},
              {"width": 129}, {"n": 0}, {"n": 7}, {"type": 3}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")}, {"rows": 0x7fffff00 // 64 * 64, "heads": 65536}):
        a = attention(**k)
        refused(lib.htgs_attention(ctypes.byref(a), 64, None, None, None))
        refused(lib.htgs_attention_backward(ctypes.byref(a), 64, None, 64, 64, 32, 16, 64, 64, 64, 64, 1 << 40, None))
        assert lib.htgs_attention_backward_workspace_bytes(ctypes.byref(a)) == 0
    a = attention()
    refused(lib.htgs_attention(ctypes.byref(a), None, None, None, None))
    refused(lib.htgs_attention(None, 64, None, None, None))
    for at in range(7):
        pointers = [None if i == at else 64 for i in range(7)]
        refused(lib.htgs_attention_backward(ctypes.byref(a), pointers[0], None, *pointers[1:3], 32, 16, *pointers[3:], 1 << 30, None), SMALL if at == 6 else BAD)
    refused(lib.htgs_attention_backward(ctypes.byref(a), 64, None, 64, 64, -1, 16, 64, 64, 64, 64, 1 << 30, None))
    refused(lib.htgs_attention_backward(ctypes.byref(a), 64, None, 64, 64, 32, 16, 64, 64, 64, 64, 16, None), SMALL)
    refused(lib.htgs_attention_backward(ctypes.byref(a), 64, None, 64, 64, 32, 16, 64, 64, 64, 72, 1 << 30, None), SMALL)
    assert lib.htgs_attention(ctypes.byref(attention(rows=0)), 64, None, None, None) == 0
    refused(lib.htgs_attention_status(-1))
    refused(lib.htgs_attention_status(64))


def test_attention_workspace_holds_the_tiles_of_every_packing():
    """Tiles of 128 rows that sequences share with none of the others, whatever their lengths."""
    for rows, n in ((1, 1), (127, 3), (128, 1), (1000, 7), (300, 300)):
        size = _native.lib().htgs_attention_backward_workspace_bytes(ctypes.byref(attention(rows=rows, n=n, offsets=64)))
        longest = (rows // 128 + n) * 128           # one row in all sequences but one
        assert size >= longest * 2 * 8
    assert _native.lib().htgs_attention_backward_workspace_bytes(ctypes.byref(attention(rows=300, n=3))) >= 3 * 128 * 2 * 8


def step(**k):
    values = {"q": 64, "k": 64, "v": 64, "keys": 64, "values": 128, "lengths": 64, "qs": 32, "ks": 16, "vs": 16, "qh": 16, "kh": 16, "vh": 16, "keys_s": 1600, "values_s": 1600, "keys_r": 16,
              "values_r": 16, "keys_h": 16, "values_h": 16, "capacity": 100, "batch": 2, "heads": 2, "key_heads": 1, "width": 16, "type": 2, "window": -1, "scale": 0.25} | k
    return _native.HtgsAttentionStep(*values.values())


def test_step_checks_its_arguments():
    lib = _native.lib()
    for k in ({"q": None}, {"k": None}, {"v": None}, {"keys": None}, {"values": None}, {"lengths": None}, {"qs": -1}, {"keys_s": -1}, {"values_r": -1}, {"capacity": -1}, {"capacity": 1 << 31},
              {"batch": -1}, {"heads": 0}, {"heads": 3, "key_heads": 2}, {"key_heads": 0}, {"width": 0}, {"width": 129}, {"type": 3}, {"scale": 0.0}, {"scale": float("nan")},
              {"batch": 0x7fffffff}):
        refused(lib.htgs_attention_step(ctypes.byref(step(**k)), 64, 64, 1 << 30, None))
        assert lib.htgs_attention_step_workspace_bytes(ctypes.byref(step(**k))) == 0
    refused(lib.htgs_attention_step(ctypes.byref(step()), None, 64, 1 << 30, None))
    refused(lib.htgs_attention_step(None, 64, 64, 1 << 30, None))
    long = step(capacity=100000)
    size = lib.htgs_attention_step_workspace_bytes(ctypes.byref(long))
    assert size > 0
    refused(lib.htgs_attention_step(ctypes.byref(long), 64, None, 0, None), SMALL)
    refused(lib.htgs_attention_step(ctypes.byref(long), 64, 64, size - 1, None), SMALL)
    refused(lib.htgs_attention_step(ctypes.byref(long), 64, 72, size, None), SMALL)
    assert lib.htgs_attention_step(ctypes.byref(step(batch=0)), 64, None, 0, None) == 0
