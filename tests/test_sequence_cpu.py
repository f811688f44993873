"""CPU: the sequence operators refuse what they cannot take before anything is launched, in Python and at the C entry."""
import ctypes

import pytest
import torch

from htgs_b200 import _native, sequence as seq


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.ones(8)
    for call in (lambda: seq.add_rms_norm(x, w), lambda: seq.add_rms_norm_fp8(x, w), lambda: seq.quantize_fp8(x), lambda: seq.fp8_linear(x, x),
                 lambda: seq.gated_scan(x, x), lambda: seq.gated_scan_step(x, x, x),
                 lambda: seq.Fp8Matrix(torch.zeros(4, 16, dtype=torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.float8_e8m0fnu))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        seq.fp8_matmul(x, x)
    with pytest.raises(TypeError):
        seq.add_rms_norm([1.0], w)


def _refused(code, rc):
    assert rc == code and _native.last_error()


def test_c_entries_check_their_arguments():
    lib = _native.lib()
    BAD, SMALL = _native.HTGS_ERR_INVALID_ARGUMENT, _native.HTGS_ERR_WORKSPACE_TOO_SMALL
    norm = lambda **k: lib.htgs_add_rms_norm(*({"x": 64, "xs": 8, "r": None, "rs": 0, "w": 64, "type": 0, "rows": 4, "width": 8, "eps": 1e-6, "y": 64,  # noqa: E731
                                               "ys": 8, "sum": None, "ss": 0, "rstd": None, "codes": None, "cs": 0, "scales": None, "scs": 0, "stream": None} | k).values())
    for k in ({"type": 3}, {"type": -1}, {"rows": -1}, {"rows": 1 << 31}, {"width": 0}, {"width": 8193}, {"eps": -1.0}, {"eps": float("nan")}, {"x": None},
              {"w": None}, {"y": None}, {"codes": 64}, {"y": None, "codes": 64}):
        _refused(BAD, norm(**k))
    assert norm(rows=0) == 0
    assert lib.htgs_add_rms_norm_backward_scratch_bytes(0, 8) == 0 and lib.htgs_add_rms_norm_backward_scratch_bytes(100, 8) >= 32
    _refused(SMALL, lib.htgs_add_rms_norm_backward(64, 8, None, 0, 64, 8, None, 0, 64, 64, 0, 4, 8, 64, 8, 64, 64, 8, None))
    _refused(BAD, lib.htgs_add_rms_norm_backward(64, 8, None, 0, 64, 8, None, 0, 64, 64, 0, 4, 8, 64, 8, None, 64, 1 << 20, None))
    quantize = lambda rps=1, rows=4, codes=64, scales=64, t=0: lib.htgs_quantize_fp8(64, 8, t, rows, 8, rps, codes, 16, scales, 4, None, 0, None, 0, None)  # noqa: E731
    for k in ({"rps": 2}, {"rows": -1}, {"codes": None}, {"scales": None}, {"t": 7}):
        _refused(BAD, quantize(**k))
    assert quantize(rows=0) == 0

    def matrix(**k):
        return _native.HtgsFp8Matrix(*({"codes": 1024, "scales": 1024, "rows": 4, "width": 200, "cs": 208, "ss": 4, "rps": 1} | k).values())
    product = lambda a, b, out=64, stride=4, t=0: lib.htgs_fp8_matmul(ctypes.byref(a), ctypes.byref(b), out, stride, t, None)  # noqa: E731
    for k in ({"codes": 1025}, {"codes": None}, {"scales": 1026}, {"scales": None}, {"cs": 200}, {"cs": 192}, {"ss": 2}, {"rps": 64}, {"rows": -1}, {"width": 1 << 31}):
        _refused(BAD, product(matrix(**k), matrix()))
        _refused(BAD, product(matrix(), matrix(**k)))
    _refused(BAD, product(matrix(), matrix(width=128)))
    _refused(BAD, product(matrix(), matrix(), t=5))
    _refused(BAD, product(matrix(), matrix(), out=None))
    _refused(BAD, product(matrix(), matrix(), stride=3))
    assert product(matrix(rows=0), matrix()) == 0
    values = lambda b, x=64, t=0, rows=4, out=64, stride=4, o=0: lib.htgs_fp8_matmul_values(x, 200, t, rows, ctypes.byref(b), out, stride, o, None)  # noqa: E731
    for k in ({"x": None}, {"t": 3}, {"rows": 9}, {"rows": -1}, {"out": None}, {"stride": 3}, {"o": -1}):
        _refused(BAD, values(matrix(), **k))
    _refused(BAD, values(matrix(codes=1025)))
    _refused(BAD, values(matrix(width=9000, cs=9008, ss=72)))
    assert values(matrix(), rows=0) == 0
    _refused(BAD, lib.htgs_dequantize_fp8(ctypes.byref(matrix(rps=3)), 64, 200, 0, None))
    _refused(BAD, lib.htgs_dequantize_fp8(None, 64, 200, 0, None))

    def scan(**k):
        return _native.HtgsScan(*({"x": 64, "gate": 64, "initial": None, "offsets": None, "xs": 8, "gs": 8, "rows": 300, "width": 8, "n": 1, "type": 0,
                                   "reverse": 0} | k).values())
    forward = lambda s, h=64, last=64, ws=64, size=1 << 30: lib.htgs_gated_scan(ctypes.byref(s), h, 8, last, None, ws, size, None)  # noqa: E731
    for k in ({"x": None}, {"gate": None}, {"rows": -1}, {"rows": 1 << 31}, {"width": 0}, {"width": 65537}, {"n": 0}, {"n": 7}, {"type": 4}, {"xs": -8}, {"gs": (1 << 22) + 1}):
        _refused(BAD, forward(scan(**k)))
        _refused(BAD, lib.htgs_gated_scan_backward(ctypes.byref(scan(**k)), 64, 64, 8, None, 64, 8, 64, 8, None, 64, 1 << 30, None))
    _refused(BAD, forward(scan(), h=None))
    _refused(BAD, forward(scan(), last=None))
    _refused(SMALL, forward(scan(), size=16))
    _refused(SMALL, forward(scan(), ws=8))
    _refused(BAD, lib.htgs_gated_scan_backward(ctypes.byref(scan()), None, 64, 8, None, 64, 8, 64, 8, None, 64, 1 << 30, None))
    _refused(BAD, lib.htgs_gated_scan_step(64, 8, 64, 8, None, 8, 64, 8, 0, 4, 8, None))
    _refused(BAD, lib.htgs_gated_scan_step(64, 8, 64, 8, 64, 8, 64, 8, 9, 4, 8, None))
    assert lib.htgs_gated_scan_step(64, 8, 64, 8, 64, 8, 64, 8, 0, 0, 8, None) == 0


def test_workspace_sizes():
    lib = _native.lib()
    assert lib.htgs_gated_scan_workspace_bytes(0, 64) == 0 and lib.htgs_gated_scan_state_bytes(-1, 64) == 0
    for rows, width in ((1, 1), (128, 64), (129, 7), (1_000_000, 128)):
        assert lib.htgs_gated_scan_state_bytes(rows, width) == -(-rows // 8) * width * 4            # a state for every eight rows
        assert lib.htgs_gated_scan_workspace_bytes(rows, width) >= -(-rows // 64) * width * 12      # a map and a state for each chunk
