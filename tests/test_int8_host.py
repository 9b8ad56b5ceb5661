"""Eight-bit Linear layers: arguments the C entry points refuse on the host (no GPU)."""
import ctypes

import pytest
import torch


def test_entry_points_refuse_bad_arguments():
    from vqa_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def q(x=p, ld=64, M=2, K=60, dt=0, out=p, ldq=128, s=p):
        return lib.vqaf_quantize_rows(x, ld, M, K, dt, out, ldq, s, None)
    assert q(x=None) == -5 and q(out=None) == -5 and q(s=None) == -5
    assert q(M=0) == -1 and q(K=0) == -1 and q(ldq=48) == -1 and q(ldq=72) == -1 and q(ld=-1) == -1
    assert q(dt=3) == -2 and q(out=p + 8) == -3 and q(x=p + 2) == -3

    def y(x=p, ldx=64, xd=1, w=p, ldw=64, ws=p, b=None, bd=0, M=10, N=8, K=60, out=p, ldy=8, yd=1, wk=p, wb=1 << 15):
        return lib.vqaf_int8_linear(x, ldx, xd, w, ldw, ws, b, bd, M, N, K, out, ldy, yd, wk, wb, None)
    assert y(x=None) == -5 and y(w=None) == -5 and y(ws=None) == -5 and y(out=None) == -5 and y(wk=None) == -5
    assert y(M=0) == -1 and y(N=0) == -1 and y(K=0) == -1 and y(K=131073, ldw=131088) == -1
    assert y(ldw=48) == -1 and y(ldw=72) == -1 and y(ldy=7) == -1 and y(wb=16) == -1
    assert y(xd=2) == -2 and y(yd=5) == -2 and y(b=p, bd=9) == -2
    assert y(w=p + 4) == -3 and y(x=p + 1) == -3 and y(out=p + 1) == -3 and y(wk=p + 8) == -3 and y(b=p + 1, bd=1) == -3
    assert lib.vqaf_int8_linear_workspace_bytes(1, 768) == 0
    assert lib.vqaf_int8_linear_workspace_bytes(100, 768) >= 100 * 768 + 400


def test_cpu_tensors_are_refused():
    from vqa_amd import ops
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.quantize_rows(torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.int8_linear(torch.zeros(2, 4), torch.zeros(3, 4, dtype=torch.int8), torch.ones(3))
