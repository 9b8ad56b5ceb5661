"""Answer scores and distillation: what is refused, decided on the host (no GPU)."""
import ctypes

import pytest
import torch


def _ops():
    from vqa_amd import ops
    return ops


def test_cpu_tensors_are_refused():
    ops = _ops()
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.token_logprobs(torch.zeros(2, 5))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.distill_loss(torch.zeros(2, 5), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.long))
    with pytest.raises(ValueError, match="classes"):
        ops.token_logprobs(torch.zeros(()))
    with pytest.raises(ValueError, match="reduction"):
        ops.distill_loss(torch.zeros(2, 5), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.long), reduction="max")


@pytest.mark.parametrize("t", [0.0, -1.0, float("nan"), float("inf"), 1e-9])
def test_temperatures(t):
    with pytest.raises(ValueError, match="temperature"):
        _ops()._temperature(t)


class _Fake:
    """Stands in for device addresses: the entry points check their arguments before any launch."""

    def __init__(self):
        self.buf = ctypes.create_string_buffer(4096)
        self.p = (ctypes.addressof(self.buf) + 63) // 64 * 64


def test_entry_points_refuse_bad_arguments():
    from vqa_amd import _lib
    lib, f = _lib.load(), _Fake()
    p = f.p

    def lp(x=p, ld=8, tg=p, R=2, C=8, T=1, K=2, dt=0, t=1.0, out=p, tl=p, ti=p):
        return lib.vqaf_token_logprobs(x, ld, tg, R, C, T, K, dt, t, out, p, tl, ti, None, None)
    assert lp(x=None) == -5 and lp(tg=None) == -5 and lp(tl=None) == -5
    assert lp(R=0) == -1 and lp(C=0) == -1 and lp(K=9) == -1 and lp(K=129, C=500) == -1 and lp(T=129) == -1 and lp(ld=-1) == -1
    assert lp(t=0.0) == -1 and lp(t=float("nan")) == -1 and lp(dt=2) == -2
    assert lp(x=p + 2) == -3 and lp(x=p + 1, dt=1) == -3

    def lb(st=p, ent=p, g=p + 64, ldg=8, ge=p, tg=p, ti=p, x=p):
        return lib.vqaf_token_logprobs_bwd(x, 8, tg, ti, 2, 8, 1, 2, 0, 1.0, st, ent, p, ge, p, g, ldg, None)
    assert lb(st=None) == -5 and lb(ent=None) == -5 and lb(tg=None) == -5 and lb(ti=None) == -5 and lb(g=None) == -5
    assert lb(g=p + 68) == -3 and lb(ldg=9) == -3 and lb(ldg=4) == -3

    def d(x=p, te=p, idx=p, R=2, C=8, K=2, dt=0, t=1.0, rows=p, g=None, ldg=0):
        return lib.vqaf_distill(x, 8, te, idx, R, C, K, dt, t, 0, rows, None, g, ldg, 1.0, None, None)
    assert d(x=None) == -5 and d(te=None) == -5 and d(idx=None) == -5 and d(rows=None) == -5
    assert d(K=0) == -1 and d(K=129, C=500) == -1 and d(t=-2.0) == -1 and d(dt=7) == -2 and d(g=p + 4, ldg=8) == -3
    assert lib.vqaf_distill(p, 400000, p, p, 2, 400000, 4, 0, 1.0, 1, p, None, None, 0, 1.0, None, None) == -1

    def db(step=0, up=p, g=p, ldg=8):
        return lib.vqaf_distill_bwd(p, 8, p, p, 2, 8, 2, 0, 1.0, p, up, step, 0, 1.0, g, ldg, None)
    assert db(step=2) == -1 and db(up=None) == -5 and db(ldg=10) == -3 and db(g=p + 4) == -3


def test_module_loads_without_torch_s_private_names():
    """A torch without the quick ways to the current device and stream: the module imports and checks its arguments."""
    import subprocess
    import sys

    from conftest import ROOT
    code = ("import torch\n"
            "for n in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    if hasattr(torch._C, n): delattr(torch._C, n)\n"
            "from vqa_amd import ops\n"
            "try: ops.token_logprobs(torch.zeros(2, 5))\n"
            "except RuntimeError as e: print(e)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "GPU only" in r.stdout, r.stderr


@pytest.mark.parametrize("top", [0, -1, 129])
def test_distillation_needs_answers(top):
    """Refused before anything runs: a list of no answers used to end inside the first batch, in an AttributeError."""
    from vqa_amd import loops
    net = torch.nn.Linear(2, 3).eval()
    with pytest.raises(ValueError, match="top"):
        loops.distill(net, torch.nn.Linear(2, 3), [], torch.optim.SGD(net.parameters(), 0.1), "cpu", top=top)
    assert not net.training
