"""Linear layers in eight-bit integers at the ends of the f32 range, and with scales that lie apart."""
import math

import pytest
import torch

from oracle import int8_oracle as io
from test_gpu_int8 import _close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


# tokens of one launch, of the few-token product and of every tile size
@pytest.mark.parametrize("M,N", [(3, 40), (50, 40), (130, 100), (2000, 2000), (4609, 1800)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tokens_near_the_end_of_the_range(dev, M, N, dtype):
    """The sum times the token's scale may lie past the f32 range where the channel's scale brings it back."""
    from vqa_amd import ops
    K = 96
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).abs() + 0.5                 # sums of one sign: up to 2^20
    w = (torch.randn(N, K, generator=g).abs() + 0.5) * 1e-6
    big = torch.finfo(dtype).max / float(x.abs().amax()) / 2
    rows = torch.arange(M) % 3
    x[rows == 0] *= big
    x[rows == 1] *= 2.0 ** 101                                     # scales to both sides of 2^96
    x = x.to(dtype)
    w[N // 2] *= 1e-30                                             # a channel of tiny weights
    w[N - 1] *= 1e20                                               # ... and of ones whose outputs are infinite
    wq, ws = ops.quantize_rows(w.to(dev))
    bias = torch.linspace(-1, 1, N)
    for b in (bias, None):
        y = ops.int8_linear(x.to(dev), wq, ws, None if b is None else b.to(dev), out_dtype=torch.float32).cpu()
        want, tol = io.linear(x, wq.cpu(), ws.cpu(), b, torch.float32)
        far = want.abs() > torch.finfo(torch.float32).max
        near = (want.abs() * (1 - 2.0 ** -20) <= torch.finfo(torch.float32).max) & \
               (want.abs() * (1 + 2.0 ** -20) >= torch.finfo(torch.float32).max)
        assert bool(far.any()) and not bool(far[:, 0].any())
        assert bool(torch.isinf(y[far & ~near]).all())
        ok = ~far & ~near
        _close(y[ok], want[ok], tol[ok], f"{M} {N}")


def test_rows_do_not_depend_on_their_neighbours(dev):
    """A row of large numbers in a tile changes no other row's bits."""
    from vqa_amd import ops
    for M, N, K in ((4, 40, 96), (50, 40, 96), (130, 100, 200), (2000, 2000, 130), (4609, 1800, 64)):
        g = torch.Generator().manual_seed(M)
        x = torch.randn(M, K, generator=g)
        wq, ws = ops.quantize_rows(torch.randn(N, K, generator=g).to(dev))
        bias = torch.linspace(-1, 1, N, device=dev)
        want = ops.int8_linear(x.to(dev), wq, ws, bias)
        x[1] *= 1e37
        got = ops.int8_linear(x.to(dev), wq, ws, bias)
        keep = torch.arange(M) != 1
        assert torch.equal(got[keep.to(dev)], want[keep.to(dev)])


def _next_to_borders(steps):
    """Rows whose scale is an odd multiple of 2^-149 below 2^-125, of the values that f32 has next to the borders between
    two steps: down to half a unit (2^-150) to either side."""
    x = torch.zeros(len(steps), 254)
    for r, k in enumerate(steps):                     # the scale is k 2^-149
        border = [(2 * q + 1) * k // 2 for q in range(-63, 63)]          # (q + 1/2) k, rounded down
        vals = [127 * k] + border + [b + 1 for b in border] + [0]
        x[r] = torch.tensor(vals, dtype=torch.float64).mul(2.0 ** -149).float()
    return x


def test_borders_of_subnormal_steps(dev):
    """The quotient is rounded as if it were exact also where half a step is no f32 number."""
    from vqa_amd import ops
    x = _next_to_borders([2 ** 23 + 1, 2 ** 23 + 7, 2 ** 23 + 12345, 2 ** 24 - 1, 2 ** 24 - 4321])
    want_q, want_s = io.quantize_rows(x)
    assert bool((want_s < 2.0 ** -125).all())
    half = (x.double() / want_s[:, None]).abs() % 1 - 0.5
    assert bool((half[:, 1:253] != 0).all()) and float(half[:, 1:253].abs().max()) < 2.0 ** -18    # next to a tie, never one
    q, s = ops.quantize_rows(x.to(dev))
    assert torch.equal(s.cpu().double(), want_s) and torch.equal(q.cpu().double(), want_q)
    # one token quantised in the product's own launch
    w = torch.eye(254, 256, dtype=torch.int8, device=dev)[:, :254]
    ones = torch.full((254,), 2.0 ** 100, device=dev)
    for m in range(x.shape[0]):
        y = ops.int8_linear(x[m:m + 1].to(dev), w, ones)
        assert torch.equal(torch.round(y.cpu().double() / (want_s[m] * 2.0 ** 100)), want_q[m:m + 1])


@pytest.mark.parametrize("M", [3, 40, 200])
def test_strided_scales(dev, M, monkeypatch):
    """Scales that lie apart, while other allocations take whatever is free between the call's preparation and its launch
    (another thread's, on the same stream)."""
    from vqa_amd import ops
    K, N = 100, 70
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).to(dev)
    wq, ws = ops.quantize_rows(torch.randn(N, K, generator=g).to(dev))
    bias = torch.linspace(-1, 1, N, device=dev)
    apart, wide = torch.stack([ws, ws + 1], 1)[:, 0], torch.stack([bias, bias], 1)[:, 1]
    shared = ws[:1].expand(N)
    want, want_shared = ops.int8_linear(x, wq, ws, bias), ops.int8_linear(x, wq, shared.contiguous(), bias)
    real, taken = ops._launch, []

    def launch(device, entry, *args):
        taken.extend(torch.full((n,), math.nan, device=dev) for n in (N, N, 128, 128))
        return real(device, entry, *args)
    monkeypatch.setattr(ops, "_launch", launch)
    assert not apart.is_contiguous() and not wide.is_contiguous() and not shared.is_contiguous()
    assert torch.equal(ops.int8_linear(x, wq, apart, wide), want)
    assert torch.equal(ops.int8_linear(x, wq, shared, bias), want_shared)
