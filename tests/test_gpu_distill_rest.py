"""The distillation loss with the teacher's rest as an event (tail=True), where the student leaves next to nothing outside
the list: the mass there may lie below every f32, or every f64, while loss and gradient are ordinary numbers."""
import math

import pytest
import torch

from oracle import answers_oracle as ao
from test_gpu_answers import _check_distill, _close

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]
SHORT, LONG = [17, 430, 1024], [1025, 30522, 50265, 70001]   # a wave to a row, a workgroup to a row


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def _rows(C, gap, T, dtype):
    """Sixteen listed answers and, `gap` temperatures below the best of them, everything else; the teacher's rest is 0.1,
    or 0.4 where an answer is named twice."""
    R, K = 6, 16
    g = torch.Generator().manual_seed(C + int(gap))
    x = 20.0 - gap * T + torch.randn(R, C, generator=g) * T
    idx = torch.stack([torch.randperm(C, generator=g)[:K] for _ in range(R)])
    x.scatter_(1, idx, 20.0 - torch.rand(R, K, generator=g) * 4 * T)
    v = torch.log_softmax(torch.randn(R, K, generator=g), 1) + math.log(0.9)
    out = torch.ones(C, dtype=torch.bool)
    out[idx[1]] = False
    ruled = torch.nonzero(out)[:, 0]
    x[1, ruled[:: 2]] = -math.inf                      # half of the rest is masked (all of it where it is one class)
    x[2, ruled[0]] = 20.0 if int(ruled[0]) not in idx[2].tolist() else x[2, ruled[0]]   # one class outside is as likely
    idx[3, 5] = idx[3, 2]
    v[3] -= math.log(1.5)
    x[4].clamp_(min=20.0 - gap * T)                    # ties at the bottom
    idx[5, 9:] = -1
    return x.to(dtype), v.float(), idx


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [0.25, 1.0, 2.0 ** -12])
@pytest.mark.parametrize("gap", [-95, 60, 80, 87, 95, 100, 110, 300, 800])
@pytest.mark.parametrize("C", SHORT + LONG)
def test_rest_far_below_the_list(dev, C, gap, T, dtype):
    x, v, idx = _rows(C, gap, T, dtype)
    loss, _, g, _ = ao.distill(x, v, idx, T, True)
    finite = (x > -math.inf).all(1)
    assert bool(torch.isfinite(loss[finite]).all()) and bool(torch.isfinite(g).all())   # by the definition
    _check_distill(x, x.to(dev), v, idx, T, True, dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [SHORT[1], LONG[1]])
def test_rest_masked_by_large_numbers(dev, C, dtype):
    """Masks of -500, -1e4 and the type's lowest value in the place of -inf: the rest is shared by what they leave equal."""
    T = 0.5
    x, v, idx = _rows(C, 10, T, dtype)
    on = torch.zeros(x.shape, dtype=torch.bool).scatter_(1, idx.clamp_min(0), True)
    for r, low in enumerate((-500.0, -1e4, torch.finfo(dtype).min)):
        x[r] = torch.where(on[r], x[r], torch.tensor(low, dtype=dtype))
    x[4] = torch.finfo(dtype).min                      # the whole row
    _check_distill(x, x.to(dev), v, idx, T, True, dev)


@pytest.mark.parametrize("C", [SHORT[1], LONG[0], LONG[3]])
def test_rest_of_rows_that_hold_no_numbers(dev, C):
    """NaN and infinities on either side of the list, alone and with everything else masked."""
    x, v, idx = _rows(C, 100, 1.0, torch.float32)
    x = x.repeat(2, 1)
    v, idx = v.repeat(2, 1), idx[:1].repeat(12, 1)
    out = torch.ones(C, dtype=torch.bool)
    out[idx[0]] = False
    far = torch.nonzero(out)[3, 0]
    x[0, idx[0, 4]] = math.nan
    x[1, far] = math.nan
    x[2, idx[0, 4]] = math.inf
    x[3, far] = math.inf
    x[4] = -math.inf
    x[5] = -math.inf
    x[5, far] = math.nan
    x[6] = -math.inf
    x[6, idx[0, 0]] = math.nan
    x[7, out] = -math.inf                              # nothing outside the list
    x[8, out] = -math.inf
    x[8, far] = math.nan
    x[9] = -math.inf
    x[9, far] = 1.0                                    # nothing on it
    idx[10] = -1
    x[11, idx[0]] = -math.inf
    _check_distill(x, x.to(dev), v, idx, 1.0, True, dev)


@pytest.mark.parametrize("C", [11, 430, 1500])
def test_gradient_against_differences(dev, C):
    """Central differences of the 64-bit definition, a hundred temperatures between the list and the rest."""
    from vqa_amd import ops
    T = 1.25
    g = torch.Generator().manual_seed(C)
    x = torch.randn(2, C, generator=g) - 100 * T
    idx = torch.tensor([[1, 4, 0, 9], [2, 8, 5, 3]])
    x.scatter_(1, idx, torch.randn(2, 4, generator=g))
    v = torch.log_softmax(torch.randn(2, 4, generator=g), 1) + math.log(0.7)
    xd = x.to(dev).requires_grad_()
    got, = torch.autograd.grad(ops.distill_loss(xd, v.to(dev), idx.to(dev), temperature=T, tail=True, reduction="sum"), xd)
    h = 1e-4   # the third derivative's h^2 / 6, about 1e-8; sums of 64 bits near 100 add 1e-14 / h
    for r in range(2):
        for j in (0, 1, 2, 6, 7, C - 1):
            hi, lo = x.double().clone(), x.double().clone()
            hi[r, j] += h
            lo[r, j] -= h
            want = float(ao.distill(hi, v, idx, T, True)[0].sum() - ao.distill(lo, v, idx, T, True)[0].sum()) / (2 * h)
            assert abs(float(got[r, j]) - want) < 2e-6


def test_replayed_graph_and_second_stream(dev):
    """The loss and both of its backward passes captured once, replayed on new rows, and beside another stream's."""
    from vqa_amd import ops
    for C in (430, 30522):
        x, v, idx = _rows(C, 100, 1.0, torch.float32)
        xs = [x.to(dev), _rows(C, 300, 1.0, torch.float32)[0].to(dev), x.flip(0).to(dev)]
        vd, idxd = v.to(dev), idx.to(dev)
        leaf = xs[0].clone().requires_grad_()

        def step():
            loss = ops.distill_loss(leaf, vd, idxd, tail=True)
            rows = ops.distill_loss(leaf, vd, idxd, tail=True, reduction="none")
            ga, = torch.autograd.grad(loss, leaf, ops.unit_gradient(loss))
            gb, = torch.autograd.grad(rows, leaf, torch.full_like(rows, 0.3))
            return [loss.detach(), rows.detach(), ga, gb]
        eager = []
        for y in xs:
            with torch.no_grad():
                leaf.copy_(y)
            eager.append([t.clone() for t in step()])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        side = torch.cuda.Stream()
        for _ in range(3):
            for y, want in zip(xs, eager):
                with torch.no_grad():
                    leaf.copy_(y)
                graph.replay()
                with torch.cuda.stream(side):
                    other = ops.distill_loss(xs[1], vd, idxd, tail=True)
                torch.cuda.synchronize()
                for a, b in zip(out, want):
                    assert torch.equal(a, b)
                assert torch.equal(other, eager[1][0])


def test_one_class_outside(dev):
    """C = K + 1: the whole rest meets one class, at every gap."""
    for gap in (0.0, 50.0, 90.0, 1000.0):
        for C in (2, 17, 129):
            K = C - 1
            x = torch.zeros(3, C)
            x[:, -1] = -gap
            v = torch.full((3, K), math.log(0.5 / K))
            idx = torch.arange(K).repeat(3, 1)
            _check_distill(x, x.to(dev), v, idx, 1.0, True, dev)
            loss, tol, _, _ = ao.distill(x, v, idx, 1.0, True)
            # q log(q / p) on the list and 0.5 log(0.5 / p) outside, by hand
            z = math.log(K + math.exp(-gap)) if gap < 700 else math.log(K)
            by_hand = 0.5 * (math.log(0.5 / K) + z) + 0.5 * (math.log(0.5) + gap + z)
            _close(loss[:1], torch.tensor([by_hand], dtype=torch.float64), tol[:1] + 1e-6, "oracle")   # (v is f32: 2^-24 each)
