"""Answer scores and the distillation loss (csrc/answers.hip) against their 64-bit statements: every row length class,
type, alignment, mask and edge of the definitions, with the error bounds that oracle/answers_oracle.py derives."""
import math

import pytest
import torch

from oracle import answers_oracle as ao

pytestmark = pytest.mark.gpu

# a wave's rows (1 to 16 registers), the workgroup shapes of both types and the rows that are read again
CLASSES = [1, 2, 13, 64, 65, 127, 430, 600, 1024, 1025, 1031, 4090, 4097, 8190, 16001, 30522, 50265, 65541, 70001]
DTYPES = [torch.bfloat16, torch.float32]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def _logits(R, C, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, C, generator=g) * spread
    x[torch.arange(R), torch.randint(0, C, (R,), generator=g)] += 5.0
    return x.to(dtype)


def _close(got, want, tol, what):
    got, want, tol = got.detach().double().cpu(), want.double(), tol.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    ok = ~(torch.isnan(want) | inf)
    off = ((got - want).abs() - tol)[ok]
    assert off.numel() == 0 or float(off.max()) <= 0, \
        f"{what}: off by {float((got - want).abs()[ok].max())}, {float(off.max())} over the bound"


def _check_logprobs(x, targets, top, T, dev, xd=None):
    from vqa_amd import ops
    want = ao.token_logprobs(x, targets, top, T)
    got = ops.token_logprobs(x.to(dev) if xd is None else xd, None if targets is None else targets.to(dev), top=top,
                             temperature=T)
    _close(got.entropy, want["entropy"], want["entropy_tol"], "entropy")
    if targets is not None:
        assert got.logprobs.shape == targets.shape
        _close(got.logprobs.reshape(x.shape[0], -1), want["logprobs"], want["logprobs_tol"], "logprobs")
    else:
        assert got.logprobs is None
    if top:
        assert torch.equal(got.top_indices.cpu(), want["top_indices"]), "top indices"
        _close(got.top_logprobs, want["top_logprobs"], want["top_logprobs_tol"], "top_logprobs")
    else:
        assert got.top_logprobs is None and got.top_indices is None
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", CLASSES)
def test_logprobs_every_row_length(dev, C, dtype):
    R = 5
    x = _logits(R, C, dtype, C)
    for T, top in ((1.0, min(C, 5)), (2.0, min(C, 20)), (0.7, min(C, 128)), (1.0, 0)):
        _check_logprobs(x, torch.arange(R) % C, top, T, dev)
    several = torch.randint(0, C, (R, 3), generator=torch.Generator().manual_seed(C))
    several[0] = torch.tensor([-100, C - 1, 0])
    several[1, 1] = C                      # past the classes
    _check_logprobs(x, several, min(C, 1), 1.0, dev)
    _check_logprobs(x, None, min(C, 64), 1.0, dev)


def _views(R, C, dtype, seed, dev):
    """The same rows in other layouts: a padded pitch, a row that starts off every alignment, columns first."""
    x = _logits(R, C, dtype, seed)
    base = x.to(dev)
    pad = torch.full((R, C + 3), 77.0, dtype=dtype, device=dev)
    pad[:, :C] = base
    off = torch.full((R, C + 5), float("nan"), dtype=dtype, device=dev)
    off[:, 3:3 + C] = base
    flat = torch.full((R * C + 1,), float("nan"), dtype=dtype, device=dev)
    flat[1:] = base.reshape(-1)
    yield x, pad[:, :C]
    yield x, off[:, 3:3 + C]
    yield x, flat[1:].view(R, C)
    yield x, base.t().contiguous().t()
    yield x[:1].expand(R, C).contiguous(), base[:1].expand(R, C)
    yield x[:1], flat[1:1 + C].view(1, C)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [7, 430, 1025, 4091, 30522, 65600])
def test_layouts_forward_and_gradient(dev, C, dtype):
    from vqa_amd import ops
    k = min(C, 9)
    for x, xd in _views(4, C, dtype, 3 * C, dev):
        R = x.shape[0]
        _check_logprobs(x, torch.arange(R) % C, k, 1.0, dev, xd)
        xg = xd.detach().requires_grad_() if xd.stride(0) != 0 else xd.detach()
        if xd.stride(0) == 0:
            continue
        tg = (torch.arange(R) * 3 % C)
        r = ops.token_logprobs(xg, tg.to(dev), top=k, temperature=1.5)
        up = [torch.linspace(-1, 2, R), torch.linspace(0.5, -0.5, R), torch.linspace(-1, 1, R * k).view(R, k)]
        g, = torch.autograd.grad((r.logprobs, r.entropy, r.top_logprobs), xg, [u.to(dev) for u in up])
        want, tol = ao.token_logprobs_grad(x, 1.5, tg, up[0], up[1], r.top_indices.cpu(), up[2])
        assert g.dtype == dtype and g.shape == xg.shape
        _close(g, want, tol, "gradient")
        v, idx = r.top_logprobs.detach(), r.top_indices
        _check_distill(x, xg, v.cpu(), idx.cpu(), 1.5, C > k, dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [5, 430, 1023, 1030, 9001, 30522, 66000])
def test_masked_rows_ties_and_broken_rows(dev, C, dtype):
    low = torch.finfo(dtype).min
    x = _logits(16, C, dtype, C + 1)
    x[12] = 0.0                                           # a few above one long tie
    x[12, [0, C // 2, C - 1]] = torch.tensor([1.0, 2.0, 1.0], dtype=dtype)
    x[13] = torch.arange(C) % 3 == 1                      # ties spread over the row
    x[14] = -torch.arange(C).to(dtype) / 64               # all negative, sorted
    x[15] = -5.0                                          # negative and tied, NaN with a sign bit among them
    x[15, C // 4] = -math.nan
    x[0] = -math.inf                                      # a mask that leaves nothing
    x[1] = low                                            # masks of the type's lowest value, everywhere
    x[2, 1:] = low                                        # one live entry
    x[3, : C // 2] = -math.inf
    x[4] = 1.0                                            # one long tie
    x[5, ::2] = -0.0
    x[5, 1::2] = 0.0                                      # zeros of both signs are equal
    x[6, C // 2] = math.nan
    x[7, C - 1] = math.inf
    x[8] = torch.linspace(4, -4, C).to(dtype)             # sorted: the best lie together
    x[9] = math.nan
    x[10] = -math.inf
    x[10, C // 3] = -3.0                                  # one live entry among masked ones
    x[11, : C - 1] = torch.finfo(dtype).max / 2           # the range's far ends
    x[11, C - 1] = low
    tg = torch.full((16,), C // 3)
    for top in sorted({1, min(C, 3), min(C, 40), min(C, 128)}):
        _check_logprobs(x, tg, top, 1.0, dev)
    from vqa_amd import ops
    xd = x.to(dev).requires_grad_()
    r = ops.token_logprobs(xd, tg.to(dev), temperature=0.5)
    up = torch.linspace(-1, 1, 16)
    g, = torch.autograd.grad((r.logprobs, r.entropy), xd, (up.to(dev), up.flip(0).to(dev)))
    want, tol = ao.token_logprobs_grad(x, 0.5, tg, up, up.flip(0))
    _close(g, want, tol, "gradient")


def test_gradient_of_targets_named_twice_and_none(dev):
    from vqa_amd import ops
    for C in (50, 2000):
        x = _logits(4, C, torch.float32, 5)
        tg = torch.tensor([[3, 3, 7, -1], [0, 0, 0, 0], [-1, -1, -1, -1], [C - 1, 3, C - 1, 1]])
        up = torch.arange(16.0).view(4, 4) / 7 - 1
        xd = x.to(dev).requires_grad_()
        lp = ops.token_logprobs(xd, tg.to(dev), top=5).logprobs
        g, = torch.autograd.grad(lp, xd, up.to(dev))
        want, tol = ao.token_logprobs_grad(x, 1.0, tg, up)
        _close(g, want, tol, "gradient")
        assert float(g[2].abs().max()) == 0.0


def test_gradients_against_differences(dev):
    """The analytic gradients against central differences of the 64-bit definitions."""
    from vqa_amd import ops
    for C in (11, 1100):
        x = _logits(2, C, torch.float32, 17)
        tg = torch.tensor([2, C - 1])
        xd = x.to(dev).requires_grad_()
        r = ops.token_logprobs(xd, tg.to(dev), temperature=1.3)
        g, = torch.autograd.grad((r.logprobs.sum() * 0.7 + r.entropy.sum() * 0.4), xd)
        v, idx = torch.randn(2, 4, generator=torch.Generator().manual_seed(1)) - 2, torch.tensor([[1, 4, 0, 9], [2, 8, 5, 3]])
        xd2 = x.to(dev).requires_grad_()
        loss = ops.distill_loss(xd2, v.to(dev), idx.to(dev), temperature=1.3, tail=True, reduction="sum")
        gd, = torch.autograd.grad(loss, xd2)
        h = 1e-4   # central differences: the third derivative's h^2 / 6, about 1e-8
        for j in (0, 1, 2, 5, C - 1):
            for r_ in range(2):
                hi, lo = x.double().clone(), x.double().clone()
                hi[r_, j] += h
                lo[r_, j] -= h

                def f(y):
                    o = ao.token_logprobs(y, tg, 0, 1.3)
                    return o["logprobs"].sum() * 0.7 + o["entropy"].sum() * 0.4

                def d(y):
                    return ao.distill(y, v, idx, 1.3, True)[0].sum()
                assert abs(float(g[r_, j]) - float(f(hi) - f(lo)) / (2 * h)) < 1e-6
                assert abs(float(gd[r_, j]) - float(d(hi) - d(lo)) / (2 * h)) < 2e-6


def _teacher(x, K, T, seed):
    g = torch.Generator().manual_seed(seed)
    z = (x.double().nan_to_num(0.0, 0.0, -20.0).clamp(-30, 30) + torch.randn(x.shape, generator=g)) / T
    v, idx = torch.log_softmax(z, 1).topk(K, 1)
    return v.float(), idx


def _check_distill(x, xd, v, idx, T, tail, dev):
    """Rows, sums and gradients for the incoming gradients of every path."""
    from vqa_amd import ops
    R = x.shape[0]
    loss, ltol, g, gtol = ao.distill(x, v, idx, T, tail)
    half = torch.finfo(x.dtype).eps / 2
    kw = dict(temperature=T, tail=tail)
    vd, idxd = v.to(dev), idx.to(dev)
    xd = xd.detach().requires_grad_()

    def grad_close(got, scale, what):
        s = torch.as_tensor(scale, dtype=torch.float64)
        s = s[:, None] if s.dim() else s
        want, tol = g * s, gtol * s.abs() + 3 * ao.U * (g * s).abs()
        _close(got, want, tol + half * (want.abs() + tol) + 2 * torch.finfo(x.dtype).tiny, what)
        assert got.dtype == x.dtype
    rows = ops.distill_loss(xd, vd, idxd, reduction="none", **kw)
    _close(rows, loss, ltol, "row losses")
    up = torch.linspace(-1.0, 2.0, R)
    got, = torch.autograd.grad(rows, xd, up.to(dev))
    grad_close(got, up, "gradient of the rows")
    with torch.no_grad():
        assert torch.equal(ops.distill_loss(xd, vd, idxd, reduction="none", **kw).nan_to_num(1e30), rows.nan_to_num(1e30))
    for reduction, scale in (("mean", 1.0 / R), ("sum", 1.0)):
        whole = ops.distill_loss(xd, vd, idxd, reduction=reduction, **kw)
        _close(whole.reshape(1), (loss.sum() * scale).reshape(1),
               (ltol.sum() * scale + 2 * ao.U * abs(float(loss.sum()) * scale)).reshape(1), reduction)
        got, = torch.autograd.grad(whole, xd, ops.unit_gradient(whole), retain_graph=True)
        grad_close(got, scale, f"{reduction}, unit gradient")
        kept = got.clone()
        again, = torch.autograd.grad(whole, xd, ops.unit_gradient(whole), retain_graph=True)
        assert again.data_ptr() != got.data_ptr()
        grad_close(again, scale, f"{reduction}, second backward")
        other, = torch.autograd.grad(whole * -3.0, xd)
        grad_close(other, -3.0 * scale, f"{reduction}, times -3")
        assert torch.equal(got.nan_to_num(1e30), kept.nan_to_num(1e30))
        whole = ops.distill_loss(xd, vd, idxd, reduction=reduction, **kw)
        got, = torch.autograd.grad(whole, xd)               # the usual loss.backward(): a 1 made by autograd
        grad_close(got, scale, f"{reduction}, fresh unit gradient")
        whole = ops.distill_loss(xd, vd, idxd, reduction=reduction, **kw)
        got, = torch.autograd.grad(whole * 0.25, xd)
        grad_close(got, 0.25 * scale, f"{reduction}, a quarter")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", CLASSES)
def test_distill_every_row_length(dev, C, dtype, tail):
    x = _logits(5, C, dtype, C + 7)
    for T, K in ((1.0, min(C, 16)), (4.0, 1), (1.5, min(C, 128))):
        v, idx = _teacher(x, K, T, C)
        _check_distill(x, x.to(dev), v, idx, T, tail, dev)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [9, 430, 1500, 30522, 66000])
def test_distill_edges(dev, C, dtype, tail):
    K = 8
    x = _logits(12, C, dtype, C + 2)
    v, idx = _teacher(x, K, 1.0, 3)
    x[0] = -math.inf                                   # the student's mask leaves nothing
    x[1, idx[1, 0]] = -math.inf                        # ... or not what the teacher says
    out = torch.ones(C, dtype=torch.bool)
    out[idx[2]] = False
    x[2, out] = -math.inf                              # nothing outside the list
    idx[3] = -1                                        # a row that teaches nothing
    x[3, 0] = math.nan
    idx[4, 2:] = -100                                  # a padded list
    idx[5, 3] = C                                      # past the classes
    idx[6] = idx[6, 0]                                 # one answer eight times
    v[6] -= 3.0
    idx[7, 4] = idx[7, 1]
    v[7] -= 1.0
    v[8, 1:] = -math.inf                               # a teacher who is sure
    v[8, 0] = 0.0
    x[9, C // 2] = math.nan
    idx[10, :] = -1
    x[10] = -math.inf                                  # a padded row on both sides
    v[11] = -math.inf
    _check_distill(x, x.to(dev), v, idx, 2.0, tail, dev)


def test_distill_broken_teacher(dev):
    from vqa_amd import ops
    x = _logits(3, 100, torch.float32, 1).to(dev).requires_grad_()
    v, idx = torch.full((3, 4), -2.0), torch.arange(4).repeat(3, 1)
    v[1, 2] = math.nan
    for tail in (False, True):
        rows = ops.distill_loss(x, v.to(dev), idx.to(dev), tail=tail, reduction="none")
        assert torch.isnan(rows).tolist() == [False, True, False]
        g, = torch.autograd.grad(rows.sum(), x)
        assert torch.isnan(g).any(1).tolist() == [False, True, False]


def test_lists_that_cover_every_class(dev):
    for C in (3, 100, 128):
        x = _logits(4, C, torch.float32, C)
        v, idx = _teacher(x, C, 1.0, 9)
        _check_distill(x, x.to(dev), v, idx, 1.0, True, dev)


@pytest.mark.parametrize("C", [13, 430, 5000])
def test_no_rows_and_leading_dimensions(dev, C):
    from vqa_amd import ops
    e = torch.empty(0, C, device=dev, requires_grad=True)
    r = ops.token_logprobs(e, torch.empty(0, dtype=torch.int64, device=dev), top=3)
    assert r.logprobs.shape == (0,) and r.entropy.shape == (0,) and r.top_logprobs.shape == (0, 3)
    assert r.top_indices.shape == (0, 3) and r.top_indices.dtype == torch.int64
    (r.logprobs.sum() + r.entropy.sum()).backward()
    assert e.grad.shape == (0, C)
    rows = ops.distill_loss(e, torch.empty(0, 2, device=dev), torch.empty(0, 2, dtype=torch.int64, device=dev), reduction="none")
    assert rows.shape == (0,)
    x = _logits(6, C, torch.bfloat16, 4).view(2, 3, C)
    xd = x.to(dev).requires_grad_()
    tg = torch.arange(6).view(2, 3) % C
    r = ops.token_logprobs(xd, tg.to(dev), top=4)
    assert r.logprobs.shape == (2, 3) and r.entropy.shape == (2, 3) and r.top_logprobs.shape == (2, 3, 4)
    flat = ops.token_logprobs(xd.detach().view(6, C), tg.to(dev).view(6), top=4)
    assert torch.equal(r.logprobs.view(6), flat.logprobs) and torch.equal(r.top_indices.view(6, 4), flat.top_indices)
    many = ops.token_logprobs(xd, tg.to(dev)[..., None].expand(2, 3, 2))
    assert many.logprobs.shape == (2, 3, 2) and torch.equal(many.logprobs[..., 1], r.logprobs)
    loss = ops.distill_loss(xd, r.top_logprobs, r.top_indices, reduction="none")
    assert loss.shape == (2, 3)
    loss.sum().backward()
    assert xd.grad.shape == x.shape


def test_strided_incoming_gradients_and_entropy_alone(dev):
    from vqa_amd import ops
    x = _logits(6, 777, torch.float32, 8)
    xd = x.to(dev).requires_grad_()
    r = ops.token_logprobs(xd, torch.arange(6, device=dev))
    g, = torch.autograd.grad(r.entropy.sum(), xd)         # an expanded scalar comes back
    want, tol = ao.token_logprobs_grad(x, 1.0, None, None, torch.ones(6))
    _close(g, want, tol, "entropy gradient")
    assert ops.token_logprobs(xd, entropy=False).entropy is None
    only = ops.token_logprobs(xd, torch.arange(6, device=dev), entropy=False)
    g, = torch.autograd.grad(only.logprobs.sum(), xd)
    want, tol = ao.token_logprobs_grad(x, 1.0, torch.arange(6), torch.ones(6))
    _close(g, want, tol, "logprob gradient")


def test_replayed_graph_equals_eager_calls(dev):
    """Forward and backward captured once and replayed with new inputs, eager work of the program in between."""
    from vqa_amd import ops
    for C in (430, 30522):
        xs = [_logits(33, C, torch.bfloat16, 50 + i).to(dev) for i in range(4)]
        tg = (torch.arange(33, device=dev) * 5) % C
        x = xs[0].clone().requires_grad_()

        def step():
            r = ops.token_logprobs(x, tg, top=7, temperature=2.0)
            loss = ops.distill_loss(x, r.top_logprobs.detach(), r.top_indices.roll(1, 0), temperature=2.0, tail=True)
            ga, = torch.autograd.grad(r.logprobs.mean() + 0.1 * r.entropy.mean(), x)
            gb, = torch.autograd.grad(loss, x, ops.unit_gradient(loss))
            return [r.logprobs.detach(), r.entropy.detach(), r.top_indices, loss.detach(), ga, gb]
        eager = []
        for v in xs:
            with torch.no_grad():
                x.copy_(v)
            eager.append([t.clone() for t in step()])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for _ in range(3):
            for v, want in zip(xs, eager):
                with torch.no_grad():
                    x.copy_(v)
                graph.replay()
                torch.cuda.synchronize()
                for a, b in zip(out, want):
                    assert torch.equal(a, b)
                ops.token_logprobs(v, tg, top=3)


def test_two_streams_at_once(dev):
    from vqa_amd import ops
    a, b = _logits(200, 30522, torch.bfloat16, 1).to(dev), _logits(200, 430, torch.float32, 2).to(dev)
    wa, wb = ops.token_logprobs(a, top=9), ops.token_logprobs(b, top=9)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s):
            ra = ops.token_logprobs(a, top=9)
        with torch.cuda.stream(t):
            rb = ops.token_logprobs(b, top=9)
        got.append((ra, rb))
    torch.cuda.synchronize()
    for ra, rb in got:
        for x, y in zip(ra[1:], wa[1:]):
            assert torch.equal(x, y)
        for x, y in zip(rb[1:], wb[1:]):
            assert torch.equal(x, y)


def test_row_past_32_bit_offsets(dev):
    """A matrix of more than 2^31 elements: rows behind the border are read and written where they are."""
    from vqa_amd import ops
    C, R = 65536, 32769 + 2
    x = torch.empty(R, C, dtype=torch.bfloat16, device=dev).normal_()
    last = _logits(3, C, torch.bfloat16, 3)
    x[-3:] = last.to(dev)
    x.requires_grad_()
    r = ops.token_logprobs(x, torch.full((R,), 5, device=dev), top=4)
    want = ao.token_logprobs(last, torch.full((3,), 5), 4, 1.0)
    _close(r.logprobs[-3:], want["logprobs"][:, 0], want["logprobs_tol"][:, 0], "logprobs")
    assert torch.equal(r.top_indices[-3:].cpu(), want["top_indices"])
    up = torch.zeros(R, device=dev)
    up[-3:] = 1.0
    g, = torch.autograd.grad(r.logprobs, x, up)
    wg, tol = ao.token_logprobs_grad(last, 1.0, torch.full((3,), 5), torch.ones(3))
    _close(g[-3:], wg, tol, "gradient")
    assert float(g[:1000].abs().max()) == 0.0


def test_one_row_without_a_batch(dev):
    from vqa_amd import ops
    x = _logits(1, 77, torch.float32, 2)
    xd = x[0].to(dev).requires_grad_()
    r = ops.token_logprobs(xd, torch.tensor(4, device=dev), top=3)
    assert r.logprobs.shape == () and r.entropy.shape == () and r.top_indices.shape == (3,)
    many = ops.token_logprobs(xd, torch.tensor([4, 5], device=dev))
    assert many.logprobs.shape == (2,) and torch.equal(many.logprobs[0], r.logprobs)
    none = ops.token_logprobs(xd, torch.empty(0, dtype=torch.int64, device=dev))
    assert none.logprobs.shape == (0,)
    loss = ops.distill_loss(xd, r.top_logprobs, r.top_indices)
    g, = torch.autograd.grad(loss + none.entropy * 0, xd)
    _, _, want, tol = ao.distill(x, r.top_logprobs.detach().cpu()[None], r.top_indices.cpu()[None])
    _close(g, want[0], tol[0] + 2.0 ** -23 * (want[0].abs() + tol[0]), "gradient")


@pytest.mark.parametrize("C", [40, 3000])
def test_gradient_of_one_row_shared_by_all(dev, C):
    """A broadcast row: the gradient of every row, added."""
    from vqa_amd import ops
    x = _logits(1, C, torch.float32, 6)
    leaf = x.to(dev).requires_grad_()
    tg = torch.arange(5) * 3
    r = ops.token_logprobs(leaf.expand(5, C), tg.to(dev))
    g, = torch.autograd.grad(r.logprobs.sum(), leaf)
    want, tol = ao.token_logprobs_grad(x.expand(5, C), 1.0, tg, torch.ones(5))
    _close(g, want.sum(0, keepdim=True), tol.sum(0, keepdim=True) + 4 * ao.U * want.abs().sum(0, keepdim=True), "shared row")


def test_no_gradient_of_a_gradient(dev):
    from vqa_amd import ops
    x = _logits(3, 50, torch.float32, 1).to(dev).requires_grad_()
    g, = torch.autograd.grad(ops.token_logprobs(x).entropy.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        torch.autograd.grad(g.sum(), x)
    v, idx = torch.full((3, 2), -1.0, device=dev), torch.tensor([[0, 1]] * 3, device=dev)
    g, = torch.autograd.grad(ops.distill_loss(x, v, idx), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        torch.autograd.grad(g.sum(), x)


def test_logits_changed_in_place_are_noticed(dev):
    from vqa_amd import ops
    x = _logits(3, 50, torch.float32, 1).to(dev).requires_grad_()
    y = x * 1.0
    r = ops.token_logprobs(y)
    y.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.entropy.sum().backward()


def test_refusals(dev):
    from vqa_amd import ops
    x = torch.zeros(4, 10, device=dev)
    tg, v, idx = torch.zeros(4, dtype=torch.long, device=dev), torch.zeros(4, 2, device=dev), torch.zeros(4, 2, dtype=torch.long, device=dev)
    for kw in (dict(targets=tg[:3]), dict(targets=tg.cpu()), dict(top=11), dict(top=-1), dict(temperature=0.0),
               dict(targets=tg[:, None].expand(4, 129))):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, **kw)
    for kw in (dict(targets=tg.float()), dict(targets=tg.bool())):
        with pytest.raises(TypeError):
            ops.token_logprobs(x, **kw)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.half())
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(4, 200, device=dev), top=129)
    for a, b, kw in ((v[:3], idx, {}), (v, idx[:, :1], {}), (v[:, :0], idx[:, :0], {}), (v, idx.cpu(), {}), (v, idx, dict(temperature=-1)),
                     (v[0], idx[0], {}), (torch.zeros(4, 129, device=dev), torch.zeros(4, 129, dtype=torch.long, device=dev), {})):
        with pytest.raises(ValueError):
            ops.distill_loss(x, a, b, **kw)
    for a, b in ((v.long(), idx), (v, idx.float())):
        with pytest.raises(TypeError):
            ops.distill_loss(x, a, b)


def test_backward_replayed_without_its_forward(dev):
    """The forward and the backward captured into graphs of their own, the backward replayed with other incoming
    gradients: nothing of the replay before may be left in the gradient."""
    from vqa_amd import ops
    for C in (430, 30522):
        x = _logits(9, C, torch.bfloat16, 7).to(dev).requires_grad_()
        v, i = ops.token_logprobs(_logits(9, C, torch.bfloat16, 8).to(dev), top=5)[2:]
        up = torch.ones((), device=dev)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        fwd, bwd = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(fwd, stream=s):
            loss = ops.distill_loss(x, v, i, reduction="sum")
        with torch.cuda.graph(bwd, pool=fwd.pool(), stream=s):
            got, = torch.autograd.grad(loss, x, up)
        ups = (2.0, 1.0, 0.5, 1.0, -3.0, 1.0)
        kept = []
        fwd.replay()
        for u in ups:
            up.fill_(u)
            bwd.replay()
            kept.append(got.clone())
        torch.cuda.synchronize()
        del loss
        for u, g in zip(ups, kept):
            xe = x.detach().clone().requires_grad_()
            le = ops.distill_loss(xe, v, i, reduction="sum")
            torch.autograd.grad(le, xe, retain_graph=True)   # takes the forward's gradient: the next is formed as the graph's
            want, = torch.autograd.grad(le, xe, torch.full((), u, device=dev))
            assert torch.equal(g, want), u


def test_more_rows_than_a_launch_takes(dev):
    """Rows in several launches (a launch has fewer than 2^32 threads): the rows on both sides of a border and the last."""
    from vqa_amd import ops
    R = (1 << 25) + 9          # a wave each
    few = _logits(64, 3, torch.bfloat16, 3).to(dev)
    x = few.repeat(R // 64 + 1, 1)[:R].requires_grad_()
    at = torch.tensor([0, 1, (1 << 25) - 1, 1 << 25, (1 << 25) + 1, R - 1], device=dev)
    f = few[at % 64].requires_grad_()
    # (against the definition: the order of a row's sums follows its alignment and the kernel that its row count takes)
    big, want = ops.token_logprobs(x, top=2), ao.token_logprobs(few[at % 64].cpu(), top=2)
    for name in ("entropy", "top_logprobs"):
        _close(getattr(big, name)[at], want[name], want[name + "_tol"], name)
    assert torch.equal(big.top_indices[at].cpu(), want["top_indices"])
    ga, = torch.autograd.grad(big.entropy.sum(), x)
    g, tol = ao.token_logprobs_grad(few[at % 64].cpu(), 1.0, g_entropy=torch.ones(6))
    _close(ga[at], g, tol, "entropy gradient")
    v, i = big.top_logprobs.detach().roll(1, 0), big.top_indices
    del big, ga
    la, lb = (ops.distill_loss(a, b, c, reduction="none") for a, b, c in ((x, v, i), (f, v[at], i[at])))
    assert torch.equal(la[at], lb)
    ga, = torch.autograd.grad(la.sum(), x)
    gb, = torch.autograd.grad(lb.sum(), f)
    assert torch.equal(ga[at], gb)
    del x, v, i, la, ga
    R = (1 << 23) + 3          # a workgroup each: one row repeated
    one = _logits(1, 1025, torch.bfloat16, 4).to(dev)
    x = one.expand(R, 1025).requires_grad_()
    got = ops.token_logprobs(x, top=1)
    want = ops.token_logprobs(one, top=1)
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a[-4:], b.expand(4, *b.shape[1:])) and torch.equal(a[:1], b)
    loss = ops.distill_loss(x, got.top_logprobs.detach(), got.top_indices, tail=True, reduction="sum")
    g, = torch.autograd.grad(loss, x, ops.unit_gradient(loss))
    assert bool((g[0] != 0).any())
    assert torch.equal(g[-4:], g[:1].expand(4, 1025)) and torch.equal(g[(1 << 23) - 1:(1 << 23) + 1], g[:1].expand(2, 1025))
    ge, = torch.autograd.grad(got.entropy.sum(), x)
    assert bool((ge[0] != 0).any())
    assert torch.equal(ge[-4:], ge[:1].expand(4, 1025))


def test_more_rows_or_classes_than_an_int_holds(dev):
    from vqa_amd import ops
    z = torch.zeros(1, device=dev)
    with pytest.raises(ValueError, match="rows"):
        ops.token_logprobs(z.expand(2 ** 32 + 5))
    with pytest.raises(ValueError, match="rows"):
        ops.token_logprobs(z.view(1, 1).expand(2 ** 32 + 5, 1))
    with pytest.raises(ValueError, match="rows"):
        ops.distill_loss(z.view(1, 1).expand(2 ** 32 + 5, 1), z.view(1, 1).expand(2 ** 32 + 5, 1),
                         torch.zeros(1, 1, dtype=torch.int64, device=dev).expand(2 ** 32 + 5, 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [1, 2, 7, 13, 64, 65, 127, 128, 200, 257, 320, 385, 430, 448, 511, 512])
def test_many_short_rows(dev, C, dtype):
    """Row counts from which rows share a wave: masked, tied and broken rows next to ordinary ones, any alignment."""
    from vqa_amd import ops
    few = _logits(37, C, dtype, C)
    few[1] = -math.inf
    few[2, : C - 1] = -math.inf
    few[3] = 0.25                                        # a tie of all
    few[4, ::2] = torch.finfo(dtype).min
    few[5, C // 2] = math.nan
    few[6, 0] = math.inf
    few[7] = math.nan
    few[8] = -few[8].abs() - 1                           # nothing above zero
    few[9, C // 3:] = few[9].max()                       # a long tie
    few[10, C // 2:] = -math.inf
    few[11] = -math.inf
    few[11, -1] = -math.nan
    few[12, ::3] = -0.0
    few[12, 1::3] = 0.0
    few[13] *= 1000
    R = 8192 + 5
    idx = (torch.arange(R) * 11) % 37
    tg = (torch.arange(37)[:, None] * 5 + torch.arange(19)) % (C + 1) - 1
    for top, T, off, ld in ((0, 1.0, 0, C), (1, 0.7, 0, C), (min(3, C), 1.0, 1, C + 3), (min(8, C), 4.0, 3, C + 1), (min(5, C), 1.0, 5, C)):
        want = ao.token_logprobs(few, tg, top, T)
        buf = torch.full((off + R * ld,), math.nan, dtype=dtype, device=dev)
        x = buf.as_strided((R, C), (ld, 1), off)
        x.copy_(few[idx].to(dev))
        got = ops.token_logprobs(x, tg[idx].to(dev), top=top, temperature=T)
        for name in ("entropy", "logprobs") + (("top_logprobs",) if top else ()):
            _close(getattr(got, name), want[name][idx].reshape(getattr(got, name).shape),
                   want[name + "_tol"][idx].nan_to_num(0.0).reshape(getattr(got, name).shape), name)
        if top:   # (no bound, a broken row: no target there is exactly 0)
            assert torch.equal(got.top_indices.cpu(), want["top_indices"][idx])
    x = few[idx].to(dev).requires_grad_()
    ok = ~torch.isnan(few).any(1) & ~(few == math.inf).any(1)
    g, = torch.autograd.grad(ops.token_logprobs(x).entropy.sum(), x)
    want, tol = ao.token_logprobs_grad(few, 1.0, None, None, torch.ones(37))
    _close(g[ok[idx].to(dev)], want[idx[ok[idx]]], tol[idx[ok[idx]]], "entropy gradient")
