"""Linear layers in eight-bit integers (csrc/int8.hip) against their 64-bit statement: every kernel, odd sizes, strides,
types, rows at the edges of the number range."""
import math

import pytest
import torch

from oracle import int8_oracle as io

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def _x(M, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g)
    x[:, :: max(1, K // 3)] *= 5.0
    return x.to(dtype)


def _close(got, want, tol, what=""):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    ok = ~torch.isnan(want)
    off = ((got - want).abs() - tol)[ok]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max())} over the bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 5), (5, 8), (7, 63), (4, 100), (9, 128), (6, 129), (130, 512), (33, 768), (5, 1000),
                                 (3, 1025), (6, 2049), (3, 4096), (3, 4097), (2, 9001)])
def test_quantize_rows_is_exact(dev, M, K, dtype):
    from vqa_amd import ops
    x = _x(M, K, dtype, K)
    want_q, want_s = io.quantize_rows(x)
    q, s = ops.quantize_rows(x.to(dev))
    assert q.dtype == torch.int8 and q.shape == (M, K) and s.shape == (M,)
    assert torch.equal(s.cpu().double(), want_s) and torch.equal(q.cpu().double(), want_q)
    base = q._base if q._base is not None else q
    assert int(base.reshape(M, -1)[:, K:].abs().sum()) == 0          # the rows' rest is zero
    # a row pitch and a start off every alignment
    wide = torch.full((M, K + 5), 9.0, dtype=dtype, device=dev)
    wide[:, 3:3 + K] = x.to(dev)
    q2, s2 = ops.quantize_rows(wide[:, 3:3 + K])
    assert torch.equal(q2, q) and torch.equal(s2, s)
    q3, s3 = ops.quantize_rows(x.to(dev).t().contiguous().t())
    assert torch.equal(q3, q) and torch.equal(s3, s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_borders_between_steps_and_the_range_s_ends(dev, dtype):
    from vqa_amd import ops
    K = 300
    x = torch.zeros(10, K, dtype=dtype)
    x[0, :260] = torch.arange(-130, 130).clamp(-127, 126).to(dtype) / 2 + 0.0   # quotients of k / 2: every other one a tie
    x[0, 299] = 127.0
    x[1] = x[0] * 2.0 ** -100
    x[2, 7] = torch.finfo(dtype).tiny                     # below what a scale can hold: steps of 2^-126
    x[3, 5] = -torch.finfo(dtype).max
    x[3, 6] = torch.finfo(dtype).max / 254                # half a step
    x[4, 0] = math.nan
    x[5, K - 1] = math.inf
    x[6, 3] = -math.inf
    x[7] = -0.0
    g = torch.Generator().manual_seed(3)
    x[8] = (torch.randint(-254, 255, (K,), generator=g).float() / 2 * 0.7371).to(dtype)   # quotients next to ties
    x[8, 0] = 0.7371 * 127
    x[9] = torch.randn(K, generator=g).to(dtype) * torch.finfo(dtype).tiny * 20
    want_q, want_s = io.quantize_rows(x)
    q, s = ops.quantize_rows(x.to(dev))
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(want_s))
    ok = ~torch.isnan(want_s)
    assert torch.equal(s.cpu().double()[ok], want_s[ok])
    assert torch.equal(q.cpu().double(), want_q)


SHAPES = [(1, 1, 1), (1, 768, 2304), (2, 100, 17), (4, 8192, 33), (4, 8200, 5), (5, 64, 16), (16, 130, 430), (17, 768, 48),
          (33, 200, 100), (64, 1024, 64), (64, 40, 3), (65, 768, 64), (100, 129, 65), (129, 16, 130), (300, 768, 768),
          (257, 4096, 31), (1000, 1024, 430), (1920, 768, 512), (2500, 256, 2050), (4100, 100, 1030),
          (3000, 200, 3001), (9300, 64, 1001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_every_size_class(dev, M, K, N, dtype):
    from vqa_amd import ops
    x, w = _x(M, K, dtype, M + K), _x(N, K, torch.float32, N) * K ** -0.5
    wq, ws = ops.quantize_rows(w.to(dev))
    bias = torch.linspace(-1, 1, N).to(dtype)
    for b, out in ((bias, None), (None, torch.float32 if dtype == torch.bfloat16 else torch.bfloat16)):
        y = ops.int8_linear(x.to(dev), wq, ws, None if b is None else b.to(dev), out_dtype=out)
        want, tol = io.linear(x, wq.cpu(), ws.cpu(), b, out or dtype)
        assert y.dtype == (out or dtype) and y.is_contiguous()
        _close(y, want, tol, f"{M} {K} {N}")


@pytest.mark.parametrize("M", [3, 40, 200])
def test_layouts_of_tokens_and_weights(dev, M):
    from vqa_amd import ops
    K, N = 200, 70
    x, w = _x(M, K, torch.bfloat16, 1), _x(N, K, torch.float32, 2)
    xd = x.to(dev)
    wq, ws = ops.quantize_rows(w.to(dev))
    want = ops.int8_linear(xd, wq, ws)
    wide = torch.full((M, K + 7), float("nan"), dtype=torch.bfloat16, device=dev)
    wide[:, 1:1 + K] = xd
    assert torch.equal(ops.int8_linear(wide[:, 1:1 + K], wq, ws), want)
    assert torch.equal(ops.int8_linear(xd.t().contiguous().t(), wq, ws), want)
    assert torch.equal(ops.int8_linear(xd.view(1, M, K), wq, ws), want.view(1, M, N))
    tight = wq.contiguous()                                   # rows of 200 bytes: not whole pieces, copied
    assert tight.stride(0) == K and torch.equal(ops.int8_linear(xd, tight, ws), want)
    dirty = torch.full((N, 256), 111, dtype=torch.int8, device=dev)   # what follows column K is never counted
    dirty[:, :K] = wq
    assert torch.equal(ops.int8_linear(xd, dirty[:, :K], ws), want)
    last = torch.full((N * 208,), 55, dtype=torch.int8, device=dev)   # the last row ends with its last piece
    view = last.view(N, 208)[:, :K]
    view.copy_(wq)
    assert torch.equal(ops.int8_linear(xd, view, ws), want)
    off = torch.zeros(N * 256 + 8, dtype=torch.int8, device=dev)[8:].view(N, 256)[:, :K]
    off.copy_(wq)
    assert torch.equal(ops.int8_linear(xd, off, ws), want)
    one = ops.int8_linear(xd, wq[:1], ws[:1])
    assert torch.equal(one, want[:, :1])


def test_rows_that_are_broken_or_empty(dev):
    from vqa_amd import ops
    for M in (4, 20, 100):
        x = _x(M, 96, torch.float32, 5)
        x[0, 3] = math.nan
        x[1, 4] = math.inf
        x[2] = 0.0
        wq, ws = ops.quantize_rows(_x(20, 96, torch.float32, 6).to(dev))
        bias = torch.arange(20.0)
        y = ops.int8_linear(x.to(dev), wq, ws, bias.to(dev)).cpu()
        assert torch.isnan(y[:2]).all() and torch.equal(y[2], bias) and torch.isfinite(y[3:]).all()
    assert ops.int8_linear(torch.empty(0, 96, device=dev), wq, ws).shape == (0, 20)
    q, s = ops.quantize_rows(torch.empty(0, 96, device=dev))
    assert q.shape == (0, 96) and s.shape == (0,)


def test_refusals(dev):
    from vqa_amd import ops
    x = torch.zeros(4, 32, device=dev)
    wq, ws = ops.quantize_rows(torch.ones(8, 32, device=dev))
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.int8_linear(x.clone().requires_grad_(), wq, ws)
    with torch.no_grad():
        ops.int8_linear(x.clone().requires_grad_(), wq, ws)
    for bad in (dict(x=x[:, :31]), dict(weight_scale=ws[:7]), dict(weight_scale=ws.double()), dict(bias=ws[:3]),
                dict(weight_scale=ws.cpu())):
        with pytest.raises(ValueError):
            ops.int8_linear(**{"x": x, "weight": wq, "weight_scale": ws, **bad})
    for bad in (dict(weight=wq.float()), dict(x=x.half()), dict(out_dtype=torch.float16), dict(bias=ws.half())):
        with pytest.raises(TypeError):
            ops.int8_linear(**{"x": x, "weight": wq, "weight_scale": ws, **bad})


def test_replayed_graph_and_streams(dev):
    from vqa_amd import ops
    wq, ws = ops.quantize_rows(_x(2304, 256, torch.float32, 6).to(dev))
    xs = [[_x(M, 256, torch.bfloat16, 10 * M + i).to(dev) for i in range(3)] for M in (2, 40, 500, 5000)]
    want = [[ops.int8_linear(x, wq, ws) for x in row] for row in xs]
    buf = [row[0].clone() for row in xs]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [ops.int8_linear(b, wq, ws) for b in buf]
    for _ in range(2):
        for i in range(3):
            for b, row in zip(buf, xs):
                b.copy_(row[i])
            graph.replay()
            torch.cuda.synchronize()
            for o, w in zip(out, want):
                assert torch.equal(o, w[i])
            ops.int8_linear(xs[2][1], wq, ws)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for st in (s, t):
            with torch.cuda.stream(st):
                got.append(ops.int8_linear(xs[2][2], wq, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[2][2]) for g in got)


def test_more_rows_than_a_launch_takes(dev):
    """Rows in several launches (a launch has fewer than 2^32 threads): the rows on both sides of a border and the last."""
    from vqa_amd import ops
    M = (1 << 25) + 9
    few = _x(64, 5, torch.bfloat16, 3).to(dev)
    at = torch.tensor([0, 1, (1 << 25) - 1, 1 << 25, (1 << 25) + 1, M - 1], device=dev)
    q, s = ops.quantize_rows(few.repeat(M // 64 + 1, 1)[:M])
    wq, ws = ops.quantize_rows(few)
    assert torch.equal(q[at], wq[at % 64]) and torch.equal(s[at], ws[at % 64])


def test_more_rows_than_an_int_holds(dev):
    from vqa_amd import ops
    z = torch.zeros(1, 1, device=dev)
    w, s = ops.quantize_rows(z)
    with pytest.raises(ValueError, match="rows"):
        ops.quantize_rows(z.expand(2 ** 32 + 5, 1))
    with pytest.raises(ValueError, match="rows"):
        ops.int8_linear(z.expand(2 ** 32 + 5, 1), w, s)
    with pytest.raises(ValueError, match="fit"):
        ops.int8_linear(z, w.expand(2 ** 32 + 5, 1), s)


def test_weight_rows_far_apart(dev):
    """Rows of weights whose offsets inside one tile pass 32 bits."""
    from vqa_amd import ops
    N, K, pitch = 160, 200, 1 << 25
    w, s = ops.quantize_rows(_x(N, K, torch.float32, 1).to(dev))
    buf = torch.empty(N * pitch, dtype=torch.int8, device=dev)
    far = buf.as_strided((N, K), (pitch, 1))
    far.copy_(w)
    for M in (3, 40, 70, 20000, 37000):   # the last ones on 128 x 128 and 256 x 256 tiles
        x = _x(M, K, torch.bfloat16, M).to(dev)
        assert torch.equal(ops.int8_linear(x, far, s), ops.int8_linear(x, w, s))


@pytest.mark.parametrize("M,N", [(130, 100), (2000, 2000), (4609, 1800)])
def test_every_number_of_stages(dev, M, N):
    """Short and long contractions on each tile size: the ring's start, its steady turns and its end, whole and partial
    last stages.  The integer sum stays below 2^24, so two f32 products are all that follows it."""
    from vqa_amd import ops
    for K in (1, 63, 64, 65, 127, 128, 129, 192, 255, 256, 257, 319, 320, 321, 384, 449, 512, 576, 577, 640, 704, 769, 1000):
        x, w = _x(M, K, torch.bfloat16, K).to(dev), _x(N, K, torch.float32, K + 1).to(dev)
        q, sx = ops.quantize_rows(x)
        wq, sw = ops.quantize_rows(w)
        want = (q.double() @ wq.double().t()).float() * sx[:, None] * sw
        assert torch.equal(ops.int8_linear(x, wq, sw, out_dtype=torch.float32), want), K
