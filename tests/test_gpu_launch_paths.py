"""How the answer operators find the device and the stream that they launch on."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def test_public_ways_to_the_stream(dev, monkeypatch):
    """What stands in for torch's private names gives the same launches, on a stream of one's own too."""
    from vqa_amd import ops
    x = torch.randn(40, 430, device=dev)
    want = ops.token_logprobs(x, top=3)
    for name in ("_raw_stream", "_current_device"):
        assert callable(getattr(ops, name))
    side = torch.cuda.Stream()
    assert ops._raw_stream(0) == torch.cuda.current_stream(0).cuda_stream and ops._current_device() == torch.cuda.current_device()
    with torch.cuda.stream(side):
        assert ops._raw_stream(0) == side.cuda_stream == torch.cuda.current_stream(0).cuda_stream
    monkeypatch.setattr(ops, "_raw_stream", lambda i: torch.cuda.current_stream(i).cuda_stream)
    monkeypatch.setattr(ops, "_current_device", torch.cuda.current_device)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = ops.token_logprobs(x, top=3)
    torch.cuda.synchronize()
    assert torch.equal(got.top_indices, want.top_indices) and torch.equal(got.entropy, want.entropy)


class _Busy:
    """The library, with other allocations of index tensors made between a call's preparation and its launch."""

    def __init__(self, lib, sizes, dev):
        self.lib, self.sizes, self.dev, self.taken = lib, sizes, dev, []

    def __getattr__(self, name):
        def call(*args):
            self.taken += [torch.zeros(n, dtype=torch.int64, device=self.dev) for n in self.sizes for _ in range(2)]
            return getattr(self.lib, name)(*args)
        return call


def test_copies_of_indices_outlive_the_launch(dev, monkeypatch):
    """Targets of another type or stride, and strided swap positions, are copied; the copies stay until the launch, whatever
    is allocated meanwhile.  (Every index of every tensor here lies inside both lists.)"""
    from vqa_amd import ops
    g = torch.Generator().manual_seed(0)
    B, C, K, R, n = 24, 430, 40, 40, 6
    logits = torch.randn(B, C, generator=g).to(dev)
    targets = torch.randint(1, C, (B,), generator=g).to(dev)
    want = ops.cross_entropy_mean(logits, targets)
    top = torch.stack([torch.randperm(K, generator=g) for _ in range(B)]).to(dev)
    bottom = torch.stack([torch.randperm(R, generator=g) + K for _ in range(B)]).to(dev)
    pos = torch.stack([torch.randperm(K, generator=g)[:n] for _ in range(B)]).to(dev)
    src = torch.stack([torch.randperm(R, generator=g)[:n] for _ in range(B)]).to(dev)
    a, b = top.clone(), bottom.clone()
    ops.adv_swap_(a, b, pos, src)
    busy = _Busy(ops.load(), (B, B * n), dev)
    monkeypatch.setattr(ops, "load", lambda: busy)
    assert torch.equal(ops.cross_entropy_mean(logits, targets.to(torch.int32)), want)
    assert torch.equal(ops.cross_entropy_mean(logits, targets.repeat_interleave(2)[::2]), want)
    c, d = top.clone(), bottom.clone()
    ops.adv_swap_(c, d, pos.t().contiguous().t(), src.t().contiguous().t())
    assert torch.equal(a, c) and torch.equal(b, d)
