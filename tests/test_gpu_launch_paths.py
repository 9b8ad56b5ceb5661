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
