"""Forward-mode derivatives through the answer and eight-bit operators: refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


@pytest.mark.parametrize("C", [40, 3000])
@pytest.mark.parametrize("recorded", [True, False])
def test_tangents_are_refused(dev, C, recorded):
    from vqa_amd import ops
    x = torch.randn(4, C, device=dev)
    said = ops.token_logprobs(x, top=3)
    w, s = ops.quantize_rows(torch.randn(8, C, device=dev))
    b = torch.zeros(8, device=dev)
    plain = ops.int8_linear(x, w, s, b)
    with torch.set_grad_enabled(recorded), fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            ops.token_logprobs(d, torch.zeros(4, dtype=torch.int64, device=dev))
        with pytest.raises(NotImplementedError):
            ops.token_logprobs(d.view(2, 2, C))
        for reduction in ("mean", "none"):
            with pytest.raises(NotImplementedError):
                ops.distill_loss(d, said.top_logprobs, said.top_indices, reduction=reduction)
        for args in ((d, w, s, b), (x, w, fw.make_dual(s, s), b), (x, w, s, fw.make_dual(b, b))):
            with pytest.raises(RuntimeError, match="gradient"):
                ops.int8_linear(*args)
        # without a tangent the calls are what they are outside the level
        assert torch.equal(ops.token_logprobs(x, top=3).top_logprobs, said.top_logprobs)
        assert torch.equal(ops.int8_linear(x, w, s, b), plain)
