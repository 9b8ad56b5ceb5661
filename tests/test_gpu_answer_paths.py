"""The answer scores, the distillation loss and the eight-bit layers where the package uses them: scoring loops, the
distillation loop, quantised encoders and the three of them in a row."""
import functools

import numpy as np
import pytest
import torch
import torch.nn as nn

from oracle import answers_oracle as ao
from oracle import int8_oracle as io

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


class Toy(nn.Module):
    """A model with VQAModel.forward's arguments whose logits are one Linear of the images."""

    def __init__(self, inner, classes, seed):
        super().__init__()
        torch.manual_seed(seed)
        self.head = nn.Linear(inner, classes)

    def forward(self, images, input_ids, attention_mask):
        return self.head(images.flatten(1))


def _loader(batches, B, inner, classes, seed):
    g = torch.Generator().manual_seed(seed)
    return [{"image": torch.randn(B, inner, generator=g), "answer": torch.randint(0, classes, (B,), generator=g),
             "inputs": {"input_ids": torch.zeros(B, 2, dtype=torch.long), "attention_mask": torch.ones(B, 2, dtype=torch.long)}}
            for _ in range(batches)]


def _labels(teacher, x, top, T):
    with torch.no_grad():
        z = teacher.head(x)
        from vqa_amd import ops
        r = ops.token_logprobs(z, top=top, temperature=T, entropy=False)
    return r.top_logprobs.cpu(), r.top_indices.cpu()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("hard", [0.0, 0.3])
def test_distillation_epoch_takes_the_gradient_of_its_loss(dev, tail, hard):
    from vqa_amd import loops
    inner, C, B, T, top = 24, 43, 9, 2.0, 6
    student, teacher = Toy(inner, C, 1).to(dev), Toy(inner, C, 2).to(dev)
    loader = _loader(1, B, inner, C, 3)
    x, y = loader[0]["image"], loader[0]["answer"]
    before = {n: p.detach().double().cpu().clone() for n, p in student.named_parameters()}
    with torch.no_grad():
        z = student.head(x.to(dev)).cpu()
    v, idx = _labels(teacher, x.to(dev), top, T)
    loss, ltol, g, gtol = ao.distill(z, v, idx, T, tail)
    want_loss, want_g, tol_g = loss.mean() * (1 - hard), g * (1 - hard) / B, gtol / B
    if hard:
        lp = torch.log_softmax(z.double(), 1)
        ce = -lp[torch.arange(B), y].mean()
        dce = (lp.exp() - torch.nn.functional.one_hot(y, C)) / B
        want_loss, want_g = want_loss + hard * ce, want_g + hard * dce
    # the loss's own bounds; a gradient that leaves through f32 products of B rows (cross-entropy: 2^-20 of the row)
    avg, agree = loops.distill(student, teacher, loader, torch.optim.SGD(student.parameters(), lr=1.0), dev, top=top,
                               temperature=T, tail=tail, hard_weight=hard)
    assert abs(avg - float(want_loss)) <= float(ltol.mean()) + 2.0 ** -20 * (1 + abs(float(want_loss)))
    assert 0.0 <= agree <= 100.0
    for name, want, tol in (("head.weight", want_g.t() @ x.double(), (tol_g + 2.0 ** -20 * want_g.abs()).t() @ x.double().abs()),
                            ("head.bias", want_g.sum(0), (tol_g + 2.0 ** -20 * want_g.abs()).sum(0))):
        after = dict(student.named_parameters())[name].detach().double().cpu()
        got = before[name] - after
        bound = tol + (B + 4) * 2.0 ** -24 * (want_g.abs().t() @ x.double().abs() if want.dim() == 2 else want_g.abs().sum(0))
        assert float(((got - want).abs() - bound - 2.0 ** -23 * before[name].abs()).max()) <= 0, name


def test_distillation_steps_a_private_optimizer_as_a_plain_one(dev):
    """Without noise and with a clipping bound nothing reaches, the DP step is the plain step."""
    from vqa_amd import dp, loops
    inner, C, B = 32, 21, 16
    teacher = Toy(inner, C, 5).to(dev)
    loader = _loader(2, B, inner, C, 6) + [None]
    plain, private = Toy(inner, C, 7).to(dev), Toy(inner, C, 7).to(dev)
    loops.distill(plain, teacher, [b for b in loader if b is not None], torch.optim.SGD(plain.parameters(), lr=0.1), dev, top=4)
    gsm = dp.GradSampleModule(private.head)
    private.head = gsm
    opt = dp.DPOptimizer(torch.optim.SGD(gsm.parameters(), lr=0.1), gsm, noise_multiplier=0.0, max_grad_norm=1e6,
                         expected_batch_size=B)
    loops.distill(private, teacher, loader, opt, dev, top=4)
    a, b = plain.head.weight.detach().cpu(), gsm._module.weight.detach().cpu()
    # two f32 sums of 16 products in different orders, two steps
    assert float((a - b).abs().max()) <= 64 * 2.0 ** -24 * float(a.abs().max())


def test_distillation_loop_arguments(dev):
    from vqa_amd import loops
    t = Toy(4, 3, 0).to(dev)
    with pytest.raises(ValueError, match="hard_weight"):
        loops.distill(t, t, [], torch.optim.SGD(t.parameters(), lr=0.1), dev, hard_weight=1.0)
    assert loops.distill(t, t, [], torch.optim.SGD(t.parameters(), lr=0.1), dev) == (0.0, 0.0)


def test_entropy_scores_of_a_loader(dev):
    from vqa_amd import mia
    m = Toy(8, 430, 3).to(dev)
    loader = _loader(3, 5, 8, 430, 4)
    r = mia.evaluate_privacy_entropy(m, loader, dev, threshold=5.9, is_member=False)
    with torch.no_grad():
        z = torch.cat([m.head(b["image"].to(dev)) for b in loader]).cpu()
    want = ao.token_logprobs(z)
    assert r["entropies"].shape == (15,) and r["ground_truth"].sum() == 0
    assert (np.abs(r["entropies"] - want["entropy"].numpy()) <= want["entropy_tol"].numpy()).all()
    assert (r["predictions"] == (r["entropies"] <= 5.9)).all()
    a = mia.score_answers(z.to(dev), torch.zeros(15, dtype=torch.long, device=dev), top=3)
    assert torch.equal(a.top_indices.cpu(), ao.order(z, 3))


def _stacks(dev):
    from vqa_amd import encoders
    torch.manual_seed(11)
    bert = encoders.Bert(hidden_dim=64, config=encoders.BertConfig(hidden_size=128, num_hidden_layers=2, num_attention_heads=2,
                                                                   intermediate_size=256, vocab_size=50, max_position_embeddings=16))
    vit = encoders.ViT(out_features=64, config=encoders.ViTConfig(hidden_size=128, num_hidden_layers=2, num_attention_heads=2,
                                                                  intermediate_size=200, image_size=32))
    ids = torch.randint(1, 50, (3, 11))
    mask = torch.ones(3, 11, dtype=torch.long)
    mask[1, 7:] = 0
    return [(bert.to(dev).eval(), (ids.to(dev), mask.to(dev))), (vit.to(dev).eval(), (torch.randn(3, 3, 32, 32).to(dev),))]


def test_quantised_encoders_follow_the_definition(dev, monkeypatch):
    """The stack on the integer kernels against the same stack with every such layer computed from its definition.  A
    layer's outputs differ in roundings to bf16 that fall the other way (2^-8, rarely), which shift later steps by one in
    127: the tolerance of the encoder stacks, 1e-2."""
    from vqa_amd import encoders, ops
    for enc, inputs in _stacks(dev):
        linears = sum(type(m) is nn.Linear for m in enc.modules())
        enc = encoders.quantize_int8(enc)
        left = [n for n, m in enc.named_modules() if type(m) is nn.Linear]
        packed = sum(isinstance(m, encoders.Int8Linear) for m in enc.modules())
        assert left == [] and packed == linears - 2 * 2     # two blocks whose three projections became one
        with torch.no_grad():
            got = enc(*inputs)
        calls = []

        def plain(x, weight, scale, bias=None, out_dtype=None):
            calls.append(1)
            y, _ = io.linear(x.reshape(-1, x.shape[-1]).cpu(), weight.cpu(), scale.cpu(), None if bias is None else bias.cpu())
            return y.to(x.dtype).to(x.device).view(*x.shape[:-1], -1)
        with monkeypatch.context() as mp, torch.no_grad():
            mp.setattr(ops, "int8_linear", plain)
            want = enc(*inputs)
        assert len(calls) >= packed
        for a, b in zip(got, want):
            assert a.dtype == b.dtype == torch.float32
            assert float((a - b).norm() / b.norm()) < 1e-2
        with pytest.raises(RuntimeError, match="no gradient"):
            enc(*inputs)


def test_quantised_layer_moves_and_casts(dev):
    from vqa_amd import encoders
    torch.manual_seed(1)
    lin = nn.Linear(100, 30).to(dev)
    q = encoders.Int8Linear.from_linear(lin)
    x = torch.randn(7, 100, device=dev)
    with torch.no_grad():
        y = q(x)
        state = {k: v.clone() for k, v in q.state_dict().items()}
        again = encoders.Int8Linear(100, 30).to(dev)
        again.load_state_dict(state)
        assert torch.equal(again(x), y)
        q.to(torch.bfloat16)
        assert q.dtype == torch.bfloat16 and q.bias.dtype == torch.bfloat16 and q.weight_scale.dtype == torch.float32
        assert q(x.bfloat16()).dtype == torch.bfloat16
        q.cpu()
        assert q.weight_scale.device.type == "cpu"
        q.to(dev)
        assert torch.equal(q.weight_scale.cpu(), state["weight_scale"].cpu())
    from vqa_amd import dp
    with pytest.raises(RuntimeError, match="eval"):
        encoders.quantize_int8(nn.Sequential(nn.Linear(4, 4)).to(dev))
    with pytest.raises(TypeError):
        encoders.quantize_int8(lin.eval())
    with pytest.raises(RuntimeError, match="DP-SGD"):
        encoders.quantize_int8(nn.Sequential(dp.GradSampleModule(nn.Linear(4, 4).to(dev))).eval())


def test_a_teacher_in_eight_bits_labels_scores_and_teaches(dev):
    """The three operators as they are used together on a VQAModel: the quantised teacher's answers are scored, reduced to
    its best ones, and a student takes an epoch on them."""
    from vqa_amd import encoders, loops, mia, model
    vis = functools.partial(encoders.ViT, config=encoders.ViTConfig(hidden_size=128, num_hidden_layers=1, num_attention_heads=2,
                                                                    intermediate_size=256, image_size=32))
    txt = functools.partial(encoders.Bert, config=encoders.BertConfig(hidden_size=128, num_hidden_layers=1, num_attention_heads=2,
                                                                      intermediate_size=256, vocab_size=60, max_position_embeddings=16))

    def make(seed):
        torch.manual_seed(seed)
        return model.VQAModel(vis, txt, fusion_type="co_attention", hidden_dim=64, num_classes=43).to(dev)
    teacher, student = encoders.quantize_int8(make(1).eval()), make(2)
    g = torch.Generator().manual_seed(9)
    loader = [{"image": torch.randn(6, 3, 32, 32, generator=g), "answer": torch.randint(0, 43, (6,), generator=g),
               "inputs": {"input_ids": torch.randint(1, 60, (6, 8), generator=g),
                          "attention_mask": torch.ones(6, 8, dtype=torch.long)}} for _ in range(2)]
    scores = mia.evaluate_privacy_entropy(teacher, loader, dev)
    losses = mia.evaluate_privacy_loss(teacher, loader, dev)
    assert np.isfinite(scores["entropies"]).all() and np.isfinite(losses["losses"]).all() and scores["entropies"].shape == (12,)
    before = {n: p.detach().clone() for n, p in student.named_parameters()}
    avg, agree = loops.distill(student, teacher, loader, torch.optim.AdamW(student.parameters(), lr=1e-3), dev, top=5)
    assert np.isfinite(avg)
    moved = [n for n, p in student.named_parameters() if not torch.equal(p, before[n])]
    assert any(n.startswith("classifier") for n in moved) and any(n.startswith("vision_encoder") for n in moved)
    assert all(torch.isfinite(p).all() for p in student.parameters())


def test_distillation_with_a_common_module(dev):
    """A module that student and teacher share runs in eval mode for the labels and in training mode for the student."""
    from vqa_amd import loops

    class Common(nn.Linear):
        def forward(self, x):
            modes.append((torch.is_grad_enabled(), self.training))
            return super().forward(x)
    modes = []
    a, b = Toy(4, 3, 0).to(dev), Toy(4, 3, 1).to(dev)
    a.head = b.head = Common(4, 3).to(dev)
    loops.distill(a, b, _loader(2, 5, 4, 3, 2), torch.optim.SGD(a.parameters(), lr=0.1), dev, top=2)
    assert modes == [(False, False), (True, True)] * 2 and a.training
    modes.clear()
    loops.distill(a, a, _loader(1, 5, 4, 3, 2), torch.optim.SGD(a.parameters(), lr=0.1), dev, top=2)
    assert modes == [(False, False), (True, True)]


def test_adapters_of_a_quantised_stack_do_not_merge(dev):
    """The plain weights are gone: the call says so, and works as before on a stack that has them."""
    from vqa_amd.encoders import BertConfig, BertModel, add_lora, merged_lora_weights, quantize_int8
    stack = BertModel(BertConfig(vocab_size=50, hidden_size=64, num_hidden_layers=1, num_attention_heads=1,
                                 intermediate_size=128, max_position_embeddings=16))
    add_lora(stack)
    assert set(merged_lora_weights(stack)) == {f"encoder.layer.0.attention.self.{t}.weight" for t in ("query", "value")}
    stack = quantize_int8(stack.to(dev).eval())
    with pytest.raises(RuntimeError, match="quantize_int8"):
        merged_lora_weights(stack)
