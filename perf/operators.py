"""What the answer-scoring, distillation and eight-bit operators cost, and what they compute.

Three operators that work on what a model answers:

  logprobs  log probabilities of given tokens, the entropy of the answer distribution and its top alternatives
            (`ops.token_logprobs`), with the gradient of the first two
  distill   the distillation loss against a teacher's top answers, with its gradient (`ops.distill_loss`)
  int8      a Linear layer in eight-bit integers, a scale for each token and each output channel (`ops.int8_linear`)

`own` chooses between the plain form of each (elementary torch operations in 32 bits, 64 where 32 lose what
matters) and the calls of this package.
"""
import math

import torch

own = False

F32, BF16 = torch.float32, torch.bfloat16


# --------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------
def listed():
    return [
        # one question answered over the 430 answers of COCO-QA: a few microseconds of work, latency is all
        {"name": "lp_one", "op": "logprobs", "rows": 1, "classes": 430, "dtype": "bf16", "top": 5,
         "temperature": 1.0, "masked": 0.0, "train": False},
        # a scoring pass over a shard of 25000 samples, f32 answers, some answers ruled out by the question's type
        {"name": "lp_shard", "op": "logprobs", "rows": 25000, "classes": 430, "dtype": "f32", "top": 3,
         "temperature": 1.0, "masked": 0.2, "train": False},
        # 64 questions of 30 tokens over BERT's vocabulary: the labels a distillation reads
        {"name": "lp_words", "op": "logprobs", "rows": 1920, "classes": 30522, "dtype": "bf16", "top": 20,
         "temperature": 2.0, "masked": 0.0, "train": False},
        # training on log probabilities with an entropy term over RoBERTa's vocabulary, an odd number of rows
        {"name": "lp_train", "op": "logprobs", "rows": 1001, "classes": 50265, "dtype": "bf16", "top": 0,
         "temperature": 1.0, "masked": 0.0, "train": True},
        # one small training batch of a student over 430 answers
        {"name": "kd_step", "op": "distill", "rows": 64, "classes": 430, "dtype": "bf16", "top": 16,
         "temperature": 2.0, "tail": False, "reduction": "mean"},
        # a DP-size batch, f32, with the teacher's remaining mass as one more event
        {"name": "kd_batch", "op": "distill", "rows": 1024, "classes": 430, "dtype": "f32", "top": 32,
         "temperature": 1.0, "tail": True, "reduction": "mean"},
        # 64 x 30 tokens over BERT's vocabulary
        {"name": "kd_words", "op": "distill", "rows": 1920, "classes": 30522, "dtype": "bf16", "top": 64,
         "temperature": 2.0, "tail": True, "reduction": "mean"},
        # rows weighted one by one (a padded batch) over RoBERTa's vocabulary, f32, odd sizes
        {"name": "kd_rows", "op": "distill", "rows": 511, "classes": 50265, "dtype": "f32", "top": 100,
         "temperature": 1.5, "tail": False, "reduction": "none"},
        # the query / key / value projection of a single token
        {"name": "q8_one", "op": "int8", "rows": 1, "inner": 768, "outer": 2304, "dtype": "bf16", "bias": True},
        # a text encoder's output projection at 64 x 30 tokens
        {"name": "q8_text", "op": "int8", "rows": 1920, "inner": 768, "outer": 768, "dtype": "bf16", "bias": True},
        # a vision encoder's query / key / value projection at 64 x 197 tokens
        {"name": "q8_vit", "op": "int8", "rows": 12608, "inner": 768, "outer": 2304, "dtype": "bf16", "bias": True},
        # a wide layer over many tokens, ragged row count: as much arithmetic as these layers meet
        {"name": "q8_wide", "op": "int8", "rows": 8191, "inner": 4096, "outer": 4096, "dtype": "bf16", "bias": False},
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_CLASSES = (13, 430, 30522, 50265)


def _rows_and_classes(rng, most):
    c = rng.choice(_CLASSES) if rng.random() < 0.4 else _between(rng, 2, 50265)
    return _between(rng, 1, max(1, min(25000, most // c))), c


def draw(rng):
    op = rng.choice(["logprobs", "distill", "int8"])
    dtype = rng.choice(["bf16", "f32"])
    if op == "logprobs":
        train = rng.random() < 0.4
        rows, classes = _rows_and_classes(rng, 25_000_000)
        top = 0 if train and rng.random() < 0.5 else min(classes, _between(rng, 1, 128))
        return {"op": op, "rows": rows, "classes": classes, "dtype": dtype, "top": top,
                "temperature": rng.choice([1.0, 1.0, 0.7, 2.0, 4.0]), "masked": rng.choice([0.0, 0.0, 0.2, 0.9]),
                "train": train}
    if op == "distill":
        rows, classes = _rows_and_classes(rng, 25_000_000)
        return {"op": op, "rows": rows, "classes": classes, "dtype": dtype, "top": min(classes, _between(rng, 1, 128)),
                "temperature": rng.choice([1.0, 1.5, 2.0, 4.0]), "tail": rng.random() < 0.5,
                "reduction": rng.choice(["mean", "mean", "none"])}
    while True:
        rows, inner, outer = _between(rng, 1, 16384), _between(rng, 16, 4096), _between(rng, 8, 4096)
        if rows * inner * outer <= 40_000_000_000 and rows * max(inner, outer) <= 40_000_000:
            return {"op": op, "rows": rows, "inner": inner, "outer": outer, "dtype": dtype, "bias": rng.random() < 0.7}


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    return g


def _dtype(case):
    return BF16 if case["dtype"] == "bf16" else F32


def _answers(g, rows, classes):
    """Logits as a trained head gives them: a spread of a few units and a handful of likely answers."""
    x = torch.randn(rows, classes, device="cuda", generator=g) * 2.0
    hot = torch.randint(0, classes, (rows, 4), device="cuda", generator=g)
    return x.scatter_add_(1, hot, torch.rand(rows, 4, device="cuda", generator=g) * 6.0), hot


def prepare(case, seed):
    g, dt = _generator(seed), _dtype(case)
    if case["op"] == "int8":
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        x = torch.randn(rows, inner, device="cuda", generator=g)
        x[:, :: max(1, inner // 3)] *= 6.0  # a few channels run larger, as they do behind a LayerNorm
        w = torch.randn(outer, inner, device="cuda", generator=g) * inner ** -0.5
        scale = (w.abs().amax(1) / 127.0).clamp_min(torch.finfo(F32).tiny)
        # the weights are laid out once: rows of whole 16-byte pieces
        packed = torch.zeros(outer, (inner + 15) // 16 * 16, dtype=torch.int8, device="cuda")
        packed[:, :inner] = (w.double() / scale.double()[:, None]).round().clamp(-127, 127).to(torch.int8)
        bias = torch.randn(outer, device="cuda", generator=g).to(dt) if case["bias"] else None
        return {"case": case, "x": x.to(dt), "weight": packed[:, :inner], "scale": scale, "bias": bias}
    rows, classes, top = case["rows"], case["classes"], case["top"]
    x, hot = _answers(g, rows, classes)
    state = {"case": case}
    if case["op"] == "logprobs":
        if case["masked"]:
            # answers ruled out for a row; the given token itself stays
            out = torch.rand(rows, classes, device="cuda", generator=g) < case["masked"]
            out.scatter_(1, hot[:, :1], False)
            x.masked_fill_(out, -math.inf)
        state["targets"] = hot[:, 0].contiguous()
        if case["train"]:
            state["up_logprob"] = -torch.rand(rows, device="cuda", generator=g) / rows
            state["up_entropy"] = torch.full((rows,), -0.01 / rows, device="cuda")
        state["logits"] = x.to(dt).requires_grad_(case["train"])
        return state
    # a teacher that mostly agrees with the student: log probabilities of its top answers at the temperature
    noise = torch.randn(rows, classes, device="cuda", generator=g)
    z = torch.add(x, noise).div_(case["temperature"])
    val, idx = z.topk(top, dim=1)
    state["teacher"] = (val - torch.logsumexp(z, 1, keepdim=True)).contiguous()
    state["indices"] = idx.contiguous()
    state["logits"] = x.to(dt).requires_grad_()
    if case["reduction"] == "none":
        live = (torch.rand(rows, device="cuda", generator=g) < 0.9).float()
        state["weights"] = live / rows
    return state


# --------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _OWN[case["op"]](state, case)
    return _PLAIN[case["op"]](state, case)


def _own_logprobs(s, case):
    from vqa_amd import ops
    r = ops.token_logprobs(s["logits"], s["targets"], top=case["top"], temperature=case["temperature"])
    out = {"logprobs": r.logprobs.detach(), "entropy": r.entropy.detach()}
    if case["top"]:
        out["top_logprobs"], out["top_indices"] = r.top_logprobs.detach(), r.top_indices
    if case["train"]:
        out["grad"], = torch.autograd.grad((r.logprobs, r.entropy), s["logits"], (s["up_logprob"], s["up_entropy"]))
    return out


def _own_distill(s, case):
    from vqa_amd import ops
    loss = ops.distill_loss(s["logits"], s["teacher"], s["indices"], temperature=case["temperature"],
                            tail=case["tail"], reduction=case["reduction"])
    up = s["weights"] if case["reduction"] == "none" else ops.unit_gradient(loss)
    grad, = torch.autograd.grad(loss, s["logits"], up)
    return {"loss": loss.detach(), "grad": grad}


def _own_int8(s, case):
    from vqa_amd import ops
    return ops.int8_linear(s["x"], s["weight"], s["scale"], s["bias"])


_OWN = {"logprobs": _own_logprobs, "distill": _own_distill, "int8": _own_int8}


def _log_softmax(z):
    """log softmax over the classes of rows that have a live entry each."""
    z = z - z.amax(1, keepdim=True)
    return z - z.exp().sum(1, keepdim=True).log()


def _plain_logprobs(s, case):
    x = s["logits"].detach().float()
    lp = _log_softmax(x / case["temperature"])
    p = lp.exp()
    plogp = torch.where(p > 0, p * lp, 0.0)
    entropy = -plogp.sum(1)
    t = s["targets"][:, None]
    out = {"logprobs": lp.gather(1, t)[:, 0], "entropy": entropy}
    if case["top"]:
        # ties go to the lowest index: the order-preserving integer of the value above the inverted index
        bits = x.view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7fffffff, bits).to(torch.int64) << 32
        key = key + (0x7fffffff - torch.arange(x.shape[1], device=x.device))
        out["top_indices"] = 0x7fffffff - (key.topk(case["top"], dim=1).values & 0xffffffff)
        out["top_logprobs"] = lp.gather(1, out["top_indices"])
    if case["train"]:
        a, b = s["up_logprob"][:, None], s["up_entropy"][:, None]
        g = -a * p - b * (plogp + p * entropy[:, None])
        g = g.scatter_add(1, t, a) / case["temperature"]
        out["grad"] = g.to(s["logits"].dtype)
    return out


def _plain_distill(s, case):
    x, t, idx = s["logits"].detach().float(), case["temperature"], s["indices"]
    rows, classes = x.shape
    z = x / t
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    # the loss is the small difference of large terms: its sums and logarithms are taken in 64 bits
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    lp = x.gather(1, idx).double() / t - top.double() - total.log()
    lq = s["teacher"].double()
    if not case["tail"]:
        lq = lq - lq.exp().sum(1, keepdim=True).log()
    q = lq.exp()
    loss = (q * (lq - lp)).sum(1)
    p = e / total.float()
    mass, slope = q.sum(1), None
    if case["tail"]:
        rest = 1.0 - mass
        # the teacher's log probabilities are f32: a remainder below 2^-20 is their rounding
        rest = torch.where(rest > 2.0 ** -20, rest, 0.0) * (idx.shape[1] < classes)
        live = rest > 0
        p_rest = e.scatter(1, idx, 0.0).sum(1, dtype=torch.float64) / total[:, 0]
        loss = loss + torch.where(live, rest * (rest.log() - p_rest.log()), 0.0)
        mass = mass + rest
        slope = mass - torch.where(live, rest / p_rest, 0.0)
    # d loss / d x = T (p mass - q) on the teacher's answers and T p (mass - rest / p_rest) elsewhere
    at = (p.gather(1, idx).double() * mass[:, None] - q).float()
    g = (p * (mass if slope is None else slope)[:, None].float()).scatter(1, idx, at)
    loss = loss * (t * t)
    if case["reduction"] == "mean":
        return {"loss": loss.mean().float(), "grad": (g * (t / rows)).to(s["logits"].dtype)}
    return {"loss": loss.float(), "grad": (g * (t * s["weights"])[:, None]).to(s["logits"].dtype)}


def _plain_int8(s, case):
    x = s["x"].float()
    scale = (x.abs().amax(1) / 127.0).clamp_min(torch.finfo(F32).tiny)
    # next to a border between two steps the quotient is taken in 64 bits
    q = (x.double() / scale.double()[:, None]).round().clamp(-127, 127).float()
    y = (q @ s["weight"].float().t()) * scale[:, None] * s["scale"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


_PLAIN = {"logprobs": _plain_logprobs, "distill": _plain_distill, "int8": _plain_int8}


# --------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "int8":
        m, k, n = case["rows"], case["inner"], case["outer"]
        return {"bytes": m * k * e + n * k + 4 * n + (e * n if case["bias"] else 0) + m * n * e, "flops": 2 * m * n * k}
    r, c, k = case["rows"], case["classes"], case["top"]
    if case["op"] == "logprobs":
        grad = case["train"]
        return {"bytes": r * c * e * (2 if grad else 1) + r * 8 + r * 8 + r * k * 12 + (r * 8 if grad else 0),
                "flops": r * c * (12 if grad else 6)}
    return {"bytes": r * c * e * 2 + r * k * 12 + r * 4, "flops": r * c * 10}


# --------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "int8":
        x = s["x"].double()
        # the token's scale is the f32 nearest to max|x| / 127; a step is half-even
        scale = torch.clamp((x.abs().amax(1) / 127.0).float(), min=torch.finfo(F32).tiny).double()
        q = torch.clamp(torch.round(x / scale[:, None]), -127, 127)
        y = torch.mm(q, s["weight"].double().t().contiguous()) * torch.outer(scale, s["scale"].double())
        return y if s["bias"] is None else y + s["bias"].double()
    x = s["logits"].detach().double()
    rows, classes = x.shape
    t = case["temperature"]
    if case["op"] == "logprobs":
        lse = torch.logsumexp(x / t, 1, keepdim=True)
        lp = x / t - lse
        p = torch.exp(lp)
        h = torch.special.entr(p).sum(1)
        out = {"logprobs": lp[torch.arange(rows, device=x.device), s["targets"]], "entropy": h}
        if case["top"]:
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : case["top"]]
            out["top_indices"], out["top_logprobs"] = order, torch.take_along_dim(lp, order, 1)
        if case["train"]:
            a, b = s["up_logprob"].double(), s["up_entropy"].double()
            # d logprob_t / dz = onehot - p;  dH / dz = entr(p) - p H
            g = b[:, None] * (torch.special.entr(p) - p * h[:, None]) - a[:, None] * p
            g[torch.arange(rows, device=x.device), s["targets"]] += a
            out["grad"] = g / t
        return out
    # the teacher's events and the student's, and the divergence between them
    lp = torch.log_softmax(x / t, 1)
    k = s["indices"].shape[1]
    lq = s["teacher"].double()
    if not case["tail"]:
        lq = lq - torch.logsumexp(lq, 1, keepdim=True)
    q = torch.exp(lq)
    target = torch.zeros_like(x).scatter_(1, s["indices"], q)
    loss = (q * (lq - torch.take_along_dim(lp, s["indices"], 1))).sum(1)
    p = torch.exp(lp)
    slope = p * q.sum(1, keepdim=True) - target
    if case["tail"] and k < classes:
        outside = torch.ones_like(x, dtype=torch.bool).scatter_(1, s["indices"], False)
        rest = 1.0 - q.sum(1)
        rest = torch.where(rest > 2.0 ** -20, rest, torch.zeros_like(rest))
        held = (p * outside).sum(1)
        some = rest > 0
        loss = loss + torch.where(some, rest * (torch.log(rest) - torch.log(held)), torch.zeros_like(rest))
        share = torch.where(some, rest / held, torch.zeros_like(rest))
        slope = slope + p * rest[:, None] - p * outside * share[:, None]
    if case["reduction"] == "mean":
        return {"loss": (loss * t * t).mean(), "grad": slope * (t / rows)}
    return {"loss": loss * t * t, "grad": slope * (t * s["weights"].double())[:, None]}
