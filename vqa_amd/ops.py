"""Tensor-level wrappers over the libvqafuse C ABI.

Every function here takes and returns torch tensors that live on a HIP device, enqueues the
kernels on torch's current stream and never synchronises with the host.  torch is used for
device memory, streams and autograd bookkeeping only; the arithmetic is in the kernels.
"""
from __future__ import annotations

import weakref
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check, dtype_code, load, ptr, stream_ptr


# --------------------------------------------------------------------------------------------
# Device-side counter-based RNG state {seed, counter}
# --------------------------------------------------------------------------------------------
class PhiloxState:
    """Four 64-bit words in device memory: {seed, counter, ticket, reserved}.

    Kernels that draw random numbers read {seed, counter} and address each draw by
    (seed, counter, element); ``advance()`` bumps the counter on the stream, so a captured HIP
    graph draws fresh numbers on every replay.  Kernels that bump the counter themselves (their last
    workgroup does it) count arrivals in `ticket`, which is zero between launches.
    """

    def __init__(self, device: torch.device, seed: Optional[int] = None, stream_salt: int = 0):
        if seed is None:
            seed = torch.initial_seed()
        self.seed = (int(seed) + 0x9E3779B97F4A7C15 * int(stream_salt)) & 0xFFFFFFFFFFFFFFFF
        signed = self.seed - (1 << 64) if self.seed >= (1 << 63) else self.seed
        self.state = torch.tensor([signed, 0, 0, 0], dtype=torch.int64, device=device)

    def advance(self, delta: int = 1) -> None:
        check(load().vqaf_rng_advance(ptr(self.state), delta, stream_ptr(self.state.device)),
              "vqaf_rng_advance")


_default_states: dict = {}


def default_rng(device: torch.device) -> PhiloxState:
    """Per-device state seeded from torch's global seed (re-made after torch.manual_seed)."""
    key = (device.type, device.index if device.index is not None else torch.cuda.current_device())
    seed = torch.initial_seed()
    st = _default_states.get(key)
    if st is None or st[0] != seed:
        st = (seed, PhiloxState(device, seed))
        _default_states[key] = st
    return st[1]


ADVANCE_RNG_IN_FOLD = True  # the query-fold launch of fused_prune_pool advances the generator state on the side
IN_KERNEL_RNG_BUMP = False  # let vqaf_fused_prune_pool_multi advance its generator state itself
FUSED_ONE_PASS = False  # True: the one-launch pruning branch takes the one-pass kernel where it applies (D = 512, N <= 208)

# Optional measurement probe: bench.py installs a callable (name, phase) -> None that records
# stream events around a named kernel launch; None in normal use.
PROBE = None


def _probe(name: str, phase: str) -> None:
    if PROBE is not None:
        PROBE(name, phase)


def require_gpu(*tensors: torch.Tensor) -> None:
    """Raises the library's "GPU only" error for CPU tensors (there is no CPU fallback)."""
    for t in tensors:
        if t is not None and not t.is_cuda:
            ptr(t)


def _noise_kind(noise_type: Optional[str]) -> int:
    if noise_type is None:
        return _lib.NOISE_NONE
    if noise_type == "gaussian":
        return _lib.NOISE_GAUSSIAN
    if noise_type == "uniform":
        return _lib.NOISE_UNIFORM
    # same message as utils/fusion.py:111 of the reference
    raise ValueError(f"Unsupported noise type: {noise_type}")


# --------------------------------------------------------------------------------------------
# Scoring and selection (no gradients flow through these: the weights only feed indices)
# --------------------------------------------------------------------------------------------
@torch.no_grad()
def attention_scores(q: torch.Tensor, seq: torch.Tensor, in_proj_weight: torch.Tensor,
                     in_proj_bias: torch.Tensor, num_heads: int) -> torch.Tensor:
    """Head-averaged single-query attention weights (B,N) f32; see vqaf_score."""
    B, N, D = seq.shape
    seq = seq.contiguous()
    q = q.reshape(B, D).to(seq.dtype).contiguous()
    w_ = in_proj_weight.detach().contiguous()
    b_ = in_proj_bias.detach().to(w_.dtype).contiguous()
    lib = load()
    nbytes = lib.vqaf_score_workspace_bytes(B, N, D, num_heads)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=seq.device)
    out = torch.empty(B, N, dtype=torch.float32, device=seq.device)
    check(lib.vqaf_score(ptr(q), ptr(seq), ptr(w_), ptr(b_), B, N, D, num_heads, dtype_code(seq),
                         dtype_code(w_), ptr(ws), nbytes, ptr(out), stream_ptr(seq.device)),
          "vqaf_score")
    return out


@torch.no_grad()
def head_score_matrix(q: torch.Tensor, seq: torch.Tensor, in_proj_weight: torch.Tensor,
                      in_proj_bias: torch.Tensor, num_heads: int) -> torch.Tensor:
    """Raw scaled per-head scores s (B,N,H) f32 (query fold + one pass over the tokens); the
    softmax / head mean is left to `select_indices`, which fuses it with the ranking."""
    B, N, D = seq.shape
    H = num_heads
    seq = seq.contiguous()
    ptr(seq)  # fails loudly on CPU tensors before any device call
    q = q.reshape(B, D).to(seq.dtype).contiguous()
    w_ = in_proj_weight.detach().contiguous()
    b_ = in_proj_bias.detach().to(w_.dtype).contiguous()
    lib, st, dev = load(), stream_ptr(seq.device), seq.device
    qp = torch.empty(B, D, dtype=torch.float32, device=dev)
    u = torch.empty(B, H, D, dtype=torch.float32, device=dev)
    check(lib.vqaf_fold_query(ptr(q), ptr(w_), ptr(b_), B, D, H, dtype_code(seq), dtype_code(w_), ptr(qp),
                              ptr(u), st), "vqaf_fold_query")
    s = torch.empty(B, N, H, dtype=torch.float32, device=dev)
    check(lib.vqaf_head_scores(ptr(seq), ptr(u), B, N, D, H, dtype_code(seq), ptr(s), st),
          "vqaf_head_scores")
    return s


@torch.no_grad()
def select_indices(k: int, *, scores: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                   k_adv: int = 0, pos: Optional[torch.Tensor] = None, src: Optional[torch.Tensor] = None,
                   rng: Optional["PhiloxState"] = None, want_weights: bool = False,
                   want_bottom: bool = False, record: bool = False, salt: int = 0,
                   advance: bool = True) -> dict:
    """Keep indices in one launch (vqaf_select): softmax/head-mean of `scores` (B,N,H) or given
    `weights` (B,N), ranking, and the adversarial swap -- injected (`pos`, `src`), drawn in the
    kernel (`rng`), or none (k_adv == 0)."""
    if (scores is None) == (weights is None):
        raise ValueError("pass exactly one of scores / weights")
    if scores is not None:
        scores = scores.contiguous()
        B, N, H = scores.shape
        dev = scores.device
    else:
        if weights.dim() == 3:
            weights = weights.squeeze(1)
        weights = weights.to(torch.float32).contiguous()
        (B, N), H, dev = weights.shape, 0, weights.device
    mode = 0
    if k_adv > 0:
        mode = 1 if pos is not None else 2
        if mode == 1:
            pos, src = pos.to(torch.int64).contiguous(), src.to(torch.int64).contiguous()
        elif rng is None:
            rng = default_rng(dev)
    out = {"top": torch.empty(B, k, dtype=torch.int64, device=dev), "bottom": None, "weights": None,
           "pos": None, "src": None}
    if want_bottom and N > k:
        out["bottom"] = torch.empty(B, N - k, dtype=torch.int64, device=dev)
    if want_weights:
        out["weights"] = torch.empty(B, N, dtype=torch.float32, device=dev)
    if record and mode == 2:
        out["pos"] = torch.empty(B, k_adv, dtype=torch.int64, device=dev)
        out["src"] = torch.empty(B, k_adv, dtype=torch.int64, device=dev)
    check(load().vqaf_select(ptr(scores), ptr(weights), B, N, H, k, mode, k_adv,
                             ptr(pos) if mode == 1 else None, ptr(src) if mode == 1 else None,
                             ptr(rng.state) if mode == 2 else None, int(salt), ptr(out["weights"]),
                             ptr(out["top"]), ptr(out["bottom"]), ptr(out["pos"]), ptr(out["src"]),
                             stream_ptr(dev)), "vqaf_select")
    out["drew"] = mode == 2
    if mode == 2 and advance:
        rng.advance()
    return out


@torch.no_grad()
def score_select_multi(specs, rng: Optional["PhiloxState"] = None):
    """Scoring + keep-index selection for several modalities that share batch, width, head count
    and dtypes (CoAttention's two branches) in FOUR launches in total: two for all query folds, one
    for all token scoring passes, one for all selections.

    specs: list of dicts(q, seq, in_proj_weight, in_proj_bias, num_heads, k, k_adv, pos, src, salt).
    Returns (list of keep-index tensors (B,k_i) int64, drew) where `drew` tells whether random
    numbers were consumed (the caller advances `rng` once)."""
    import ctypes
    n = len(specs)
    seq0 = specs[0]["seq"]
    B, _, D = seq0.shape
    H = specs[0]["num_heads"]
    dev = seq0.device
    ptr(seq0.contiguous())  # fails loudly on CPU tensors before any device call
    lib, st = load(), stream_ptr(dev)
    w_dt = specs[0]["in_proj_weight"].dtype
    keep = []  # keeps every temporary alive until the launches are enqueued
    folds = (_lib.FoldDesc * n)()
    scores = (_lib.ScoresDesc * n)()
    sels = (_lib.SelectDesc * n)()
    tops, drew = [], False
    for i, sp in enumerate(specs):
        seq = sp["seq"].contiguous()
        N = seq.shape[1]
        q = sp["q"].reshape(B, D).to(seq.dtype).contiguous()
        w_ = sp["in_proj_weight"].detach().contiguous()
        b_ = sp["in_proj_bias"].detach().to(w_.dtype).contiguous()
        qp = torch.empty(B, D, dtype=torch.float32, device=dev)
        u = torch.empty(B, H, D, dtype=torch.float32, device=dev)
        sc = torch.empty(B, N, H, dtype=torch.float32, device=dev)
        top = torch.empty(B, sp["k"], dtype=torch.int64, device=dev)
        k_adv = int(sp.get("k_adv", 0))
        pos, src = sp.get("pos"), sp.get("src")
        mode = 0
        if k_adv > 0:
            mode = 1 if pos is not None else 2
            if mode == 1:
                pos, src = pos.to(torch.int64).contiguous(), src.to(torch.int64).contiguous()
            else:
                drew = True
        keep.append((seq, q, w_, b_, qp, u, sc, pos, src))
        folds[i] = _lib.FoldDesc(ptr(q), ptr(w_), ptr(b_), ptr(qp), ptr(u))
        scores[i] = _lib.ScoresDesc(ptr(seq), ptr(u), ptr(sc), N)
        sels[i] = _lib.SelectDesc(ptr(sc), None, ptr(pos) if mode == 1 else None, ptr(src) if mode == 1 else None,
                                  None, ptr(top), None, None, None, int(sp.get("salt", i)), N, sp["k"], mode, k_adv)
        tops.append(top)
    if drew and rng is None:
        rng = default_rng(dev)
    check(lib.vqaf_fold_query_multi(ctypes.cast(folds, ctypes.c_void_p), n, B, D, H, dtype_code(seq0),
                                    _lib.BF16 if w_dt == torch.bfloat16 else _lib.F32, st), "vqaf_fold_query_multi")
    check(lib.vqaf_head_scores_multi(ctypes.cast(scores, ctypes.c_void_p), n, B, D, H, dtype_code(seq0), st),
          "vqaf_head_scores_multi")
    check(lib.vqaf_select_multi(ctypes.cast(sels, ctypes.c_void_p), n, B, H, ptr(rng.state) if drew else None, st),
          "vqaf_select_multi")
    return tops, drew


@torch.no_grad()
def topk_indices(w: torch.Tensor, k: int, need_bottom: bool = True
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(top (B,k) int64 weight-descending, bottom (B,N-k) int64 weight-ascending)."""
    if w.dim() == 3:
        w = w.squeeze(1)
    w = w.to(torch.float32).contiguous()
    B, N = w.shape
    top = torch.empty(B, k, dtype=torch.int64, device=w.device)
    bottom = torch.empty(B, N - k, dtype=torch.int64, device=w.device) if (need_bottom and N > k) else None
    check(load().vqaf_topk(ptr(w), B, N, k, ptr(top), ptr(bottom), stream_ptr(w.device)), "vqaf_topk")
    return top, bottom


@torch.no_grad()
def adv_swap_(top: torch.Tensor, bottom: torch.Tensor, pos: torch.Tensor, src: torch.Tensor) -> None:
    B, K = top.shape
    R = bottom.shape[1]
    k_adv = pos.shape[1]
    pos, src = pos.contiguous(), src.contiguous()   # (copies have to outlive the launch)
    check(load().vqaf_adv_swap(ptr(top), ptr(bottom), ptr(pos), ptr(src),
                               B, K, R, k_adv, stream_ptr(top.device)), "vqaf_adv_swap")


@torch.no_grad()
def adv_swap_random_(top: torch.Tensor, bottom: torch.Tensor, k_adv: int, rng: PhiloxState,
                     record: bool = False):
    B, K = top.shape
    R = bottom.shape[1]
    pos = src = None
    if record:
        pos = torch.empty(B, k_adv, dtype=torch.int64, device=top.device)
        src = torch.empty(B, k_adv, dtype=torch.int64, device=top.device)
    check(load().vqaf_adv_swap_random(ptr(top), ptr(bottom), B, K, R, k_adv, ptr(rng.state),
                                      ptr(pos), ptr(src), stream_ptr(top.device)),
          "vqaf_adv_swap_random")
    rng.advance()
    return pos, src


# --------------------------------------------------------------------------------------------
# Gather + noise + mix token (differentiable w.r.t. seq)
# --------------------------------------------------------------------------------------------
class _GatherMix(torch.autograd.Function):
    @staticmethod
    def forward(ctx, seq, idx, noise, noise_kind, noise_scale, rng_state, alpha, out_dtype):
        B, N, D = seq.shape
        K = idx.shape[1]
        seq_c = seq.contiguous()
        idx_c = idx.contiguous()
        kout = K + (1 if alpha > 0 else 0)
        out = torch.empty(B, kout, D, dtype=out_dtype, device=seq.device)
        noise_c = noise.to(torch.float32).contiguous() if noise is not None else None
        check(load().vqaf_gather_mix(ptr(seq_c), ptr(idx_c), ptr(noise_c), noise_kind,
                                     float(noise_scale), ptr(rng_state), float(alpha), B, N, K, D,
                                     dtype_code(seq_c), dtype_code(out), ptr(out),
                                     stream_ptr(seq.device)), "vqaf_gather_mix")
        ctx.save_for_backward(idx_c)
        ctx.meta = (B, N, K, D, float(alpha), seq.dtype)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        (idx_c,) = ctx.saved_tensors
        B, N, K, D, alpha, sdt = ctx.meta
        g = grad_out.contiguous()
        if g.dtype not in (torch.float32, torch.bfloat16):
            g = g.float()
        grad_seq = torch.empty(B, N, D, dtype=sdt, device=g.device)
        check(load().vqaf_gather_mix_bwd(ptr(g), ptr(idx_c), alpha, B, N, K, D, dtype_code(g),
                                         dtype_code(grad_seq), ptr(grad_seq), stream_ptr(g.device)),
              "vqaf_gather_mix_bwd")
        return grad_seq, None, None, None, None, None, None, None


def gather_mix(seq: torch.Tensor, idx: torch.Tensor, alpha: float, noise: Optional[torch.Tensor] = None,
               noise_type: Optional[str] = None, noise_scale: float = 0.0,
               rng: Optional[PhiloxState] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """out (B,K+1,D) (or (B,K,D) if alpha <= 0); see vqaf_gather_mix."""
    kind = _noise_kind(noise_type) if noise is None else _lib.NOISE_NONE
    state = None
    if kind != _lib.NOISE_NONE:
        rng = rng or default_rng(seq.device)
        state = rng.state
    out = _GatherMix.apply(seq, idx, noise, kind, noise_scale, state, alpha, out_dtype or seq.dtype)
    if kind != _lib.NOISE_NONE:
        rng.advance()
    return out


def prune_mix_supported(n_tokens: int, width: int, dtype: torch.dtype) -> bool:
    """Whether vqaf_prune_mix takes a (.., n_tokens, width) sequence of this dtype."""
    if dtype not in (torch.float32, torch.bfloat16):
        return False
    return bool(load().vqaf_prune_mix_supported(int(n_tokens), int(width),
                                                _lib.BF16 if dtype == torch.bfloat16 else _lib.F32))


class _PruneMix(torch.autograd.Function):
    """Selection + gather + noise + mix token of one sequence in one launch (vqaf_prune_mix)."""

    @staticmethod
    def forward(ctx, seq, w, K, mode, k_adv, pos, src, rng_state, salt, noise, noise_kind, noise_scale,
                noise_off, alpha, out_dtype):
        B, N, D = seq.shape
        seq_c = seq.contiguous()
        kout = K + (1 if alpha > 0 else 0)
        out = torch.empty(B, kout, D, dtype=out_dtype, device=seq.device)
        idx = torch.empty(B, K, dtype=torch.int64, device=seq.device)
        noise_c = noise.to(torch.float32).contiguous() if noise is not None else None
        need_noise_state = noise_c is None and noise_kind != _lib.NOISE_NONE
        check(load().vqaf_prune_mix(ptr(seq_c), ptr(w), B, N, K, D, dtype_code(seq_c), mode, k_adv,
                                    ptr(pos) if mode == 1 else None, ptr(src) if mode == 1 else None,
                                    ptr(rng_state) if mode == 2 else None, int(salt), ptr(noise_c), noise_kind,
                                    float(noise_scale), ptr(rng_state) if need_noise_state else None,
                                    int(noise_off), float(alpha), dtype_code(out), ptr(out), ptr(idx),
                                    stream_ptr(seq.device)), "vqaf_prune_mix")
        ctx.save_for_backward(idx)
        ctx.meta = (B, N, K, D, float(alpha), seq.dtype)
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)
        return out, idx

    @staticmethod
    def backward(ctx, grad_out, _grad_idx):
        if grad_out is None:
            return (None,) * 15
        (idx,) = ctx.saved_tensors
        B, N, K, D, alpha, sdt = ctx.meta
        g = grad_out.contiguous()
        if g.dtype not in (torch.float32, torch.bfloat16):
            g = g.float()
        grad_seq = torch.empty(B, N, D, dtype=sdt, device=g.device)
        check(load().vqaf_gather_mix_bwd(ptr(g), ptr(idx), alpha, B, N, K, D, dtype_code(g),
                                         dtype_code(grad_seq), ptr(grad_seq), stream_ptr(g.device)),
              "vqaf_gather_mix_bwd")
        return (grad_seq,) + (None,) * 14


def prune_mix(seq: torch.Tensor, weights: torch.Tensor, k: int, alpha: float, k_adv: int = 0,
              pos: Optional[torch.Tensor] = None, src: Optional[torch.Tensor] = None,
              noise: Optional[torch.Tensor] = None, noise_type: Optional[str] = None, noise_scale: float = 0.0,
              rng: Optional[PhiloxState] = None, out_dtype: Optional[torch.dtype] = None, salt: int = 0):
    """(out (B,K+1,D) or (B,K,D) if alpha <= 0, keep indices (B,K) int64) from attention weights in
    ONE launch.  Same results and the same random streams as select_indices() followed by
    gather_mix(): the adversarial draws come from the state's current counter, the noise from the
    next one when both are drawn, and the state then advances once per stream used."""
    if weights.dim() == 3:
        weights = weights.squeeze(1)
    w = weights.detach().to(torch.float32).contiguous()
    mode = 0
    if k_adv > 0:
        mode = 1 if pos is not None else 2
        if mode == 1:
            pos, src = pos.to(torch.int64).contiguous(), src.to(torch.int64).contiguous()
    kind = _noise_kind(noise_type) if noise is None else _lib.NOISE_NONE
    draws_noise = kind != _lib.NOISE_NONE
    state = None
    if mode == 2 or draws_noise:
        rng = rng or default_rng(seq.device)
        state = rng.state
    noise_off = 1 if (mode == 2 and draws_noise) else 0
    out, idx = _PruneMix.apply(seq, w, int(k), mode, int(k_adv), pos, src, state, salt, noise, kind,
                               noise_scale, noise_off, alpha, out_dtype or seq.dtype)
    if state is not None:
        rng.advance((1 if mode == 2 else 0) + (1 if draws_noise else 0))
    return out, idx


class _MeanPool(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        B, M, D = x.shape
        xc = x.contiguous()
        out = torch.empty(B, D, dtype=x.dtype, device=x.device)
        check(load().vqaf_mean_pool(ptr(xc), B, M, D, dtype_code(xc), ptr(out), D, 0, dtype_code(out),
                                    stream_ptr(x.device)), "vqaf_mean_pool")
        ctx.meta = (B, M, D, x.dtype)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        B, M, D, dt = ctx.meta
        g = grad_out.contiguous()
        if g.dtype not in (torch.float32, torch.bfloat16):
            g = g.float()
        gx = torch.empty(B, M, D, dtype=dt, device=g.device)
        check(load().vqaf_mean_pool_bwd(ptr(g), D, 0, dtype_code(g), B, M, D, dtype_code(gx), ptr(gx),
                                        stream_ptr(g.device)), "vqaf_mean_pool_bwd")
        return gx


def mean_pool(x: torch.Tensor) -> torch.Tensor:
    """x.mean(dim=1) for (B,M,D) tokens."""
    return _MeanPool.apply(x)


class _PrunedPool(torch.autograd.Function):
    """fused[:, off:off+D] = mean_j prune(seq_m, idx_m)[:, j, :] for each modality m, without
    writing the pruned token tensors.  Inputs: a list of (seq, idx, alpha, noise, kind, scale,
    rng_state) flattened; output (B, sum D_m).  Modalities that share dtype and width (the vision
    and text halves of CoAttention) go through ONE launch forward and ONE backward."""

    @staticmethod
    def forward(ctx, n_mod, out_dtype, *flat):
        import ctypes
        mods = [flat[i * 7:(i + 1) * 7] for i in range(n_mod)]
        B = mods[0][0].shape[0]
        dev = mods[0][0].device
        widths = [m[0].shape[2] for m in mods]
        ld = sum(widths)
        out = torch.empty(B, ld, dtype=out_dtype, device=dev)
        lib, st = load(), stream_ptr(dev)
        col0 = 0
        saved, metas, keep = [], [], []
        for (seq, idx, alpha, noise, kind, scale, state), D in zip(mods, widths):
            seq_c, idx_c = seq.contiguous(), idx.contiguous()
            noise_c = noise.to(torch.float32).contiguous() if noise is not None else None
            keep.append((seq_c, idx_c, noise_c, state, float(alpha), int(kind), float(scale)))
            saved.append(idx_c)
            metas.append((seq.shape[1], idx.shape[1], D, float(alpha), seq.dtype, col0))
            col0 += D
        uniform = n_mod > 1 and n_mod <= 4 and len(set(widths)) == 1 and len({m[0].dtype for m in mods}) == 1
        if uniform:
            arr = (_lib.PoolMod * n_mod)()
            for i, ((seq_c, idx_c, noise_c, state, alpha, kind, scale), meta) in enumerate(zip(keep, metas)):
                arr[i] = _lib.PoolMod(ptr(seq_c), ptr(idx_c), ptr(noise_c), ptr(state), scale, alpha, kind,
                                      meta[0], meta[1], meta[5])
            _probe("gather_mix_pool_multi", "begin")
            check(lib.vqaf_gather_mix_pool_multi(ctypes.cast(arr, ctypes.c_void_p), n_mod, B, widths[0],
                                                 dtype_code(keep[0][0]), ptr(out), ld, dtype_code(out), st),
                  "vqaf_gather_mix_pool_multi")
            _probe("gather_mix_pool_multi", "end")
        else:
            for i, ((seq_c, idx_c, noise_c, state, alpha, kind, scale), (N, K, D, _a, _dt, c0)) in \
                    enumerate(zip(keep, metas)):
                _probe(f"gather_mix_pool:{i}", "begin")
                check(lib.vqaf_gather_mix_pool(ptr(seq_c), ptr(idx_c), ptr(noise_c), kind, scale, ptr(state),
                                               alpha, B, N, K, D, dtype_code(seq_c), ptr(out), ld, c0,
                                               dtype_code(out), st), "vqaf_gather_mix_pool")
                _probe(f"gather_mix_pool:{i}", "end")
        for (_s, _i, _n, state, _al, kind, _sc) in keep:
            if state is not None and kind != _lib.NOISE_NONE:  # next consumer gets a fresh stream
                check(lib.vqaf_rng_advance(ptr(state), 1, st), "vqaf_rng_advance")
        ctx.save_for_backward(*saved)
        ctx.metas = metas
        ctx.B, ctx.ld, ctx.n_mod, ctx.uniform = B, ld, n_mod, uniform
        return out

    @staticmethod
    def backward(ctx, grad_out):
        import ctypes
        g = grad_out.contiguous()
        if g.dtype not in (torch.float32, torch.bfloat16):
            g = g.float()
        lib, st = load(), stream_ptr(g.device)
        grads = [None, None]
        outs = []
        for i, (N, K, D, alpha, sdt, col0) in enumerate(ctx.metas):
            need = ctx.needs_input_grad[2 + 7 * i]
            outs.append(torch.empty(ctx.B, N, D, dtype=sdt, device=g.device) if need else None)
        if ctx.uniform and any(o is not None for o in outs):
            arr = (_lib.PoolBwdMod * ctx.n_mod)()
            for i, (idx_c, (N, K, D, alpha, sdt, col0)) in enumerate(zip(ctx.saved_tensors, ctx.metas)):
                arr[i] = _lib.PoolBwdMod(ptr(idx_c), ptr(outs[i]), alpha, N, K, col0)
            sdt0 = ctx.metas[0][4]
            check(lib.vqaf_gather_mix_pool_bwd_multi(ptr(g), ctx.ld, dtype_code(g), ctypes.cast(arr, ctypes.c_void_p),
                                                     ctx.n_mod, ctx.B, ctx.metas[0][2],
                                                     _lib.BF16 if sdt0 == torch.bfloat16 else _lib.F32, st),
                  "vqaf_gather_mix_pool_bwd_multi")
        else:
            for i, (idx_c, (N, K, D, alpha, sdt, col0)) in enumerate(zip(ctx.saved_tensors, ctx.metas)):
                if outs[i] is not None:
                    check(lib.vqaf_gather_mix_pool_bwd(ptr(g), ctx.ld, col0, dtype_code(g), ptr(idx_c), alpha,
                                                       ctx.B, N, K, D, dtype_code(outs[i]), ptr(outs[i]), st),
                          "vqaf_gather_mix_pool_bwd")
        for o in outs:
            grads.extend([o, None, None, None, None, None, None])
        return tuple(grads)


FUSED_WIDTHS = (64, 128, 256, 512, 1024)


def fused_prune_pool_supported(specs) -> bool:
    """True when vqaf_fused_prune_pool_multi covers these modalities (bf16 tokens of one width and
    batch, at most 8 heads, per-sample state within 64 KiB of LDS)."""
    s0 = specs[0]["seq"]
    B, _, D = s0.shape
    H = specs[0]["num_heads"]
    if not (1 <= len(specs) <= 4) or s0.dtype != torch.bfloat16 or D not in FUSED_WIDTHS or H > 8:
        return False
    for sp in specs:
        seq = sp["seq"]
        if seq.dtype != torch.bfloat16 or seq.shape[0] != B or seq.shape[2] != D or sp["num_heads"] != H:
            return False
        N = seq.shape[1]
        NP = 64
        while NP < N:
            NP *= 2
        lds = max(32 * (D + 8), 16384) + 8 * NP + N * H * 4 + 12 * N + 8 * max(1, sp.get("k_adv", 0)) + 512
        if N > 4096 or lds > 64 * 1024:
            return False
    return True


class _FusedPrunePool(torch.autograd.Function):
    """Scoring + selection + pooled prune/mix of several modalities: two launches for the query
    folds, ONE for everything that touches tokens.  Returns (fused (B, n*D), idx_0, idx_1, ...).
    The backward is the pooled prune/mix backward (scores and indices carry no gradient)."""

    @staticmethod
    def forward(ctx, n_mod, out_dtype, rng_state, rng_advance, sel_draws, *flat):
        import ctypes
        per = 14
        mods = [flat[i * per:(i + 1) * per] for i in range(n_mod)]
        seq0 = mods[0][0]
        B, _, D = seq0.shape
        dev = seq0.device
        H = mods[0][4]
        lib, st = load(), stream_ptr(dev)
        w_dt = mods[0][2].dtype
        ld = n_mod * D
        out = torch.empty(B, ld, dtype=out_dtype, device=dev)
        folds = (_lib.FoldDesc * n_mod)()
        fm = (_lib.FusedMod * n_mod)()
        keep, idxs, metas = [], [], []
        for i, (seq, q, w, bia, _h, k, k_adv, pos, src, salt, alpha, noise, kind, scale_state) in enumerate(mods):
            noise_scale, noise_state = scale_state
            seq_c = seq.contiguous()
            N = seq_c.shape[1]
            q_c = q.reshape(B, D).to(seq_c.dtype).contiguous()
            w_c = w.detach().contiguous()
            b_c = bia.detach().to(w_c.dtype).contiguous()
            qp = torch.empty(B, D, dtype=torch.float32, device=dev)
            u = torch.empty(B, H, D, dtype=torch.float32, device=dev)
            idx = torch.empty(B, k, dtype=torch.int64, device=dev)
            mode = 0
            if k_adv > 0:
                mode = 1 if pos is not None else 2
                if mode == 1:
                    pos, src = pos.to(torch.int64).contiguous(), src.to(torch.int64).contiguous()
            noise_c = noise.to(torch.float32).contiguous() if noise is not None else None
            keep.append((seq_c, q_c, w_c, b_c, qp, u, pos, src, noise_c, noise_state))
            folds[i] = _lib.FoldDesc(ptr(q_c), ptr(w_c), ptr(b_c), ptr(qp), ptr(u))
            fm[i] = _lib.FusedMod(ptr(seq_c), ptr(u), ptr(pos) if mode == 1 else None, ptr(src) if mode == 1 else None,
                                  ptr(noise_c), ptr(noise_state), ptr(idx), None, int(salt), float(alpha),
                                  float(noise_scale), int(kind), N, int(k), mode, int(k_adv), i * D,
                                  int(sel_draws and rng_state is not None and noise_state is not None
                                      and noise_state.data_ptr() == rng_state.data_ptr()))
            idxs.append(idx)
            metas.append((N, int(k), D, float(alpha), seq.dtype, i * D))
        if rng_advance < 0:  # the fold launch advances the generator state for the launch behind it
            check(lib.vqaf_fold_query_multi_advance(ctypes.cast(folds, ctypes.c_void_p), n_mod, B, D, H,
                                                    dtype_code(seq0), _lib.BF16 if w_dt == torch.bfloat16 else _lib.F32,
                                                    ptr(rng_state), -int(rng_advance), st),
                  "vqaf_fold_query_multi_advance")
        else:
            check(lib.vqaf_fold_query_multi(ctypes.cast(folds, ctypes.c_void_p), n_mod, B, D, H, dtype_code(seq0),
                                            _lib.BF16 if w_dt == torch.bfloat16 else _lib.F32, st),
                  "vqaf_fold_query_multi")
        _probe("fused_prune_pool", "begin")
        entry = lib.vqaf_fused_prune_pool_multi
        if FUSED_ONE_PASS:
            ns = (ctypes.c_int * n_mod)(*[m[0].shape[1] for m in mods])
            if lib.vqaf_fused_prune_pool_onepass_supported(n_mod, ctypes.cast(ns, ctypes.c_void_p), D, H):
                entry = lib.vqaf_fused_prune_pool_onepass_multi
        check(entry(ctypes.cast(fm, ctypes.c_void_p), n_mod, B, D, H, dtype_code(seq0),
                    ptr(rng_state), int(rng_advance), ptr(out), ld, dtype_code(out), st),
              "vqaf_fused_prune_pool_multi")
        _probe("fused_prune_pool", "end")
        if not rng_advance:  # the kernel did not bump the counter itself: one launch per noise stream
            for (_s, _q, _w, _b, _qp, _u, _p, _sr, noise_c, noise_state), m in zip(keep, mods):
                if noise_state is not None and m[12] != _lib.NOISE_NONE and noise_c is None:
                    check(lib.vqaf_rng_advance(ptr(noise_state), 1, st), "vqaf_rng_advance")
        ctx.save_for_backward(*idxs)
        ctx.metas = metas
        ctx.B, ctx.ld, ctx.n_mod, ctx.per = B, ld, n_mod, per
        ctx.mark_non_differentiable(*idxs)
        ctx.set_materialize_grads(False)  # no zero-filled int64 "gradients" for the index outputs
        return (out, *idxs)

    @staticmethod
    def backward(ctx, grad_out, *_unused):
        import ctypes
        if grad_out is None:
            return (None,) * (5 + ctx.per * ctx.n_mod)
        g = grad_out.contiguous()
        if g.dtype not in (torch.float32, torch.bfloat16):
            g = g.float()
        lib, st = load(), stream_ptr(g.device)
        outs = []
        for i, (N, K, D, alpha, sdt, col0) in enumerate(ctx.metas):
            need = ctx.needs_input_grad[5 + ctx.per * i]
            outs.append(torch.empty(ctx.B, N, D, dtype=sdt, device=g.device) if need else None)
        if any(o is not None for o in outs):
            arr = (_lib.PoolBwdMod * ctx.n_mod)()
            for i, (idx_c, (N, K, D, alpha, sdt, col0)) in enumerate(zip(ctx.saved_tensors, ctx.metas)):
                arr[i] = _lib.PoolBwdMod(ptr(idx_c), ptr(outs[i]), alpha, N, K, col0)
            check(lib.vqaf_gather_mix_pool_bwd_multi(ptr(g), ctx.ld, dtype_code(g), ctypes.cast(arr, ctypes.c_void_p),
                                                     ctx.n_mod, ctx.B, ctx.metas[0][2], _lib.BF16, st),
                  "vqaf_gather_mix_pool_bwd_multi")
        grads = [None, None, None, None, None]
        for o in outs:
            grads.extend([o] + [None] * (ctx.per - 1))
        return tuple(grads)


def fused_prune_pool(specs, out_dtype: torch.dtype, rng: Optional["PhiloxState"] = None):
    """specs: list of dicts(q, seq, in_proj_weight, in_proj_bias, num_heads, k, k_adv, pos, src, salt,
    alpha, noise, noise_type, noise_scale, noise_rng).  Returns (fused, [keep indices], drew)."""
    flat, drew, noise_states = [], False, []
    dev = specs[0]["seq"].device
    for i, sp in enumerate(specs):
        kind = _noise_kind(sp.get("noise_type")) if sp.get("noise") is None else _lib.NOISE_NONE
        state = None
        if kind != _lib.NOISE_NONE:
            state = (sp.get("noise_rng") or default_rng(dev)).state
            noise_states.append(state)
        k_adv = int(sp.get("k_adv", 0))
        if k_adv > 0 and sp.get("pos") is None:
            drew = True
        flat.extend([sp["seq"], sp["q"], sp["in_proj_weight"], sp["in_proj_bias"], sp["num_heads"], sp["k"], k_adv,
                     sp.get("pos"), sp.get("src"), sp.get("salt", i), sp["alpha"], sp.get("noise"), kind,
                     (sp.get("noise_scale", 0.0), state)])
    if drew and rng is None:
        rng = default_rng(dev)
    # Every stream this launch draws from: the selection's and the in-kernel noise streams.  When
    # they are one and the same state the kernel's last workgroup bumps its counter (once per
    # stream position consumed) and no counter launch follows; the caller then has nothing to advance.
    streams = list(noise_states) + ([rng.state] if drew else [])
    # (off by default: the bump costs every workgroup a returning device-scope atomic at its end, which
    # at thousands of workgroups per launch is slower than the one-thread launch it saves)
    one_state = bool(streams) and all(t.data_ptr() == streams[0].data_ptr() for t in streams)
    in_kernel = IN_KERNEL_RNG_BUMP and one_state and streams[0].numel() >= 4
    # (the default) the query-fold launch in front of the token launch advances the counter on the side, and
    # the token launch draws from the positions in front of the advance: same values, no counter launch
    ahead = ADVANCE_RNG_IN_FOLD and one_state and not in_kernel
    res = _FusedPrunePool.apply(len(specs), out_dtype,
                                streams[0] if (in_kernel or ahead) else (rng.state if drew else None),
                                len(streams) if in_kernel else (-len(streams) if ahead else 0), drew, *flat)
    return res[0], list(res[1:]), drew and not (in_kernel or ahead)


def pruned_pool(mods, out_dtype: torch.dtype) -> torch.Tensor:
    """mods: list of dicts(seq, idx, alpha, noise, noise_type, noise_scale, rng)."""
    flat = []
    for m in mods:
        kind = _noise_kind(m.get("noise_type")) if m.get("noise") is None else _lib.NOISE_NONE
        state = None
        if kind != _lib.NOISE_NONE:
            state = (m.get("rng") or default_rng(m["seq"].device)).state
        flat.extend([m["seq"], m["idx"], m["alpha"], m.get("noise"), kind, m.get("noise_scale", 0.0), state])
    return _PrunedPool.apply(len(mods), out_dtype, *flat)


# --------------------------------------------------------------------------------------------
# Small helpers used by the DP-SGD engine and the MIA scorer
# --------------------------------------------------------------------------------------------
@torch.no_grad()
def ce_conf(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, want_loss: bool = True,
            want_conf: bool = True, want_pred: bool = False, grad_scale: Optional[float] = None,
            grad_dtype: torch.dtype = torch.float32):
    """Per-sample cross-entropy, max-softmax confidence, argmax and (optionally) the gradient of
    grad_scale * sum_i CE_i w.r.t. the logits (f32, or bf16 on request).  Returns (loss, conf, pred, grad)."""
    B, C = logits.shape
    lg = logits.contiguous()
    dev = lg.device
    loss = torch.empty(B, dtype=torch.float32, device=dev) if (want_loss and targets is not None) else None
    conf = torch.empty(B, dtype=torch.float32, device=dev) if want_conf else None
    pred = torch.empty(B, dtype=torch.int64, device=dev) if want_pred else None
    grad = torch.empty(B, C, dtype=grad_dtype, device=dev) if grad_scale is not None else None
    tg = targets.to(torch.int64).contiguous() if targets is not None else None
    check(load().vqaf_ce_conf(ptr(lg), ptr(tg), B, C, dtype_code(lg), ptr(loss), ptr(conf), ptr(pred),
                              ptr(grad), dtype_code(grad) if grad is not None else 0, float(grad_scale or 0.0),
                              stream_ptr(dev)), "vqaf_ce_conf")
    return loss, conf, pred, grad


_ce_tickets: dict = {}
_zero_padded: dict = {}  # id(buffer) -> weak reference: (B, ld) buffers whose columns past the logical width are zero


def zero_padded_pitch(t: torch.Tensor) -> Optional[int]:
    """Row pitch of `t` if it is the leading-columns view of one of the zero-padded gradient buffers the
    mean cross-entropy hands out (the library's bf16 GEMMs may then read whole 16-byte chunks past its
    logical width), else None."""
    base = t._base
    if base is None or t.dim() != 2 or t.stride(1) != 1 or t.storage_offset() != 0:
        return None
    ref = _zero_padded.get(id(base))
    if ref is None or ref() is not base or t.stride(0) != base.shape[1] or t.shape[0] != base.shape[0]:
        return None
    return int(t.stride(0))


class _MeanCE(torch.autograd.Function):
    """Mean cross-entropy (nn.CrossEntropyLoss() as the training loop uses it, train.py:104,
    utils/src.py:96) with its logits gradient produced by the same kernel launch."""

    @staticmethod
    def forward(ctx, logits, targets):
        B = logits.shape[0]
        # the gradient is written in the logits' dtype: with the usual incoming gradient of 1 it is handed on as is
        gdt = logits.dtype if logits.dtype in (torch.float32, torch.bfloat16) else torch.float32
        lg = logits.contiguous()
        dev = lg.device
        C = lg.shape[1]
        loss = torch.empty(B, dtype=torch.float32, device=dev)
        # bf16 gradient rows are padded with zeros to a multiple of 8 elements (16 bytes): a 430-class head's
        # backprop is then a legal operand of the library's own bf16 GEMMs (input gradient, clipped sum)
        ldg = (C + 7) // 8 * 8 if gdt == torch.bfloat16 else C
        buf = torch.empty(B, ldg, dtype=gdt, device=dev)
        if ldg != C:
            _zero_padded[id(buf)] = weakref.ref(buf, lambda _r, k=id(buf): _zero_padded.pop(k, None))
        grad = buf[:, :C]
        mean = torch.empty((), dtype=torch.float32, device=dev)
        # one self-resetting ticket word per device, made before any graph capture can be under way (a
        # tensor allocated during a capture would live in that graph's memory pool); mean losses computed
        # on different streams of one device must not overlap
        ticket = _ce_tickets.get(dev)
        if ticket is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("cross_entropy_mean: run one step eagerly before capturing a HIP graph")
            ticket = _ce_tickets[dev] = torch.zeros(1, dtype=torch.int32, device=dev)
        tg = targets.to(torch.int64).contiguous()   # (a copy has to outlive the launch)
        check(load().vqaf_ce_mean(ptr(lg), ptr(tg), B, C, dtype_code(lg), ptr(loss),
                                  ptr(buf), ldg, dtype_code(buf), 1.0 / B, ptr(mean), ptr(ticket), stream_ptr(dev)),
              "vqaf_ce_mean")
        ctx.buf = buf  # the unit-gradient backward hands on a view of it (its base stays this object)
        ctx.save_for_backward(grad)
        ctx.in_dtype = logits.dtype
        # kept for the rare backward with a non-unit incoming gradient (see backward); no copy is made
        ctx.logits, ctx.targets = (logits.detach(), targets) if gdt != torch.float32 else (None, None)
        return mean

    @staticmethod
    def backward(ctx, grad_out):
        (grad,) = ctx.saved_tensors
        if grad_out is _unit_grads.get((grad_out.device, grad_out.dtype)) and grad.dtype == ctx.in_dtype:
            # loss.backward(gradient=unit_gradient(loss)): the factor is exactly 1
            return ctx.buf[:, :grad.shape[1]], None
        if grad.dtype == torch.float32 and ctx.in_dtype in (torch.float32, torch.bfloat16) and grad_out.numel() == 1:
            # one launch: the product is rounded straight into the logits' dtype
            out = torch.empty(grad.shape, dtype=ctx.in_dtype, device=grad.device)
            go = grad_out.reshape(1).to(torch.float32)  # a view for the usual f32 scalar
            check(load().vqaf_scale_cast(ptr(grad), ptr(go), grad.numel(), dtype_code(out), ptr(out),
                                         stream_ptr(grad.device)), "vqaf_scale_cast")
            return out, None
        # bf16 logits and another incoming gradient (a weighted or scaled loss): the saved gradient was
        # rounded to bf16 for the unit-gradient hand-over, so scaling it would round twice; form it again
        # from the logits in f32 and round the product once
        if grad.dtype != torch.float32 and ctx.logits is not None:
            _, _, _, g32 = ce_conf(ctx.logits, ctx.targets, want_loss=False, want_conf=False,
                                   grad_scale=1.0 / grad.shape[0], grad_dtype=torch.float32)
            return (g32 * grad_out.float()).to(ctx.in_dtype), None
        return (grad.float() * grad_out).to(ctx.in_dtype), None


def cross_entropy_mean(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    return _MeanCE.apply(logits, targets)


_unit_grads: dict = {}


def unit_gradient(loss: torch.Tensor) -> torch.Tensor:
    """A cached scalar 1 of the loss's dtype and device for `loss.backward(gradient=...)`: what
    `loss.backward()` uses, without the fill launch autograd spends on making it every step."""
    key = (loss.device, loss.dtype)
    one = _unit_grads.get(key)
    if one is None:
        one = torch.ones((), dtype=loss.dtype, device=loss.device)
        _unit_grads[key] = one
    return one


# --------------------------------------------------------------------------------------------
# Answer scores and distillation
# --------------------------------------------------------------------------------------------
ANSWERS_MAX = 128  # given tokens, alternatives and teacher's answers per row
ANSWERS_MAX_CLASSES = 2 ** 28


class TokenLogprobs(NamedTuple):
    """What `token_logprobs` returns; None where it was not asked for."""
    logprobs: Optional[torch.Tensor]
    entropy: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]


# Of a device index without building a stream object, where torch has it (a build without GPU support does not)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(device: torch.device, entry: str, *args) -> None:
    """Calls a C entry point whose last argument is the stream, on `device`'s current stream.  A launch goes to the
    current device whatever its stream, so another device is made current around it."""
    lib = load()
    index = device.index
    if index == _current_device():
        status = getattr(lib, entry)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = getattr(lib, entry)(*args, _raw_stream(index))
    if status != 0:
        check(status, entry)


def _first_order(backward):
    """once_differentiable without its cost where nothing records gradients of gradients."""
    recorded = once_differentiable(backward)

    def run(ctx, *grads):
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a forward-mode derivative comes with any of them.  These operators have none: autograd's function refuses
    it, so a tensor that carries one takes that way whether gradients are recorded or not."""
    if getattr(forward_ad, "_current_level", 0) < 0:   # no level is open (asking a tensor costs 0.7 us)
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _answer_rows(logits: torch.Tensor):
    """(logits as (R,C) with unit inner stride, its row pitch)."""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits need a dimension of classes, got shape {tuple(logits.shape)}")
    require_gpu(logits)
    dtype_code(logits)
    x = logits
    C = logits.shape[-1]
    if C > ANSWERS_MAX_CLASSES or logits.numel() // C >= 2 ** 31:
        raise ValueError(f"logits of at most 2^31 - 1 rows of {ANSWERS_MAX_CLASSES} classes, got shape {tuple(logits.shape)}")
    if x.dim() == 2 and x.is_contiguous():
        return x, C
    if x.dim() != 2:
        x = x.reshape(-1, C)
    if C > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, (x.stride(0) if x.shape[0] > 1 else C)


def _grad_rows(x: torch.Tensor, ld: int) -> torch.Tensor:
    """An (R,C) tensor of x's dtype whose rows lie on the 16-byte grid as x's do."""
    R, C = x.shape
    if ld == C and x.data_ptr() % 16 == 0:
        return torch.empty((R, C), dtype=x.dtype, device=x.device)
    per = 16 // x.element_size()
    off, ldg = (x.data_ptr() // x.element_size()) % per, C + (ld - C) % per
    buf = torch.empty(off + R * ldg, dtype=x.dtype, device=x.device)
    return buf.as_strided((R, C), (ldg, 1), off)


def _grad_pitch(x: torch.Tensor, ld: int) -> int:
    """Row pitch of _grad_rows(x, ld)."""
    C = x.shape[1]
    return C if ld == C else C + (ld - C) % (16 // x.element_size())


def _temperature(t: float) -> float:
    t = float(t)
    if not 2.0 ** -20 <= t <= 2.0 ** 20:
        raise ValueError(f"temperature has to be in [2^-20, 2^20], got {t}")
    return t


def _f32(g: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if g is None or (g.dtype is torch.float32 and g.is_contiguous()):
        return g
    return g.to(torch.float32).contiguous()


def _addr(t: Optional[torch.Tensor]) -> Optional[int]:
    """Address of a tensor made or checked here (None passes NULL)."""
    return None if t is None else t.data_ptr()


def _logprobs_forward(x, targets, call, stats):
    """One launch; (logprobs, entropy, top_logprobs, top_indices, stats), None where not asked for, in the shapes that the
    caller returns.  call: (row pitch, leading dimensions, targets of a row, alternatives, temperature, entropy)."""
    ld, lead, T, top, temperature, entropy = call
    R, C = x.shape
    dev, f32 = x.device, torch.float32
    lp = None if targets is None else torch.empty(targets.shape, dtype=f32, device=dev)
    ent = torch.empty(lead, dtype=f32, device=dev) if entropy else None
    tl = torch.empty((*lead, top), dtype=f32, device=dev) if top else None
    ti = torch.empty((*lead, top), dtype=torch.int64, device=dev) if top else None
    st = torch.empty((R, 2), dtype=f32, device=dev) if stats else None
    _launch(dev, "vqaf_token_logprobs", x.data_ptr(), ld, _addr(targets), R, C, T, top, dtype_code(x), temperature,
            _addr(lp), _addr(ent), _addr(tl), _addr(ti), _addr(st))
    return lp, ent, tl, ti, st


def _token_indices(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise TypeError(f"{what} are token indices, got {t.dtype}")
    return t.to(torch.int64)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, targets, call):
        lp, ent, tl, ti, ctx.stats = _logprobs_forward(x, targets, call, True)
        ctx.save_for_backward(x, targets, ti, ent)
        ctx.call = call
        ctx.set_materialize_grads(False)
        if ti is not None:
            ctx.mark_non_differentiable(ti)
        return lp, ent, tl, ti

    @staticmethod
    @_first_order
    def backward(ctx, g_lp, g_ent, g_top, _g_idx):
        if g_lp is None and g_ent is None and g_top is None:
            return None, None, None
        x, targets, ti, ent = ctx.saved_tensors
        ld, _, T, top, temperature, _ = ctx.call
        R, C = x.shape
        g_lp, g_ent, g_top = _f32(g_lp), _f32(g_ent), _f32(g_top)
        grad = _grad_rows(x, ld)
        _launch(x.device, "vqaf_token_logprobs_bwd", x.data_ptr(), ld, _addr(targets), _addr(ti), R, C, T, top,
                dtype_code(x), temperature, ctx.stats.data_ptr(), _addr(ent), _addr(g_lp), _addr(g_ent), _addr(g_top),
                grad.data_ptr(), _grad_pitch(x, ld))
        return grad, None, None


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top: int = 0, temperature: float = 1.0,
                   entropy: bool = True) -> TokenLogprobs:
    """Log probabilities of given tokens under softmax(logits / temperature), the entropy of that distribution and its
    `top` most probable tokens, from one read of the logits (vqaf_token_logprobs).

    logits (..., C) f32 or bf16.  targets (...) or (..., T) int64, at most 128 for each row: a negative one is none
    (log probability 0, no gradient), one past the classes gives NaN.  Results are f32 with the leading dimensions of
    `logits`; alternatives come in falling order, ties by the lowest index.  The log probabilities and the entropy are
    differentiable, once and in reverse mode.  Rows of nothing but -inf have log probabilities -inf, entropy 0 and no
    gradient; a NaN or +inf makes its row NaN."""
    x, ld = _answer_rows(logits)
    R, C = x.shape
    lead = logits.shape[:-1]
    temperature = _temperature(temperature)
    top = int(top)
    if not 0 <= top <= min(C, ANSWERS_MAX):
        raise ValueError(f"top has to be in [0, {min(C, ANSWERS_MAX)}], got {top}")
    T, tg = 0, None
    if targets is not None:
        given = targets.shape
        if given != lead and given[:-1] != lead:
            raise ValueError(f"targets of shape {tuple(given)} do not fit logits of shape {tuple(logits.shape)}")
        if targets.dtype is not torch.int64:
            targets = _token_indices(targets, "targets")
        if targets.device != logits.device:
            raise ValueError(f"targets are on {targets.device}, logits on {logits.device}")
        T = 1 if given == lead else given[-1]
        if T > ANSWERS_MAX:
            raise ValueError(f"at most {ANSWERS_MAX} targets for each row, got {T}")
        tg = targets.contiguous()
    if R == 0:
        z = x.sum(1, dtype=torch.float32).view(lead)
        lp = None if tg is None else (z if given == lead else z[..., None].expand(given)) * 1.0
        ent, tl = (z if entropy else None), (z[..., None].expand(*lead, top) * 1.0 if top else None)
        ti = torch.empty((*lead, top), dtype=torch.int64, device=x.device) if top else None
        return TokenLogprobs(lp, ent, tl, ti)
    call = (ld, lead, T, top, temperature, bool(entropy))
    if (x.requires_grad and torch.is_grad_enabled()) or _has_tangent(x):
        return TokenLogprobs(*_TokenLogprobs.apply(x, tg, call))
    return TokenLogprobs(*_logprobs_forward(x, tg, call, False)[:4])


def _distill_forward(x, ld, teacher, indices, temperature, tail, scale, needs):
    """(row losses, or their sum times `scale`; statistics; gradient of that sum).  The last two are None unless a
    backward needs them, the gradient also where there is no sum."""
    R, C = x.shape
    dev = x.device
    if scale is None:
        rows = torch.empty(R, dtype=torch.float32, device=dev)
        stats = torch.empty(5 * R, dtype=torch.float64, device=dev) if needs else None
        _launch(dev, "vqaf_distill", x.data_ptr(), ld, teacher.data_ptr(), indices.data_ptr(), R, C, teacher.shape[1],
                dtype_code(x), temperature, tail, rows.data_ptr(), _addr(stats), None, 0, 1.0, None)
        return rows, stats, None
    loss = torch.empty((), dtype=torch.float32, device=dev)
    room = torch.empty(6 * R if needs else R, dtype=torch.float64, device=dev)   # 5 R statistics, R row losses behind them
    at = room.data_ptr()
    grad = _grad_rows(x, ld) if needs else None
    _launch(dev, "vqaf_distill", x.data_ptr(), ld, teacher.data_ptr(), indices.data_ptr(), R, C, teacher.shape[1],
            dtype_code(x), temperature, tail, at + 40 * R if needs else at, at if needs else None, _addr(grad),
            _grad_pitch(x, ld), scale, loss.data_ptr())
    return loss, room, grad


class _Distill(torch.autograd.Function):
    """Row losses, or their sum / mean with the gradient for an incoming gradient of 1 formed in the same pass."""

    @staticmethod
    def forward(ctx, x, ld, teacher, indices, temperature, tail, scale):
        out, stats, ctx.unit = _distill_forward(x, ld, teacher, indices, temperature, tail, scale, True)
        ctx.recorded = torch.cuda.is_current_stream_capturing()
        ctx.save_for_backward(x, teacher, indices, stats)
        ctx.meta = (ld, temperature, scale)
        return out

    @staticmethod
    @_first_order
    def backward(ctx, up):
        grad, ctx.unit = ctx.unit, None   # handed out once: a second backward forms its own
        ready = grad is not None
        recording = torch.cuda.is_current_stream_capturing()
        if recording and not ctx.recorded:
            ready = False   # the graph replays without this forward: it forms the gradient itself every time
        if not ready or up is not _unit_grads.get((up.device, up.dtype)):
            x, teacher, indices, stats = ctx.saved_tensors   # (also tells of logits changed in place since)
            ld, temperature, scale = ctx.meta
            if not ready:
                grad = _grad_rows(x, ld)
            up = _f32(up)
            _launch(x.device, "vqaf_distill_bwd", x.data_ptr(), ld, teacher.data_ptr(), indices.data_ptr(), x.shape[0],
                    x.shape[1], teacher.shape[1], dtype_code(x), temperature, stats.data_ptr(), up.data_ptr(),
                    int(scale is None), int(ready and not recording), 1.0 if scale is None else scale, grad.data_ptr(), _grad_pitch(x, ld))
        return grad, None, None, None, None, None, None


def distill_loss(logits: torch.Tensor, teacher: torch.Tensor, indices: torch.Tensor, temperature: float = 1.0,
                 tail: bool = False, reduction: str = "mean") -> torch.Tensor:
    """temperature^2 * KL(teacher || softmax(logits / temperature)) over a teacher's top answers (vqaf_distill).

    logits (..., C) f32 or bf16; teacher (..., K) the teacher's log probabilities AT THIS TEMPERATURE of the answers
    `indices` (..., K) int64, K <= 128 -- top_logprobs and top_indices of `token_logprobs(teacher_logits, top=K,
    temperature=temperature)`.  tail=False divides them by their sum (any constant per row cancels); tail=True keeps
    them and takes the mass that they leave as one more event, met by all other classes together.  A negative index is
    no answer, and a row without answers has no loss and no gradient; an index past the classes makes its row NaN.
    reduction: "mean" over the rows, "sum", or "none" (f32, the leading dimensions of `logits`).  The teacher's side is
    constant.  `loss.backward(gradient=unit_gradient(loss))` hands on the gradient that the forward pass formed; any
    other incoming gradient forms it again, rounded once."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction has to be mean, sum or none, got {reduction!r}")
    x, ld = _answer_rows(logits)
    R, C = x.shape
    shape, dev = teacher.shape, logits.device
    lead, K = logits.shape[:-1], shape[-1] if shape else 0
    temperature = _temperature(temperature)
    if indices.shape != shape or len(shape) != len(lead) + 1 or shape[:-1] != lead:
        raise ValueError(f"teacher {tuple(shape)} and indices {tuple(indices.shape)} do not fit logits of shape "
                         f"{tuple(logits.shape)}")
    if not 1 <= K <= ANSWERS_MAX:
        raise ValueError(f"between 1 and {ANSWERS_MAX} answers for each row, got {K}")
    if not teacher.dtype.is_floating_point:
        raise TypeError(f"teacher holds log probabilities, got {teacher.dtype}")
    if indices.dtype is not torch.int64:
        indices = _token_indices(indices, "indices")
    if teacher.device != dev or indices.device != dev:
        raise ValueError(f"logits are on {dev}, teacher on {teacher.device}, indices on {indices.device}")
    if R == 0:
        rows = x.sum(1, dtype=torch.float32)
        return rows.view(lead) if reduction == "none" else rows.sum() if reduction == "sum" else rows.mean()
    v, idx = _f32(teacher.detach() if teacher.requires_grad else teacher), indices.contiguous()
    if len(lead) != 1:
        v, idx = v.reshape(R, K), idx.reshape(R, K)
    scale = 1.0 / R if reduction == "mean" else 1.0 if reduction == "sum" else None
    if (x.requires_grad and torch.is_grad_enabled()) or _has_tangent(x):
        out = _Distill.apply(x, ld, v, idx, temperature, int(bool(tail)), scale)
    else:
        out = _distill_forward(x, ld, v, idx, temperature, int(bool(tail)), scale, False)[0]
    return out.view(lead) if scale is None and len(lead) != 1 else out


def gemm_bf16_supported(lda: int, a_kmajor: bool, ldb: int, b_kmajor: bool, M: int, N: int, K: int) -> bool:
    return bool(load().vqaf_gemm_bf16_supported(lda, int(a_kmajor), ldb, int(b_kmajor), M, N, K))


@torch.no_grad()
def gemm_bf16(A: torch.Tensor, a_kmajor: bool, B: torch.Tensor, b_kmajor: bool, M: int, N: int, K: int,
              out: torch.Tensor, bias: Optional[torch.Tensor] = None, accumulate: bool = False,
              colsum: Optional[torch.Tensor] = None, name: Optional[str] = None) -> torch.Tensor:
    """out (M,N) = op(A) op(B) (+ bias) on bf16 MFMA (vqaf_gemm_bf16); A, B are 2-D bf16 tensors whose
    second stride is 1 (row pitch = first stride), out f32 or bf16."""
    assert A.dtype == torch.bfloat16 and B.dtype == torch.bfloat16 and A.stride(1) == 1 and B.stride(1) == 1
    assert out.stride(1) == 1
    if name is not None:
        _probe(name, "begin")
    check(load().vqaf_gemm_bf16(A.data_ptr(), A.stride(0), int(a_kmajor), B.data_ptr(), B.stride(0), int(b_kmajor),
                                M, N, K, ptr(bias), dtype_code(bias) if bias is not None else 0, out.data_ptr(),
                                out.stride(0), dtype_code(out), int(accumulate), ptr(colsum),
                                stream_ptr(A.device)), "vqaf_gemm_bf16")
    if name is not None:
        _probe(name, "end")
    return out


@torch.no_grad()
def gemm_bf16_wgrad_group(items, K: int, accumulate: bool = False, name: Optional[str] = None) -> bool:
    """items: list of (A (K,M) bf16, B (K,N) bf16, C (M,N) f32 view, colsum (M) f32 or None).  Launches all
    C_i = A_i^T B_i in one kernel (vqaf_gemm_bf16_wgrad_group); returns False, having launched nothing, when
    the products cannot share a launch (the caller then issues them one by one)."""
    import ctypes
    n = len(items)
    if not 1 <= n <= 4:
        return False
    for A, B, Cm, cs in items:
        assert A.dtype == torch.bfloat16 and B.dtype == torch.bfloat16 and Cm.dtype == torch.float32
        assert A.stride(1) == 1 and B.stride(1) == 1 and Cm.stride(1) == 1 and A.shape[0] == K and B.shape[0] == K
    vp, lg, it = ctypes.c_void_p * n, ctypes.c_long * n, ctypes.c_int * n
    has_cs = any(cs is not None for _, _, _, cs in items)
    if name is not None:
        _probe(name, "begin")
    status = load().vqaf_gemm_bf16_wgrad_group(
        n, vp(*[A.data_ptr() for A, _, _, _ in items]), lg(*[A.stride(0) for A, _, _, _ in items]),
        vp(*[B.data_ptr() for _, B, _, _ in items]), lg(*[B.stride(0) for _, B, _, _ in items]),
        it(*[A.shape[1] for A, _, _, _ in items]), it(*[B.shape[1] for _, B, _, _ in items]), K,
        vp(*[Cm.data_ptr() for _, _, Cm, _ in items]), lg(*[Cm.stride(0) for _, _, Cm, _ in items]), int(accumulate),
        vp(*[None if cs is None else cs.data_ptr() for _, _, _, cs in items]) if has_cs else None,
        stream_ptr(items[0][0].device))
    if name is not None:
        _probe(name, "end")
    if status == -1:  # VQAF_E_SHAPE: not groupable
        return False
    check(status, "vqaf_gemm_bf16_wgrad_group")
    return True


def linear_nt_supported(x2: torch.Tensor, w: torch.Tensor, w_kmajor: bool = False) -> bool:
    """Whether y = x2 op(w) can run on vqaf_linear_nt: x2 (M,K); w (N,K), or (K,N) with w_kmajor; both bf16 with
    unit inner stride."""
    for t in (x2, w):
        if t.dtype != torch.bfloat16 or t.dim() != 2 or t.stride(1) != 1 or t.data_ptr() % 16:
            return False
    M, K = x2.shape
    N = w.shape[1] if w_kmajor else w.shape[0]
    if (w.shape[0] if w_kmajor else w.shape[1]) != K:
        return False
    return bool(load().vqaf_linear_nt_supported(x2.stride(0), w.stride(0), int(w_kmajor), N, M, N, K))


@torch.no_grad()
def linear_nt(x2: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, w_kmajor: bool = False,
              epilogue: int = 0, aux: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y (M,N) bf16 = x2 (M,K) op(w) (+ bias) on the library's large-tile bf16 MFMA kernel (vqaf_linear_nt).
    epilogue 1: aux (M,N), allocated by the caller, receives gelu(y); epilogue 2: y = (x2 op(w)) * gelu'(aux)."""
    M, K = x2.shape
    N = w.shape[1] if w_kmajor else w.shape[0]
    y = torch.empty(M, N, dtype=torch.bfloat16, device=x2.device)
    check(load().vqaf_linear_nt(x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0), int(w_kmajor), ptr(bias),
                                dtype_code(bias) if bias is not None else 0, M, N, K, y.data_ptr(), N, epilogue,
                                ptr(aux), aux.stride(0) if aux is not None else 0, stream_ptr(x2.device)),
          "vqaf_linear_nt")
    return y


def wgrad_tn_supported(gy2: torch.Tensor, x2: torch.Tensor) -> bool:
    if gy2.dtype != torch.bfloat16 or x2.dtype != torch.bfloat16 or gy2.stride(1) != 1 or x2.stride(1) != 1:
        return False
    if gy2.data_ptr() % 16 or x2.data_ptr() % 16 or gy2.shape[0] != x2.shape[0]:
        return False
    K, M = gy2.shape
    N = x2.shape[1]
    return bool(load().vqaf_wgrad_tn_supported(gy2.stride(0), x2.stride(0), N, M, N, K))


@torch.no_grad()
def wgrad_tn(gy2: torch.Tensor, x2: torch.Tensor, w_dtype: torch.dtype = torch.bfloat16,
             bias_dtype: Optional[torch.dtype] = torch.bfloat16):
    """(gy2^T x2 (M,N) `w_dtype`, column sums of gy2 (M) `bias_dtype` or None) for gy2 (K,M), x2 (K,N) bf16:
    weight and bias gradient of a Linear whose batch has K tokens (vqaf_wgrad_tn)."""
    K, M = gy2.shape
    N = x2.shape[1]
    lib = load()
    gw = torch.empty(M, N, dtype=w_dtype, device=gy2.device)
    gb = torch.empty(M, dtype=bias_dtype, device=gy2.device) if bias_dtype is not None else None
    ws = torch.empty(lib.vqaf_wgrad_tn_workspace_bytes(M, N, K), dtype=torch.uint8, device=gy2.device)
    check(lib.vqaf_wgrad_tn(gy2.data_ptr(), gy2.stride(0), x2.data_ptr(), x2.stride(0), M, N, K, gw.data_ptr(), N,
                            dtype_code(gw), ptr(gb), dtype_code(gb) if gb is not None else 0, ws.data_ptr(),
                            ws.numel(), stream_ptr(gy2.device)), "vqaf_wgrad_tn")
    return gw, gb


# --------------------------------------------------------------------------------------------
# Linear layers in eight-bit integers
# --------------------------------------------------------------------------------------------
INT8_MAX_K = 131072  # the integer sum stays inside 32 bits


def _int8_rows(x: torch.Tensor, what: str):
    require_gpu(x)
    dtype_code(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what} needs a last dimension, got shape {tuple(x.shape)}")
    if x.shape[-1] > INT8_MAX_K or x.numel() // x.shape[-1] >= 2 ** 31:
        raise ValueError(f"{what}: at most 2^31 - 1 rows of {INT8_MAX_K} columns, got {tuple(x.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.shape[1] > 1 and x2.stride(1) != 1:
        x2 = x2.contiguous()
    return x2, (x2.stride(0) if x2.shape[0] > 1 else x2.shape[1])


@torch.no_grad()
def quantize_rows(x: torch.Tensor):
    """(q (..., K) int8, scale (...) f32) with q = x / scale rounded half to even and scale = max|row| / 127
    (vqaf_quantize_rows): a Linear layer's weight (out, in), one scale for each output channel, as `int8_linear` takes
    it.  q is laid out in rows of whole 128-byte pieces."""
    x2, ld = _int8_rows(x, "quantize_rows")
    M, K = x2.shape
    pitch = (K + 127) // 128 * 128
    q = torch.empty(M, pitch, dtype=torch.int8, device=x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    if M:
        _launch(x.device, "vqaf_quantize_rows", x2.data_ptr(), ld, M, K, dtype_code(x2), q.data_ptr(), pitch,
                scale.data_ptr())
    lead = x.shape[:-1]
    return (q[:, :K] if len(lead) == 1 else q.view(*lead, pitch)[..., :K]), scale.view(lead)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x (..., K) f32 or bf16 through a Linear layer held in eight-bit integers: weight (N,K) int8 and weight_scale (N)
    f32 from `quantize_rows`, bias (N) f32 or bf16 or None; the tokens are quantised row by row on the way in
    (vqaf_int8_linear).  Returns (..., N) in out_dtype (default: x's).  Weights in rows that are not whole 16-byte
    pieces are copied into such rows first.  There is no gradient: an input that requires one is refused while
    gradients are recorded, and one with a forward-mode tangent always."""
    if ((x.requires_grad or weight_scale.requires_grad or (bias is not None and bias.requires_grad)) and
            torch.is_grad_enabled()) or _has_tangent(x, weight_scale, bias):
        raise RuntimeError("int8_linear has no gradient: call it under torch.no_grad(), or train the layer in bf16")
    x2, ld = _int8_rows(x, "int8_linear")
    if weight.dim() != 2 or weight.dtype != torch.int8:
        raise TypeError(f"weight has to be (N,K) int8, got {tuple(weight.shape)} {weight.dtype}")
    N, K = weight.shape
    M = x2.shape[0]
    if x2.shape[1] != K or not 1 <= N <= 2 ** 27:
        raise ValueError(f"x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    if weight_scale.shape != (N,) or weight_scale.dtype != torch.float32:
        raise ValueError(f"weight_scale has to be ({N},) float32, got {tuple(weight_scale.shape)} {weight_scale.dtype}")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"bias has to be ({N},), got {tuple(bias.shape)}")
    if weight.device != x.device or weight_scale.device != x.device or (bias is not None and bias.device != x.device):
        raise ValueError(f"x is on {x.device}, weight on {weight.device}, weight_scale on {weight_scale.device}"
                         + ("" if bias is None else f", bias on {bias.device}"))
    dt = out_dtype or x.dtype
    code = _lib.BF16 if dt == torch.bfloat16 else _lib.F32
    if dt not in (torch.float32, torch.bfloat16):
        raise TypeError(f"out_dtype has to be float32 or bfloat16, got {dt}")
    weight_scale = weight_scale.contiguous()   # (a copy has to outlive the launch)
    if bias is not None:
        dtype_code(bias)
        bias = bias.contiguous()
    ldw = weight.stride(0) if N > 1 else (K + 15) // 16 * 16
    fits = weight.stride(1) == 1 or K == 1
    if N == 1 and fits:   # one row: its pitch says nothing, its last piece has to be there
        fits = weight.storage_offset() + ldw <= weight.untyped_storage().nbytes()
    elif fits:
        fits = ldw % 16 == 0 and ldw >= K and weight.storage_offset() + (N - 1) * ldw + (K + 15) // 16 * 16 <= \
            weight.untyped_storage().nbytes()
    if not fits or weight.data_ptr() % 16:
        whole = torch.zeros(N, (K + 15) // 16 * 16, dtype=torch.int8, device=x.device)
        whole[:, :K] = weight
        weight, ldw = whole, whole.shape[1]
    y = torch.empty(M, N, dtype=dt, device=x.device)
    if M:
        need = load().vqaf_int8_linear_workspace_bytes(M, K)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        _launch(x.device, "vqaf_int8_linear", x2.data_ptr(), ld, dtype_code(x2), weight.data_ptr(), ldw,
                weight_scale.data_ptr(), _addr(bias), dtype_code(bias) if bias is not None else 0, M, N, K,
                y.data_ptr(), N, code, _addr(ws), need)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


def keep_count(n_tokens: int, prune_ratio: float) -> int:
    """k = max(1, int(N * (1 - prune_ratio))) in Python double arithmetic (utils/fusion.py:41)."""
    return max(1, int(n_tokens * (1 - prune_ratio)))


def adv_count(k: int, adv_ratio: float) -> int:
    """k_adv = max(1, int(k * adv_ratio)) (utils/fusion.py:54)."""
    return max(1, int(k * adv_ratio))
