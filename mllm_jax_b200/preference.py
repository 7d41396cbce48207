"""Preference loss over paired log ratios (DPO-style), beside the token losses of `ops`.

Sequences 0..P-1 of a batch are the chosen answers and sequence P + p is the rejected answer of pair p:

    lp_s = sum_t mask_st * lp_st          (averaged over the valid tokens with cfg.average)
    h_p  = (lp_p - ref_p) - (lp_(P+p) - ref_(P+p))
    "sigmoid"  -(1-e) log sigmoid(beta h) - e log sigmoid(-beta h)      e = label_smoothing
    "hinge"    max(0, 1 - beta h)
    "ipo"      (h - 1/(2 beta))^2
    loss = sum_p pair_weights_p * l_p / total_pairs

Rows and masks mean what they mean in `grpo_token_loss`; log-probs of a frozen reference model come from
`token_logprobs` or `linear_loss.lm_head_forward` (whose head may be held in 8 bits).  Positions whose mask is 0 are
neither read nor allowed to matter, whatever they hold.  The kernels run on the current stream; every call has a
workspace of its own, so calls on several streams and captured graphs do not share state.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_KINDS = {"sigmoid": 0, "hinge": 1, "ipo": 2}


@dataclass
class PreferenceConfig:
    """Attributes of the paired loss."""

    beta: float = 0.1
    loss_type: str = "sigmoid"      # "sigmoid", "hinge" or "ipo"
    label_smoothing: float = 0.0    # sigmoid only, in [0, 0.5]
    average: bool = False           # length-normalised log-probs
    softcap: Optional[float] = None


def _f32(t: Optional[torch.Tensor], dev, shapes, name: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if tuple(t.shape) not in shapes:
        raise ValueError(f"{name} must have shape {' or '.join(str(s) for s in shapes)}, got {tuple(t.shape)}")
    return t.to(device=dev, dtype=torch.float32).contiguous()


class PreferenceProblem:
    """Device buffers of one call, laid out as the C ABI wants them; keeps references so that they outlive the launch."""

    def __init__(self, sequences: int, T: int, dev, mask, ref, pair_weights, total_pairs, cfg: PreferenceConfig):
        if sequences < 2 or sequences % 2:
            raise ValueError(f"the batch holds chosen and rejected answers of pairs: {sequences} sequences is not a "
                             "positive even number")
        if T < 1:
            raise ValueError("there is no scored position")
        if cfg.loss_type not in _KINDS:
            raise ValueError(f"loss_type must be one of {sorted(_KINDS)}, got {cfg.loss_type!r}")
        if not cfg.beta > 0:
            raise ValueError(f"beta must be positive, got {cfg.beta}")
        if not 0 <= cfg.label_smoothing <= 0.5 or (cfg.label_smoothing and cfg.loss_type != "sigmoid"):
            raise ValueError("label_smoothing must lie in [0, 0.5] and belongs to the sigmoid loss")
        self.P, self.T, self.dev, self.cfg = sequences // 2, T, dev, cfg
        B = sequences
        self.mask = _f32(mask, dev, [(B, T)], "mask")
        self.ref = _f32(ref, dev, [(B, T), (B,)], "ref_per_token_logps")
        self.weights = _f32(pair_weights, dev, [(self.P,)], "pair_weights")
        self.total_dev = None
        self.total = float(self.P)
        if isinstance(total_pairs, torch.Tensor):
            self.total_dev = total_pairs.to(device=dev, dtype=torch.float32).reshape(1)
        elif total_pairs is not None:
            self.total = float(total_pairs)
        lib = _lib.load()
        nbytes = int(lib.mllm_grpo_preference_workspace_bytes(self.P, T))
        if nbytes == 0:
            raise ValueError(f"{B} x {T} scored positions are too many for one call")
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        out = torch.empty(1 + 4 * self.P, dtype=torch.float32, device=dev)
        self.loss, self.rewards, self.sequence_logps = out[0], out[1:1 + B], out[1 + B:]
        self.device_status = None
        self.grad_scale = 1.0
        a = self.a = _lib.PreferenceArgs()
        a.n_pairs, a.seq_rows, a.scored_rows = self.P, T, T
        a.kind, a.average = _KINDS[cfg.loss_type], int(cfg.average)
        a.beta, a.label_smoothing = cfg.beta, cfg.label_smoothing
        a.softcap = float(cfg.softcap) if cfg.softcap else 0.0
        a.grad_scale, a.total_pairs = 1.0, self.total
        a.mask = None if self.mask is None else self.mask.data_ptr()
        a.ref_logps = None if self.ref is None else self.ref.data_ptr()
        a.ref_per_sequence = int(self.ref is not None and self.ref.dim() == 1)
        a.pair_weights = None if self.weights is None else self.weights.data_ptr()
        a.total_pairs_dev = None if self.total_dev is None else self.total_dev.data_ptr()
        a.loss, a.rewards = out.data_ptr(), self.rewards.data_ptr()
        a.sequence_logps, a.workspace = self.sequence_logps.data_ptr(), self.workspace.data_ptr()

    def bind_logits(self, logits: torch.Tensor, ids: torch.Tensor, L: int) -> None:
        self.logits = logits
        if tuple(ids.shape) != (2 * self.P, self.T):
            raise ValueError(f"token ids must have {2 * self.P}x{self.T} elements, got shape {tuple(ids.shape)}")
        self.ids = ids.to(device=self.dev, dtype=torch.int32).contiguous()
        self.device_status = torch.zeros(1, dtype=torch.int32, device=self.dev)
        a = self.a
        a.seq_rows, a.vocab, a.row_stride = L, logits.shape[2], logits.stride(1)
        a.logits, a.chosen_ids, a.device_status = logits.data_ptr(), self.ids.data_ptr(), self.device_status.data_ptr()

    def bind_dlogits(self, dlogits: torch.Tensor) -> torch.Tensor:
        x = self.logits
        if dlogits.shape != x.shape or dlogits.stride() != x.stride() or dlogits.dtype != x.dtype or \
                dlogits.device != x.device:
            raise ValueError("dlogits must match logits in shape, strides, dtype and device")
        self.dlogits = dlogits
        self.a.dlogits = dlogits.data_ptr()
        return dlogits

    def run(self, entry: str) -> None:
        _lib.launch(entry, self.a, self.dev)

    def outputs(self) -> dict:
        P = self.P
        return {"loss": self.loss, "chosen_rewards": self.rewards[:P], "rejected_rewards": self.rewards[P:],
                "chosen_logps": self.sequence_logps[:P], "rejected_logps": self.sequence_logps[P:]}


def _from_logits(logits, token_ids, mask, ref, shifted, cfg, pair_weights, total_pairs) -> PreferenceProblem:
    if not logits.is_cuda:
        raise RuntimeError("the preference loss kernels run on a CUDA device only (no CPU path)")
    if logits.dtype != torch.bfloat16:
        raise TypeError(f"logits must be bfloat16, got {logits.dtype}")
    if logits.dim() != 3:
        raise ValueError(f"logits must be [2P, L, V], got shape {tuple(logits.shape)}")
    B, L, V = logits.shape
    if V < 1 or logits.stride(2) != 1 or logits.stride(1) < V or logits.stride(0) != L * logits.stride(1):
        raise ValueError("logits must have unit stride on the vocabulary and rows evenly spaced")
    if shifted:
        token_ids, mask = token_ids[:, 1:], None if mask is None else mask[:, 1:]
    T = L - 1 if shifted else L
    prob = PreferenceProblem(B, T, logits.device, mask, ref, pair_weights, total_pairs, cfg or PreferenceConfig())
    prob.bind_logits(logits, token_ids, L)
    return prob


def preference_value_and_grad(logits: torch.Tensor, token_ids: torch.Tensor, mask: Optional[torch.Tensor],
                              ref_per_token_logps: Optional[torch.Tensor] = None, *, shifted: bool = False,
                              cfg: Optional[PreferenceConfig] = None, pair_weights: Optional[torch.Tensor] = None,
                              total_pairs=None, grad_scale: float = 1.0, inplace: bool = False,
                              dlogits: Optional[torch.Tensor] = None) -> dict:
    """Loss, rewards and dlogits in one call (three launches).

    logits [2P, L, V] bf16.  shifted=True takes the reference layout (token_ids = input_ids [2P, L], mask = labels
    [2P, L]; row i is scored against token i + 1, the last row gets a zero gradient); shifted=False takes aligned
    [2P, L] arrays.  mask is a weight per token (0 = not part of the answer).  ref_per_token_logps: [2P, T] log-probs
    of the reference policy, [2P] sequence log-probs of it, or None (reference-free).  pair_weights [P]: 0 takes a
    padded pair out of the batch.  total_pairs: the loss's normaliser (number or scalar tensor, default P).
    Returns loss, chosen_rewards / rejected_rewards [P] (beta times the log ratio), chosen_logps / rejected_logps
    [P], dlogits and the problem (whose device_status has MLLM_GRPO_DEV_ID_CLAMPED for ids outside the vocabulary)."""
    prob = _from_logits(logits, token_ids, mask, ref_per_token_logps, shifted, cfg, pair_weights, total_pairs)
    prob.a.grad_scale = float(grad_scale)
    if dlogits is None:
        dlogits = logits if inplace else torch.empty_strided(logits.shape, logits.stride(), dtype=logits.dtype,
                                                             device=logits.device)
    prob.bind_dlogits(dlogits)
    prob.run("mllm_grpo_preference_fwd_bwd")
    out = prob.outputs()
    out["dlogits"], out["problem"] = dlogits, prob
    return out


class _PreferenceLoss(torch.autograd.Function):
    """Forward keeps (log-sum-exps, pair coefficients) in the call's workspace; backward streams the logits again."""

    @staticmethod
    def forward(ctx, logits, prob: PreferenceProblem, inplace_backward: bool):
        prob.run("mllm_grpo_preference_fwd")
        ctx.prob, ctx.inplace, ctx.spent = prob, inplace_backward, False
        ctx.save_for_backward(logits)  # a change of the logits between the sweeps is an error
        ctx.mark_non_differentiable(prob.rewards, prob.sequence_logps)
        return prob.loss.clone(), prob.rewards, prob.sequence_logps

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _g_rewards, _g_logps):
        prob: PreferenceProblem = ctx.prob
        (logits,) = ctx.saved_tensors
        if ctx.spent:
            raise RuntimeError("the first backward has overwritten the logits (inplace_backward=True)")
        ctx.spent = ctx.inplace
        scale = grad_loss.to(torch.float32).reshape(1).contiguous()
        prob.a.grad_scale_dev = scale.data_ptr()
        prob.bind_dlogits(logits if ctx.inplace else torch.empty_strided(
            logits.shape, logits.stride(), dtype=logits.dtype, device=logits.device))
        prob.run("mllm_grpo_preference_bwd")
        return prob.dlogits, None, None


def preference_loss(logits: torch.Tensor, input_ids: torch.Tensor, labels: Optional[torch.Tensor],
                    ref_per_token_logps: Optional[torch.Tensor] = None, *, cfg: Optional[PreferenceConfig] = None,
                    pair_weights: Optional[torch.Tensor] = None, total_pairs=None,
                    inplace_backward: bool = False) -> dict:
    """Preference loss on the reference layout, differentiable with respect to the logits: logits [2P, L, V] bf16,
    input_ids / labels [2P, L], reference log-probs [2P, L-1], [2P] or None (see `preference_value_and_grad`).
    Only `loss` is differentiable; rewards and log-probs are detached."""
    prob = _from_logits(logits.detach(), input_ids, labels, ref_per_token_logps, True, cfg, pair_weights, total_pairs)
    P = prob.P
    loss, rewards, lps = _PreferenceLoss.apply(logits, prob, inplace_backward)
    return {"loss": loss, "chosen_rewards": rewards[:P], "rejected_rewards": rewards[P:], "chosen_logps": lps[:P],
            "rejected_logps": lps[P:]}


def preference_logps_value_and_grad(per_token_logps: torch.Tensor, mask: Optional[torch.Tensor],
                                    ref_per_token_logps: Optional[torch.Tensor] = None, *,
                                    cfg: Optional[PreferenceConfig] = None,
                                    pair_weights: Optional[torch.Tensor] = None, total_pairs=None,
                                    grad_scale: float = 1.0) -> dict:
    """The same loss from per-token log-probs [2P, T] (any floating type, read in f32) with `dlogps` [2P, T] f32, its
    gradient with respect to them; exact zeros where the mask is 0.  cfg.softcap has no meaning here."""
    x = per_token_logps
    if not x.is_cuda:
        raise RuntimeError("the preference loss kernels run on a CUDA device only (no CPU path)")
    if x.dim() != 2:
        raise ValueError(f"per_token_logps must be [2P, T], got shape {tuple(x.shape)}")
    prob = PreferenceProblem(x.shape[0], x.shape[1], x.device, mask, ref_per_token_logps, pair_weights, total_pairs,
                             cfg or PreferenceConfig())
    prob.logps = x.detach().to(torch.float32).contiguous()
    dlogps = torch.empty_like(prob.logps)
    prob.a.token_logps, prob.a.dtoken_logps = prob.logps.data_ptr(), dlogps.data_ptr()
    prob.a.grad_scale = float(grad_scale)
    prob.run("mllm_grpo_preference_logps")
    out = prob.outputs()
    out["dlogps"], out["problem"] = dlogps, prob
    return out


class _PreferenceLogpsLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, mask, ref, kwargs):
        out = preference_logps_value_and_grad(logps, mask, ref, **kwargs)
        prob = out["problem"]
        ctx.save_for_backward(out["dlogps"])
        ctx.dtype = logps.dtype
        ctx.mark_non_differentiable(prob.rewards, prob.sequence_logps)
        return prob.loss.clone(), prob.rewards, prob.sequence_logps

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _g_rewards, _g_logps):
        (d,) = ctx.saved_tensors
        return (grad_loss * d).to(ctx.dtype), None, None, None


def preference_loss_from_logps(per_token_logps: torch.Tensor, mask: Optional[torch.Tensor],
                               ref_per_token_logps: Optional[torch.Tensor] = None, *,
                               cfg: Optional[PreferenceConfig] = None, pair_weights: Optional[torch.Tensor] = None,
                               total_pairs=None) -> dict:
    """`preference_logps_value_and_grad` as a differentiable function of the log-probs (the gradient is formed with
    the loss; backward applies the cotangent)."""
    P = per_token_logps.shape[0] // 2
    loss, rewards, lps = _PreferenceLogpsLoss.apply(per_token_logps, mask, ref_per_token_logps,
                                                    dict(cfg=cfg, pair_weights=pair_weights, total_pairs=total_pairs))
    return {"loss": loss, "chosen_rewards": rewards[:P], "rejected_rewards": rewards[P:], "chosen_logps": lps[:P],
            "rejected_logps": lps[P:]}
