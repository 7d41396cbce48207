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
    if t.shape not in shapes:
        raise ValueError(f"{name} must have shape {' or '.join(str(tuple(s)) for s in shapes)}, got {tuple(t.shape)}")
    if t.dtype is torch.float32 and t.device == dev and t.is_contiguous():
        return t
    return t.to(device=dev, dtype=torch.float32).contiguous()


def _rows(t: torch.Tensor, dev, dtypes) -> torch.Tensor:
    """A [B, T] tensor of one of `dtypes` whose rows are contiguous and any distance apart (a view where possible)."""
    if t.dtype not in dtypes or t.device != dev:
        t = t.to(device=dev, dtype=dtypes[0])
    B, T = t.shape
    if (T > 1 and t.stride(1) != 1) or (B > 1 and t.stride(0) < T):
        t = t.contiguous()
    return t


class PreferenceProblem:
    """Device buffers of one call, laid out as the C ABI wants them; keeps references so that they outlive the launch."""

    def __init__(self, sequences: int, T: int, dev, mask, ref, pair_weights, total_pairs, cfg: PreferenceConfig):
        B, P = sequences, sequences // 2
        if B < 2 or B % 2:
            raise ValueError(f"the batch holds chosen and rejected answers of pairs: {B} sequences is not a "
                             "positive even number")
        if T < 1:
            raise ValueError("there is no scored position")
        kind = _KINDS.get(cfg.loss_type)
        if kind is None:
            raise ValueError(f"loss_type must be one of {sorted(_KINDS)}, got {cfg.loss_type!r}")
        if not cfg.beta > 0:
            raise ValueError(f"beta must be positive, got {cfg.beta}")
        if not 0 <= cfg.label_smoothing <= 0.5 or (cfg.label_smoothing and kind != 0):
            raise ValueError("label_smoothing must lie in [0, 0.5] and belongs to the sigmoid loss")
        self.P, self.T, self.dev, self.cfg = P, T, dev, cfg
        self.mask = None
        if mask is not None:
            if mask.shape != (B, T):
                raise ValueError(f"mask must have shape {(B, T)}, got {tuple(mask.shape)}")
            self.mask = _rows(mask, dev, (torch.float32, torch.int32))
        self.ref = _f32(ref, dev, ((B, T), (B,)), "ref_per_token_logps")
        self.weights = _f32(pair_weights, dev, ((P,),), "pair_weights")
        self.total_dev = None
        self.total = float(P)
        if isinstance(total_pairs, torch.Tensor):
            self.total_dev = total_pairs.to(device=dev, dtype=torch.float32).reshape(1)
        elif total_pairs is not None:
            self.total = float(total_pairs)
        nbytes = _lib.load().mllm_grpo_preference_workspace_bytes(P, T)
        if nbytes == 0:
            raise ValueError(f"{B} x {T} scored positions are too many for one call")
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        self.out = torch.empty(2 + 4 * P, dtype=torch.float32, device=dev)  # rewards, log-probs, loss, status
        o = self.out.data_ptr()
        self.a = _lib.PreferenceArgs(
            n_pairs=P, seq_rows=T, scored_rows=T, kind=kind, average=bool(cfg.average), beta=cfg.beta,
            label_smoothing=cfg.label_smoothing, softcap=float(cfg.softcap) if cfg.softcap else 0.0, grad_scale=1.0,
            total_pairs=self.total, rewards=o, sequence_logps=o + 4 * B, loss=o + 8 * B, call_status=o + 8 * B + 4,
            workspace=self.workspace.data_ptr())
        a = self.a
        if self.mask is not None:
            a.mask, a.mask_int = self.mask.data_ptr(), self.mask.dtype is torch.int32
            a.mask_stride = self.mask.stride(0) if B > 1 else 0
        if self.ref is not None:
            a.ref_logps, a.ref_per_sequence = self.ref.data_ptr(), self.ref.dim() == 1
        if self.weights is not None:
            a.pair_weights = self.weights.data_ptr()
        if self.total_dev is not None:
            a.total_pairs_dev = self.total_dev.data_ptr()

    @property
    def device_status(self) -> torch.Tensor:
        """MLLM_GRPO_DEV_* bits of the forward (an int32 on the device; nothing raises one from log-probs)."""
        return self.out[-1:].view(torch.int32)

    def bind_logits(self, logits: torch.Tensor, ids: torch.Tensor, L: int, row_stride: int) -> None:
        self.logits = logits
        if ids.shape != (2 * self.P, self.T):
            raise ValueError(f"token ids must have {2 * self.P}x{self.T} elements, got shape {tuple(ids.shape)}")
        if ids.dtype is torch.int64:
            ids = ids.clamp(-1, 2 ** 31 - 1)  # an id beyond 32 bits must not wrap to a valid one
        self.ids = _rows(ids, self.dev, (torch.int32,))
        a = self.a
        a.seq_rows, a.vocab, a.row_stride = L, logits.shape[2], row_stride
        a.logits, a.chosen_ids, a.ids_stride = logits.data_ptr(), self.ids.data_ptr(), self.ids.stride(0)

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
        good, bad, good_lp, bad_lp, _ = self.out.split_with_sizes((P, P, P, P, 2))
        return {"loss": self.out.select(0, -2), "chosen_rewards": good, "rejected_rewards": bad, "chosen_logps": good_lp,
                "rejected_logps": bad_lp}


def _shifted(t: torch.Tensor, B: int, L: int, name: str) -> torch.Tensor:
    if t.shape != (B, L):
        raise ValueError(f"{name} must have shape {(B, L)}, got {tuple(t.shape)}")
    return t.narrow(1, 1, L - 1) if L > 1 else t[:, 1:]


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device)


def _from_logits(logits, token_ids, mask, ref, shifted, cfg, pair_weights, total_pairs) -> PreferenceProblem:
    if not logits.is_cuda:
        raise RuntimeError("the preference loss kernels run on a CUDA device only (no CPU path)")
    if logits.dtype != torch.bfloat16:
        raise TypeError(f"logits must be bfloat16, got {logits.dtype}")
    if logits.dim() != 3:
        raise ValueError(f"logits must be [2P, L, V], got shape {tuple(logits.shape)}")
    B, L, V = logits.shape
    row = logits.stride(0) if L == 1 else logits.stride(1)
    if V < 1 or (V > 1 and logits.stride(2) != 1) or row < V or logits.stride(0) != L * row:
        raise ValueError("logits must have unit stride on the vocabulary and rows evenly spaced")
    if shifted:
        token_ids, mask = _shifted(token_ids, B, L, "token ids"), None if mask is None else _shifted(mask, B, L, "mask")
    T = L - 1 if shifted else L
    prob = PreferenceProblem(B, T, logits.device, mask, ref, pair_weights, total_pairs, cfg or PreferenceConfig())
    prob.bind_logits(logits, token_ids, L, row)
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
    given = inplace or dlogits is not None
    if dlogits is None:
        dlogits = logits if inplace else _like(logits)
    prob.bind_dlogits(dlogits)
    prob.run("mllm_grpo_preference_fwd_bwd")
    if given:
        _lib.written(dlogits)
    out = prob.outputs()
    out["dlogits"], out["problem"] = dlogits, prob
    return out


class _PreferenceLoss(torch.autograd.Function):
    """Forward keeps (log-sum-exps, pair coefficients) in the call's workspace; backward streams the logits again."""

    @staticmethod
    def forward(ctx, logits, prob: PreferenceProblem, inplace_backward: bool):
        prob.run("mllm_grpo_preference_fwd")
        ctx.prob, ctx.inplace, ctx.spent = prob, inplace_backward, False
        # a change of what the backward reads again, between the sweeps, is an error
        ctx.save_for_backward(logits, prob.ids, *(() if prob.mask is None else (prob.mask,)))
        return prob.out.select(0, -2).clone()

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        prob: PreferenceProblem = ctx.prob
        if ctx.spent:
            raise RuntimeError("the first backward has overwritten the logits (inplace_backward=True)")
        _lib.no_tangent(grad_loss, "the loss's cotangent")
        ctx.spent = ctx.inplace
        logits = ctx.saved_tensors[0]
        scale = grad_loss.to(torch.float32).reshape(1).contiguous()
        prob.a.grad_scale_dev = scale.data_ptr()
        prob.bind_dlogits(logits if ctx.inplace else _like(logits))
        prob.run("mllm_grpo_preference_bwd")
        if ctx.inplace:
            _lib.written(logits)  # another backward that needs what they held is an error
        return prob.dlogits, None, None


def preference_loss(logits: torch.Tensor, input_ids: torch.Tensor, labels: Optional[torch.Tensor],
                    ref_per_token_logps: Optional[torch.Tensor] = None, *, cfg: Optional[PreferenceConfig] = None,
                    pair_weights: Optional[torch.Tensor] = None, total_pairs=None,
                    inplace_backward: bool = False) -> dict:
    """Preference loss on the reference layout, differentiable with respect to the logits: logits [2P, L, V] bf16,
    input_ids / labels [2P, L], reference log-probs [2P, L-1], [2P] or None (see `preference_value_and_grad`).
    Only `loss` is differentiable; rewards and log-probs are detached."""
    prob = _from_logits(logits.detach(), input_ids, labels, ref_per_token_logps, True, cfg, pair_weights, total_pairs)
    loss = _PreferenceLoss.apply(logits, prob, inplace_backward)
    return {**prob.outputs(), "loss": loss, "problem": prob}


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
    prob.logps = _f32(x.detach() if x.requires_grad else x, x.device, (x.shape,), "per_token_logps")
    dlogps = torch.empty_like(prob.logps)
    prob.a.token_logps, prob.a.dtoken_logps = prob.logps.data_ptr(), dlogps.data_ptr()
    prob.a.grad_scale = float(grad_scale)
    prob.run("mllm_grpo_preference_logps")
    out = prob.outputs()
    out["dlogps"], out["problem"] = dlogps, prob
    return out


class _PreferenceLogpsLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, out):
        ctx.save_for_backward(out["dlogps"])
        ctx.dtype = logps.dtype
        return out["loss"].clone()

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        (d,) = ctx.saved_tensors
        return (grad_loss * d).to(ctx.dtype), None


def preference_loss_from_logps(per_token_logps: torch.Tensor, mask: Optional[torch.Tensor],
                               ref_per_token_logps: Optional[torch.Tensor] = None, *,
                               cfg: Optional[PreferenceConfig] = None, pair_weights: Optional[torch.Tensor] = None,
                               total_pairs=None) -> dict:
    """`preference_logps_value_and_grad` as a differentiable function of the log-probs (the gradient is formed with
    the loss; backward applies the cotangent)."""
    out = preference_logps_value_and_grad(per_token_logps, mask, ref_per_token_logps, cfg=cfg, pair_weights=pair_weights,
                                          total_pairs=total_pairs)
    return {**{k: v for k, v in out.items() if k != "dlogps"}, "loss": _PreferenceLogpsLoss.apply(per_token_logps, out)}
