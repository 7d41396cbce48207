"""Plain 64-bit forms of the preference loss, the embedding table and the block-scaled 8-bit operators, on whatever
device their inputs are, and the error bounds the tests hold the kernels to.

Roundings: to nearest is off by at most finfo(t).eps / 2 relative to the value (bf16 2^-8, f16 2^-11, f32 2^-24,
e4m3 2^-4)."""
from __future__ import annotations

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# smallest normal numbers: below them a rounding is off by half a subnormal step
TINY_STEP = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}

# Error of one log-prob.  A term 2^a of the row sum: the exponent a = y log2e - mk is rounded once (|a| <= 32 for every
# term that matters: 2^-20 absolute, times ln 2), ex2.approx is off by 2^-22 relative; a thread adds up to 80 terms of
# one sign (80 * 2^-24) and ten more additions merge them: under 7e-6 altogether, relative to the sum, i.e. absolute in
# its logarithm.  The logarithm and the difference are double precision.
LP_ERR = 7e-6
# A soft-capped logit is off by 2.6e-7 * cap (odd polynomial) on top, in the chosen logit and in the sum.
CAP_ERR = 2 * 2.6e-7


def preference(logits, ids, mask, ref, *, kind="sigmoid", beta=0.1, smooth=0.0, average=False, softcap=0.0,
               weights=None, total=None, logps=None):
    """logits [2P, T, V] (or logps [2P, T] in their place) aligned with ids / mask [2P, T]; everything in 64 bits.
    Returns loss, rewards [2P], seq_logps [2P], coef [2P, T] = dloss/dlp, dh [P], dlogits or None."""
    if logps is None:
        x = logits.double()
        y = softcap * torch.tanh(x / softcap) if softcap else x
        lp = (y - torch.logsumexp(y, -1, keepdim=True)).gather(-1, ids.long()[..., None])[..., 0]
    else:
        lp = logps.double()
    B = lp.shape[0]
    P = B // 2
    m = torch.ones_like(lp) if mask is None else mask.double()
    live = m != 0
    zero = torch.zeros_like(lp)
    n = torch.where(live, m, zero).sum(1)
    inv = torch.where(n != 0, 1 / n, torch.zeros_like(n)) if average else torch.ones_like(n)
    seq = (torch.where(live, lp, zero) * m).sum(1) * inv
    if ref is None:
        d = seq
    elif ref.dim() == 1:
        d = seq - ref.double()
    else:
        d = (torch.where(live, lp - ref.double(), zero) * m).sum(1) * inv
    h = d[:P] - d[P:]
    z = beta * h
    if kind == "sigmoid":
        sp = torch.nn.functional.softplus
        term = (1 - smooth) * sp(-z) + smooth * sp(z)
        dh = -beta * ((1 - smooth) * torch.sigmoid(-z) - smooth * torch.sigmoid(z))
    elif kind == "hinge":
        term = (1 - z).clamp_min(0)
        dh = torch.where(z < 1, -beta, 0.0).double()
    else:
        term = (h - 0.5 / beta) ** 2
        dh = 2 * (h - 0.5 / beta)
    w = torch.ones(P, dtype=torch.float64, device=lp.device) if weights is None else weights.double()
    tot = float(P) if total is None else float(total)
    loss = torch.where(w != 0, w * term, torch.zeros_like(w)).sum() / tot
    c = torch.where(w != 0, w * dh, torch.zeros_like(w)) / tot
    coef = torch.cat([c, -c])[:, None] * torch.where(live, m, zero) * inv[:, None]
    out = {"loss": loss, "rewards": beta * d, "seq_logps": seq, "coef": coef, "dh": dh, "h": h, "n": n, "inv": inv, "w": w, "total": tot}
    if logps is None:
        g = torch.softmax(y, -1).neg_()
        g.scatter_add_(-1, ids.long()[..., None], torch.ones_like(lp)[..., None])
        if softcap:
            g = g * (1 - (y / softcap) ** 2)
        out["dlogits"] = torch.where(coef[..., None] != 0, coef[..., None] * g, torch.zeros((), dtype=torch.float64, device=lp.device))
    return out


def preference_bounds(r, mask, lp_err, *, kind, beta):
    """Bounds on the error of loss, rewards, seq_logps and coef that an error of lp_err per log-prob allows (plus the
    f32 rounding of what is returned)."""
    n = r["n"].abs() if mask is not None else r["n"]
    e_seq = lp_err * n * r["inv"].abs()
    P = r["h"].shape[0]
    e_h = e_seq[:P] + e_seq[P:]
    slope = {"sigmoid": beta, "hinge": beta}.get(kind)
    e_term = (r["dh"].abs() * e_h + e_h ** 2) if kind == "ipo" else slope * e_h
    curve = {"sigmoid": beta * beta / 4, "hinge": 0.0, "ipo": 2.0}[kind]
    e_c = (r["w"].abs() * curve * e_h / r["total"])
    e_coef = torch.cat([e_c, e_c])[:, None] * torch.where(r["coef"] != 0, 1.0, 0.0).double() * r["inv"].abs()[:, None]
    f = 2.0 ** -23
    return {"loss": (r["w"].abs() * e_term).sum() / r["total"] + f * r["loss"].abs(),
            "rewards": beta * e_seq + f * r["rewards"].abs(), "seq_logps": e_seq + f * r["seq_logps"].abs(),
            "coef": e_coef + 4 * 2.0 ** -24 * r["coef"].abs()}


def assert_within(got, ref, bound, what=""):
    got, ref, bound = got.double(), ref.double(), torch.as_tensor(bound, dtype=torch.float64, device=ref.device)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaNs in other places"
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), f"{what}: infinities differ"
    over = ((got - ref).abs() - bound)[fine]
    assert over.numel() == 0 or over.max() <= 0, f"{what}: off by {(got - ref).abs()[fine].max():.3e}, {over.max():.3e} over the bound"


def e4m3(y):
    """The nearest e4m3 value (ties to even, saturating), in 64 bits."""
    a = y.abs().clamp_max(448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.copysign(torch.round(a / step) * step, y)


def quantize(x, block_rows):
    """(values, scales, quotients) in 64 bits; scales as the f32 they are stored in."""
    R, C = x.shape
    br = block_rows
    nr, nc = -(-R // br), -(-C // 128)
    p = torch.zeros(nr * br, nc * 128, dtype=torch.float64, device=x.device)
    p[:R, :C] = x.double()
    p = p.view(nr, br, nc, 128)
    top = torch.nan_to_num(p.abs(), nan=0.0, posinf=float("inf")).amax(dim=(1, 3)).clamp_min(448.0 * 2.0 ** -126)
    y = (448.0 * p / top[:, None, :, None]).view(nr * br, nc * 128)[:R, :C]
    # 64-bit quotient rounded once: the f32 division (torch divides a CUDA tensor by a number through its reciprocal)
    return e4m3(y), (top / 448.0).float(), y


def spread(scales, block_rows, R, C):
    s = scales.double().repeat_interleave(128, 1)[:, :C]
    return s if block_rows == 1 else s.repeat_interleave(128, 0)[:R]


def product(xv, xs, wv, ws):
    """(x w^T, sum of the absolute products) in 64 bits from e4m3 values and scales."""
    x = xv.double() * spread(xs, 1, *xv.shape)
    w = wv.double() * spread(ws, 128, *wv.shape)
    return x @ w.t(), x.abs() @ w.abs().t()


def product_bound(y, mag, K):
    """The products of two e4m3 numbers are exact in f32; a block's 128 of them and then the blocks are added in f32
    (at worst truncated: 2^-23 of the running magnitude each), each block is scaled by a product of two rounded f32."""
    return (min(K, 128) + -(-K // 128) + 4) * 2.0 ** -23 * mag
