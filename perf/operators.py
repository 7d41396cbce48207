"""Cases for measuring the operators at the vocabulary end of a model: the preference loss over paired log ratios, the
scaled embedding lookup and its gradient, quantising to 8-bit floating point by blocks, and the block-scaled 8-bit
product (plain, and folded into the softmax statistics of the loss).

`run` computes a case in plain torch (32 bits, 64 where 32 lose what matters) or, with `own` set, through the package.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 128
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # the loss alone, from log-probs a folded head has produced: latency of a small call
        dict(name="pref logps 8x255", op="pref_logps", pairs=8, rows=255, kind="sigmoid", beta=0.1, smooth=0.0, mean=False, ref=True),
        # one micro-batch of four pairs, 256 positions (151936 vocabulary)
        dict(name="pref 4x256 v151936", op="pref", pairs=4, rows=256, vocab=151936, kind="sigmoid", beta=0.1, smooth=0.0, mean=False, ref=True),
        # eight long pairs, length-normalised squared loss (128256 vocabulary)
        dict(name="pref 8x512 v128256", op="pref", pairs=8, rows=512, vocab=128256, kind="ipo", beta=0.1, smooth=0.0, mean=True, ref=True),
        # one decoding step of 16 sequences
        dict(name="embed 16 h3584", op="embed", tokens=16, vocab=151936, hidden=3584, dtype="bf16", scale=1.0),
        # the tokens of a training batch, scaled by the root of the width (256000 vocabulary)
        dict(name="embed 32768 h3584", op="embed", tokens=32768, vocab=256000, hidden=3584, dtype="bf16", scale=59.75),
        # the table's gradient for a small model's batch of 2048 tokens
        dict(name="embed grad 2048 h896", op="embed_grad", tokens=2048, vocab=151936, hidden=896, dtype="bf16", scale=1.0),
        # the same for 32768 tokens of a large one
        dict(name="embed grad 32768 h3584", op="embed_grad", tokens=32768, vocab=151936, hidden=3584, dtype="bf16", scale=1.0),
        # activations in front of an 8-bit product, a ragged last block
        dict(name="quant 1x128 1999x1000", op="quant", rows=1999, cols=1000, dtype="bf16", tall=False),
        # a whole head's weight
        dict(name="quant 128x128 151936x3584", op="quant", rows=151936, cols=3584, dtype="bf16", tall=True),
        # logits of a single token
        dict(name="fp8 1x151936x3584", op="matmul", rows=1, vocab=151936, hidden=3584, out="f32"),
        # logits of a batch of prompts
        dict(name="fp8 4096x151936x3584", op="matmul", rows=4096, vocab=151936, hidden=3584, out="bf16"),
        # log-probs of a frozen reference model, rows that end inside a tile
        dict(name="fp8 head 2041x151936x896", op="head", rows=2041, vocab=151936, hidden=896),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pref_logps", "pref", "pref", "embed", "embed_grad", "quant", "matmul", "matmul", "head"])
    kind = rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"])
    loss = dict(kind=kind, beta=rng.choice([0.05, 0.1, 0.3]), smooth=rng.choice([0.0, 0.1]) if kind == "sigmoid" else 0.0,
                mean=kind == "ipo" or rng.random() < 0.2, ref=rng.random() < 0.8)
    if op == "pref_logps":
        return dict(op=op, pairs=_log(rng, 1, 512), rows=_log(rng, 8, 4096), **loss)
    if op == "pref":
        pairs, vocab = _log(rng, 1, 16), _log(rng, 129, 256000)
        return dict(op=op, pairs=pairs, rows=_log(rng, 8, max(9, min(2048, 8 * 512 * 128256 // (pairs * vocab)))), vocab=vocab, **loss)
    if op in ("embed", "embed_grad"):
        hidden = _log(rng, 64, 4096) if rng.random() < 0.5 else 64 * _log(rng, 1, 64)
        vocab = _log(rng, 129, min(256000, 151936 * 1792 // hidden))
        return dict(op=op, tokens=_log(rng, 1, min(131072, 32768 * 1792 // hidden)), vocab=vocab, hidden=hidden,
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), scale=rng.choice([1.0, math.sqrt(hidden)]))
    if op == "quant":
        cols = _log(rng, 16, 8192)
        return dict(op=op, rows=_log(rng, 1, min(151936, 151936 * 1792 // cols)), cols=cols, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    tall=rng.random() < 0.5)
    hidden = 16 * _log(rng, 4, 224)
    vocab = _log(rng, 129, 151936)
    if op == "matmul":
        return dict(op=op, rows=_log(rng, 1, 4096), vocab=vocab, hidden=hidden, out=rng.choice(["bf16", "f32"]))
    return dict(op=op, rows=_log(rng, 1, 2048), vocab=vocab, hidden=hidden)


def _pair_masks(pairs, rows, g):
    """Labels [2*pairs, rows + 1]: a prompt of a quarter, then an answer that ends between half and the whole length."""
    start = rows // 4
    end = torch.randint(max(start + 1, rows // 2), rows + 1, (2 * pairs, 1), device=DEV, generator=g)
    at = torch.arange(rows, device=DEV)[None, :]
    live = ((at >= start) & (at < end)).to(torch.int32)
    return torch.cat([torch.zeros(2 * pairs, 1, dtype=torch.int32, device=DEV), live], 1)


def _token_ids(n, vocab, g):
    """Token ids as text has them: a few very frequent ones, a long tail, and the padding id at the end of the batch."""
    u = torch.rand(n, device=DEV, generator=g)
    ids = (torch.exp(u * math.log(vocab)) - 1).long().clamp_(0, vocab - 1)
    ids[n - n // 8:] = 0
    return (ids * 48271 + 11) % vocab


def _quantised(x, tall):
    """(values, scales) of x in e4m3 with one scale for each 1 x 128 or 128 x 128 block: scale = max(amax / 448, 2^-126).

    The quotient x / scale is formed as 448 x / amax in 64 bits: with inputs of few bits it is often the middle between
    two e4m3 values, and a scale rounded to 32 bits first would move it to either side."""
    r, c = x.shape
    br = BLOCK if tall else 1
    nr, nc = -(-r // br), -(-c // BLOCK)
    p = torch.nn.functional.pad(x.float(), (0, nc * BLOCK - c, 0, nr * br - r)).view(nr, br, nc, BLOCK)
    top = p.abs().amax(dim=(1, 3)).clamp_min(E4M3_MAX * 2.0 ** -126)
    y = (p * E4M3_MAX).double() / top[:, None, :, None]
    q = y.to(torch.float8_e4m3fn).view(nr * br, nc * BLOCK)[:r, :c].contiguous()
    return q, top / E4M3_MAX


def _values(q, s, tall):
    r, c = q.shape
    s = s.repeat_interleave(BLOCK, 1)[:, :c]
    if tall:
        s = s.repeat_interleave(BLOCK, 0)[:r]
    return q.float() * s


def _head_weight(vocab, hidden, g):
    """A head's weight whose rows and column blocks differ in size, as trained ones do."""
    w = torch.randn(vocab, hidden, device=DEV, generator=g) * (2.0 / math.sqrt(hidden))
    return w * (0.5 + torch.rand(vocab, 1, device=DEV, generator=g))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    s = dict(case=case)
    op = case["op"]
    if op in ("pref", "pref_logps"):
        B, T = 2 * case["pairs"], case["rows"]
        s["labels"] = _pair_masks(case["pairs"], T, g)
        drift = 0.1 * torch.randn(B, 1, device=DEV, generator=g)
        noise = 0.5 * torch.randn(B, T, device=DEV, generator=g) + drift
        if op == "pref":
            V = case["vocab"]
            logits = torch.empty(B, T + 1, V, dtype=torch.bfloat16, device=DEV)
            for b in range(B):
                logits[b] = 2.0 * torch.randn(T + 1, V, device=DEV, generator=g)
            s["logits"] = logits
            s["input_ids"] = torch.randint(0, V, (B, T + 1), device=DEV, generator=g, dtype=torch.int32)
            chosen = logits[:, :-1].gather(2, s["input_ids"][:, 1:].long()[..., None])[..., 0].float()
            s["ref"] = chosen - (math.log(V) + 2.0) + noise  # 2.0: half the variance, as log-sum-exp of such logits has it
        else:
            s["logps"] = -2.0 * torch.rand(B, T, device=DEV, generator=g).add_(1e-3).log_().abs_()
            s["ref"] = s["logps"] + noise
        if not case["ref"]:
            s["ref"] = None
    elif op in ("embed", "embed_grad"):
        V, H, N = case["vocab"], case["hidden"], case["tokens"]
        s["ids"] = _token_ids(N, V, g).to(torch.int32)
        x = torch.empty(V if op == "embed" else N, H, dtype=DTYPES[case["dtype"]], device=DEV)
        for i in range(0, x.shape[0], 16384):
            x[i:i + 16384] = 0.02 * torch.randn(x[i:i + 16384].shape, device=DEV, generator=g)
        s["x"] = x
    elif op == "quant":
        s["x"] = (torch.randn(case["rows"], case["cols"], device=DEV, generator=g) * torch.exp(
            torch.randn(case["rows"], 1, device=DEV, generator=g))).to(DTYPES[case["dtype"]])
    else:
        M, V, H = case["rows"], case["vocab"], case["hidden"]
        s["wq"], s["ws"] = _quantised(_head_weight(V, H, g), True)
        x = torch.randn(M, H, device=DEV, generator=g).to(torch.bfloat16)
        if op == "matmul":
            s["xq"], s["xs"] = _quantised(x, False)
        else:
            s["hidden"] = x.view(1, M, H)
            s["ids"] = torch.randint(0, V, (1, M), device=DEV, generator=g, dtype=torch.int32)
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import mllm_jax_b200 as G
    from mllm_jax_b200.linear_loss import lm_head_forward

    case = s["case"]
    op = case["op"]
    if op in ("pref", "pref_logps"):
        cfg = G.PreferenceConfig(beta=case["beta"], loss_type=case["kind"], label_smoothing=case["smooth"], average=case["mean"])
        if op == "pref":
            out = G.preference_value_and_grad(s["logits"], s["input_ids"], s["labels"], s["ref"], shifted=True, cfg=cfg)
            return [out["loss"], out["chosen_rewards"], out["rejected_rewards"], out["dlogits"]]
        out = G.preference_logps_value_and_grad(s["logps"], s["labels"][:, 1:], s["ref"], cfg=cfg)
        return [out["loss"], out["chosen_rewards"], out["rejected_rewards"], out["dlogps"]]
    if op == "embed":
        return G.embedding_lookup(s["ids"], s["x"], scale=case["scale"])
    if op == "embed_grad":
        return G.embedding_grad(s["x"], s["ids"], case["vocab"], scale=case["scale"])
    if op == "quant":
        q = G.quantize_fp8(s["x"], block=(BLOCK, BLOCK) if case["tall"] else (1, BLOCK))
        return [q.values, q.scales]
    weight = G.Fp8Blocks(s["wq"], s["ws"], (BLOCK, BLOCK))
    if op == "matmul":
        return G.fp8_matmul(G.Fp8Blocks(s["xq"], s["xs"], (1, BLOCK)), weight, out_dtype=DTYPES[case["out"]])
    out = lm_head_forward(s["hidden"], weight, s["ids"])
    return [out["per_token_logps"], out["token_entropy"], out["lse"]]


def _pair_terms(case, lp, m, ref):
    """loss, rewards of both sides and d loss / d lp (all in 64 bits) from per-token log-probs in 64 bits."""
    P, b, e = case["pairs"], case["beta"], case["smooth"]
    live = m != 0
    d = torch.where(live, lp if ref is None else lp - ref.double(), 0.0)
    n = m.double().sum(1, keepdim=True) if case["mean"] else torch.ones(2 * P, 1, dtype=torch.float64, device=m.device)
    seq = (d * m).sum(1) / n[:, 0]
    h = seq[:P] - seq[P:]
    if case["kind"] == "sigmoid":
        z = b * h
        loss = (1 - e) * torch.log1p(torch.exp(-z.abs())) + (1 - e) * (-z).clamp_min(0) + e * torch.log1p(torch.exp(-z.abs())) + e * z.clamp_min(0)
        dh = -b * ((1 - e) / (1 + torch.exp(z)) - e / (1 + torch.exp(-z)))
    elif case["kind"] == "hinge":
        loss = (1 - b * h).clamp_min(0)
        dh = torch.where(b * h < 1, -b, 0.0).double()
    else:
        loss = (h - 0.5 / b) ** 2
        dh = 2 * (h - 0.5 / b)
    coef = torch.cat([dh, -dh])[:, None] / P * m / n
    return loss.sum() / P, b * seq[:P], b * seq[P:], coef


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "pref":
        ids, m = s["input_ids"][:, 1:].long(), s["labels"][:, 1:]
        x = s["logits"][:, :-1].float()
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - top)
        total = p.sum(-1, keepdim=True, dtype=torch.float64)
        lp = (x.gather(2, ids[..., None]).double() - top.double() - total.log())[..., 0]
        loss, good, bad, coef = _pair_terms(case, lp, m, s["ref"])
        del x
        p *= (-coef[..., None] / total).float()
        p.scatter_add_(2, ids[..., None], coef[..., None].float())
        d = torch.zeros_like(s["logits"])
        d[:, :-1] = p
        return [loss.float(), good.float(), bad.float(), d]
    if op == "pref_logps":
        loss, good, bad, coef = _pair_terms(case, s["logps"].double(), s["labels"][:, 1:], s["ref"])
        return [loss.float(), good.float(), bad.float(), coef.float()]
    if op == "embed":
        return (s["x"][s["ids"].long()].float() * case["scale"]).to(s["x"].dtype)
    if op == "embed_grad":
        out = torch.zeros(case["vocab"], case["hidden"], device=s["x"].device)
        return out.index_add_(0, s["ids"].long(), s["x"].float()).mul_(case["scale"])
    if op == "quant":
        return list(_quantised(s["x"], case["tall"]))
    w = _values(s["wq"], s["ws"], True)
    if op == "matmul":
        return (_values(s["xq"], s["xs"], False) @ w.t()).to(DTYPES[case["out"]])
    q, qs = _quantised(s["hidden"][0], False)
    y = _values(q, qs, False) @ w.t()
    top = y.amax(-1, keepdim=True)
    p = torch.exp(y - top)
    total = p.sum(-1, dtype=torch.float64)
    lse = top[:, 0].double() + total.log()
    lp = y.gather(1, s["ids"][0].long()[:, None])[:, 0].double() - lse
    entropy = lse - (p * y).sum(-1, dtype=torch.float64) / total
    return [lp.float()[None], entropy.float()[None], lse.float()[None]]


def work(case):
    op = case["op"]
    if op == "pref":  # half of the scored rows carry the answer: only those need their logits
        n = 2 * case["pairs"] * (case["rows"] + 1) * case["vocab"]
        return {"bytes": 3.0 * n, "flops": 5.0 * n}
    if op == "pref_logps":
        n = 2 * case["pairs"] * case["rows"]
        return {"bytes": (4 + 4 + 4 + (4 if case["ref"] else 0)) * n, "flops": 4 * n}
    if op == "embed":
        n = case["tokens"] * case["hidden"]
        return {"bytes": 2 * n * SIZE[case["dtype"]] + 4 * case["tokens"], "flops": n}
    if op == "embed_grad":
        n = case["tokens"] * case["hidden"]
        return {"bytes": n * SIZE[case["dtype"]] + 4 * case["vocab"] * case["hidden"] + 4 * case["tokens"], "flops": 2 * n}
    if op == "quant":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (SIZE[case["dtype"]] + 1) + n // (BLOCK * BLOCK if case["tall"] else BLOCK) * 4, "flops": 3 * n}
    M, V, H = case["rows"], case["vocab"], case["hidden"]
    if op == "matmul":
        return {"bytes": M * H + V * H + M * V * SIZE[case["out"]], "flops": 2 * M * V * H}
    return {"bytes": 2 * M * H + V * H + 16 * M, "flops": 2 * M * V * H}


def _e4m3_64(y):
    """y rounded to the nearest e4m3 value (ties to even), computed and held in 64 bits."""
    a = y.abs().clamp_max(E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.sign(y) * (torch.round(a / step) * step)


def _blocks_64(x, tall):
    """(values, scales) of the quantiser's definition in 64 bits, block column by block column."""
    x = x.double()
    r, c = x.shape
    values, scales = torch.empty_like(x), []
    for j in range(0, c, BLOCK):
        col = x[:, j:j + BLOCK]
        top = col.abs().amax(1)
        if tall:
            top = torch.stack([t.max() for t in top.split(BLOCK)])
        top = torch.clamp(top, min=E4M3_MAX * 2.0 ** -126)
        scales.append(top / E4M3_MAX)
        each = top.repeat_interleave(BLOCK)[:r] if tall else top
        values[:, j:j + BLOCK] = _e4m3_64(E4M3_MAX * col / each[:, None])
    return values, torch.stack(scales, 1)


def _product_64(xv, xs, wv, ws):
    """sum over blocks of sx * sw * (inner sum), in 64 bits: each operand's values times its scale."""
    xd, wd = xv.double(), wv.double()
    for j in range(xs.shape[1]):
        cols = slice(j * BLOCK, (j + 1) * BLOCK)
        xd[:, cols] *= xs[:, j:j + 1].double()
        wd[:, cols] *= ws[:, j].double().repeat_interleave(BLOCK)[:wd.shape[0], None]
    return xd @ wd.t()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("pref", "pref_logps"):
        P, b, e = case["pairs"], case["beta"], case["smooth"]
        m = s["labels"][:, 1:].double()
        grad = torch.zeros(s["logits"].shape if op == "pref" else s["logps"].shape, dtype=torch.float64, device=DEV)
        lp = s["logps"].double() if op == "pref_logps" else torch.stack([
            torch.log_softmax(s["logits"][i, :-1].double(), -1).gather(1, s["input_ids"][i, 1:].long()[:, None])[:, 0]
            for i in range(2 * P)])
        lp.requires_grad_(True)
        gap = lp if s["ref"] is None else lp - s["ref"].double()
        reward = (gap * m).sum(1)
        if case["mean"]:
            reward = reward / m.sum(1)
        h = reward[:P] - reward[P:]
        sig = torch.nn.functional.logsigmoid
        loss = {"sigmoid": -(1 - e) * sig(b * h) - e * sig(-b * h), "hinge": torch.relu(1 - b * h),
                "ipo": (h - 1 / (2 * b)).square()}[case["kind"]].mean()
        loss.backward()
        if op == "pref_logps":
            grad = lp.grad
        else:
            for i in range(2 * P):
                p = torch.softmax(s["logits"][i, :-1].double(), -1).neg_()
                p.scatter_add_(1, s["input_ids"][i, 1:].long()[:, None], torch.ones_like(p[:, :1]))
                grad[i, :-1] = p * lp.grad[i][:, None]
        return [loss.detach(), b * reward[:P].detach(), b * reward[P:].detach(), grad]
    if op == "embed":
        return torch.index_select(s["x"], 0, s["ids"].long()).double() * case["scale"]
    if op == "embed_grad":
        order = torch.argsort(s["ids"], stable=True)
        lengths = torch.bincount(s["ids"].long(), minlength=case["vocab"])
        rows = (s["x"].double() * case["scale"])[order]
        return torch.segment_reduce(rows, "sum", lengths=lengths, axis=0, initial=0)
    if op == "quant":
        return list(_blocks_64(s["x"], case["tall"]))
    if op == "matmul":
        return _product_64(s["xq"], s["xs"], s["wq"], s["ws"])
    out = _product_64(*_blocks_64(s["hidden"][0], False), s["wq"], s["ws"])
    lse = torch.logsumexp(out, 1)
    lp = out.gather(1, s["ids"][0].long()[:, None])[:, 0] - lse
    entropy = -(torch.exp(out - lse[:, None]) * (out - lse[:, None])).sum(1)
    return [lp[None], entropy[None], lse[None]]
