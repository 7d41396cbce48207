"""One preference-training step at the vocabulary end of a small tied model, with every operator in its place:
scaled embedding lookup -> trunk -> logits of the tied table -> paired loss against the log-probs of a frozen reference
model whose head is held in 8 bits -> gradients of both uses of the table, added up in f32."""
import pytest
import torch

import mllm_jax_b200 as G
from tests import operator_reference as R

pytestmark = pytest.mark.gpu

P, L, V, H = 3, 24, 2011, 96


def _model(dev):
    g = torch.Generator().manual_seed(11)
    table = (0.3 * torch.randn(V, H, generator=g)).to(torch.bfloat16).to(dev)
    mix = (torch.randn(H, H, generator=g) / H ** 0.5).to(torch.bfloat16).to(dev)
    frozen = (0.3 * torch.randn(V, H, generator=g)).to(torch.bfloat16).to(dev)
    ids = torch.randint(0, V, (2 * P, L), generator=g).to(dev)
    labels = (torch.rand(2 * P, L, generator=g) < 0.7).to(torch.int64).to(dev)
    labels[-1] = 0  # an empty answer
    return table, mix, frozen, ids, labels


def test_step(cuda):
    table, mix, frozen, ids, labels = _model(cuda)
    scale, cfg = H ** 0.5, G.PreferenceConfig(beta=0.2, label_smoothing=0.05)
    # the reference model: its head in 8 bits, log-probs without logits in memory
    ref_head = G.quantize_fp8(frozen, block=(128, 128))
    ref_hidden = torch.tanh(G.embedding_lookup(ids, frozen, scale=scale) @ mix)[:, :-1]
    ref = G.lm_head_forward(ref_hidden, ref_head, ids[:, 1:], cfg=G.LossConfig(compute_entropy=False))["per_token_logps"]
    q = G.quantize_fp8(ref_hidden.reshape(-1, H))
    y, mag = R.product(q.values, q.scales, ref_head.values, ref_head.scales)
    lp = torch.log_softmax(y, -1).gather(1, ids[:, 1:].reshape(-1)[:, None])[:, 0]
    # both logits are off by at most the product's bound; the row's sum by 2^-17 (exponents below 32 rounded once)
    R.assert_within(ref.reshape(-1), lp, 2 * R.product_bound(y, mag, H).amax(1) + 2.0 ** -17, "reference log-probs")

    # the step by hand: gradients of the table's two uses meet in one f32 buffer
    emb = G.embedding_lookup(ids, table, scale=scale)
    pre = emb @ mix
    hidden = torch.tanh(pre)
    logits = hidden @ table.t()
    out = G.preference_value_and_grad(logits, ids, labels, ref, shifted=True, cfg=cfg)
    d = out["dlogits"].view(-1, V)
    dtable = d.t().float() @ hidden.view(-1, H).float()
    dhidden = d.float() @ table.float()
    demb = ((dhidden * (1 - hidden.view(-1, H).float() ** 2)) @ mix.float().t()).view(2 * P, L, H)
    by_head = dtable.clone()
    assert G.embedding_grad(demb, ids, V, scale=scale, out=dtable) is dtable
    want = R.preference(logits[:, :-1], ids[:, 1:], labels[:, 1:], ref, beta=0.2, smooth=0.05)
    b = R.preference_bounds(want, labels[:, 1:], R.LP_ERR, kind="sigmoid", beta=0.2)
    R.assert_within(out["loss"], want["loss"], b["loss"], "loss")
    R.assert_within(out["dlogits"][:, :-1], want["dlogits"],
                    (want["coef"].abs() * (2.0 ** -18 + 2 * R.LP_ERR) + b["coef"])[..., None] + 2.0 ** -8 * 1.01 * want["dlogits"].abs(), "dlogits")
    flat = ids.reshape(-1)
    x = demb.reshape(-1, H).double() * torch.tensor(scale, dtype=torch.float32).double()
    total = by_head.double().index_add(0, flat, x)
    size = by_head.double().abs().index_add(0, flat, x.abs())
    n = torch.bincount(flat, minlength=V)[:, None].double()
    R.assert_within(dtable, total, (n + 3) * 2.0 ** -24 * size, "table gradient")
    untouched = n[:, 0] == 0
    assert torch.equal(dtable[untouched], by_head[untouched])

    # the same step through autograd
    leaf = table.clone().requires_grad_(True)
    hid = torch.tanh(G.embedding_lookup(ids, leaf, scale=scale) @ mix)
    res = G.preference_loss(hid @ leaf.t(), ids, labels, ref, cfg=cfg)
    res["loss"].backward()
    assert torch.equal(res["loss"].detach(), out["loss"]) and torch.equal(res["chosen_rewards"], out["chosen_rewards"])
    # bf16 gradients: dhidden, the tanh's derivative (a square, a difference, a product), demb, the two uses' results and
    # their sum are rounded to bf16 where the hand-made step kept f32: ten half steps of what is added up cover them
    size = (d.float().abs().t() @ hidden.view(-1, H).float().abs()).double()
    chain = ((d.float().abs() @ table.float().abs()) @ mix.float().abs().t()).double() * scale
    size = size.index_add(0, flat, chain)
    R.assert_within(leaf.grad, dtable.double(), 10 * 2.0 ** -8 * size + 2.0 ** -126, "autograd")


def test_step_from_log_probs(cuda):
    """The forward of a policy whose head is folded too: loss and rewards from log-probs alone equal those from logits."""
    table, mix, frozen, ids, labels = _model(cuda)
    head = G.quantize_fp8(table, block=(128, 128))
    hidden = torch.tanh(G.embedding_lookup(ids, table) @ mix)[:, :-1]
    lp = G.lm_head_forward(hidden, head, ids[:, 1:])["per_token_logps"]
    ref = torch.zeros_like(lp) - 7.0
    out = G.preference_logps_value_and_grad(lp, labels[:, 1:], ref)
    x = lp.clone().requires_grad_(True)
    res = G.preference_loss_from_logps(x, labels[:, 1:], ref)
    res["loss"].backward()
    assert torch.equal(res["loss"].detach(), out["loss"]) and torch.equal(x.grad, out["dlogps"])
    want = R.preference(None, None, labels[:, 1:], ref, logps=lp)
    b = R.preference_bounds(want, labels[:, 1:], 0.0, kind="sigmoid", beta=0.1)
    R.assert_within(out["loss"], want["loss"], b["loss"], "loss")
    R.assert_within(out["dlogps"], want["coef"], b["coef"], "dlogps")
