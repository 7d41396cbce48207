"""Preference loss over paired log ratios against its 64-bit form: every loss type, masks that leave sequences empty,
garbage in masked places, strides and alignments, few and many rows, autograd, streams, graphs."""
import pytest
import torch

import mllm_jax_b200 as G
from tests import operator_reference as R

pytestmark = pytest.mark.gpu


def _case(P, T, V, seed, device, ref="token", prompt=True, sigma=2.0):
    g = torch.Generator().manual_seed(seed)
    B = 2 * P
    logits = (torch.randn(B, T, V, generator=g) * sigma).to(torch.bfloat16)
    ids = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32)
    end = torch.randint(max(1, T // 2), T + 1, (B, 1), generator=g)
    at = torch.arange(T)[None]
    mask = ((at < end) & (at >= (T // 4 if prompt else 0))).to(torch.int32)
    x = logits.double()
    lp = (x - torch.logsumexp(x, -1, keepdim=True)).gather(-1, ids.long()[..., None])[..., 0]
    rf = (lp + 0.5 * torch.randn(B, T, generator=g)).float()
    if ref == "sequence":
        rf = (rf * mask).sum(1)
    elif ref is None:
        rf = None
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    return to(logits), to(ids), to(mask), to(rf)


def _check(out, logits, ids, mask, ref, cfg, weights=None, total=None, grad_scale=1.0, scored=None):
    kw = dict(kind=cfg.loss_type, beta=cfg.beta)
    x = logits if scored is None else logits[:, :scored]
    r = R.preference(x, ids, mask, ref, smooth=cfg.label_smoothing, average=cfg.average, softcap=cfg.softcap or 0.0,
                     weights=weights, total=total, **kw)
    lp_err = R.LP_ERR + (R.CAP_ERR * cfg.softcap if cfg.softcap else 0.0)
    b = R.preference_bounds(r, mask, lp_err, **kw)
    P = logits.shape[0] // 2
    R.assert_within(out["loss"], r["loss"], b["loss"], "loss")
    R.assert_within(torch.cat([out["chosen_rewards"], out["rejected_rewards"]]), r["rewards"], b["rewards"], "rewards")
    R.assert_within(torch.cat([out["chosen_logps"], out["rejected_logps"]]), r["seq_logps"], b["seq_logps"], "log-probs")
    assert out["chosen_rewards"].shape == (P,)
    if "dlogits" in out:
        d = out["dlogits"]
        if scored is not None:
            assert not d[:, scored:].any(), "rows that are not scored have no gradient"
            d = d[:, :scored]
        ref_d = r["dlogits"] * grad_scale
        coef, e_coef = r["coef"].abs() * abs(grad_scale), b["coef"] * abs(grad_scale)
        # the softmax from a rounded log-sum-exp and exponent: 2^-18 of it, plus what the soft-cap's logits are off;
        # then one rounding to bf16 (a half step of a subnormal at least)
        rel = 2.0 ** -18 + 2 * lp_err
        bound = ((coef * rel + e_coef)[..., None] * (1 + 0 * ref_d) + (2.0 ** -8) * (1 + 2.0 ** -7) * ref_d.abs() + 2.0 ** -126)
        R.assert_within(d, ref_d, bound, "dlogits")
        dead = (coef == 0)[..., None].expand_as(d)
        assert not d[dead].any(), "a row without a coefficient is exactly zero"


CASES = [
    (1, 1, 2, {}),                                        # one token, two logits
    (1, 2, 7, {}),
    (2, 9, 129, dict(loss_type="hinge")),
    (3, 33, 1000, dict(loss_type="ipo", average=True)),
    (2, 40, 4099, dict(label_smoothing=0.1)),
    (1, 3, 32007, dict(beta=0.5)),                        # few rows: a row split over CTAs, odd width
    (5, 17, 20000, dict(average=True)),                   # split_cols above the small kernels' limit
    (300, 2, 64, dict(beta=0.3)),                         # many pairs
    (2, 11, 5000, dict(softcap=30.0)),
    (1, 4, 256000, dict(softcap=30.0, loss_type="ipo", average=True)),
]


@pytest.mark.parametrize("P,T,V,kw", CASES)
@pytest.mark.parametrize("ref", ["token", "sequence", None])
def test_matches_the_64_bit_form(cuda, P, T, V, kw, ref):
    cfg = G.PreferenceConfig(**kw)
    logits, ids, mask, rf = _case(P, T, V, 100 + V, cuda, ref)
    if ref == "sequence" and cfg.average:
        rf = rf / mask.sum(1).clamp_min(1)
    out = G.preference_value_and_grad(logits, ids, mask, rf, cfg=cfg)
    torch.cuda.synchronize()
    assert int(out["problem"].device_status.item()) == 0
    _check(out, logits, ids, mask, rf, cfg)


def test_reference_layout_weights_and_normaliser(cuda):
    """shifted layout, pair weights with a padded pair of NaN logits' weight 0, a device normaliser, a grad scale."""
    logits, ids, mask, rf = _case(4, 21, 777, 5, cuda)
    weights = torch.tensor([1.0, 0.5, 0.0, 2.0], device=cuda)
    logits[2] = float("nan")
    cfg = G.PreferenceConfig(beta=0.2)
    total = torch.tensor(3.5, device=cuda)
    out = G.preference_value_and_grad(logits, ids, mask, rf[:, :-1], shifted=True, cfg=cfg, pair_weights=weights,
                                      total_pairs=total, grad_scale=-1.5)
    torch.cuda.synchronize()
    clean = logits.clone()
    clean[2] = 0
    r = R.preference(clean[:, :-1], ids[:, 1:], mask[:, 1:], rf[:, :-1], beta=0.2, weights=weights, total=3.5)
    b = R.preference_bounds(r, mask, R.LP_ERR, kind="sigmoid", beta=0.2)
    R.assert_within(out["loss"], r["loss"], b["loss"], "loss")
    assert not out["dlogits"][2].any() and not out["dlogits"][6].any() and not out["dlogits"][:, -1].any()
    assert torch.isfinite(out["dlogits"]).all()
    live = [0, 1, 3]
    sel = lambda t: torch.cat([t[live], t[[4, 5, 7]]])  # noqa: E731
    sub = {k: out[k][live] for k in ("chosen_rewards", "rejected_rewards", "chosen_logps", "rejected_logps")}
    sub["loss"], sub["dlogits"] = out["loss"], sel(out["dlogits"])
    _check(sub, sel(logits), sel(ids)[:, 1:], sel(mask)[:, 1:], sel(rf)[:, :-1], cfg, weights=weights[live], total=3.5,
           grad_scale=-1.5, scored=20)


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
def test_empty_masks_and_garbage_in_masked_places(cuda, average, kind):
    logits, ids, mask, rf = _case(3, 12, 500, 9, cuda)
    mask[1] = 0            # a chosen answer without tokens
    mask[2] = 0
    mask[5] = 0            # a pair without any
    dead = mask == 0
    logits[dead] = float("nan")
    rf[dead] = float("inf")
    ids[dead] = -7         # not an id: not looked at
    logits[0, 4, 10] = float("-inf")  # a forbidden token in a live row
    cfg = G.PreferenceConfig(loss_type=kind, average=average)
    out = G.preference_value_and_grad(logits, ids, mask, rf, cfg=cfg)
    torch.cuda.synchronize()
    assert int(out["problem"].device_status.item()) == 0
    clean, rclean, iclean = logits.clone(), rf.clone(), ids.clone()
    clean[dead], rclean[dead], iclean[dead] = 0, 0, 0
    _check(out, clean, iclean, mask, rclean, cfg)


def test_fractional_masks_and_no_mask(cuda):
    logits, ids, mask, rf = _case(2, 8, 300, 10, cuda)
    w = torch.rand(4, 8, device=cuda)
    w[0, 3] = 0
    for m in (w, None):
        for average in (False, True):
            cfg = G.PreferenceConfig(average=average)
            out = G.preference_value_and_grad(logits, ids, m, rf, cfg=cfg)
            torch.cuda.synchronize()
            _check(out, logits, ids, m, rf, cfg)


def test_extreme_margins(cuda):
    """Log-ratios far beyond what exp holds in 32 bits: the loss is linear, the gradient saturates, nothing overflows."""
    logits, ids, mask, _ = _case(2, 6, 100, 11, cuda)
    ref = torch.tensor([3e4, -3e4, -3e4, 3e4], device=cuda)
    for kw in (dict(), dict(label_smoothing=0.2), dict(loss_type="hinge"), dict(loss_type="ipo")):
        cfg = G.PreferenceConfig(beta=0.7, **kw)
        out = G.preference_value_and_grad(logits, ids, mask, ref, cfg=cfg)
        torch.cuda.synchronize()
        assert torch.isfinite(out["loss"])
        _check(out, logits, ids, mask, ref, cfg)


def test_ids_outside_the_vocabulary_are_clamped_and_reported(cuda):
    logits, ids, mask, rf = _case(1, 6, 50, 12, cuda, prompt=False)
    mask[:] = 1
    ids[0, 0], ids[1, 2] = -3, 50
    out = G.preference_value_and_grad(logits, ids, mask, rf)
    torch.cuda.synchronize()
    assert int(out["problem"].device_status.item()) == 1
    _check(out, logits, ids.clamp(0, 49), mask, rf, G.PreferenceConfig())


@pytest.mark.parametrize("shift", [0, 1, 3])
def test_strided_unaligned_views_and_in_place(cuda, shift):
    """Rows that start off a 16-byte boundary, a row stride beyond the vocabulary, guards that must stay as they were."""
    P, T, V, ld = 2, 5, 997, 1010
    logits, ids, mask, rf = _case(P, T, V, 13, cuda)
    big = torch.full((2 * P * T * ld + 16,), 7.0, dtype=torch.bfloat16, device=cuda)
    view = big[shift:shift + 2 * P * T * ld].view(2 * P, T, ld)[:, :, :V]
    view.copy_(logits)
    cfg = G.PreferenceConfig()
    out = G.preference_value_and_grad(view, ids, mask, rf, cfg=cfg)   # gradient buffer of its own: another phase
    torch.cuda.synchronize()
    _check(out, logits, ids, mask, rf, cfg)
    out = G.preference_value_and_grad(view, ids, mask, rf, cfg=cfg, inplace=True)
    torch.cuda.synchronize()
    _check({**out, "dlogits": view}, logits, ids, mask, rf, cfg)
    rows = big[shift:shift + 2 * P * T * ld].view(-1, ld)
    assert (rows[:, V:] == 7).all() and (big[:shift] == 7).all() and (big[shift + 2 * P * T * ld:] == 7).all()


def test_autograd_equals_value_and_grad(cuda):
    logits, ids, mask, rf = _case(3, 15, 640, 14, cuda)
    cfg = G.PreferenceConfig(label_smoothing=0.05)
    ref = G.preference_value_and_grad(logits, ids, mask, rf[:, 1:], shifted=True, cfg=cfg, grad_scale=3.0)
    x = logits.clone().requires_grad_(True)
    out = G.preference_loss(x, ids, mask, rf[:, 1:], cfg=cfg)
    assert not out["chosen_rewards"].requires_grad
    (out["loss"] * 3).backward()
    assert torch.equal(x.grad, ref["dlogits"]) and torch.equal(out["loss"].detach(), ref["loss"])
    x2 = logits.clone().requires_grad_(True)
    out = G.preference_loss(x2 * 1.0, ids, mask, rf[:, 1:], cfg=cfg, inplace_backward=True)
    (out["loss"] * 3).backward()
    assert torch.equal(x2.grad, ref["dlogits"])
    out = G.preference_loss(x2 * 1.0, ids, mask, rf[:, 1:], cfg=cfg, inplace_backward=True)
    out["loss"].backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="overwritten"):
        out["loss"].backward()


@pytest.mark.parametrize("P,T", [(1, 1), (2, 7), (33, 50), (5, 4000), (700, 31), (1, 20000)])
@pytest.mark.parametrize("kind,average", [("sigmoid", False), ("hinge", True), ("ipo", True)])
def test_from_logps(cuda, P, T, kind, average):
    g = torch.Generator().manual_seed(P + T)
    lp = -3 * torch.rand(2 * P, T, generator=g).to(cuda)
    rf = lp + 0.3 * torch.randn(2 * P, T, generator=g).to(cuda)
    mask = (torch.rand(2 * P, T, generator=g) < 0.6).float().to(cuda)
    mask[-1] = 0
    bad_lp, bad_rf = lp.clone(), rf.clone()
    bad_lp[mask == 0], bad_rf[mask == 0] = float("nan"), float("-inf")
    cfg = G.PreferenceConfig(loss_type=kind, average=average)
    r = R.preference(None, None, mask, rf, kind=kind, beta=0.1, average=average, logps=lp)
    b = R.preference_bounds(r, mask, 0.0, kind=kind, beta=0.1)
    # double precision sums: what is left is the f32 rounding of what is returned (and of 1/n, the mean's weight)
    out = G.preference_logps_value_and_grad(bad_lp, mask, bad_rf, cfg=cfg)
    torch.cuda.synchronize()
    R.assert_within(out["loss"], r["loss"], b["loss"], "loss")
    R.assert_within(torch.cat([out["chosen_rewards"], out["rejected_rewards"]]), r["rewards"], b["rewards"], "rewards")
    R.assert_within(out["dlogps"], r["coef"], b["coef"], "dlogps")
    x = lp.clone().requires_grad_(True)
    G.preference_loss_from_logps(x, mask, rf, cfg=cfg)["loss"].mul(2.0).backward()
    R.assert_within(x.grad, 2 * r["coef"], 2 * b["coef"] + 2.0 ** -23 * r["coef"].abs(), "autograd")


def test_gradient_against_differences(cuda):
    """d loss / d logits by central differences of the operator itself (loss in f32: steps large against 2^-24)."""
    logits, ids, mask, rf = _case(1, 4, 33, 15, cuda, sigma=1.0)
    mask[:] = 1
    cfg = G.PreferenceConfig(beta=1.0)
    out = G.preference_value_and_grad(logits, ids, mask, rf, cfg=cfg)
    d = out["dlogits"].double()
    for b, t, j in [(0, 0, int(ids[0, 0])), (0, 2, 5), (1, 3, int(ids[1, 3])), (1, 1, 9)]:
        step = 0.125 * max(1.0, float(logits[b, t, j].abs()))
        vals, at = [], []
        for sgn in (1, -1):
            y = logits.clone()
            y[b, t, j] += sgn * step
            at.append(float(y[b, t, j]))
            vals.append(float(G.preference_value_and_grad(y, ids, mask, rf, cfg=cfg)["loss"]))
        num = (vals[0] - vals[1]) / (at[0] - at[1])
        # third derivative of the loss along one logit is below 2 (beta = 1): the difference is off by step^2 / 3,
        # plus 2^-23 of the loss over the step, plus the gradient's own bf16 rounding
        assert abs(num - float(d[b, t, j])) <= 2 * step ** 2 / 6 + 2.0 ** -22 * abs(vals[0]) / step + 2.0 ** -8 * abs(num)


def test_streams_and_graph_replay(cuda):
    """Two calls in flight on two streams, and a captured call replayed on new inputs beside an eager one."""
    a, b = _case(2, 30, 3001, 16, cuda), _case(2, 30, 3001, 17, cuda)
    cfg = G.PreferenceConfig()
    want = [G.preference_value_and_grad(*c, cfg=cfg) for c in (a, b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = [None, None]
    for _ in range(3):
        with torch.cuda.stream(s1):
            got[0] = G.preference_value_and_grad(*a, cfg=cfg)
        with torch.cuda.stream(s2):
            got[1] = G.preference_value_and_grad(*b, cfg=cfg)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g["dlogits"], w["dlogits"]) and torch.equal(g["loss"], w["loss"])
    static = [t.clone() for t in a]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = G.preference_value_and_grad(*static, cfg=cfg)
    for src, w in ((b, want[1]), (a, want[0])):
        for t, x in zip(static, src):
            t.copy_(x)
        graph.replay()
        eager = G.preference_value_and_grad(*src, cfg=cfg)
        torch.cuda.synchronize()
        assert torch.equal(out["dlogits"], w["dlogits"]) and torch.equal(out["loss"], w["loss"])
        assert torch.equal(eager["dlogits"], w["dlogits"])


@pytest.mark.parametrize("P,T", [(8192, 1), (600, 129), (3, 128), (64, 64)])
def test_from_logps_many_or_short_pairs(cuda, P, T):
    test_from_logps(cuda, P, T, "sigmoid", False)


def test_single_rows_of_longer_sequences(cuda):
    """L = 1 as a slice: the rows are the sequences' distance apart."""
    logits, ids, mask, rf = _case(2, 5, 300, 30, cuda, prompt=False)
    cfg = G.PreferenceConfig()
    out = G.preference_value_and_grad(logits[:, 2:3], ids[:, 2:3], None, rf[:, 2:3], cfg=cfg)
    _check(out, logits[:, 2:3], ids[:, 2:3], torch.ones_like(ids[:, 2:3]), rf[:, 2:3], cfg)
    assert out["dlogits"].stride() == logits[:, 2:3].stride()


@pytest.mark.parametrize("what", ["ids", "mask", "logits"])
def test_a_change_between_the_sweeps_is_an_error(cuda, what):
    logits, ids, mask, rf = _case(2, 9, 200, 31, cuda)
    x = logits.clone().requires_grad_(True)
    y = x * 1.0
    out = G.preference_loss(y, ids, mask, rf[:, 1:])
    if what == "logits":
        with torch.no_grad():
            y.mul_(2)
    else:
        dict(ids=ids, mask=mask)[what].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out["loss"].backward()


def test_gradients_written_over_the_logits_are_seen(cuda):
    """Two losses of the same logits: once the first has written its gradient over them, the second cannot be formed."""
    logits, ids, mask, rf = _case(2, 9, 200, 32, cuda)
    x = logits.clone().requires_grad_(True)
    y = x * 1.0
    first = G.preference_loss(y, ids, mask, rf[:, 1:], inplace_backward=True)["loss"]
    second = G.preference_loss(y, ids, mask, rf[:, 1:], cfg=G.PreferenceConfig(loss_type="ipo"))["loss"]
    first.backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        second.backward()
    z = logits.clone().requires_grad_(True)
    w = z * 1.0
    loss = G.preference_loss(w, ids, mask, rf[:, 1:])["loss"]
    G.preference_value_and_grad(w.detach(), ids, mask, rf[:, 1:], shifted=True, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        G.preference_value_and_grad(logits * 1.0, ids, mask, rf[:, 1:], shifted=True, inplace=True)


def test_captured_backward(cuda):
    """Forward and backward of the differentiable forms in one graph, replayed with other logits."""
    a, ids, mask, rf = _case(2, 9, 200, 33, cuda)
    b = _case(2, 9, 200, 34, cuda)[0]
    want = [G.preference_value_and_grad(t, ids, mask, rf[:, 1:], shifted=True) for t in (a, b)]
    want = [(t["loss"].clone(), t["dlogits"].clone()) for t in want]
    static = a.clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        loss = G.preference_loss(static, ids, mask, rf[:, 1:])["loss"]
        (grad,) = torch.autograd.grad(loss, static)
    for k, t in ((1, b), (0, a)):
        with torch.no_grad():
            static.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss.detach(), want[k][0]) and torch.equal(grad, want[k][1])


@pytest.mark.parametrize("P,T,V,kw", [(1, 3, 1, {}), (7, 61, 2047, dict(loss_type="ipo")), (3, 50, 2048, {}), (3, 50, 2049, {}),
                                      (2, 17, 900, dict(softcap=30.0))])
def test_short_rows(cuda, P, T, V, kw):
    """Rows of a warp each, to the last that is and the first that is not; rows behind the scored ones."""
    logits, ids, mask, rf = _case(P, T, V, P + T + V, cuda)
    cfg = G.PreferenceConfig(**kw)
    _check(G.preference_value_and_grad(logits, ids, mask, rf, cfg=cfg), logits, ids, mask, rf, cfg)
    if T > 3:
        out = G.preference_value_and_grad(logits, ids, mask, rf[:, 1:], shifted=True, cfg=cfg)
        _check(out, logits, ids[:, 1:], mask[:, 1:], rf[:, 1:], cfg, scored=T - 1)


def _large_case(P, T, V, seed, device):
    """As `_case` with reference log-probs per token, made on the device and a sequence at a time."""
    g = torch.Generator(device).manual_seed(seed)
    B = 2 * P
    logits = torch.empty(B, T, V, dtype=torch.bfloat16, device=device)
    ids = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32, device=device)
    rf = torch.empty(B, T, device=device)
    for b in range(B):
        logits[b] = 2 * torch.randn(T, V, generator=g, device=device)
        lp = torch.log_softmax(logits[b].double(), -1).gather(-1, ids[b].long()[:, None])[:, 0]
        rf[b] = lp + 0.5 * torch.randn(T, generator=g, device=device)
    end = torch.randint(max(1, T // 2), T + 1, (B, 1), generator=g, device=device)
    at = torch.arange(T, device=device)[None]
    return logits, ids, ((at < end) & (at >= T // 4)).to(torch.int32), rf


@pytest.mark.parametrize("P,T,V,kw", [
    (37, 64, 16501, {}), (37, 64, 16501, dict(softcap=30.0, average=True)),                  # 4736 tokens: rows unsplit
    (37, 32, 33001, dict(loss_type="ipo")), (37, 32, 33001, dict(softcap=30.0)),             # two parts of 16504 columns
    (5, 158, 50001, dict(label_smoothing=0.1)), (5, 158, 50001, dict(softcap=20.0, loss_type="hinge")),  # three of 16672
])
def test_parts_of_more_than_16384_columns(cuda, P, T, V, kw):
    """So many tokens that a row, or its part, is too long for the CTAs of 128 threads: those of 512 take it."""
    cfg = G.PreferenceConfig(**kw)
    logits, ids, mask, rf = _large_case(P, T, V, P + T + V, cuda)
    ids[0, T // 4], ids[0, T // 4 + 1], ids[1, T // 4], ids[1, T // 4 + 1] = 0, V - 1, 16503 % V, 16504 % V
    out = G.preference_value_and_grad(logits, ids, mask, rf, cfg=cfg)
    torch.cuda.synchronize()
    assert int(out["problem"].device_status.item()) == 0
    _check(out, logits, ids, mask, rf, cfg)
    if P == 5:  # rows behind the scored ones, and a gradient buffer of another phase than the logits
        big = torch.full((2 * P * T * V + 8,), 7.0, dtype=torch.bfloat16, device=cuda)
        d = big[1:1 + 2 * P * T * V].view(2 * P, T, V)
        out = G.preference_value_and_grad(logits, ids, mask, rf[:, 1:], shifted=True, cfg=cfg, dlogits=d)
        _check(out, logits, ids[:, 1:], mask[:, 1:], rf[:, 1:], cfg, scored=T - 1)
        assert float(big[0]) == 7 and bool((big[1 + d.numel():] == 7).all())


def test_status_from_log_probs(cuda):
    """A problem's status word says what its kernels raised, from log-probs as well: nothing, whatever lay in the
    memory that the call was given."""
    P, T = 5, 9
    lp = -torch.rand(2 * P, T, device=cuda)
    for form in (G.preference_logps_value_and_grad, G.preference_loss_from_logps):
        dirty = [torch.full((2 + 4 * P,), -1, dtype=torch.int32, device=cuda) for _ in range(64)]
        del dirty  # the next allocations of this size
        out = form(lp, None)
        torch.cuda.synchronize()
        assert G.ops.check_device_status(out["problem"]) == 0


def test_forward_mode_cotangents_are_refused(cuda):
    import torch.autograd.forward_ad as fwd

    logits, ids, mask, rf = _case(1, 5, 40, 35, cuda)
    x = logits.clone().requires_grad_(True)
    loss = G.preference_loss(x, ids, mask, rf[:, 1:])["loss"]
    lp = torch.full((2, 5), -1.0, device=cuda, requires_grad=True)
    from_lp = G.preference_loss_from_logps(lp, mask, rf)["loss"]
    one = torch.ones((), device=cuda)
    with fwd.dual_level():
        for out, leaf in ((loss, x), (from_lp, lp)):
            dual = fwd.make_dual(one, one)
            if leaf is x:
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    torch.autograd.grad(out, leaf, dual, retain_graph=True)
            else:  # linear in the cotangent: its tangent comes through
                (g,) = torch.autograd.grad(out, leaf, dual, retain_graph=True)
                value, tangent = fwd.unpack_dual(g)
                assert torch.equal(value, tangent)
        with pytest.raises((NotImplementedError, RuntimeError)):
            G.preference_loss(fwd.make_dual(logits, torch.ones_like(logits)), ids, mask, rf[:, 1:])
        with pytest.raises((NotImplementedError, RuntimeError)):
            G.preference_loss_from_logps(fwd.make_dual(lp.detach(), torch.ones_like(lp)), mask, rf)
    (g,) = torch.autograd.grad(loss, x)
    assert torch.isfinite(g).all() and g.any()
