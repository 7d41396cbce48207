"""Block-scaled e4m3: quantising, the product, and the lm_head folded into the loss statistics, against 64-bit forms."""
import pytest
import torch

import mllm_jax_b200 as G
from mllm_jax_b200.linear_loss import lm_head_forward
from tests import operator_reference as R

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _x(r, c, dtype, seed, dev, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(r, c, generator=g) * torch.exp(spread * torch.randn(r, 1, generator=g))).to(dtype).to(dev)


def _check_quantized(q, x, block):
    values, scales, y = R.quantize(x, block[0])
    assert torch.equal(q.scales, scales.to(q.scales.device))
    got = q.values.double()
    if x.dtype == torch.float32:
        # a quotient within 2^-19 of a border may fall to either side: half a step and that much more
        a = y.abs().clamp(2.0 ** -6, 448)
        half = torch.exp2(torch.floor(torch.log2(a)) - 4)
        R.assert_within(got, y, half + 2.0 ** -18 * y.abs(), "values")
    else:
        assert torch.equal(torch.isnan(got), torch.isnan(values))
        fine = ~torch.isnan(values)
        assert torch.equal(got[fine], values[fine])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block", [(1, 128), (128, 128)])
@pytest.mark.parametrize("r,c", [(1, 1), (1, 128), (3, 127), (129, 130), (128, 256), (37, 1000), (300, 515), (257, 2048), (5, 16)])
def test_quantize(cuda, dtype, block, r, c):
    x = _x(r, c, dtype, r * 1000 + c, cuda)
    q = G.quantize_fp8(x, block=block)
    assert q.values.shape == (r, c) and q.values.dtype == torch.float8_e4m3fn
    _check_quantized(q, x, block)


def test_quantize_borders(cuda):
    """Quotients that are exactly the middle between two e4m3 values go to the even one, whatever the block's maximum."""
    for dtype in (torch.bfloat16, torch.float16):
        tops = torch.arange(129, 256, dtype=torch.float32)            # 8-bit maxima
        x = torch.zeros(tops.numel(), 128)
        x[:, 0] = tops
        x[:, 1:] = torch.arange(1, 128, dtype=torch.float32) * 2      # and all even numbers below
        x = x.to(dtype).to(cuda)
        assert (x.float().amax(1) <= 255).all()
        _check_quantized(G.quantize_fp8(x), x, (1, 128))
        _check_quantized(G.quantize_fp8(-x * 2.0 ** -9), -x * 2.0 ** -9, (1, 128))


@pytest.mark.parametrize("block", [(1, 128), (128, 128)])
def test_quantize_special_values(cuda, block):
    x = _x(130, 300, torch.bfloat16, 3, cuda)
    x[0] = 0                                        # a zero row; with tall blocks just small values
    x[1] *= 1e-38                                   # subnormal results
    x[2, :128] = 3e38
    x[5, 7] = float("nan")
    q = G.quantize_fp8(x, block=block)
    _check_quantized(q, x, block)
    z = torch.zeros(130, 300, device=cuda)
    q = G.quantize_fp8(z, block=block)
    assert not q.values.float().any() and (q.scales == 2.0 ** -126).all()
    x[9, 200] = float("-inf")
    q = G.quantize_fp8(x, block=block)
    assert torch.isinf(q.scales[9 if block[0] == 1 else 0, 1]) and torch.isnan(q.dequantize()[9, 200])


def test_quantize_strides_and_offsets(cuda):
    for shift, ld in ((0, 400), (1, 401), (2, 404), (4, 408)):
        big = torch.full((50 * ld + 8,), float("nan"), dtype=torch.bfloat16, device=cuda)
        view = big[shift:shift + 50 * ld].view(50, ld)[:, :264]
        view.copy_(_x(50, 264, torch.bfloat16, 5, cuda))
        for block in ((1, 128), (128, 128)):
            _check_quantized(G.quantize_fp8(view, block=block), view, block)
    t = _x(64, 96, torch.float32, 6, cuda).t()     # not row-major: laid out first
    _check_quantized(G.quantize_fp8(t), t, (1, 128))
    assert G.quantize_fp8(torch.empty(0, 40, device=cuda)).values.shape == (0, 40)


def _operands(M, N, K, seed, dev):
    x = _x(M, K, torch.bfloat16, seed, dev, 0.5)
    w = _x(N, K, torch.bfloat16, seed + 1, dev, 0.5) * (K ** -0.5)
    return G.quantize_fp8(x), G.quantize_fp8(w, block=(128, 128))


SHAPES = [
    (1, 1, 16), (1, 128, 128), (1, 1000, 896), (2, 4099, 272), (7, 300, 3584), (8, 129, 64), (9, 640, 1040), (16, 2048, 512),
    (17, 257, 384), (33, 513, 160), (64, 1024, 2048), (128, 256, 128), (129, 255, 144), (300, 1111, 400), (257, 4096, 1792),
    (1000, 20000, 256), (257, 19001, 144), (300, 30000, 16), (128, 40000, 400), (140, 38000, 1056),
]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("out", TYPES)
def test_matmul(cuda, M, N, K, out):
    x, w = _operands(M, N, K, M + N + K, cuda)
    y = G.fp8_matmul(x, w, out_dtype=out)
    assert y.shape == (M, N) and y.dtype == out
    ref, mag = R.product(x.values, x.scales, w.values, w.scales)
    R.assert_within(y, ref, R.product_bound(ref, mag, K) + ref.abs() * R.HALF_STEP[out] + R.TINY_STEP[out], f"{M}x{N}x{K}")
    assert torch.equal(y, G.fp8_matmul(x, w, out_dtype=out))


@pytest.mark.parametrize("M", [1, 12, 200])
def test_matmul_views(cuda, M):
    """Operands that are rows of wider buffers, an output with guards around its rows, a tensor quantised on the way."""
    N, K, ld = 333, 208, 256
    x, w = _operands(M, N, K, 77, cuda)
    wide = lambda t, r: torch.full((r, ld), 0x7F, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)  # noqa: E731  (NaNs)
    bx, bw = wide(x, M), wide(w, N)
    bx[:, :K].copy_(x.values)
    bw[:, :K].copy_(w.values)
    want = G.fp8_matmul(x, w, out_dtype=torch.float32)
    got = G.fp8_matmul(G.Fp8Blocks(bx[:, :K], x.scales, (1, 128)), G.Fp8Blocks(bw[:, :K], w.scales), out_dtype=torch.float32)
    assert torch.equal(got, want)
    for dtype, off, pad in ((torch.bfloat16, 1, 3), (torch.float32, 0, 0), (torch.float32, 4, 11)):
        buf = torch.full((M * (N + pad) + off + 8,), 7.0, dtype=dtype, device=cuda)
        view = buf[off:off + M * (N + pad)].view(M, N + pad)[:, :N]
        assert G.fp8_matmul(x, w, out=view) is view
        assert torch.equal(view, want.to(dtype))
        assert (buf[:off] == 7).all() and (buf[off:off + M * (N + pad)].view(M, -1)[:, N:] == 7).all() and (buf[-8:] == 7).all()
    raw = _x(M, K, torch.bfloat16, 77, cuda, 0.5)
    assert torch.equal(G.fp8_matmul(raw, w, out_dtype=torch.float32), want)
    assert G.fp8_matmul(G.quantize_fp8(raw[:0]), w).shape == (0, N)


@pytest.mark.parametrize("M", [3, 150])
def test_matmul_non_finite(cuda, M):
    """A NaN or an infinite block reaches its own row or its own columns and no others."""
    N, K = 300, 256
    x, w = _operands(M, N, K, 80, cuda)
    ref, mag = R.product(x.values, x.scales, w.values, w.scales)
    x.values[1, 5] = float("nan")
    w.scales[1, 0] = float("inf")
    y = G.fp8_matmul(x, w, out_dtype=torch.float32).double()
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[:, 128:256]).any()
    rows = [m for m in range(M) if m != 1]
    for cols in (slice(0, 128), slice(256, 300)):
        R.assert_within(y[rows][:, cols], ref[rows][:, cols], R.product_bound(ref, mag, K)[rows][:, cols] + 2.0 ** -24 * ref[rows][:, cols].abs())


HEADS = [(1, 1, 64, 256, None), (1, 5, 16, 7, None), (2, 75, 192, 1000, None), (1, 130, 128, 10240, None), (3, 50, 896, 4099, None),
         (1, 300, 80, 2500, 30.0)]


@pytest.mark.parametrize("B,T,H,V,cap", HEADS)
def test_folded_head(cuda, B, T, H, V, cap):
    g = torch.Generator().manual_seed(B + T + H + V)
    hidden = torch.randn(B, T, H, generator=g).to(torch.bfloat16).to(cuda)
    w = G.quantize_fp8((torch.randn(V, H, generator=g) * 3 / H ** 0.5).to(cuda), block=(128, 128))
    ids = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32).to(cuda)
    edges = [0, V - 1] + [e for e in (127, 128, 255, 256, 511, 2047) if e < V]
    ids.view(-1)[:min(len(edges), B * T)] = torch.tensor(edges[:B * T], dtype=torch.int32, device=cuda)
    out = lm_head_forward(hidden, w, ids, cfg=G.LossConfig(softcap=cap))
    torch.cuda.synchronize()
    assert G.ops.check_device_status(out["problem"]) == 0
    q = G.quantize_fp8(hidden.view(-1, H))
    y, mag = R.product(q.values, q.scales, w.values, w.scales)
    err = R.product_bound(y, mag, H)
    if cap:
        y = cap * torch.tanh(y / cap)
        err = err + 2.6e-7 * cap
    lse = torch.logsumexp(y, 1)
    lp = y.gather(1, ids.view(-1).long()[:, None])[:, 0] - lse
    p = torch.exp(y - lse[:, None])
    ent = -(p * (y - lse[:, None])).sum(1)
    worst = err.amax(1)
    # a term of the sum: its exponent is rounded twice (2^-19 each while |y log2e| <= 64), ex2.approx 2^-22, and at
    # most V / 64 + 600 additions in f32; the logarithm, the merged maximum and the result are f32 numbers below 64
    e_sum = 3 * 2.0 ** -20 + 2.0 ** -22 + (min(V, 16384) / 64 + 600) * 2.0 ** -24 + 4 * 2.0 ** -19
    R.assert_within(out["lse"].view(-1), lse, worst + e_sum, "lse")
    R.assert_within(out["per_token_logps"].view(-1), lp, 2 * worst + e_sum, "log-probs")
    # the two-step form (combine after the partials, as a loss or a sharded head takes it) agrees
    full = lm_head_forward(hidden, w, ids, None, torch.ones(B, device=cuda), cfg=G.LossConfig(softcap=cap))
    R.assert_within(full["per_token_logps"].view(-1), out["per_token_logps"].view(-1).double(), 4 * 2.0 ** -19, "combined")
    R.assert_within(full["token_entropy"].view(-1), out["token_entropy"].view(-1).double(), 4 * 2.0 ** -19, "combined entropy")
    cold = lm_head_forward(hidden, w, ids, cfg=G.LossConfig(softcap=cap, temperature=0.5, compute_entropy=False))
    assert cold["token_entropy"] is None and torch.equal(cold["per_token_logps"], 2 * out["per_token_logps"])
    # entropy = lse - U / S: U has the terms' relative error times |y|
    R.assert_within(out["token_entropy"].view(-1), ent, 2 * worst * (1 + y.abs().amax(1)) + e_sum * (2 + (p * y.abs()).sum(1)), "entropy")


def test_folded_head_feeds_the_loss_and_shards(cuda):
    """The whole forward of the token loss on an 8-bit head equals the loss on its dequantised logits; two vocabulary
    shards merged by hand give the unsharded log-probs."""
    B, T, H, V = 2, 40, 256, 1536
    g = torch.Generator().manual_seed(5)
    hidden = torch.randn(B, T, H, generator=g).to(torch.bfloat16).to(cuda)
    wt = (torch.randn(V, H, generator=g) * 0.2).to(cuda)
    w = G.quantize_fp8(wt, block=(128, 128))
    ids = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32).to(cuda)
    mask = (torch.rand(B, T, generator=g) < 0.7).float().to(cuda)
    adv = torch.randn(B, generator=g).to(cuda)
    old = lm_head_forward(hidden, w, ids)["per_token_logps"] + 0.1
    out = lm_head_forward(hidden, w, ids, mask, adv, mask.sum(), old)
    q = G.quantize_fp8(hidden.view(-1, H))
    y = R.product(q.values, q.scales, w.values, w.scales)[0].view(B, T, V)
    lp = torch.log_softmax(y, -1).gather(-1, ids.long()[..., None])[..., 0]
    ratio = torch.exp(lp - old.double())
    a = adv.double()[:, None]
    loss = -(torch.minimum(ratio * a, ratio.clamp(0.8, 1.3) * a) * mask).sum() / mask.sum()
    assert abs(float(out["loss"]) - float(loss)) <= 1e-4 * abs(float(loss)) + 1e-6
    from mllm_jax_b200 import _lib
    from mllm_jax_b200.fp8 import _bind
    lib = _lib.load()
    parts = []
    for a0, b0 in ((0, 640), (640, V)):
        shard = G.quantize_fp8(wt[a0:b0], block=(128, 128))
        args = _bind(q, shard)
        buf = torch.empty(lib.mllm_lm_head_fp8_partials_bytes(B * T, b0 - a0), dtype=torch.uint8, device=cuda)
        args.vocab_start, args.vocab_total = a0, V
        args.chosen_ids, args.partials = ids.data_ptr(), buf.data_ptr()
        _lib.call("mllm_lm_head_fp8_partials", args, torch.cuda.current_stream().cuda_stream)
        parts.append(buf[:16 * B * T].view(torch.float32).view(B * T, 4).double())
    top = torch.maximum(parts[0][:, 0], parts[1][:, 0])
    total = sum(p[:, 1] * torch.exp(p[:, 0] - top) for p in parts)
    merged = sum(p[:, 3] for p in parts) - top - total.log()
    assert (merged - lp.view(-1)).abs().max() <= 1e-4


def test_streams_and_graph_replay(cuda):
    for M in (4, 200):
        x, w = _operands(M, 3000, 512, 90, cuda)
        x2 = G.quantize_fp8(_x(M, 512, torch.bfloat16, 91, cuda))
        want = [G.fp8_matmul(t, w) for t in (x, x2)]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
        for _ in range(3):
            for k, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[k] = G.fp8_matmul((x, x2)[k], w)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        raw = _x(M, 512, torch.bfloat16, 90, cuda, 0.5)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = G.fp8_matmul(raw, w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0])
        raw.copy_(_x(M, 512, torch.bfloat16, 91, cuda))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[1])


def test_product_reports_and_marks_what_it_writes(cuda):
    x, w = _operands(20, 300, 256, 95, cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.empty(20, 300, dtype=torch.bfloat16, device=cuda)
    version = out._version
    assert G.fp8_matmul(x, w, out=out, device_status=status) is out
    assert out._version > version and int(status) == 0 and torch.equal(out, G.fp8_matmul(x, w))
    with pytest.raises(ValueError, match="device_status"):
        G.fp8_matmul(x, w, device_status=torch.zeros(1, dtype=torch.int32))


def test_folded_head_clamps_ids_beyond_32_bits(cuda):
    B, T, H, V = 1, 6, 64, 300
    hidden = _x(T, H, torch.bfloat16, 96, cuda).view(B, T, H)
    w = G.quantize_fp8(_x(V, H, torch.bfloat16, 97, cuda), block=(128, 128))
    ids = torch.tensor([[0, 5, 2 ** 32 + 5, -(2 ** 32) + 5, V, V - 1]], device=cuda)
    near = torch.tensor([[0, 5, V - 1, 0, V - 1, V - 1]], device=cuda)
    out, want = lm_head_forward(hidden, w, ids), lm_head_forward(hidden, w, near)
    assert torch.equal(out["per_token_logps"], want["per_token_logps"])
    assert int(out["problem"].device_status) == 1 and int(want["problem"].device_status) == 0


@pytest.mark.parametrize("M,N,K", [(1, 40003, 16), (3, 38017, 288), (8, 40000, 1024), (2, 38000, 1296), (5, 4800, 528), (7, 4736, 400)])
def test_few_rows_split_by_the_inner_size(cuda, M, N, K):
    """Each way of giving K to the warps of a CTA: one, two, four and eight of them."""
    x, w = _operands(M, N, K, 98, cuda)
    ref, mag = R.product(x.values, x.scales, w.values, w.scales)
    out = G.fp8_matmul(x, w, out_dtype=torch.float32)
    R.assert_within(out, ref, R.product_bound(ref, mag, K) + ref.abs() * R.HALF_STEP[torch.float32], f"{M}x{N}x{K}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,c", [(40001, 129), (3001, 546), (777, 2976), (70, 1)])
def test_quantize_rows_by_the_four(cuda, dtype, r, c):
    """Rows whose blocks do not come in fours, odd widths, more than one wave of CTAs."""
    x = _x(r, c, dtype, 99, cuda)
    _check_quantized(G.quantize_fp8(x), x, (1, 128))


@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("M,N", [(33, 300), (300, 515), (260, 33000)])
@pytest.mark.parametrize("shift", range(8))
def test_product_at_every_address(cuda, out_dtype, M, N, shift):
    """Rows of out that start at every place between 16-byte boundaries, with values behind them that stay."""
    if M * N > 10 ** 6 and shift not in (0, 1, 6):
        return
    x, w = _operands(M, N, 144, 101, cuda)
    want = G.fp8_matmul(x, w, out_dtype=out_dtype)
    for stride in (N + shift, N + 8 + (shift & 3)):
        buf = torch.full((shift + M * stride + 16,), 3.0, dtype=out_dtype, device=cuda)
        out = buf[shift:shift + M * stride].view(M, stride)
        G.fp8_matmul(x, w, out=out[:, :N])
        assert torch.equal(out[:, :N], want)
        assert bool((out[:, N:] == 3).all()) and bool((buf[:shift] == 3).all()) and bool((buf[shift + M * stride:] == 3).all())


def test_call_status_beside_a_running_one(cuda):
    """The call's own bits are set, not added up, and the caller's running word collects them (through the C ABI)."""
    from mllm_jax_b200 import _lib
    from mllm_jax_b200.fp8 import _bind
    N, V, H = 5, 200, 32
    x, w = _operands(N, V, H, 102, cuda)
    buf = torch.empty(_lib.load().mllm_lm_head_fp8_partials_bytes(N, V), dtype=torch.uint8, device=cuda)
    mine, running = torch.full((1,), 77, dtype=torch.int32, device=cuda), torch.full((1,), 4, dtype=torch.int32, device=cuda)
    a = _bind(x, w)
    a.partials, a.call_status, a.device_status = buf.data_ptr(), mine.data_ptr(), running.data_ptr()
    for ids, bits, total in (([0, 1, 2, 3, 4], 0, 4), ([0, 1, 2, 3, V], 1, 5), ([0, 1, 2, 3, 4], 0, 5)):
        chosen = torch.tensor(ids, dtype=torch.int32, device=cuda)
        a.chosen_ids = chosen.data_ptr()
        _lib.launch("mllm_lm_head_fp8_partials", a, x.device)
        assert int(mine) == bits and int(running) == total


def test_folded_head_workspaces_and_refusals(cuda):
    from mllm_jax_b200 import _lib
    B, T, H, V = 2, 9, 48, 500
    wide = _x(B * T, 2 * H, torch.bfloat16, 103, cuda).view(B, T, 2 * H)
    w = G.quantize_fp8(_x(V, H, torch.bfloat16, 104, cuda), block=(128, 128))
    ids = torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(105)).to(cuda)
    want = lm_head_forward(wide[..., :H].contiguous(), w, ids)
    room = torch.full((_lib.load().mllm_lm_head_fp8_partials_bytes(B * T, V) + 32,), 9, dtype=torch.uint8, device=cuda)
    for hidden, kw in ((wide[..., :H], {}), (wide[..., :H].transpose(1, 2).contiguous().transpose(1, 2), {}),
                       (wide[..., :H], dict(workspace=room[:-32]))):
        got = lm_head_forward(hidden, w, ids, **kw)
        for k in ("per_token_logps", "token_entropy", "lse"):
            assert torch.equal(got[k], want[k])
        assert int(got["problem"].device_status) == 0
    assert bool((room[-32:] == 9).all())
    with pytest.raises(ValueError, match="multiple of 16"):
        lm_head_forward(wide[..., :40], G.quantize_fp8(_x(V, 40, torch.bfloat16, 104, cuda), block=(128, 128)), ids)
    with pytest.raises(ValueError, match="workspace"):
        lm_head_forward(wide[..., :H], w, ids, workspace=room[:64])
    with pytest.raises(ValueError, match="blocks"):
        lm_head_forward(wide[..., :H], G.quantize_fp8(_x(V, H, torch.bfloat16, 104, cuda)), ids)
    with pytest.raises(ValueError, match="do not match"):
        lm_head_forward(wide, w, ids)


@pytest.mark.parametrize("M,N,K", [(2050, 300, 272), (4200, 300, 144), (4200, 1500, 272), (2305, 2200, 128)])
def test_product_of_many_rows(cuda, M, N, K):
    """More than 2048 rows: several groups of row tiles, the last of them shorter; an odd number of row tiles for pairs."""
    x, w = _operands(M, N, K, M + N, cuda)
    ref, mag = R.product(x.values, x.scales, w.values, w.scales)
    for out_dtype in (torch.float32, torch.bfloat16):
        out = G.fp8_matmul(x, w, out_dtype=out_dtype)
        R.assert_within(out, ref, R.product_bound(ref, mag, K) + ref.abs() * R.HALF_STEP[out_dtype] + R.TINY_STEP[out_dtype], f"{M}x{N}x{K}")


# rows, width, columns, tiles of 256 columns in a range
LONG_HEADS = [(70, 64, 40000, 2), (128, 80, 76801, 3), (300, 48, 40000, 5), (2300, 64, 2000, None)]


@pytest.mark.parametrize("N,H,V,per", LONG_HEADS)
@pytest.mark.parametrize("cap", [None, 30.0])
def test_folded_head_of_several_tiles_per_range(cuda, N, H, V, per, cap):
    """Ranges of several tiles and a shorter last one, with logits that rise from tile to tile for half of the rows and
    fall for the other half, chosen columns in first and last tiles; more rows than one group of row tiles."""
    from mllm_jax_b200 import _lib
    tiles = -(-V // 256)
    if per is not None:
        entries = _lib.load().mllm_lm_head_fp8_partials_bytes(N, V) // (16 * N) - 1
        assert entries == 2 * -(-tiles // per) and tiles % per, "the case is meant for another plan"
    g = torch.Generator().manual_seed(N + V)
    side = torch.where(torch.arange(N) % 2 == 0, 1.0, -1.0)[:, None]
    hidden = torch.randn(N, H, generator=g)
    hidden[:, :16] = side
    wt = torch.randn(V, H, generator=g) * 2 / H ** 0.5
    wt[:, :16] = 0.6 * torch.arange(V)[:, None] / V          # +- 9.6 from the first column to the last
    hidden, w = hidden.to(torch.bfloat16).to(cuda), G.quantize_fp8(wt.to(cuda), block=(128, 128))
    ids = torch.randint(0, V, (N,), generator=g, dtype=torch.int32)
    edges = [0, V - 1, 255, 256, 511, 512, V - 257, (tiles - 1) * 256, V // 2, 1279, 1280]
    ids[:len(edges)] = torch.tensor(edges, dtype=torch.int32)
    ids = ids.to(cuda)
    out = lm_head_forward(hidden, w, ids, cfg=G.LossConfig(softcap=cap))
    torch.cuda.synchronize()
    assert G.ops.check_device_status(out["problem"]) == 0
    q = G.quantize_fp8(hidden)
    y, mag = R.product(q.values, q.scales, w.values, w.scales)
    worst = R.product_bound(y, mag, H).amax(1)
    if cap:
        y, worst = cap * torch.tanh(y / cap), worst + 2.6e-7 * cap
    lse = torch.logsumexp(y, 1)
    lp = y.gather(1, ids.long()[:, None])[:, 0] - lse
    p = torch.exp(y - lse[:, None])
    ent = -(p * (y - lse[:, None])).sum(1)
    # a term's exponent is rounded twice (2^-19 each while |y log2e| <= 64), ex2.approx is off by 2^-22; a thread adds up
    # 64 terms of a tile in each of two sums, and fewer than 600 additions in f32 follow from the tiles and ranges; every
    # further tile may raise the maximum, where the sum is multiplied by an ex2.approx (2^-22) of a rounded exponent a
    # (2^-23 a of a weight 2^-a: at most 2^-23) and rounded; logarithm, merged maximum and result are below 64 in f32
    e_sum = 3 * 2.0 ** -20 + 2.0 ** -22 + 664 * 2.0 ** -24 + (per or 8) * 2.0 ** -21 + 4 * 2.0 ** -19
    R.assert_within(out["lse"].view(-1), lse, worst + e_sum, "lse")
    R.assert_within(out["per_token_logps"].view(-1), lp, 2 * worst + e_sum, "log-probs")
    R.assert_within(out["token_entropy"].view(-1), ent, 2 * worst * (1 + y.abs().amax(1)) + e_sum * (2 + (p * y.abs()).sum(1)), "entropy")


def _gathered(monkeypatch, ranks, record):
    """all_gather_into_tensor of `ranks` ranks in one process: records what this call sends, or hands out what each sent."""
    import torch.distributed as dist

    def gather(parts, mine, group=None):
        if ranks == 1:
            record.append(mine.clone())
            parts.copy_(mine)
        else:
            torch.cat(record, out=parts)

    monkeypatch.setattr(dist, "get_world_size", lambda group=None: ranks)
    monkeypatch.setattr(dist, "all_gather_into_tensor", gather)


@pytest.mark.parametrize("cap", [None, 25.0])
def test_folded_head_over_a_group(cuda, monkeypatch, cap):
    """The group branch with an 8-bit weight: the merged records of two vocabulary shards, gathered rank by rank, give
    the log-probs, entropies, log-sum-exps and the loss of the whole head."""
    B, T, H, V, cut = 2, 33, 64, 2304, 896
    g = torch.Generator().manual_seed(110)
    hidden = torch.randn(B, T, H, generator=g).to(torch.bfloat16).to(cuda)
    w = G.quantize_fp8((torch.randn(V, H, generator=g) * 0.4).to(cuda), block=(128, 128))
    shards = [(0, G.Fp8Blocks(w.values[:cut], w.scales[:cut // 128])), (cut, G.Fp8Blocks(w.values[cut:], w.scales[cut // 128:]))]
    ids = torch.randint(0, V, (B, T), generator=g).to(cuda)
    ids[0, :4] = torch.tensor([0, cut - 1, cut, V - 1])
    mask, adv = torch.ones(B, T, device=cuda), torch.randn(B, generator=g).to(cuda)
    cfg = G.LossConfig(softcap=cap)
    want = lm_head_forward(hidden, w, ids, mask, adv, cfg=cfg)
    sent, group = [], object()
    _gathered(monkeypatch, 1, sent)
    for start, shard in shards:
        lm_head_forward(hidden, shard, ids, mask, adv, cfg=cfg, vocab_start=start, vocab_total=V, group=group)
    assert [t.numel() for t in sent] == [16 * B * T] * 2
    _gathered(monkeypatch, 2, sent)
    for start, shard in shards:
        for extra in ((mask, adv), ()):
            out = lm_head_forward(hidden, shard, ids, *extra, cfg=cfg, vocab_start=start, vocab_total=V, group=group)
            assert G.ops.check_device_status(out["problem"]) == 0
            # the same f32 tile sums, merged in another order: a few roundings of numbers below 64
            for k in ("per_token_logps", "token_entropy", "lse"):
                R.assert_within(out[k], want[k].double(), 6 * 2.0 ** -18, k)
            if extra:
                R.assert_within(out["loss"], want["loss"].double(), 2.0 ** -17 * (1 + float(adv.abs().max())), "loss")


def test_folded_head_over_a_process_group_of_one(cuda, tmp_path):
    import torch.distributed as dist

    B, T, H, V = 1, 20, 32, 700
    hidden = _x(T, H, torch.bfloat16, 111, cuda).view(B, T, H)
    w = G.quantize_fp8(_x(V, H, torch.bfloat16, 112, cuda), block=(128, 128))
    ids = torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(113)).to(cuda)
    want = lm_head_forward(hidden, w, ids, advantages=torch.zeros(B, device=cuda))
    dist.init_process_group("nccl", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        out = lm_head_forward(hidden, w, ids, group=dist.group.WORLD)
        torch.cuda.synchronize()
    finally:
        dist.destroy_process_group()
    for k in ("per_token_logps", "token_entropy", "lse"):
        assert torch.equal(out[k], want[k])


# rows, columns, output tiles multiplied by a CTA (pair) before it stops, whether some of the product is there
@pytest.mark.parametrize("M,N,tiles,some", [(40, 700, 0, False), (300, 515, 0, False), (260, 33001, 1, True), (2049, 33000, 0, False)])
@pytest.mark.parametrize("out_dtype", TYPES)
def test_what_a_run_out_wait_leaves_is_nan(cuda, out_dtype, M, N, tiles, some):
    """A wait that runs out makes every element that was not reached a NaN, with a status word or without one, and
    nothing outside of out is written; the next call is as ever."""
    if M * N > 10 ** 6 and out_dtype != torch.bfloat16:
        return
    from mllm_jax_b200 import _lib
    lib = _lib.load()
    x, w = _operands(M, N, 272, 120, cuda)
    want = G.fp8_matmul(x, w, out_dtype=out_dtype)
    stride = N + 3
    buf = torch.full((M * stride + 16,), 3.0, dtype=out_dtype, device=cuda)
    out = buf[8:8 + M * stride].view(M, stride)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    lib.mllm_lm_head_fp8_stop_after(tiles)
    try:
        G.fp8_matmul(x, w, out=out[:, :N], device_status=status if M != 40 else None)
        torch.cuda.synchronize()
    finally:
        lib.mllm_lm_head_fp8_stop_after(-1)
    assert M == 40 or int(status) == _lib.DEV_WAIT_TIMEOUT
    void = torch.isnan(out[:, :N])
    assert torch.equal(torch.where(void, want, out[:, :N]), want) and bool(void.any()) and bool((~void).any()) == some
    assert bool((out[:, N:] == 3).all()) and bool((buf[:8] == 3).all()) and bool((buf[8 + M * stride:] == 3).all())
    assert torch.equal(G.fp8_matmul(x, w, out_dtype=out_dtype), want)


@pytest.mark.parametrize("temperature", [0.0, 1e-60, -1.0, float("nan")])
def test_a_temperature_that_is_not_positive_is_refused(cuda, temperature):
    """By heads of both kinds, with and without the loss (1e-60 is 0 in the 32 bits that the kernels take)."""
    B, T, H, V = 1, 4, 64, 256
    hidden, plain = _x(T, H, torch.bfloat16, 114, cuda).view(B, T, H), _x(V, H, torch.bfloat16, 115, cuda)
    ids = torch.zeros(B, T, dtype=torch.int32, device=cuda)
    cfg = G.LossConfig(temperature=temperature, compute_entropy=False)
    for weight in (plain, G.quantize_fp8(plain, block=(128, 128))):
        for adv in (None, torch.ones(B, device=cuda)):
            with pytest.raises((ValueError, G.GrpoError)):
                lm_head_forward(hidden, weight, ids, advantages=adv, cfg=cfg)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_workspaces_of_any_type(cuda, monkeypatch, kind):
    """A workspace of floats serves as one of bytes, alone and where a part of it is gathered; one of the host is refused."""
    from mllm_jax_b200 import _lib
    B, T, H, V = 1, 10, 64, 512
    hidden, plain = _x(T, H, torch.bfloat16, 130, cuda).view(B, T, H), _x(V, H, torch.bfloat16, 131, cuda)
    weight = plain if kind == "bf16" else G.quantize_fp8(plain, block=(128, 128))
    ids = torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(132)).to(cuda)
    lib = _lib.load()
    nbytes = (lib.mllm_lm_head_partials_bytes if kind == "bf16" else lib.mllm_lm_head_fp8_partials_bytes)(T, V)
    room = torch.empty(nbytes // 4, device=cuda)
    sent = []
    _gathered(monkeypatch, 1, sent)
    adv = torch.zeros(B, device=cuda)
    want = lm_head_forward(hidden, weight, ids, advantages=adv)
    for extra in ({}, dict(group=object())):
        out = lm_head_forward(hidden, weight, ids, advantages=adv, workspace=room, **extra)
        for k in ("per_token_logps", "token_entropy", "lse"):
            assert torch.equal(out[k], want[k])
    assert sent[0].dtype == torch.uint8
    with pytest.raises(ValueError, match="workspace"):
        lm_head_forward(hidden, weight, ids, workspace=torch.empty(nbytes, dtype=torch.uint8))


def test_folded_head_with_a_loss_clamps_ids_beyond_32_bits(cuda):
    """As without one: such an id is the vocabulary's end and is reported, not the id that its lower 32 bits spell."""
    B, T, H, V = 1, 6, 64, 300
    hidden = _x(T, H, torch.bfloat16, 96, cuda).view(B, T, H)
    w = G.quantize_fp8(_x(V, H, torch.bfloat16, 97, cuda), block=(128, 128))
    ids = torch.tensor([[0, 5, 2 ** 32 + 5, -(2 ** 32) + 5, V, V - 1]], device=cuda)
    near = torch.tensor([[0, 5, V - 1, 0, V - 1, V - 1]], device=cuda)
    adv = torch.ones(B, device=cuda)
    out, want = (lm_head_forward(hidden, w, i, advantages=adv) for i in (ids, near))
    assert torch.equal(out["per_token_logps"], want["per_token_logps"])
    assert G.ops.check_device_status(out["problem"]) == 1 and G.ops.check_device_status(want["problem"]) == 0
