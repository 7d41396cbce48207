"""Embedding lookup and its gradient by sorted tokens against 64-bit forms: types, odd widths, strides, no tokens, one
id for all of them, ids of other shards and outside the vocabulary, accumulation into a tied head's gradient."""
import pytest
import torch

import mllm_jax_b200 as G
from mllm_jax_b200 import _lib
from tests import operator_reference as R

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rows(n, h, dtype, seed, dev, stride=None, offset=0):
    """[n, h] with rows `stride` apart, `offset` elements into a buffer filled with NaN."""
    stride = stride or h
    g = torch.Generator().manual_seed(seed)
    buf = torch.full((n * stride + offset + 8,), float("nan"), dtype=dtype, device=dev)
    view = buf[offset:offset + n * stride].view(n, stride)[:, :h]
    view.copy_(torch.randn(n, h, generator=g).to(dtype))
    return view


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,H,stride,offset", [
    (1, 1, 1, None, 0), (7, 5, 3, None, 0), (33, 129, 64, None, 0), (100, 1000, 897, None, 0), (64, 50, 200, 203, 1),
    (40, 90, 128, 136, 2), (4096, 4099, 1024, None, 0), (3000, 777, 1792, 1800, 0),
])
def test_lookup(cuda, dtype, N, V, H, stride, offset):
    w = _rows(V, H, dtype, N + H, cuda, stride, offset)
    g = torch.Generator().manual_seed(N)
    ids = torch.randint(0, V, (N,), generator=g)
    ids[0], ids[-1] = V - 1, 0
    for scale in (1.0, 59.75, -0.3):
        for t in (ids.to(torch.int32).to(cuda), ids.to(cuda)):
            out = G.embedding_lookup(t, w, scale=scale)
            assert out.dtype == dtype and out.shape == (N, H)
            ref = w[t.long()].double() * torch.tensor(scale, dtype=torch.float32).double()
            # one product rounded to f32, then to the type
            R.assert_within(out, ref, ref.abs() * (R.HALF_STEP[dtype] + 2.0 ** -23) + R.TINY_STEP[dtype], "lookup")


def test_lookup_shapes_shards_and_reports(cuda):
    V, H = 60, 48
    w = _rows(V, H, torch.bfloat16, 1, cuda)
    ids = torch.tensor([[3, 59, 0], [10, 44, 20]], device=cuda)
    whole = G.embedding_lookup(ids, w)
    assert whole.shape == (2, 3, H)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    parts = [G.embedding_lookup(ids, w[a:b], vocab_start=a, vocab_total=V, device_status=status) for a, b in ((0, 20), (20, 60))]
    assert torch.equal(parts[0] + parts[1], whole) and int(status.item()) == 0
    bad = torch.tensor([5, -1, 60, 2 ** 31 + 5, -2 ** 40, 7], device=cuda)
    out = G.embedding_lookup(bad, w, device_status=status)
    assert int(status.item()) == _lib.DEV_ID_IGNORED
    assert torch.equal(out[[0, 5]], w[[5, 7]]) and not out[1:5].any()
    assert G.embedding_lookup(ids[:0], w).shape == (0, 3, H)
    # NaN and infinities of the table come through, of other rows do not
    w[10, 3], w[11] = float("inf"), float("nan")
    out = G.embedding_lookup(ids, w)
    assert torch.isinf(out[1, 0, 3]) and torch.isfinite(out[0]).all()


def _grad_ref(g, ids, V, scale, start=0):
    """(sum, sum of magnitudes, most terms of a row) in 64 bits."""
    H = g.shape[-1]
    local = ids.long().reshape(-1) - start
    keep = (local >= 0) & (local < V)
    x = g.reshape(-1, H).double()[keep] * torch.tensor(scale, dtype=torch.float32).double()
    z = torch.zeros(V, H, dtype=torch.float64, device=g.device)
    n = torch.bincount(local[keep], minlength=V).double()
    return z.index_add(0, local[keep], x), z.index_add(0, local[keep], x.abs()), n


def _grad_bound(ref, mag, n, dtype):
    # at most n additions in f32 (2^-24 of the magnitudes each) and the scale's product, then one rounding
    return mag * (n[:, None] + 2) * 2.0 ** -24 + ref.abs() * R.HALF_STEP[dtype] + R.TINY_STEP[dtype]


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                             (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("N,V,H,kind", [
    (0, 5, 8, "any"), (1, 1, 1, "any"), (5, 3, 7, "any"), (31, 1000, 64, "any"), (32, 129, 64, "one"), (33, 129, 65, "one"),
    (1000, 70, 130, "any"), (1023, 512, 33, "one"), (1024, 511, 96, "one"), (5000, 4099, 256, "text"), (9001, 300000, 16, "text"),
    (40000, 151936, 24, "pad"), (33000, 2, 40, "any"),
])
def test_grad(cuda, dtype, out_dtype, N, V, H, kind):
    gen = torch.Generator().manual_seed(N + V)
    ids = torch.randint(0, V, (N,), generator=gen)
    if kind == "one":
        ids[:] = V - 1
    elif kind == "text":
        ids = (torch.rand(N, generator=gen) ** 4 * V).long()
    elif kind == "pad":
        ids[N // 3:] = 17
    ids = ids.to(torch.int32).to(cuda)
    x = _rows(N, H, dtype, N + H, cuda) if N else torch.empty(0, H, dtype=dtype, device=cuda)
    out = G.embedding_grad(x, ids, V, scale=0.7, dtype=out_dtype)
    ref, mag, n = _grad_ref(x, ids, V, 0.7)
    assert out.dtype == out_dtype
    R.assert_within(out, ref, _grad_bound(ref, mag, n, out_dtype), "dweight")
    assert not out[n == 0].any()
    again = G.embedding_grad(x, ids, V, scale=0.7, dtype=out_dtype)
    assert torch.equal(out, again), "the sums' order depends on the ids alone"
    if out_dtype == torch.float32:
        base = _rows(V, H, torch.float32, 3, cuda, stride=H + 5)
        acc = base.clone()
        view = torch.empty(V, H + 5, device=cuda)[:, :H]
        view.copy_(base)
        assert G.embedding_grad(x, ids, V, scale=0.7, out=view) is view
        assert torch.equal(view[n == 0], acc[n == 0])
        R.assert_within(view, acc.double() + ref, _grad_bound(ref, mag, n, torch.float32) + 2.0 ** -23 * (acc.double().abs() + ref.abs()),
                        "accumulated")


@pytest.mark.parametrize("H,stride,offset", [(64, 64, 0), (64, 67, 1), (63, 64, 0), (62, 62, 0)])
def test_grad_strides_shards_and_ignored_ids(cuda, H, stride, offset):
    N, V = 300, 90
    x = _rows(N, H, torch.bfloat16, 8, cuda, stride, offset)
    ids = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(2)).to(cuda)
    ids[5], ids[6], ids[7] = -1, V, 2 ** 35 + 3
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    whole = G.embedding_grad(x, ids, V, device_status=status)
    assert int(status.item()) == _lib.DEV_ID_IGNORED
    ref, mag, n = _grad_ref(x, ids, V, 1.0)
    R.assert_within(whole, ref, _grad_bound(ref, mag, n, torch.float32), "dweight")
    status.zero_()
    ids[5:8] = 0
    whole = G.embedding_grad(x, ids, V, device_status=status)
    parts = [G.embedding_grad(x, ids, b - a, vocab_start=a, vocab_total=V, device_status=status) for a, b in ((0, 31), (31, 90))]
    assert int(status.item()) == 0
    # a shard sorts other places to runs of 32: the same terms in f32, grouped differently
    ref, mag, n = _grad_ref(x, ids, V, 1.0)
    R.assert_within(torch.cat(parts), ref, _grad_bound(ref, mag, n, torch.float32), "shards")
    R.assert_within(whole, ref, _grad_bound(ref, mag, n, torch.float32), "whole")


def test_grad_keeps_non_finite_values_in_their_rows(cuda):
    x = _rows(6, 16, torch.float32, 1, cuda)
    x[2, 3], x[4] = float("inf"), float("nan")
    ids = torch.tensor([1, 0, 2, 1, 3, 0], device=cuda)
    out = G.embedding_grad(x, ids, 5)
    assert torch.isfinite(out[[0, 1, 4]]).all() and torch.isinf(out[2, 3]) and torch.isnan(out[3]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd(cuda, dtype):
    V, H = 211, 56
    w = _rows(V, H, dtype, 5, cuda).clone().requires_grad_(True)
    ids = torch.randint(0, V, (3, 50), generator=torch.Generator().manual_seed(4)).to(cuda)
    out = G.embedding_lookup(ids, w, scale=2.5)
    g = _rows(150, H, dtype, 6, cuda).reshape(3, 50, H)
    out.backward(g)
    assert w.grad.dtype == dtype
    ref, mag, n = _grad_ref(g, ids, V, 2.5)
    R.assert_within(w.grad, ref, _grad_bound(ref, mag, n, dtype), "weight.grad")
    w.grad = None
    G.embedding_lookup(ids, w).sum().backward()     # an expanded cotangent
    assert torch.equal(w.grad.float(), n[:, None].expand(V, H).float())
    assert not G.embedding_lookup(ids, w.detach()).requires_grad
    with torch.no_grad():
        assert not G.embedding_lookup(ids, w).requires_grad


def test_gradient_against_differences(cuda):
    """sum(c * out) is linear in the table: differences are exact up to the f32 sums of the comparison."""
    V, H = 9, 5
    w = _rows(V, H, torch.float32, 7, cuda)
    ids = torch.tensor([0, 3, 3, 8, 3], device=cuda)
    c = _rows(5, H, torch.float32, 8, cuda)
    grad = G.embedding_grad(c, ids, V, scale=1.5)
    for v, j in ((0, 0), (3, 2), (8, 4), (5, 1)):
        f = []
        for s in (0.5, -0.5):
            y = w.clone()
            y[v, j] += s
            f.append((G.embedding_lookup(ids, y, scale=1.5).double() * c.double()).sum().item())
        # each of the (at most five) terms is a product of f32 numbers below 16, rounded once
        assert abs(f[0] - f[1] - grad[v, j].item()) <= 2.0 ** -23 * 16 * 10


def test_streams_and_graph_replay(cuda):
    V, H, N = 5000, 320, 3000
    w = _rows(V, H, torch.bfloat16, 9, cuda)
    gen = torch.Generator().manual_seed(9)
    ids = [torch.randint(0, V, (N,), generator=gen, dtype=torch.int32).to(cuda) for _ in range(2)]
    x = _rows(N, H, torch.bfloat16, 10, cuda)
    want = [(G.embedding_lookup(i, w), G.embedding_grad(x, i, V)) for i in ids]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = (G.embedding_lookup(ids[k], w), G.embedding_grad(x, ids[k], V))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    static = ids[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = (G.embedding_lookup(static, w), G.embedding_grad(x, static, V))
    for k in (1, 0):
        static.copy_(ids[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[k][0]) and torch.equal(out[1], want[k][1])


def test_sums_added_to_a_saved_tensor_are_seen(cuda):
    """A gradient added into a tensor that autograd has saved makes that backward an error, not a wrong result."""
    V, H = 40, 16
    ids = torch.arange(5, device=cuda)
    x = _rows(5, H, torch.float32, 11, cuda)
    w = torch.ones(V, H, device=cuda, requires_grad=True)
    buf = torch.zeros(V, H, device=cuda)
    loss = (w * buf).sum()
    G.embedding_grad(x, ids, V, out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_captured_backward(cuda):
    V, H = 70, 24
    gen = torch.Generator().manual_seed(12)
    ids = [torch.randint(0, V, (4, 30), generator=gen).to(cuda) for _ in range(2)]
    c = _rows(120, H, torch.bfloat16, 12, cuda).reshape(4, 30, H)
    want = [G.embedding_grad(c, i, V, scale=2.0, dtype=torch.bfloat16) for i in ids]
    w = _rows(V, H, torch.bfloat16, 13, cuda).clone().requires_grad_(True)
    static = ids[0].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        (grad,) = torch.autograd.grad(G.embedding_lookup(static, w, scale=2.0), w, c)
    for k in (1, 0):
        static.copy_(ids[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want[k])


@pytest.mark.parametrize("H,out_dtype", [(2048, torch.float32), (2047, torch.float32), (4096, torch.bfloat16)])
def test_grad_of_many_wide_rows(cuda, H, out_dtype):
    """So many wide rows may have tokens that only the first ones get their zeros beside the sort."""
    V, N = 30000, 9001
    gen = torch.Generator().manual_seed(14)
    ids = torch.randint(0, V, (N,), generator=gen)
    ids[100:300], ids[4000:4020], ids[-1], ids[0] = 29990, 20000, V - 1, 0
    ids = ids.to(cuda)
    x = _rows(N, H, torch.bfloat16, 14, cuda)
    poison = torch.full((V, H), float("nan"), dtype=out_dtype, device=cuda)  # the next allocation of this size
    del poison
    out = G.embedding_grad(x, ids, V, scale=0.5, dtype=out_dtype)
    ref, mag, n = _grad_ref(x, ids, V, 0.5)
    R.assert_within(out, ref, _grad_bound(ref, mag, n, out_dtype), "dweight")


def test_grad_beyond_2_to_31_words(cuda):
    """Rows of an odd width, more elements than 32 bits of them count."""
    V, H = 70001, 32769
    ids = torch.tensor([0, 65535, V - 1, 65533, 65534], device=cuda)
    x = _rows(5, H, torch.bfloat16, 15, cuda)
    out = G.embedding_grad(x, ids, V, dtype=torch.bfloat16)
    assert torch.equal(out[ids], x)
    out[ids] = 0
    assert not any(part.any() for part in out.split(4096))


@pytest.mark.parametrize("N", [0, 40, 9000])
@pytest.mark.parametrize("H,stride,offset", [(63, 66, 1), (64, 72, 0), (2047, 2049, 3), (5, 5, 1), (5, 5, 0)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_grad_into_strided_rows(cuda, N, H, stride, offset, out_dtype):
    """The whole gradient into rows some distance apart, at any address (through the C ABI): what lies between and
    behind them stays."""
    from mllm_jax_b200 import _lib
    V = 21001 if H > 2000 else 1003
    gen = torch.Generator().manual_seed(16)
    ids = torch.randint(0, V, (N,), generator=gen, dtype=torch.int32).to(cuda)
    x = _rows(N, H, torch.bfloat16, 16, cuda) if N else torch.empty(0, H, dtype=torch.bfloat16, device=cuda)
    buf = torch.full((offset + V * stride + 8,), 7.0, dtype=out_dtype, device=cuda)
    a = _lib.EmbeddingArgs()
    a.n_tokens, a.vocab, a.hidden, a.weight_stride, a.token_stride, a.scale = N, V, H, stride, H, 1.0
    a.dtype, a.out_dtype = _lib.DTYPE_BF16, _lib.DTYPE_F32 if out_dtype is torch.float32 else _lib.DTYPE_BF16
    work = torch.empty(_lib.load().mllm_grpo_embedding_workspace_bytes(N, H, V), dtype=torch.uint8, device=cuda)
    a.ids, a.grad_out, a.workspace = ids.data_ptr(), x.data_ptr(), work.data_ptr()
    a.dweight = buf.data_ptr() + offset * buf.element_size()
    _lib.launch("mllm_grpo_embedding_grad", a, x.device)
    rows = buf[offset:offset + V * stride].view(V, stride)
    ref, mag, n = _grad_ref(x, ids.long(), V, 1.0)
    R.assert_within(rows[:, :H], ref, _grad_bound(ref, mag, n, out_dtype), "dweight")
    assert bool((rows[:, H:] == 7).all()) and bool((buf[:offset] == 7).all()) and bool((buf[offset + V * stride:] == 7).all())


@pytest.mark.parametrize("N", [5, 1100])
def test_grad_in_several_fills(cuda, N):
    """More than 2^31 words of two bytes, in rows some distance apart at an odd address, so that zeros go out an element at
    a time in several launches: all of them beside the sort, or (more tokens) most behind it."""
    from mllm_jax_b200 import _lib
    V, H, stride = 70001, 32769, 32771
    per_launch = 2 ** 31 // H
    gen = torch.Generator().manual_seed(20)
    ids = torch.randperm(V, generator=gen)[:N]
    first = 0 if N == 5 else ((128 << 20) + N * 4096) // (H * 2) + 1   # rows whose zeros are written beside the sort
    assert (N * H * 2 > 64 << 20) == (first > 0)
    edges = torch.tensor([per_launch - 1, per_launch, V - 1, 0] if N == 5 else
                         [first - 1, first, first + per_launch - 1, first + per_launch, V - 1, 0])
    ids = torch.cat([ids[~torch.isin(ids, edges)][:N - len(edges)], edges]).to(cuda)
    x = _rows(ids.numel(), H, torch.float16, 20, cuda)
    buf = torch.full((1 + V * stride,), 7.0, dtype=torch.float16, device=cuda)
    a = _lib.EmbeddingArgs()
    n = ids.numel()
    a.n_tokens, a.vocab, a.hidden, a.weight_stride, a.token_stride, a.scale = n, V, H, stride, H, 1.0
    a.dtype = a.out_dtype = _lib.DTYPE_F16
    work = torch.empty(_lib.load().mllm_grpo_embedding_workspace_bytes(n, H, V), dtype=torch.uint8, device=cuda)
    ids32 = ids.to(torch.int32)
    a.ids, a.grad_out, a.workspace, a.dweight = ids32.data_ptr(), x.data_ptr(), work.data_ptr(), buf.data_ptr() + 2
    _lib.launch("mllm_grpo_embedding_grad", a, x.device)
    rows = buf[1:].view(V, stride)
    assert torch.equal(rows[ids, :H], x)
    rows[ids, :H] = 0
    assert not any(part.any() for part in rows[:, :H].split(4096))
    assert bool((rows[:, H:] == 7).all()) and float(buf[0]) == 7


@pytest.mark.parametrize("N", [65537, 131072, 200003])
@pytest.mark.parametrize("V", [300, 100000, 300000])   # one, two and three digits
@pytest.mark.parametrize("kind", ["any", "one", "pad"])
def test_grad_of_many_tokens(cuda, N, V, kind):
    """More than 65536 tokens: a CTA of the sort has several tiles."""
    gen = torch.Generator().manual_seed(N + V)
    ids = torch.randint(0, V, (N,), generator=gen)
    if kind == "one":
        ids[:] = V - 1
    elif kind == "pad":
        ids[N // 3:] = 17
        ids[5], ids[N - 1] = V - 1, 0
    ids = ids.to(cuda)
    x = _rows(N, 16, torch.bfloat16, N, cuda)
    out = G.embedding_grad(x, ids, V)
    ref, mag, n = _grad_ref(x, ids, V, 1.0)
    R.assert_within(out, ref, _grad_bound(ref, mag, n, torch.float32), "dweight")
    assert torch.equal(out, G.embedding_grad(x, ids, V))


@pytest.mark.parametrize("H,dtype", [(4096, torch.bfloat16), (1030, torch.bfloat16), (1028, torch.float32), (1033, torch.float16)])
def test_grad_added_to_many_heavy_rows(cuda, H, dtype):
    """Sums added to a table whose rows have tens of tokens each, its columns in several parts."""
    N, V = 20011, 431
    gen = torch.Generator().manual_seed(21)
    ids = (torch.rand(N, generator=gen) ** 2 * (V - 3)).long()   # a few hundred rows, the last three without tokens
    ids[4000:7000] = 11
    ids = ids.to(cuda)
    x = _rows(N, H, dtype, 21, cuda)
    base = _rows(V, H, torch.float32, 22, cuda)
    out = base.clone()
    assert G.embedding_grad(x, ids, V, scale=1.5, out=out) is out
    ref, mag, n = _grad_ref(x, ids, V, 1.5)
    assert int((n > 16).sum()) > 200
    R.assert_within(out, base.double() + ref, _grad_bound(ref, mag, n, torch.float32) + 2.0 ** -23 * (base.double().abs() + ref.abs()), "accumulated")
    assert torch.equal(out[V - 3:], base[V - 3:])
    R.assert_within(G.embedding_grad(x, ids, V, scale=1.5), ref, _grad_bound(ref, mag, n, torch.float32), "new")


def test_forward_mode_tangents_are_refused(cuda):
    """A tensor that carries a forward-mode tangent is an error, not a result that has lost it: in the lookup, with and
    without gradients recorded, in its gradient, and in a backward pass whose cotangent has one."""
    import torch.autograd.forward_ad as fwd

    V, H = 11, 8
    w, c = _rows(V, H, torch.float32, 30, cuda), _rows(5, H, torch.float32, 31, cuda)
    ids = torch.tensor([0, 3, 3, 10, 7], device=cuda)
    leaf = w.clone().requires_grad_(True)
    out = G.embedding_lookup(ids, leaf)
    with fwd.dual_level():
        dual, cotangent = fwd.make_dual(w, torch.ones_like(w)), fwd.make_dual(c, torch.ones_like(c))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            G.embedding_lookup(ids, dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            G.embedding_lookup(ids, dual)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            G.embedding_grad(cotangent, ids, V)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, leaf, cotangent, retain_graph=True)
        assert torch.equal(G.embedding_lookup(ids, w), w[ids])   # a tensor without one
    (g,) = torch.autograd.grad(out, leaf, c)
    assert torch.equal(g, G.embedding_grad(c, ids, V))
