"""Preference loss, embedding table and 8-bit operators without a GPU: struct layouts, workspace sizes, the status codes
of every refused call (validation runs before any CUDA call), and the Python wrappers' refusals."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import mllm_jax_b200 as G
from mllm_jax_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = [("mllm_grpo_preference_args", _lib.PreferenceArgs), ("mllm_grpo_embedding_args", _lib.EmbeddingArgs),
           ("mllm_lm_head_fp8_quantize_args", _lib.Fp8QuantizeArgs), ("mllm_lm_head_fp8_args", _lib.Fp8Args)]


@pytest.mark.parametrize("name,mirror", STRUCTS)
def test_struct_matches_c_layout(tmp_path, name, mirror):
    fields = [f[0] for f in mirror._fields_]
    src = tmp_path / "layout.c"
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "mllm_grpo.h"', "int main(void){",
             f'printf("%zu\\n", sizeof({name}));']
    lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields]
    src.write_text("\n".join(lines + ["return 0;}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{os.path.join(ROOT, 'include')}", str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert int(out[0]) == C.sizeof(mirror)
    for f, off in zip(fields, out[1:]):
        assert getattr(mirror, f).offset == int(off), f


def _status(name, a):
    return getattr(_lib.load(), name)(C.byref(a), None)


def _pref(**kw):
    a = _lib.PreferenceArgs()
    a.struct_size = C.sizeof(a)
    a.n_pairs, a.seq_rows, a.scored_rows, a.vocab, a.row_stride = 2, 5, 4, 64, 64
    a.beta, a.total_pairs, a.grad_scale = 0.1, 2.0, 1.0
    a.logits = a.dlogits = a.chosen_ids = a.token_logps = a.loss = a.rewards = a.workspace = 0x1000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("fields,status", [
    (dict(struct_size=8), 4), (dict(n_pairs=0), 2), (dict(scored_rows=0), 2), (dict(scored_rows=6), 2), (dict(vocab=0), 2),
    (dict(row_stride=63), 2), (dict(n_pairs=1 << 30), 8), (dict(seq_rows=1 << 31), 8), (dict(kind=3), 3), (dict(kind=-1), 3),
    (dict(beta=0.0), 3), (dict(beta=float("nan")), 3), (dict(softcap=-1.0), 3), (dict(softcap=float("nan")), 3),
    (dict(label_smoothing=0.6), 3), (dict(label_smoothing=0.1, kind=1), 3), (dict(total_pairs=0.0), 3), (dict(logits=None), 1),
    (dict(chosen_ids=None), 1), (dict(loss=None), 1), (dict(rewards=None), 1), (dict(dlogits=None), 1), (dict(workspace=None), 1),
    (dict(workspace=0x1008), 5), (dict(logits=0x1001), 5), (dict(mask=0x1002), 5), (dict(ref_logps=0x1001), 5),
])
def test_preference_refusals(built_lib, fields, status):
    assert _status("mllm_grpo_preference_fwd_bwd", _pref(**fields)) == status


def test_preference_entry_points_ask_for_what_they_read(built_lib):
    lib = _lib.load()
    for name in ("fwd", "bwd", "fwd_bwd", "logps"):
        assert getattr(lib, f"mllm_grpo_preference_{name}")(None, None) == 1
    assert _status("mllm_grpo_preference_fwd", _pref(loss=None)) == 1
    assert _status("mllm_grpo_preference_bwd", _pref(dlogits=None)) == 1
    assert _status("mllm_grpo_preference_logps", _pref(token_logps=None)) == 1
    assert lib.mllm_grpo_preference_workspace_bytes(0, 4) == 0 and lib.mllm_grpo_preference_workspace_bytes(1 << 30, 4) == 0
    n = 2 * 3 * 7
    # terms, coefficients, log-sum-exps, chosen logits and the split sums of every token
    assert lib.mllm_grpo_preference_workspace_bytes(3, 7) >= 3 * 8 + 6 * 4 + n * 8 + n * 8


def _emb(**kw):
    a = _lib.EmbeddingArgs()
    a.struct_size = C.sizeof(a)
    a.n_tokens, a.vocab, a.hidden, a.weight_stride, a.token_stride, a.scale = 3, 10, 8, 8, 8, 1.0
    a.ids = a.weight = a.out = a.grad_out = a.dweight = a.workspace = 0x1000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("entry", ["lookup", "grad"])
@pytest.mark.parametrize("fields,status", [
    (dict(struct_size=8), 4), (dict(n_tokens=-1), 2), (dict(vocab=0), 2), (dict(hidden=0), 2), (dict(weight_stride=7), 2),
    (dict(token_stride=7), 2), (dict(vocab_start=-1), 2), (dict(vocab_total=9), 2), (dict(vocab=1 << 31), 8),
    (dict(n_tokens=1 << 31), 8), (dict(hidden=1 << 21, weight_stride=1 << 21, token_stride=1 << 21), 8), (dict(dtype=3), 3),
    (dict(scale=float("nan")), 3), (dict(ids=0x1002), 5), (dict(ids=None), 1), (dict(device_status=0x1001), 5),
])
def test_embedding_refusals(built_lib, entry, fields, status):
    assert _status(f"mllm_grpo_embedding_{entry}", _emb(**fields)) == status


def test_embedding_entry_points_ask_for_what_they_read(built_lib):
    lib = _lib.load()
    assert lib.mllm_grpo_embedding_lookup(None, None) == 1 and lib.mllm_grpo_embedding_grad(None, None) == 1
    for f in ("weight", "out"):
        assert _status("mllm_grpo_embedding_lookup", _emb(**{f: None})) == 1
        assert _status("mllm_grpo_embedding_lookup", _emb(**{f: 0x1001})) == 5
    for f in ("grad_out", "dweight", "workspace"):
        assert _status("mllm_grpo_embedding_grad", _emb(**{f: None})) == 1
        assert _status("mllm_grpo_embedding_grad", _emb(**{f: 0x1001})) == 5
    assert _status("mllm_grpo_embedding_grad", _emb(accumulate=1, out_dtype=0)) == 3
    assert _status("mllm_grpo_embedding_grad", _emb(out_dtype=4)) == 3
    assert _status("mllm_grpo_embedding_lookup", _emb(n_tokens=0, ids=None, weight=None, out=None)) == 0  # nothing to do
    for bad in ((-1, 8, 5), (5, 0, 5), (5, 8, 0), (1 << 31, 8, 5), (5, 8, 1 << 31)):
        assert lib.mllm_grpo_embedding_workspace_bytes(*bad) == 0
    assert lib.mllm_grpo_embedding_workspace_bytes(0, 8, 5) >= 5
    # marks of 777 rows, four lists of tokens, a record per row that may have some, the sums of 128 runs
    assert lib.mllm_grpo_embedding_workspace_bytes(4096, 100, 777) >= 777 + 4 * 4096 * 4 + 4096 * 16 + 128 * 100 * 4


def _quant(**kw):
    a = _lib.Fp8QuantizeArgs()
    a.struct_size = C.sizeof(a)
    a.rows, a.cols, a.x_stride, a.q_stride, a.block_rows = 4, 100, 100, 100, 1
    a.x = a.q = a.scales = 0x1000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("fields,status", [
    (dict(struct_size=8), 4), (dict(rows=-1), 2), (dict(cols=0), 2), (dict(x_stride=99), 2), (dict(q_stride=99), 2),
    (dict(block_rows=64), 3), (dict(dtype=3), 3), (dict(x=None), 1), (dict(q=None), 1), (dict(scales=None), 1),
    (dict(x=0x1001), 5), (dict(dtype=2, x=0x1002), 5), (dict(scales=0x1002), 5), (dict(rows=1 << 33), 8),
    (dict(cols=1 << 40, x_stride=1 << 40, q_stride=1 << 40), 8), (dict(rows=0, x=None, q=None, scales=None), 0),
])
def test_quantize_refusals(built_lib, fields, status):
    assert _status("mllm_lm_head_fp8_quantize", _quant(**fields)) == status


def _fp8(**kw):
    a = _lib.Fp8Args()
    a.struct_size = C.sizeof(a)
    a.n_rows, a.vocab, a.hidden_dim, a.hidden_stride, a.weight_stride, a.out_stride = 4, 100, 128, 128, 128, 100
    a.hidden = a.weight = a.hidden_scales = a.weight_scales = a.out = a.chosen_ids = a.partials = 0x1000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("entry", ["matmul", "partials"])
@pytest.mark.parametrize("fields,status", [
    (dict(struct_size=8), 4), (dict(n_rows=-1), 2), (dict(vocab=0), 2), (dict(hidden_dim=0), 2), (dict(hidden_stride=112), 2),
    (dict(weight_stride=112), 2), (dict(n_rows=1 << 31), 8), (dict(vocab=1 << 31, out_stride=1 << 31), 8),
    (dict(hidden_dim=120), 7), (dict(hidden_stride=136), 7), (dict(weight_stride=136), 7), (dict(hidden=None), 1),
    (dict(weight=None), 1), (dict(hidden_scales=None), 1), (dict(weight_scales=None), 1), (dict(hidden=0x1008), 5),
    (dict(weight=0x1004), 5), (dict(hidden_scales=0x1001), 5), (dict(weight_scales=0x1002), 5),
])
def test_fp8_product_refusals(built_lib, entry, fields, status):
    assert _status(f"mllm_lm_head_fp8_{entry}", _fp8(**fields)) == status


def test_fp8_entry_points_ask_for_what_they_read(built_lib):
    lib = _lib.load()
    assert _status("mllm_lm_head_fp8_matmul", _fp8(out_stride=99)) == 2
    assert _status("mllm_lm_head_fp8_matmul", _fp8(out_dtype=3)) == 3
    assert _status("mllm_lm_head_fp8_matmul", _fp8(out=None)) == 1
    assert _status("mllm_lm_head_fp8_matmul", _fp8(out=0x1001)) == 5
    assert _status("mllm_lm_head_fp8_matmul", _fp8(n_rows=0, hidden=None, hidden_scales=None, out=None)) == 0
    assert _status("mllm_lm_head_fp8_partials", _fp8(n_rows=0)) == 2
    assert _status("mllm_lm_head_fp8_partials", _fp8(chosen_ids=None)) == 1
    assert _status("mllm_lm_head_fp8_partials", _fp8(partials=None)) == 1
    assert _status("mllm_lm_head_fp8_partials", _fp8(partials=0x1008)) == 5
    assert _status("mllm_lm_head_fp8_partials", _fp8(vocab_start=1, vocab_total=100)) == 2
    assert _status("mllm_lm_head_fp8_partials", _fp8(softcap=-1.0)) == 3
    assert _status("mllm_lm_head_fp8_partials", _fp8(temperature=-1.0)) == 3
    assert _status("mllm_lm_head_fp8_partials", _fp8(temperature=0.7, token_entropy=0x1000)) == 7
    assert _status("mllm_lm_head_fp8_partials", _fp8(vocab_total=200, lse=0x1000)) == 7
    assert _status("mllm_lm_head_fp8_partials", _fp8(per_token_logps=0x1002)) == 5
    assert lib.mllm_lm_head_fp8_partials_bytes(0, 5) == 0 and lib.mllm_lm_head_fp8_partials_bytes(300, 151936) >= 300 * 16 * 2


def test_wrappers_refuse_cpu_tensors():
    bf = torch.zeros(2, 3, 8, dtype=torch.bfloat16)
    ids = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        G.preference_loss(bf, ids, ids)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        G.preference_value_and_grad(bf, ids, ids)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        G.preference_logps_value_and_grad(torch.zeros(2, 3), None)
    with pytest.raises(RuntimeError, match="CUDA"):
        G.embedding_lookup(ids, bf[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        G.embedding_grad(bf, ids, 5)
    with pytest.raises(RuntimeError, match="CUDA"):
        G.quantize_fp8(bf[0])
    q = G.Fp8Blocks(torch.zeros(2, 16, dtype=torch.float8_e4m3fn), torch.ones(2, 1), (1, 128))
    w = G.Fp8Blocks(torch.zeros(5, 16, dtype=torch.float8_e4m3fn), torch.ones(1, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        G.fp8_matmul(q, w)


def test_blocks_are_checked():
    v = torch.zeros(130, 200, dtype=torch.float8_e4m3fn)
    assert G.Fp8Blocks(v, torch.ones(2, 2)).shape == (130, 200)
    assert torch.equal(G.Fp8Blocks(v, torch.ones(130, 2), (1, 128)).dequantize(), torch.zeros(130, 200))
    with pytest.raises(ValueError, match="scales"):
        G.Fp8Blocks(v, torch.ones(1, 2))
    with pytest.raises(ValueError, match="scales"):
        G.Fp8Blocks(v, torch.ones(2, 2, dtype=torch.float64))
    with pytest.raises(ValueError, match="block"):
        G.Fp8Blocks(v, torch.ones(2, 2), (64, 128))
    with pytest.raises(TypeError, match="float8"):
        G.Fp8Blocks(v.float(), torch.ones(2, 2))


def test_preference_arguments_are_checked(built_lib):
    from mllm_jax_b200.preference import PreferenceProblem
    cpu = torch.device("cpu")
    make = lambda B=4, T=3, mask=None, ref=None, w=None, **kw: PreferenceProblem(  # noqa: E731
        B, T, cpu, mask, ref, w, None, G.PreferenceConfig(**kw))
    assert make().total == 2.0
    for bad, match in ((dict(B=3), "even"), (dict(B=0), "even"), (dict(T=0), "no scored"), (dict(loss_type="dpo"), "loss_type"),
                       (dict(beta=0.0), "beta"), (dict(label_smoothing=0.7), "label_smoothing"),
                       (dict(label_smoothing=0.1, loss_type="ipo"), "label_smoothing"), (dict(mask=torch.ones(4, 2)), "mask"),
                       (dict(ref=torch.ones(2)), "ref_per_token_logps"), (dict(w=torch.ones(4)), "pair_weights")):
        with pytest.raises(ValueError, match=match):
            make(**bad)


def test_status_words_are_checked():
    from mllm_jax_b200 import _lib
    cpu = torch.device("cpu")
    word = torch.zeros(1, dtype=torch.int32)
    assert _lib.status_word(word, cpu) == word.data_ptr()
    for bad in (torch.zeros(1), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32, device="meta")):
        with pytest.raises(ValueError, match="device_status"):
            _lib.status_word(bad, cpu)


def test_written_tensors_change_their_version():
    from mllm_jax_b200 import _lib
    t = torch.zeros(3)
    before = t._version
    _lib.written(t[1:])
    assert t._version > before
    with torch.inference_mode():
        _lib.written(torch.zeros(3))


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwd

    t = torch.zeros(3)
    _lib.no_tangent(t, "t")
    with fwd.dual_level():
        _lib.no_tangent(t, "t")
        with pytest.raises(NotImplementedError, match="t carries a forward-mode tangent"):
            _lib.no_tangent(fwd.make_dual(t, torch.ones(3)), "t")


def test_a_workspace_is_checked_before_a_kernel_writes_it():
    """Its device (an address of the host's memory would be written by the kernel), its layout, its size in bytes; of any
    type it is taken as bytes, which a gather over ranks counts."""
    from mllm_jax_b200.linear_loss import _workspace_bytes

    cpu, room = torch.device("cpu"), torch.zeros(64, dtype=torch.float32)
    got = _workspace_bytes(room, 256, cpu)
    assert got.dtype == torch.uint8 and got.shape == (256,) and got.data_ptr() == room.data_ptr()
    assert _workspace_bytes(room.view(8, 8), 200, cpu)[:16].numel() == 16
    for bad, nbytes, dev in ((room, 257, cpu), (room, 16, torch.device("cuda:0")), (room.view(8, 8)[:, :4], 16, cpu),
                             (room[1:], 16, cpu)):
        with pytest.raises(ValueError, match="workspace"):
            _workspace_bytes(bad, nbytes, dev)
