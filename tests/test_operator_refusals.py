"""What the loss without logits, the embedding and linear attention refuse, on the CPU: the C entry points' checks of
argument blocks (nothing is launched) and the Python operators' checks."""
from __future__ import annotations

import ctypes

import pytest
import torch

from lrnnx_b200 import _lib


def err(name):
    return _lib.enum(name)


def run(fn, a):
    return getattr(_lib.lib(), fn)(ctypes.byref(a), None)


ADDRESS = 1 << 20          # never read: every call here is refused


def lce():
    a = _lib.struct("b200_lce_args")()
    a.rows, a.classes, a.features, a.dtype, a.reduction, a.ignore_index = 64, 1000, 64, err("B200_BF16"), 1, -100
    a.hidden = a.weight = a.labels = a.lse = a.loss = a.count = a.dloss = a.dhidden = a.dweight = a.work = ADDRESS
    a.hidden_rs = a.weight_rs = a.dhidden_rs = a.dweight_rs = 64
    return a


def embed():
    a = _lib.struct("b200_embed_args")()
    a.tokens, a.classes, a.features, a.dtype, a.scale, a.padding_idx = 100, 1000, 64, err("B200_F32"), 1.0, -1
    a.ids = a.weight = a.dout = a.out = a.dweight = a.work = ADDRESS
    a.weight_rs = a.out_rs = a.dout_rs = a.dweight_rs = 64
    return a


def attn():
    a = _lib.struct("b200_linattn_args")()
    a.batch, a.seqlen, a.heads, a.groups, a.dk, a.dv, a.dtype, a.g_dtype = 2, 300, 4, 2, 64, 64, err("B200_BF16"), err("B200_F32")
    for f in ("q", "k", "v", "g", "out", "dout", "dq", "dk_out", "dv_out", "dg", "work"):
        setattr(a, f, ADDRESS)
    return a


def step():
    a = _lib.struct("b200_linattn_step_args")()
    a.batch, a.heads, a.groups, a.dk, a.dv, a.slots = 2, 4, 2, 64, 64, 2
    a.dtype, a.g_dtype, a.state_dtype = err("B200_BF16"), err("B200_F32"), err("B200_F32")
    for f in ("state", "q", "k", "v", "g", "out"):
        setattr(a, f, ADDRESS)
    return a


@pytest.mark.parametrize("fn,make,change,code", [
    ("b200_lce_fwd", lce, dict(hidden=0), "B200_ERR_NULL"), ("b200_lce_fwd", lce, dict(lse=0), "B200_ERR_NULL"), ("b200_lce_fwd", lce, dict(count=0), "B200_ERR_NULL"),
    ("b200_lce_fwd", lce, dict(rows=0), "B200_ERR_SHAPE"), ("b200_lce_fwd", lce, dict(features=0), "B200_ERR_SHAPE"), ("b200_lce_fwd", lce, dict(rows=1 << 31), "B200_ERR_SHAPE"),
    ("b200_lce_fwd", lce, dict(hidden_rs=63), "B200_ERR_SHAPE"), ("b200_lce_fwd", lce, dict(dtype=9), "B200_ERR_DTYPE"), ("b200_lce_fwd", lce, dict(reduction=3), "B200_ERR_DTYPE"),
    ("b200_lce_fwd", lce, dict(work=ADDRESS + 16), "B200_ERR_ALIGN"), ("b200_lce_fwd", lce, dict(work_bytes=100), "B200_ERR_TOO_LARGE"),
    ("b200_lce_bwd", lce, dict(dloss=0), "B200_ERR_NULL"), ("b200_lce_bwd", lce, dict(dhidden=0, dweight=0), "B200_ERR_NULL"), ("b200_lce_bwd", lce, dict(dweight_rs=63), "B200_ERR_SHAPE"),
    ("b200_lce_bwd", lce, dict(work_bytes=100), "B200_ERR_TOO_LARGE"),
    ("b200_embed_fwd", embed, dict(weight=0), "B200_ERR_NULL"), ("b200_embed_fwd", embed, dict(tokens=0), "B200_ERR_SHAPE"), ("b200_embed_fwd", embed, dict(dtype=-1), "B200_ERR_DTYPE"),
    ("b200_embed_bwd", embed, dict(dout=0), "B200_ERR_NULL"), ("b200_embed_bwd", embed, dict(work=0), "B200_ERR_NULL"), ("b200_embed_bwd", embed, dict(work=ADDRESS + 8), "B200_ERR_ALIGN"),
    ("b200_embed_bwd", embed, dict(work_bytes=100), "B200_ERR_TOO_LARGE"), ("b200_embed_bwd", embed, dict(tokens=1 << 31), "B200_ERR_SHAPE"),
    ("b200_embed_bwd", embed, dict(work_bytes=1 << 30, dweight_rs=65), "B200_ERR_SHAPE"), ("b200_embed_bwd", embed, dict(work_bytes=1 << 30, dweight=ADDRESS + 4), "B200_ERR_ALIGN"),
    ("b200_linattn_fwd", attn, dict(q=0), "B200_ERR_NULL"), ("b200_linattn_fwd", attn, dict(out=0), "B200_ERR_NULL"), ("b200_linattn_fwd", attn, dict(seqlen=0), "B200_ERR_SHAPE"),
    ("b200_linattn_fwd", attn, dict(dk=129), "B200_ERR_SHAPE"), ("b200_linattn_fwd", attn, dict(dv=129), "B200_ERR_SHAPE"), ("b200_linattn_fwd", attn, dict(groups=3), "B200_ERR_SHAPE"),
    ("b200_linattn_fwd", attn, dict(batch=40000), "B200_ERR_SHAPE"), ("b200_linattn_fwd", attn, dict(dtype=5), "B200_ERR_DTYPE"),
    ("b200_linattn_fwd", attn, dict(g_dtype=1), "B200_ERR_DTYPE"), ("b200_linattn_fwd", attn, dict(work=ADDRESS + 8), "B200_ERR_ALIGN"),
    ("b200_linattn_fwd", attn, dict(seqlen=20000, work_bytes=100), "B200_ERR_TOO_LARGE"), ("b200_linattn_bwd", attn, dict(dq=0), "B200_ERR_NULL"),
    ("b200_linattn_bwd", attn, dict(work_bytes=100), "B200_ERR_TOO_LARGE"),
    ("b200_linattn_step", step, dict(state=0), "B200_ERR_NULL"), ("b200_linattn_step", step, dict(dk=129), "B200_ERR_SHAPE"), ("b200_linattn_step", step, dict(groups=3), "B200_ERR_SHAPE"),
    ("b200_linattn_step", step, dict(state_dtype=1), "B200_ERR_DTYPE"), ("b200_linattn_step", step, dict(batch=0), "B200_ERR_SHAPE")])
def test_entry_points_refuse(fn, make, change, code):
    a = make()
    for k, v in change.items():
        setattr(a, k, v)
    assert run(fn, a) == err(code), _lib.lib().b200_last_error()
    assert _lib.lib().b200_last_error()


@pytest.mark.parametrize("fn", ["b200_lce_fwd", "b200_lce_bwd", "b200_embed_fwd", "b200_embed_bwd", "b200_linattn_fwd", "b200_linattn_bwd", "b200_linattn_step"])
def test_entry_points_refuse_no_arguments(fn):
    assert getattr(_lib.lib(), fn)(None, None) == err("B200_ERR_NULL")


def test_workspaces_are_bounded_and_sized():
    """The loss's backward holds at most 1 GiB of the logits' gradient (and at least 256 columns of it), its sums and copies."""
    lib = _lib.lib()
    a = lce()
    a.rows, a.classes, a.features = 16384, 50280, 768
    a.hidden_rs = a.weight_rs = a.dhidden_rs = a.dweight_rs = 768
    assert lib.b200_lce_bwd_work_bytes(ctypes.byref(a)) <= (1 << 30) + 2 * 4 * 16384 * 768
    assert lib.b200_lce_fwd_work_bytes(ctypes.byref(a)) <= 8 * 16384 * 400
    a.dtype = err("B200_F32")
    split = 2 * 3 * (16384 + 50280) * 768
    assert lib.b200_lce_bwd_work_bytes(ctypes.byref(a)) <= (1 << 30) + split + 4 * (16384 + 50280) * 768 * 2
    a.rows = 1 << 29
    a.classes = 300
    assert lib.b200_lce_bwd_work_bytes(ctypes.byref(a)) > 0
    for fn, make in (("b200_lce_fwd", lce), ("b200_embed_bwd", embed), ("b200_linattn_bwd", attn)):
        bad = make()
        setattr(bad, "dtype", 77)
        assert getattr(lib, fn + "_work_bytes")(ctypes.byref(bad)) == 0
        assert getattr(lib, fn + "_work_bytes")(None) == 0


def test_packed_blocks_have_the_structures_layout():
    for name in ("b200_lce_args", "b200_embed_args", "b200_linattn_args", "b200_linattn_step_args"):
        st = _lib.struct(name)
        values = [float(i + 1) if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(st._fields_)]
        a = st.from_buffer_copy(_lib.packer(name)(*values))
        assert [getattr(a, n) for n, _ in st._fields_] == values


def test_loss_refuses():
    from lrnnx_b200.ops import linear_cross_entropy
    h, w, y = torch.randn(4, 8), torch.randn(10, 8), torch.zeros(4, dtype=torch.long)
    for args, match in (((h, w, y), "CUDA"), ((h, w[:, :7], y), "expected"), ((h, w, y[:3]), "expected"), ((h, w[0], y), "expected"),
                        ((h, w.double(), y), "dtype"), ((h.double(), w.double(), y), "dtype")):
        with pytest.raises(RuntimeError, match=match):
            linear_cross_entropy(*args)
    with pytest.raises(RuntimeError, match="reduction"):
        linear_cross_entropy(h, w, y, reduction="max")


def test_embedding_refuses():
    from lrnnx_b200.ops import token_embedding
    ids, w = torch.zeros(3, dtype=torch.long), torch.randn(5, 4)
    for args, match in (((ids, w), "CUDA"), ((ids, w[0]), "expected"), ((ids, w[:0]), "expected"), ((ids, w.double()), "float32")):
        with pytest.raises(RuntimeError, match=match):
            token_embedding(*args)


def test_linear_attention_refuses():
    from lrnnx_b200.ops import linear_attention_fn, linear_attention_step
    q, v, g = torch.randn(2, 5, 2, 8), torch.randn(2, 5, 4, 6), -torch.rand(2, 5, 4)
    for args, match in (((q, q, v, g), "CUDA"), ((q, q[..., :7], v, g), "shape"), ((q, q, v[:, :4], g), "shape"), ((q, q, v[:, :, :3], g), "multiple"),
                        ((q, q, v, g[:, :, :3]), "g must"), ((q.double(), q.double(), v.double(), g), "dtype"), ((q, q, v, g.double()), "dtype"),
                        ((torch.randn(2, 5, 2, 129),) * 2 + (v, g), "sizes"), ((q, q, torch.randn(2, 5, 4, 129), g), "sizes"), ((q[0], q[0], v[0], g[0]), "shape")):
        with pytest.raises(RuntimeError, match=match):
            linear_attention_fn(*args)
    s = torch.zeros(2, 4, 8, 6)
    for args, match in (((s, q[:, 0], q[:, 0], v[:, 0], g[:, 0]), "CUDA"), ((s, q[:, 0], q[:, 0], v[:, 0, :3], g[:, 0, :3]), "multiple"),
                        ((s, q[:, 0], q[:, 0], v[:, 0], g[:, 0, :3]), "g must")):
        with pytest.raises(RuntimeError, match=match):
            linear_attention_step(*args)
