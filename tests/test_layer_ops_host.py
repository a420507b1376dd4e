"""Host side of rotations with several axes and of the norms around a block (CPU only): refusals before
anything touches the device, and the tables' values."""
import ctypes

import pytest
import torch

from bhaskera_col_b200 import _lib
from bhaskera_col_b200.inference import ops
from test_serving_ops_host import BATCH, CACHE, KV, NORM, POS, ROPE, TABLES, X, far, geom, t4

r = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731


def axes_of(n, pairs, stride=10):
    return _lib.RopeAxes(n, stride, (ctypes.c_uint8 * 128)(*pairs))


@pytest.mark.parametrize("rope,axes,what", [
    (ROPE, axes_of(0, [0] * 64), "axes"), (ROPE, axes_of(5, [0] * 64), "axes"),
    (ROPE, axes_of(3, [0] * 63 + [3]), "axes"), (ROPE, axes_of(1, [1] + [0] * 63), "axes"),
    (None, axes_of(1, [0] * 64), "rotation")])
def test_axes_refusals(rope, axes, what):
    lib = _lib.load()
    norm = NORM
    rc = lib.tq_qk_rope_axes(r(rope), r(axes), r(POS), r(t4(X)), r(far(X)), r(norm), None, None, None, None)
    assert rc == _lib.TQ_ERR_INVALID and what in _lib.last_error(), _lib.last_error()
    rc = lib.tq_append_ragged_axes(r(geom()), r(TABLES), r(CACHE), r(t4(KV)), r(t4(KV)), r(BATCH), r(rope),
                                   r(axes), r(norm), r(POS), None)
    assert rc == _lib.TQ_ERR_INVALID and what in _lib.last_error(), _lib.last_error()


def test_axis_of_pairs():
    f = ops.RopeTable.axis_of_pairs
    assert f((2, 1, 3)) == (0, 0, 1, 2, 2, 2)
    assert f((3, 1, 2), mixed=True) == (0, 1, 2, 0, 2, 0)
    assert f((0, 2)) == (1, 1) and f((4,)) == (0, 0, 0, 0)
    for bad in ((), (0, 0), (1, 1, 1, 1, 1), (3, -1)):
        with pytest.raises(ValueError, match="sections"):
            f(bad)


def test_axes_wrapper_checks():
    cs = torch.zeros((5, 8))
    t = ops.RopeTable(cs, axes=(0, 1, 2, 0))
    assert t.num_axes == 3 and ops.RopeTable(cs).num_axes == 1
    for bad in ((0, 1), (0, 1, 2, 4), (0, 1, 2, -1)):
        with pytest.raises(ValueError, match="axes"):
            ops.RopeTable(cs, axes=bad)
    built = ops.RopeTable.build(8, 20, device=torch.device("cpu"), axes=(0, 0, 1, 1))
    assert built.num_axes == 2 and torch.equal(built.cos_sin, ops.RopeTable.build(
        8, 20, device=torch.device("cpu")).cos_sin)
    p = ops._positions
    assert p(torch.zeros(7, dtype=torch.int64), 1, 7, t, True)[1] is None
    assert p(torch.zeros((3, 7), dtype=torch.int64), 1, 7, t, True)[1] is not None
    assert p(torch.zeros((3, 2, 7), dtype=torch.int32), 2, 7, t, False)[1] is not None
    assert p(torch.zeros((2, 7), dtype=torch.int32), 2, 7, t, False)[1] is None
    for shape, b, flat in (((2, 7), 1, True), ((3, 6), 1, True), ((3, 7), 2, False), ((4, 7), 1, True),
                           ((3, 7, 2), 2, False)):
        with pytest.raises(ValueError, match="positions must be"):
            p(torch.zeros(shape, dtype=torch.int64), b, 7, t, flat)
    with pytest.raises(ValueError, match="positions must be"):
        p(torch.zeros((3, 7), dtype=torch.int64), 1, 7, ops.RopeTable(cs), True)
    x = torch.zeros((7, 2, 8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.qk_rope(x, None, t, torch.zeros((3, 7), dtype=torch.int64))


def norm_call(x=t4((1, 1, 6, 64)), res=None, gate=None, y=None, h=None, post=None, pre=None, act=0, **kw):
    shape = tuple(x.shape)
    res = res or t4(shape, data=1 << 28)
    y = y or far(shape)
    p = lambda v: None if v is None else ctypes.pointer(v)  # noqa: E731
    a = _lib.ResidualNormArgs(p(x), p(res), p(gate), p(y), p(h), p(post), p(pre), 1.0, act)
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.load().tq_residual_norm(ctypes.byref(a), None), _lib.last_error()


RN = _lib.RowNorm(4096, 4096, _lib.TQ_F32, 1e-6, 0.0, 0)
W = (1, 1, 6, 64)
FAR2 = lambda **kw: t4(W, data=1 << 31, **kw)  # noqa: E731


@pytest.mark.parametrize("kw,what", [
    (dict(x=t4(W, data=None)), "NULL"), (dict(x=None, res=t4(W), y=far(W)), "needed"),
    (dict(pre=RN), "out comes with"), (dict(h=FAR2()), "out comes with"),
    (dict(res=t4((1, 1, 5, 64), data=1 << 28)), "disagree"), (dict(y=far((1, 1, 6, 32))), "disagree"),
    (dict(gate=t4((1, 1, 6, 32), data=1 << 29)), "disagree"),
    (dict(y=far(W, dtype=_lib.TQ_F32)), "type"), (dict(pre=RN, h=FAR2(dtype=_lib.TQ_F16)), "type"),
    (dict(post=_lib.RowNorm(4096, 4096, 5, 1e-6, 0.0, 0)), "post"),
    (dict(post=_lib.RowNorm(4098, None, 0, 1e-6, 0.0, 0)), "post"),
    (dict(pre=_lib.RowNorm(4096, None, 0, float("nan"), 0.0, 0), h=FAR2()), "pre"),
    (dict(post=_lib.RowNorm(4096, None, 0, -1.0, 0.0, 0)), "post"),
    (dict(act=3), "gate_act"), (dict(act=-1), "gate_act"),
    (dict(x=t4((1, 1, 2, 32769))), "32768"), (dict(x=t4((1, 1, 2, 0))), "32768"),
    (dict(x=t4((1, 1 << 16, 1 << 16, 8))), "2^31"),
    (dict(y=t4(W, stride=[0, 0, 0, 1], data=1 << 30)), "share memory"),
    (dict(y=t4(W, data=(1 << 28) + 128)), "overlaps"), (dict(y=t4(W)), "overlaps"),
    (dict(pre=RN, h=t4(W, data=(1 << 20) + 64)), "overlaps"), (dict(pre=RN, h=t4(W, data=1 << 28)), "overlaps"),
    (dict(pre=RN, h=t4(W, data=1 << 30)), "overlaps"),
    (dict(gate=t4(W, data=1 << 29), y=t4(W, data=1 << 29)), "overlaps"),
    (dict(res=t4(W, dtype=_lib.TQ_F32, data=(1 << 28) + 2)), "aligned"),
])
def test_residual_norm_refusals(kw, what):
    if "x" in kw and kw["x"] is None:
        a = _lib.ResidualNormArgs()
        assert _lib.load().tq_residual_norm(ctypes.byref(a), None) == _lib.TQ_ERR_INVALID
        assert what in _lib.last_error()
        return
    rc, err = norm_call(**kw)
    assert rc == _lib.TQ_ERR_INVALID and what in err, err


def test_residual_norm_wrapper_checks():
    x, n = torch.zeros((3, 64)), ops.RowNorm(torch.ones(64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.residual_norm(x, x.clone(), post_norm=n)
    for kw, what in ((dict(gate_act="relu"), "gate_act"), (dict(gate_act="tanh"), "comes with a gate"),
                     (dict(residual=torch.zeros((3, 63))), "one shape")):
        args = dict(residual=x.clone(), post_norm=n)
        args.update(kw)
        with pytest.raises(ValueError, match=what):
            ops.residual_norm(x, **args)
    for bad in (dict(weight=torch.ones((2, 3))), dict(weight=torch.ones(4).double()),
                dict(weight=torch.ones(8)[::2]), dict(weight=torch.ones(4), bias=torch.ones(5)),
                dict(weight=torch.ones(4), bias=torch.ones(4).half()), dict(eps=-1.0),
                dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            ops.RowNorm(**bad)
    w = torch.ones(4)
    n = ops.RowNorm(w)
    assert n.c.weight == w.data_ptr() and n.c.bias is None
    w.data = torch.zeros(4, dtype=torch.float16)
    assert n.c.weight == w.data_ptr() and n.c.dtype == _lib.TQ_F16
    meta = torch.zeros((3, 64), requires_grad=True)
    with pytest.raises(RuntimeError):
        ops.residual_norm(meta, x)


def diff_call(g=None, c=_lib.Cache(1 << 20, 12, 4, 0, 0, 0), q=t4((1, 8, 10, 128)), out=None, batch=BATCH,
              scale=0.1, engine=0, shared=0, halves=0, lam=1 << 40, ls=(0, 1), norm=None, t=TABLES,
              ws=1 << 20, nbytes=None):
    lib = _lib.load()
    g = g or geom()
    out = out or far((1, q.shape[1] // 2, q.shape[2], q.shape[3] * (1 if shared else 2)))
    a = _lib.DiffArgs(ctypes.pointer(q), ctypes.pointer(out), batch, scale, 1, engine, shared, halves, lam,
                      (ctypes.c_int64 * 2)(*ls), None if norm is None else ctypes.pointer(norm), 1.0)
    need = lib.tq_diff_attend_ragged_workspace_bytes(r(g), r(c), r(a))
    rc = lib.tq_diff_attend_ragged(r(g), r(t), r(c), r(a), ws, need if nbytes is None else nbytes, None)
    return rc, _lib.last_error(), need


@pytest.mark.parametrize("kw,what", [
    (dict(engine=4), "engine"), (dict(engine=-1), "engine"), (dict(g=geom(D=96), q=t4((1, 8, 10, 96))), "no kernel"),
    (dict(g=geom(kb=7)), "no kernel"), (dict(q=t4((1, 7, 10, 128)), out=far((1, 3, 10, 256))), "pairs"),
    (dict(q=t4((1, 6, 10, 128))), "multiple"), (dict(c=_lib.Cache(1 << 20, 9, 4, 0, 0, 0), q=t4((1, 6, 10, 128))),
                                                "multiple"),
    (dict(shared=1, q=t4((1, 12, 10, 128))), "multiple"), (dict(shared=1, halves=1), "next to each other"),
    (dict(out=far((1, 4, 10, 128))), "must be"), (dict(shared=1, out=far((1, 4, 10, 256))), "must be"),
    (dict(out=far((1, 4, 9, 256))), "differ in rows"), (dict(q=t4((1, 2048, 1, 128))), "1024 query heads"),
    (dict(batch=_lib.Ragged(5, 4096, 4096, 1)), "multiple"), (dict(c=_lib.Cache(1 << 20, 12, 1 << 27)), "32 bits"),
])
def test_diff_attend_refusals(kw, what):
    rc, err, need = diff_call(**kw)
    assert rc == _lib.TQ_ERR_INVALID and need == 0 and what in err, err


def test_diff_attend_refusals_of_the_call_alone():
    big = (1, 4, 10, 256)
    for kw, what in ((dict(out=t4(big, data=(1 << 20) + 256)), "overlaps"), (dict(out=t4(big)), "overlaps"),
                     (dict(out=far(big, stride=[0, 0, 1024, 1])), "share memory"), (dict(lam=None), "NULL"),
                     (dict(lam=(1 << 40) + 2), "aligned"), (dict(lam=1 << 30, ls=(4, 1)), "lambda"),
                     (dict(norm=_lib.HeadNorm(None, 0, 1e-6, 0)), "norm"),
                     (dict(norm=_lib.HeadNorm(4096, 0, -1.0, 0)), "norm"),
                     (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
                     (dict(t=_lib.Tables(*([4096] * 9))), "rot_f16")):
        rc, err, need = diff_call(**kw)
        assert rc == _lib.TQ_ERR_INVALID and need > 0 and what in err, err
    for kw in (dict(nbytes=100), dict(ws=(1 << 20) + 64), dict(ws=None)):
        rc, err, need = diff_call(**kw)
        assert rc == _lib.TQ_ERR_WORKSPACE and str(need) in err


def test_diff_wrapper_checks():
    x = torch.zeros((3, 4, 128))
    batch = ops.RaggedBatch(torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3], dtype=torch.int32), 3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.diff_attend_ragged(None, None, x, batch, ops.DiffHeads(torch.ones(2)))
    for kw in (dict(lam=torch.ones(2).double()), dict(lam=torch.ones((1, 1, 2))), dict(lam=torch.ones(2), keys="both"),
               dict(lam=torch.ones(2), pairs="odd"), dict(lam=torch.ones(2), keys="shared", pairs="halves")):
        with pytest.raises(ValueError):
            ops.DiffHeads(**kw)
    lam = ops.DiffHeads.lam_of(*(torch.full((3, 4), f) for f in (0.1, 0.2, 0.3, 0.1)), 0.5)
    want = torch.tensor(0.08, dtype=torch.float64).exp() - torch.tensor(0.12, dtype=torch.float64).exp() + 0.5
    assert lam.shape == (3,) and (lam - want).abs().max() < 2e-8 + 2.0 ** -24
    p = ops.DiffHeads(torch.ones((5, 4))[:, ::2])
    assert p.c[1:] == (4, 2) and ops.DiffHeads(torch.ones((5, 1))).c[1:] == (1, 0)
