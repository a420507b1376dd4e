"""Host side of the serving operators (CPU only): refusals of the C entries before anything touches
the device, checks of the Python wrappers, and the arithmetic the kernels rely on."""
import ctypes
import random

import pytest
import torch

from bhaskera_col_b200 import _lib
from bhaskera_col_b200.inference import ops

I64x4 = ctypes.c_int64 * 4


def t4(shape, stride=None, dtype=_lib.TQ_BF16, data=1 << 20):
    if stride is None:
        stride = [shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1]
    return _lib.Tensor4(data, dtype, I64x4(*shape), I64x4(*stride))


def far(shape, **kw):
    return t4(shape, data=1 << 30, **kw)


def rope_call(rope=None, pos=None, q=None, qo=None, qn=None, k=None, ko=None, kn=None):
    r = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
    rc = _lib.load().tq_qk_rope(r(rope), r(pos), r(q), r(qo), r(qn), r(k), r(ko), r(kn), None)
    return rc, _lib.last_error()


ROPE = _lib.Rope(4096, 100, 128, 0)
POS = _lib.Positions(4096, 64, (ctypes.c_int64 * 2)(0, 1))
NORM = _lib.HeadNorm(4096, _lib.TQ_F32, 1e-6, 0.0)
X = (1, 4, 7, 128)


@pytest.mark.parametrize("kw,what", [
    (dict(), "neither"),
    (dict(rope=ROPE, pos=POS, q=t4(X)), "come together"),
    (dict(q=t4(X), qo=far(X)), "neither a rotation nor a norm"),
    (dict(rope=ROPE, q=t4(X), qo=far(X)), "needs positions"),
    (dict(rope=_lib.Rope(4096, 100, 63, 0), pos=POS, q=t4(X), qo=far(X)), "rot_dim"),
    (dict(rope=_lib.Rope(4096, 100, 130, 0), pos=POS, q=t4(X), qo=far(X)), "rot_dim"),
    (dict(rope=_lib.Rope(4096, 100, 0, 0), pos=POS, q=t4(X), qo=far(X)), "rot_dim"),
    (dict(rope=_lib.Rope(4100, 100, 128, 0), pos=POS, q=t4(X), qo=far(X)), "table"),
    (dict(rope=_lib.Rope(4096, 0, 128, 0), pos=POS, q=t4(X), qo=far(X)), "table"),
    (dict(rope=ROPE, pos=_lib.Positions(4096, 16, POS.stride), q=t4(X), qo=far(X)), "positions"),
    (dict(rope=ROPE, pos=_lib.Positions(4100, 64, POS.stride), q=t4(X), qo=far(X)), "positions"),
    (dict(qn=_lib.HeadNorm(4096, 7, 1e-6, 0), q=t4(X), qo=far(X)), "head norm"),
    (dict(qn=_lib.HeadNorm(4096, 0, -1e-6, 0), q=t4(X), qo=far(X)), "head norm"),
    (dict(qn=_lib.HeadNorm(4096, 0, float("nan"), 0), q=t4(X), qo=far(X)), "head norm"),
    (dict(qn=NORM, q=t4(X), qo=far((1, 4, 6, 128))), "disagree"),
    (dict(qn=NORM, q=t4(X), qo=far(X, dtype=_lib.TQ_F16)), "differ in type"),
    (dict(qn=NORM, kn=NORM, q=t4(X), qo=far(X), k=t4((1, 2, 6, 128)), ko=far((1, 2, 6, 128))),
     "disagree"),
    (dict(qn=NORM, q=t4((1, 1, 1, 257)), qo=far((1, 1, 1, 257))), "head_dim"),
    (dict(qn=NORM, q=t4(X), qo=t4(X, stride=[0, 0, 128, 1], data=1 << 30)), "share memory"),
    (dict(qn=NORM, q=t4(X), qo=t4(X, stride=[0, 64, 512, 1], data=1 << 30)), "share memory"),
    (dict(qn=NORM, q=t4(X), qo=t4(X, data=(1 << 20) + 256)), "overlaps"),
    (dict(qn=NORM, q=t4(X), qo=t4(X, stride=[0, 128, 512, 1])), "overlaps"),
    (dict(qn=NORM, q=t4(X, data=None), qo=far(X)), "NULL"),
    (dict(qn=NORM, q=t4(X, data=4097), qo=far(X)), "aligned"),
    (dict(qn=NORM, q=t4(X, dtype=_lib.TQ_F32, data=4098), qo=far(X, dtype=_lib.TQ_F32)), "aligned"),
])
def test_qk_rope_refusals(kw, what):
    rc, err = rope_call(**kw)
    assert rc == _lib.TQ_ERR_INVALID and what in err, err


def geom(D=128, kb=4, vb=2, qjl=0):
    return _lib.Geom(D, kb, vb, qjl)


TABLES = _lib.Tables(*([4096] * 11))
CACHE = _lib.Cache(1 << 20, 6, 4, 0, 0, 0)                 # 3 requests x 2 heads
BATCH = _lib.Ragged(3, 4096, 4096, 9)
KV = (1, 2, 10, 128)


def entry(fn, g=None, t=TABLES, c=CACHE, batch=BATCH, k=t4(KV), v=t4(KV), rope=None, norm=None,
          pos=None):
    r = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
    lib = _lib.load()
    g = g or geom()
    if fn == "append":
        rc = lib.tq_append_ragged(r(g), r(t), r(c), r(k), r(v), r(batch), r(rope), r(norm), r(pos), None)
    else:
        rc = lib.tq_dequantize_ragged(r(g), r(t), r(c), r(batch), r(k), r(v), None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("fn", ["append", "read"])
@pytest.mark.parametrize("kw,what", [
    (dict(g=geom(D=48)), "head_dim"),
    (dict(g=geom(kb=9)), "bit widths"),
    (dict(t=_lib.Tables()), "NULL"),
    (dict(c=_lib.Cache(0, 6, 4)), "cache"),
    (dict(c=_lib.Cache(1 << 20, 6, 4, 4096, 3, 5)), "block table"),
    (dict(batch=_lib.Ragged(0, 4096, 4096, 9)), "batch"),
    (dict(batch=_lib.Ragged(3, 0, 4096, 9)), "batch"),
    (dict(batch=_lib.Ragged(3, 4096, 4098, 9)), "batch"),
    (dict(batch=_lib.Ragged(3, 4096, 4096, -1)), "batch"),
    (dict(batch=_lib.Ragged(4, 4096, 4096, 9)), "multiple"),
    (dict(k=t4((1, 3, 10, 128))), "must be"),
    (dict(v=t4((2, 2, 10, 128))), "must be"),
    (dict(k=t4((1, 2, 10, 64))), "must be"),
    (dict(k=t4((1, 2, 9, 128))), "differ in rows"),
    (dict(g=geom(D=256), k=t4((1, 2, 10, 256)), v=t4((1, 2, 10, 256))), "128"),
])
def test_ragged_store_and_read_refusals(fn, kw, what):
    rc, err = entry(fn, **kw)
    assert rc == _lib.TQ_ERR_INVALID and what in err, err


def test_more_append_and_read_refusals():
    for kw, what in ((dict(g=geom(qjl=1)), "QJL"), (dict(rope=_lib.Rope(4096, 10, 200, 0)), "rot_dim"),
                     (dict(norm=_lib.HeadNorm(None, 0, 1e-6, 0)), "head norm"),
                     (dict(pos=_lib.Positions(None, 64, POS.stride)), "positions")):
        rc, err = entry("append", **kw)
        assert rc == _lib.TQ_ERR_INVALID and what in err, err
    rc, err = entry("read", k=None, v=None)
    assert rc == _lib.TQ_ERR_INVALID and "neither" in err
    rc, err = entry("read", k=t4(KV, stride=[0, 0, 128, 1]))
    assert rc == _lib.TQ_ERR_INVALID and "share memory" in err


def attend(g=None, c=CACHE, q=t4((1, 4, 10, 128)), out=None, batch=BATCH, scale=0.1, engine=0,
           t=TABLES, ws=1 << 20, nbytes=None):
    lib = _lib.load()
    g = g or geom()
    out = out or far(tuple(q.shape))
    a = _lib.AttendArgs(ctypes.pointer(q), ctypes.pointer(out), batch, scale, 1, engine)
    need = lib.tq_attend_ragged_workspace_bytes(ctypes.byref(g), ctypes.byref(c), ctypes.byref(a))
    if nbytes is None:
        nbytes = need
    rc = lib.tq_attend_ragged(ctypes.byref(g), ctypes.byref(t), ctypes.byref(c), ctypes.byref(a), ws,
                              nbytes, None)
    return rc, _lib.last_error(), need


@pytest.mark.parametrize("kw,what", [
    (dict(engine=4), "engine"), (dict(engine=-1), "engine"),
    (dict(g=geom(D=96), q=t4((1, 4, 10, 96))), "no kernel"),
    (dict(g=geom(kb=7)), "no kernel"),
    (dict(g=geom(D=64), q=t4((1, 4, 10, 64)), engine=2), "no kernel"),
    (dict(g=geom(kb=8, vb=8), engine=3), "no kernel"),
    (dict(q=t4((1, 3, 10, 128))), "multiple"),
    (dict(q=t4((1, 4, 10, 64))), "must be"),
    (dict(batch=_lib.Ragged(5, 4096, 4096, 1)), "multiple"),
    (dict(q=t4((1, 2048, 1, 128))), "1024 query heads"),
    (dict(c=_lib.Cache(1 << 20, 6, 1 << 27)), "32 bits"),
    (dict(out=far((1, 4, 9, 128))), "differ in rows"),
    (dict(out=far((1, 2, 10, 128))), "must be"),
])
def test_attend_refusals(kw, what):
    rc, err, need = attend(**kw)
    assert rc == _lib.TQ_ERR_INVALID and need == 0 and what in err, err


def test_attend_workspace_query_without_tensors():
    lib = _lib.load()
    q, g = t4((1, 4, 10, 128)), geom()
    for a in (_lib.AttendArgs(None, ctypes.pointer(q), BATCH, 0.1, 1, 0),
              _lib.AttendArgs(ctypes.pointer(q), None, BATCH, 0.1, 1, 0)):
        assert lib.tq_attend_ragged_workspace_bytes(ctypes.byref(g), ctypes.byref(CACHE),
                                                    ctypes.byref(a)) == 0
        assert "NULL" in _lib.last_error()


def test_attend_refusals_of_the_call_alone():
    for kw, what in ((dict(out=t4((1, 4, 10, 128), data=(1 << 20) + 256)), "overlaps"),
                     (dict(out=t4((1, 4, 10, 128), dtype=_lib.TQ_F32)), "overlaps"),
                     (dict(out=t4((1, 4, 10, 128), stride=[0, 0, 128, 1])), "share memory"),
                     (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
                     (dict(t=_lib.Tables(*([4096] * 9))), "rot_f16")):
        rc, err, need = attend(**kw)
        assert rc == _lib.TQ_ERR_INVALID and need > 0 and what in err, err
    for kw in (dict(nbytes=100), dict(ws=(1 << 20) + 64), dict(ws=None)):
        rc, err, need = attend(**kw)
        assert rc == _lib.TQ_ERR_WORKSPACE and str(need) in err


def test_wrapper_checks():
    x = torch.zeros((3, 2, 128))
    table = ops.RopeTable(torch.zeros((5, 128)))
    batch = ops.RaggedBatch(torch.tensor([0, 3], dtype=torch.int32),
                            torch.tensor([3], dtype=torch.int32), 3)
    for call in (lambda: ops.qk_rope(x, None, table, torch.arange(3)),
                 lambda: ops.append_ragged(None, None, x, x, batch),
                 lambda: ops.dequantize_ragged(None, None, batch, x, x),
                 lambda: ops.attend_ragged(None, None, x, batch)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="neither"):
        ops.qk_rope(None, None, table)
    with pytest.raises(ValueError, match="positions"):
        ops.qk_rope(x, None, table)
    with pytest.raises(ValueError, match="neither"):
        ops.dequantize_ragged(None, None, batch, None, None)
    for bad in (torch.zeros((5, 128)).double(), torch.zeros((5, 127)), torch.zeros(5),
                torch.zeros((0, 128)), torch.zeros((128, 5)).t()):
        with pytest.raises(ValueError):
            ops.RopeTable(bad)
    with pytest.raises(ValueError):
        ops.RopeTable.build(64, 10, inv_freq=torch.ones(31), device="cpu")
    for kw in (dict(weight=torch.ones((2, 2))), dict(weight=torch.ones(4, dtype=torch.int32)),
               dict(weight=torch.ones(8)[::2]), dict(weight=torch.ones(4), eps=-1.0)):
        with pytest.raises(ValueError):
            ops.HeadNorm(**kw)
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    for a in ((i(0, 3), i(3, 4), 3), (i(0, 3).long(), i(3), 3), (i(0, 3), i(3).float(), 3),
              (i(0), i(), 0), (i(0, 3), i(3), -1), (i(0, 9, 3, 9)[::2], i(3), 3)):
        with pytest.raises(ValueError):
            ops.RaggedBatch(*a)


def test_descriptors_follow_their_tensors():
    """A description is frozen; memory that moved under its tensor (module.to()) is seen."""
    w = torch.nn.Parameter(torch.ones(8))
    norm = ops.HeadNorm(w)
    first = norm.c.weight
    w.data = torch.ones(8, dtype=torch.bfloat16)
    assert norm.c.weight == w.data_ptr() != first and norm.c.dtype == _lib.TQ_BF16
    with pytest.raises(AttributeError):
        norm.eps = 1.0
    batch = ops.RaggedBatch(torch.tensor([0, 3], dtype=torch.int32),
                            torch.tensor([3], dtype=torch.int32), 3)
    with pytest.raises(AttributeError):
        batch.max_q_len = 4


def tables_on(device, D=128, kb=4, vb=2):
    z = lambda *n: torch.zeros(n, device=device)  # noqa: E731
    return ops.LayerTables(D, kb, vb, False, z(1 << kb), z((1 << kb) - 1), z(1 << vb),
                           z((1 << vb) - 1), z(D, D))


def test_pages_that_do_not_fit_are_refused():
    t, dev = tables_on("cpu"), torch.device("cpu")
    pb = ops.page_bytes(128, 4, 2, False)
    pages = torch.zeros((4, 2, pb), dtype=torch.uint8)
    assert ops._pages(t, pages, dev)
    table = torch.zeros((4, 2), dtype=torch.int32)
    assert ops._pages(t, ops.PagedPages(pages[0], table), dev)
    for bad in (pages[:, ::2], pages[..., :-64], pages.float(), pages[0],
                torch.zeros((4, 2, pb + 64), dtype=torch.uint8), pages.transpose(0, 1),
                ops.PagedPages(torch.zeros((4, pb + 64), dtype=torch.uint8), table),
                ops.PagedPages(torch.zeros((4, 2 * pb), dtype=torch.uint8)[:, :pb], table)):
        with pytest.raises(ValueError, match="pages"):
            ops._pages(t, bad, dev)
    with pytest.raises(ValueError, match="tables on"):
        ops._pages(t, pages, torch.device("cuda", 0))


def test_positions_follow_the_batch():
    """A batch's positions are computed once, and again when its lengths change in place."""
    from bhaskera_col_b200.inference.vllm_turboquant import VLLMBatch
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    b = VLLMBatch(i(0, 2, 2, 5), i(7, 4, 3), torch.zeros((3, 1), dtype=torch.int32), 5, 3)
    assert b.positions().tolist() == [5, 6, 0, 1, 2]
    assert b.positions() is b.positions()
    b.seq_lens.add_(10)
    assert b.positions().tolist() == [15, 16, 10, 11, 12]
    with torch.inference_mode():
        c = VLLMBatch(i(0, 2, 2, 5), i(7, 4, 3), b.block_table, 5, 3)
        assert c.positions().tolist() == [5, 6, 0, 1, 2]
        c.seq_lens.add_(1)
        assert c.positions().tolist() == [6, 7, 1, 2, 3]


def test_rope_table_values():
    t = ops.RopeTable.build(8, 20, base=100.0, scale=2.0, device="cpu")
    p = torch.arange(20, dtype=torch.float64)[:, None]
    a = p * 100.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)
    assert torch.equal(t.cos_sin, (2 * torch.cat([a.cos(), a.sin()], -1)).float())
    f = torch.tensor([1.0, 0.5, 0.25, 0.125])
    t = ops.RopeTable.build(8, 20, inv_freq=f, interleaved=True, device="cpu")
    assert t.interleaved and torch.equal(t.cos_sin[:, :4], (p * f.double()).cos().float())


def test_division_by_multiplication_is_exact():
    """The kernels' i / d: m = ceil(2^(31 + s) / d), 2^s >= d, for every i below 2^31.  The quotient
    can go wrong only beside a multiple of d, and the error grows with i."""
    for d in list(range(1, 300)) + [511, 512, 513, 1000, 1024, 65535, 65536]:
        s = (d - 1).bit_length()
        m = -(-(1 << (31 + s)) // d)
        assert m < 1 << 32
        top = (1 << 31) - 1
        ks = {1, 2, 3, top // d, top // d - 1, top // d // 2} | {random.Random(d).randrange(1, top // d + 1)
                                                                 for _ in range(50)}
        for k in ks:
            for i in (k * d - 1, k * d, k * d + 1):
                if 0 <= i <= top:
                    assert (i * m) >> (31 + s) == i // d


def test_attention_work_list_fits_its_bounds():
    """The launch's bounds on segments and partial slots hold for any lengths: tiles are at most
    N / pcta + R, and segments of at most L = max(min, ceil(all / wanted)) key tiles add at most
    wanted / G each way."""
    rng = random.Random(0)
    for _ in range(300):
        R = rng.randrange(1, 40)
        q = [rng.choice([0, 1, rng.randrange(1, 9), rng.randrange(1, 3000)]) for _ in range(R)]
        t = [rng.choice([0, 1, rng.randrange(1, 100000)]) for _ in range(R)]
        causal = rng.random() < 0.5
        seq = [a + b for a, b in zip(q, t)] if causal else t
        pcta, keys = rng.choice([1, 2, 4, 16, 64]), rng.choice([64, 128])
        G, wanted, least = rng.choice([1, 5, 8, 64, 300]), 148 * rng.choice([3, 5]), rng.choice([4, 8])
        tiles = []
        for a, s in zip(q, seq):
            for i in range(-(-a // pcta)):
                kend = s - a + min((i + 1) * pcta, a) if causal else s
                tiles.append(max(0, -(-kend // keys)))
        L = max(least, -(-sum(tiles) * G // wanted))
        ns = [max(1, -(-n // L)) for n in tiles]
        extra = wanted // G + 1
        assert sum(ns) <= sum(q) // pcta + R + extra
        assert sum(n for n in ns if n > 1) <= 2 * extra
        for n, k in zip(tiles, ns):                        # parts cover the tile, none above L
            base, more = divmod(n, k)
            assert base + (more > 0) <= L


def vllm_batch(start, seq, n, most):
    from bhaskera_col_b200.inference.vllm_turboquant import VLLMBatch
    i = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return VLLMBatch(i(start), i(seq), torch.zeros((len(seq), 1), dtype=torch.int32), n, most)


def test_ragged_batch_follows_replaced_fields():
    """A step that replaces the batch's offsets, lengths or bound is described by the new ones."""
    b = vllm_batch([0, 2, 5], [7, 3], 5, 3)
    first = b.ragged()
    assert b.ragged() is first                             # one description for the layers of a step
    b.seq_lens = b.seq_lens + 1
    assert b.ragged().seq_lens is b.seq_lens and b.ragged().q_start is first.q_start
    b.query_start_loc = b.query_start_loc.clone()
    assert b.ragged().q_start is b.query_start_loc
    b.max_query_len = 9
    assert b.ragged().max_q_len == 9 and b.ragged().seq_lens is b.seq_lens


def test_positions_of_a_padded_batch():
    """Rows before the first request and behind the last (padding of a captured batch) are at 0, and
    so are tokens that lie before their request's start; requests without rows take no part."""
    assert vllm_batch([0, 2, 2, 3], [7, 4, 1], 6, 2).positions().tolist() == [5, 6, 0, 0, 0, 0]
    assert vllm_batch([2, 4, 5], [9, 3], 7, 2).positions().tolist() == [0, 0, 7, 8, 2, 0, 0]
    assert vllm_batch([0, 3], [1], 3, 3).positions().tolist() == [0, 0, 0]
    assert vllm_batch([0, 0], [5], 2, 0).positions().tolist() == [0, 0]
    assert vllm_batch([0, 2, 5], [7, 3], 5, 3).positions().dtype == torch.int64


def test_positions_follow_writes_that_torch_does_not_count():
    """A graph's replay and .data write lengths without a new version."""
    b = vllm_batch([0, 2, 5], [7, 3], 5, 3)
    assert b.positions().tolist() == [5, 6, 0, 1, 2]
    b.seq_lens.data.add_(4)
    assert b.positions().tolist() == [9, 10, 4, 5, 6]
    b.num_actual_tokens = 6
    assert b.positions().tolist() == [9, 10, 4, 5, 6, 0]
    with torch.inference_mode():
        assert b.positions().tolist() == [9, 10, 4, 5, 6, 0]
    assert not b.positions().is_inference()


def test_descriptors_follow_type_and_shape_at_one_address():
    """module.half() may put a weight of another type at the address of the old one."""
    buf = torch.zeros(64, dtype=torch.uint8)
    w = torch.nn.Parameter(buf[:32].view(torch.float32))
    norm = ops.HeadNorm(w)
    assert norm.c.dtype == _lib.TQ_F32
    w.data = buf[:16].view(torch.float16)
    assert norm.c.weight == buf.data_ptr() and norm.c.dtype == _lib.TQ_F16
    w.data = buf[:32].view(torch.float16)[::2]
    with pytest.raises(ValueError, match="contiguous"):
        norm.c
    buf = torch.zeros(48)
    table = ops.RopeTable(buf.view(6, 8))
    assert (table.c.positions, table.c.rot_dim) == (6, 8)
    table.cos_sin.data = buf[:16].view(4, 4)
    assert table.c.cos_sin == buf.data_ptr() and (table.c.positions, table.c.rot_dim) == (4, 4)
    buf = torch.zeros(8, dtype=torch.int32)
    batch = ops.RaggedBatch(buf[:4], buf[4:7], 1)
    assert batch.c.requests == 3
    batch.seq_lens.data, batch.q_start.data = buf[4:6], buf[:3]
    assert batch.c.requests == 2 and batch.c.q_start == buf.data_ptr()


def test_workspace_keeps_what_a_capture_has_seen(monkeypatch):
    """A captured call goes on using its buffer at every replay: growing must not give it back."""
    import gc
    import weakref
    dev, capturing = torch.device("cpu"), [False]
    monkeypatch.setattr(ops, "_capturing", lambda device: capturing[0], raising=False)
    ws = ops.DecodeWorkspace()
    first = weakref.ref(ws.get(1000, dev))
    second = weakref.ref(ws.get(2000, dev))
    gc.collect()
    assert first() is None and ws.get(1500, dev) is second()    # nothing captured: one buffer
    capturing[0] = True
    assert ws.get(1800, dev) is second()
    capturing[0] = False
    third = weakref.ref(ws.get(3000, dev))
    fourth = weakref.ref(ws.get(4000, dev))
    gc.collect()
    assert second() is not None and third() is None and ws.get(10, dev) is fourth()
    # a buffer first taken while capturing holds nothing before the graph has run: cleared for others
    ws = ops.DecodeWorkspace()
    capturing[0] = True
    own = ws.get(100, dev)
    own.fill_(7)
    assert ws.get(50, dev) is own and (own == 7).all()
    capturing[0] = False
    assert ws.get(100, dev) is own and (own == 0).all()
    own.fill_(7)
    assert ws.get(100, dev) is own and (own == 7).all()


@pytest.mark.parametrize("engine", [0, 1, 2, 3])
@pytest.mark.parametrize("dtype", [_lib.TQ_BF16, _lib.TQ_F16, _lib.TQ_F32])
def test_attend_workspace_query_accepts_what_the_call_does(dtype, engine):
    """Code widths that the query sizes a workspace for are those that the call goes on with (here up
    to its workspace check)."""
    for D in (64, 128):
        for kb in range(1, 9):
            for vb in range(1, 9):
                q = t4((1, 4, 10, D), dtype=dtype)
                rc, err, need = attend(g=geom(D, kb, vb), q=q, out=far((1, 4, 10, D), dtype=dtype),
                                       engine=engine, nbytes=0)
                assert (need > 0) == (rc == _lib.TQ_ERR_WORKSPACE), err
                assert need > 0 or "no kernel" in err
    # the protected layers of K3/V2: (5, 4)
    rc, _, need = attend(g=geom(kb=5, vb=4), q=t4((1, 4, 10, 128), dtype=dtype),
                         out=far((1, 4, 10, 128), dtype=dtype), engine=engine, nbytes=0)
    assert (need > 0) == (engine < 3)


def test_attend_needs_an_aligned_rotation():
    """The rotation is read in pieces of up to 16 bytes; a table that LayerTables is given anywhere in
    memory is moved to where that holds."""
    for dtype in (_lib.TQ_BF16, _lib.TQ_F32):
        t = _lib.Tables(*([4096] * 4), 4100, *([4096] * 6))
        rc, err, need = attend(t=t, q=t4((1, 4, 10, 128), dtype=dtype), out=far((1, 4, 10, 128), dtype=dtype),
                               nbytes=0)
        assert rc == _lib.TQ_ERR_INVALID and "rot" in err and need > 0
    z = lambda *n: torch.zeros(n)  # noqa: E731
    R = torch.arange(128.0 * 128 + 3)[3:].view(128, 128)
    assert R.data_ptr() % 16
    t = ops.LayerTables(128, 4, 2, False, z(16), z(15), z(4), z(3), R)
    assert t.rot.data_ptr() % 16 == 0 and torch.equal(t.rot, R) and torch.equal(t.rot_t, R.t())


def places(x):
    """Byte addresses of a small view's elements."""
    es = 4 if x.dtype == _lib.TQ_F32 else 2
    at = {x.data}
    for n, s in zip(x.shape, x.stride):
        at = {a + i * s * es for a in at for i in range(n)}
    return {a + b for a in at for b in range(es)}


def test_outputs_beside_inputs_in_one_buffer():
    """Slices of one buffer that share no element are taken, whatever their order; views that share one
    are refused (but for an output that is its input)."""
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(600):
        B, T, D = rng.choice([1, 1, 2]), rng.choice([1, 2, 3]), 4
        heads = [rng.choice([1, 2]) for _ in range(2)]
        row = rng.choice([4, 6, 8]) * D
        pad = rng.choice([0, 0, row])
        b0 = 1 << 20
        at = [b0 + 2 * rng.randrange(0, 2 * row, rng.choice([1, D])) for _ in range(2)]
        tr = rng.random() < 0.5                            # token-major or head-major rows
        view = lambda h, a: t4((B, h, T, D), stride=[T * row * 2 + pad, D if tr else T * row // 2,  # noqa: E731
                                                     row if tr else D, 1], data=a)
        x, y = view(heads[0], at[0]), view(heads[0], at[1])
        rc, err = rope_call(rope=_lib.Rope(4096, 9, 4, 0), pos=POS, q=x, qo=y)
        if "share memory" in err and rc == _lib.TQ_ERR_INVALID:
            continue
        shared = at[0] != at[1] and bool(places(x) & places(y))
        assert rc == (_lib.TQ_ERR_INVALID if "overlaps" in err and rc == _lib.TQ_ERR_INVALID else _lib.TQ_ERR_CUDA)
        if shared:
            assert rc == _lib.TQ_ERR_INVALID
        seen[shared] += 1
    assert min(seen) > 50
    n, D, hq, hkv = 7, 128, 4, 2
    row = (hq + 2 * hkv) * D
    fused = lambda h, first: t4((1, h, n, D), stride=[0, D, row, 1], data=(1 << 20) + 2 * first * D)  # noqa: E731
    q, k, v = fused(hq, 0), fused(hkv, hq), fused(hkv, hq + hkv)
    base = dict(rope=ROPE, pos=POS)
    other = far((1, hkv, n, D))
    for kw in (dict(q=q, qo=q, k=k, ko=k), dict(k=k, ko=v), dict(q=k, qo=v), dict(q=k, qo=v, k=q, ko=q)):
        rc, err = rope_call(**base, **kw)
        assert rc == _lib.TQ_ERR_CUDA, err                 # past the checks: there is no device here
    for kw in (dict(q=k, qo=v, k=v, ko=v), dict(q=k, qo=k, k=v, ko=k), dict(q=k, qo=other, k=v, ko=other),
               dict(q=k, qo=v, k=v, ko=other), dict(q=q, qo=fused(hq, 1))):
        rc, err = rope_call(**base, **kw)
        assert rc == _lib.TQ_ERR_INVALID and "overlaps" in err, err
    # read-back: the two outputs
    kv = lambda first: t4(KV, stride=[0, 128, 512, 1], data=(1 << 20) + 256 * first)  # noqa: E731
    assert entry("read", k=kv(0), v=kv(2))[0] == _lib.TQ_ERR_CUDA
    for v2 in (kv(0), kv(1)):
        rc, err = entry("read", k=kv(0), v=v2)
        assert rc == _lib.TQ_ERR_INVALID and "overlaps" in err
    # attention: q a slice of the fused projection, out another or itself
    a = lambda first: t4((1, 4, 10, 128), stride=[0, 128, 2048, 1], data=(1 << 20) + 256 * first)  # noqa: E731
    for first, good in ((0, True), (4, True), (12, True), (3, False), (15, False)):
        rc, err, _ = attend(q=a(0), out=a(first), nbytes=0)
        assert (rc == _lib.TQ_ERR_WORKSPACE) == good and (good or "overlaps" in err), (first, err)


def test_tangents_are_refused():
    """Forward-mode differentiation: dropping the tangent would be a wrong derivative of 0."""
    x = torch.zeros((3, 2, 128))
    w = torch.ones(128)
    table = ops.RopeTable(torch.zeros((5, 128)))
    batch = ops.RaggedBatch(torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3], dtype=torch.int32), 3)
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        d = ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.qk_rope(d, None, table, torch.arange(3)),
                     lambda: ops.qk_rope(x, None, None, q_norm=ops.HeadNorm(ad.make_dual(w, w))),
                     lambda: ops.append_ragged(None, None, x, d, batch),
                     lambda: ops.dequantize_ragged(None, None, batch, d, None),
                     lambda: ops.attend_ragged(None, None, d, batch)):
            with pytest.raises(RuntimeError, match="derivative"):
                call()
        with pytest.raises(RuntimeError, match="no CPU path"):
            ops.attend_ragged(None, None, x, batch)


def test_device_status_reads_the_word_of_its_device(monkeypatch):
    """The word is looked up on the current device: the one asked for is made current."""
    current, seen = [0], []

    class Device:                                          # torch.cuda.device without a driver
        def __init__(self, device):
            self.to = device.index

        def __enter__(self):
            self.back, current[0] = current[0], self.to

        def __exit__(self, *a):
            current[0] = self.back

    class Lib:
        @staticmethod
        def tq_device_status(word, stream):
            seen.append(current[0])
            return _lib.TQ_OK

    monkeypatch.setattr(ops._lib, "load", lambda: Lib)
    monkeypatch.setattr(ops, "_stream", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    for d in (torch.device("cuda", 1), torch.device("cuda", 0), torch.device("cuda")):
        assert ops.device_status(d) == 0
    current[0] = 2
    assert ops.device_status() == 0
    assert seen == [1, 0, 0, 2] and current == [2]
