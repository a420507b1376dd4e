"""Rotations with several position axes (qk_rope, append_ragged) and the norms around a block
(residual_norm) against their plain forms in 64 bits.

Tolerances: the rotation's and the store's as in test_gpu_serving_ops; residual_norm: half an ulp of the
result's type plus the bound of the fp32 arithmetic (layer_oracle), 2^-25 for fp16 subnormals."""
import numpy as np
import pytest
import torch

import layer_oracle as L
import serving_oracle as S
from bhaskera_col_b200 import _lib
from bhaskera_col_b200.inference import ops
from test_gpu_parity import DEV, make_tables
from test_gpu_serving_ops import (BF16, F16, F32, LENS, check_read, check_stored, contiguous, make_batch,
                                  make_paged, ok_status, randn)

pytestmark = pytest.mark.gpu


def grid_positions(n, axes, top, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, top, (axes, n), generator=g)


# --------------------------------------------------------------------------- rotations with axes
def check_axes(got, x, table, pos, norm):
    w = norm.weight if norm else None
    eps, off = (norm.eps, norm.offset) if norm else (0.0, 0.0)
    want = L.rope_axes(x, table.cos_sin, pos, table.axes, table.interleaved, w, eps, off)
    tol = S.half_ulp(x.dtype) * np.abs(want) + S.rope_slack(x, w, eps, off)
    if x.dtype == F16:
        tol = tol + 2.0 ** -25
    err = np.abs(L.arr(got) - want)
    assert (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,hq,hkv,D,sections,mixed,norm", [
    (1, 1, 1, 128, (16, 24, 24), False, False), (5, 8, 2, 128, (24, 20, 20), True, True),
    (131, 5, 1, 64, (16, 16), False, True), (33, 4, 4, 128, (1, 30, 1), False, False),
    (17, 3, 3, 96, (4, 4, 4, 4), True, True), (9, 2, 1, 256, (50, 70, 8), False, True),
    (7, 2, 2, 80, (5, 12, 7), False, False), (3, 1, 1, 8, (1, 1), True, False),
    (3, 1, 1, 2, (1,), False, False), (301, 40, 8, 128, (63, 1), False, True),
    (40, 3, 2, 64, (0, 20, 12), True, False)])
def test_rope_with_axes_matches_plain_form(n, hq, hkv, D, sections, mixed, norm, dtype, interleaved):
    axes = ops.RopeTable.axis_of_pairs(sections, mixed)
    table = ops.RopeTable.build(2 * len(axes), 3000, interleaved=interleaved, device=DEV, axes=axes)
    pos = grid_positions(n, table.num_axes, 3000, n)
    pos[0, 0], pos[-1, -1] = 0, 2999
    norms = [ops.HeadNorm(randn((D,), 7 + i, dtype if i else F32), 1e-6, float(i))
             if norm else None for i in range(2)]
    q, k = randn((n, hq, D), 1, dtype, 3), randn((n, hkv, D), 2, dtype)
    for bits in (torch.int32, torch.int64):
        qo, ko = ops.qk_rope(q, k, table, pos.to(DEV, bits), *norms)
        check_axes(qo, q, table, pos.numpy(), norms[0])
        check_axes(ko, k, table, pos.numpy(), norms[1])
    # one position of a token for all its axes: the rotation without axes, to the bit
    plain = ops.RopeTable(table.cos_sin, interleaved)
    one = pos[0].to(DEV)
    same = ops.qk_rope(q, k, plain, one, *norms)
    for got in (ops.qk_rope(q, k, table, one, *norms),
                ops.qk_rope(q, k, table, one.expand(table.num_axes, n), *norms)):
        assert all(torch.equal(a, b) for a, b in zip(got, same))
    assert ok_status() == 0


def test_rope_with_axes_batches_views_and_in_place():
    """(B, H, T, D) heads with positions (axes, B, T), (T,) and (B, T); strided positions; slices of a
    fused projection rotated in place; odd offsets."""
    axes = ops.RopeTable.axis_of_pairs((10, 12, 10))
    table = ops.RopeTable.build(64, 900, device=DEV, axes=axes)
    B, T, H, D = 2, 13, 3, 64
    raw = randn((B * T * H * D + 1,), 4)
    x = raw[1:].view(B, T, H, D).transpose(1, 2)
    pos = grid_positions(B * T, 3, 900, 5).view(3, B, T)
    for p in (pos.to(DEV), pos.permute(2, 0, 1).contiguous().to(DEV).permute(1, 2, 0)):
        y, _ = ops.qk_rope(x, None, table, p)
        for b in range(B):
            check_axes(y[b].transpose(0, 1), x[b].transpose(0, 1), table, pos[:, b].numpy(), None)
    for p in (torch.arange(T, device=DEV), torch.arange(B * T, device=DEV).view(B, T)):
        y, _ = ops.qk_rope(x, None, table, p)
        pp = p.expand(B, T).cpu().numpy()
        for b in range(B):
            check_axes(y[b].transpose(0, 1), x[b].transpose(0, 1), table, np.stack([pp[b]] * 3), None)
    n = 19
    fused = randn((n, 5 * D), 6)
    keep = fused.clone()
    q, k = fused[:, : 3 * D].view(n, 3, D), fused[:, 3 * D: 4 * D].view(n, 1, D)
    flat = grid_positions(n, 3, 900, 7)
    ops.qk_rope(q, k, table, flat.to(DEV), q_out=q, k_out=k)
    check_axes(q, keep[:, : 3 * D].view(n, 3, D), table, flat.numpy(), None)
    check_axes(k, keep[:, 3 * D: 4 * D].view(n, 1, D), table, flat.numpy(), None)
    assert torch.equal(fused[:, 4 * D:], keep[:, 4 * D:])
    e, _ = ops.qk_rope(q[:0], None, table, flat[:, :0].to(DEV))
    assert e.shape == (0, 3, D) and ok_status() == 0


def test_rope_with_axes_bad_positions():
    """An axis' position outside the table takes row 0 for that axis alone and is flagged."""
    table = ops.RopeTable.build(64, 100, device=DEV, axes=ops.RopeTable.axis_of_pairs((16, 16)))
    x = randn((1, 2, 64), 1, F32).expand(4, 2, 64).contiguous()
    bad = torch.tensor([[5, 100, 5, -1], [7, 7, 1 << 40, 7]], device=DEV)
    good = torch.tensor([[5, 0, 5, 0], [7, 7, 0, 7]], device=DEV)
    odd = torch.zeros((4, 2, 66), device=DEV)
    odd[..., 1:65] = x
    for view in (x, odd[..., 1:65]):                        # the register kernel, the other
        a, _ = ops.qk_rope(view, None, table, bad)
        assert ok_status() == _lib.DEV_BAD_POSITION
        b, _ = ops.qk_rope(view, None, table, good)
        assert torch.equal(a, b) and ok_status() == 0


@pytest.mark.parametrize("D,kb,vb,H,dtype,sections,mixed,interleaved,norm", [
    (128, 4, 2, 2, BF16, (16, 24, 24), False, False, False),
    (128, 4, 4, 8, BF16, (24, 20, 20), True, False, True),
    (128, 8, 1, 3, F32, (5, 20, 7), False, True, False),
    (64, 3, 3, 4, F16, (16, 16), False, False, True), (64, 6, 5, 2, F32, (4, 4, 4, 4), True, True, True),
    (96, 5, 7, 1, BF16, (20, 20, 8), False, False, True),
    (128, 4, 2, 2, BF16, (3, 2), False, False, False), (32, 2, 2, 2, BF16, (8, 8), True, False, False)])
@pytest.mark.parametrize("lens", sorted(LENS))
def test_append_with_axes_and_read_back(D, kb, vb, H, dtype, sections, mixed, interleaved, norm, lens):
    tables = make_tables(D, kb, vb, False)
    lens = LENS[lens]
    R = len(lens)
    batch, start, seq = make_batch(lens, lead=2)
    n = start[-1] + 3
    pages = make_paged(tables, R * H, max(seq))
    k, v = randn((n, H, D), 1, dtype, 9), randn((n, H, D), 2, dtype, 11)
    axes = ops.RopeTable.axis_of_pairs(sections, mixed)
    rope = ops.RopeTable.build(2 * len(axes), 400, interleaved=interleaved, device=DEV, axes=axes)
    w = ops.HeadNorm(1 + 0.2 * randn((D,), 3, F32), 1e-6) if norm else None
    pos = grid_positions(n, rope.num_axes, 400, 3)
    for p in (pos.to(DEV), pos.to(torch.int32).t().contiguous().to(DEV).t()):
        pages.pool.zero_()
        ops.append_ragged(tables, pages, k, v, batch, rope=rope, k_norm=w, positions=p)
        assert ok_status() == 0
        kx = L.rope_axes(k, rope.cos_sin, pos.numpy(), axes, interleaved, w.weight if w else None, 1e-6)
        check_stored(tables, pages, k, v, start, seq, R, H, kx)
    check_read(tables, pages, batch, start, seq, n, H, dtype)
    # without positions every axis is at the token's place, as without axes
    pages.pool.zero_()
    ops.append_ragged(tables, pages, k, v, batch, rope=rope, k_norm=w)
    first = pages.pool.clone()
    pages.pool.zero_()
    ops.append_ragged(tables, pages, k, v, batch, rope=ops.RopeTable(rope.cos_sin, interleaved), k_norm=w)
    assert torch.equal(first, pages.pool) and ok_status() == 0


@pytest.mark.parametrize("D,kb,dtype,interleaved,norm", [(64, 3, F16, True, False), (128, 4, BF16, False, True)])
def test_append_with_axes_codes_are_those_of_exact_arithmetic(D, kb, dtype, interleaved, norm):
    tables = make_tables(D, kb, 4, False)
    H, n = 4, (1 << 20) // (4 * D) - 5
    batch, start, seq = make_batch([(n - 700, n - 700), (700, 900)])
    pages = make_paged(tables, 2 * H, max(seq))
    k = randn((n, H, D), 21, dtype)
    axes = ops.RopeTable.axis_of_pairs((D // 2 - 20, 11, 9), True)
    rope = ops.RopeTable.build(D, n, interleaved=interleaved, device=DEV, axes=axes)
    w = ops.HeadNorm(0.2 * randn((D,), 23, F32), 1e-6, 1.0) if norm else None
    at = grid_positions(n, 3, n, 9)
    ops.append_ragged(tables, pages, k, k, batch, rope=rope, k_norm=w, positions=at.to(DEV))
    got = S.parse(tables, contiguous(pages), max(seq))
    r, pos = S.positions(start, seq, n)
    x = L.rope_axes(k, rope.cos_sin, at.numpy(), axes, interleaved, w.weight if w else None, 1e-6, 1.0)
    y = (x / np.linalg.norm(x, axis=-1, keepdims=True)) @ L.arr(tables.rot).T
    b = L.arr(tables.k_boundaries)[: (1 << kb) - 1]
    code = np.searchsorted(b, y, side="left")
    gap = np.abs(y[..., None] - b[np.clip(np.stack([code - 1, code], -1), 0, len(b) - 1)]).min(-1)
    have = got["k_idx"].reshape(2, H, -1, D)[r, :, pos]
    assert not ((have != code) & (gap > 1e-12)).any()
    assert ok_status() == 0


def test_append_with_axes_bad_positions_and_places():
    """A position outside the table turns by row 0, a token without a place is dropped whatever its
    positions say, on both kernels."""
    for D in (128, 96):
        H = 2
        tables = make_tables(D, 4, 4, False)
        batch, start, seq = make_batch([(3, 66), (2, 2)])
        n = start[-1]
        pages = make_paged(tables, 2 * H, 64)
        rope = ops.RopeTable.build(32, 50, device=DEV, axes=ops.RopeTable.axis_of_pairs((8, 8)))
        k = randn((n, H, D), 1)
        pos = torch.tensor([[1, 2, 3, 50, 5], [6, 7, 8, 9, -1]], device=DEV)
        ops.append_ragged(tables, pages, k, k, batch, rope=rope, positions=pos)
        assert ok_status() == _lib.DEV_BAD_POSITION
        bad = pages.pool.clone()
        pages.pool.zero_()
        pos[0, 3], pos[1, 4] = 0, 0
        ops.append_ragged(tables, pages, k, k, batch, rope=rope, positions=pos)
        assert torch.equal(bad, pages.pool) and ok_status() == _lib.DEV_BAD_POSITION   # 64, 65: no place


@pytest.mark.parametrize("D", [128, 64, 96])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_with_axes_looks_at_the_positions_of_stored_tokens_alone(D, interleaved):
    """Rows of no request, in front of the batch and behind it, and tokens without a place have positions
    outside the table, and so does everybody on an axis that no pair follows: nothing is flagged for them,
    whichever kernel runs and however many tiles a CTA takes."""
    H = 8
    tables = make_tables(D, 4, 4, False)
    rope = ops.RopeTable.build(32, 50, interleaved=interleaved, device=DEV,
                               axes=ops.RopeTable.axis_of_pairs((8, 0, 8)))
    for lens in ([(3, 60), (2, 2)], [(2500, 2500), (1, 70)]):
        batch, start, seq = make_batch(lens, lead=5)
        n = start[-1] + 4
        pages = make_paged(tables, 2 * H, max(seq))
        k = randn((n, H, D), 1)
        good = torch.randint(0, 50, (3, n), generator=torch.Generator().manual_seed(n)).to(DEV)
        good[1] = 0
        ops.append_ragged(tables, pages, k, k, batch, rope=rope, positions=good)
        assert ok_status() == 0
        want = pages.pool.clone()
        pos = good.clone()
        pos[:, :start[0]], pos[:, start[-1]:], pos[1] = -1, 1 << 40, 77
        pages.pool.zero_()
        ops.append_ragged(tables, pages, k, k, batch, rope=rope, positions=pos)
        assert ok_status() == 0 and torch.equal(pages.pool, want)
        pos[2, start[0] + 1] = 50                          # a stored token's own
        ops.append_ragged(tables, pages, k, k, batch, rope=rope, positions=pos)
        assert ok_status() == _lib.DEV_BAD_POSITION


# ------------------------------------------------------------------------------- residual_norm
def check_norm(got, want, err, dtype):
    tol = S.half_ulp(dtype) * np.abs(want) + err * (1 + S.half_ulp(dtype))
    if dtype == F16:
        tol = tol + 2.0 ** -25
    off = np.abs(L.arr(got) - want)
    assert got.dtype == dtype and (off <= tol).all(), (off - tol).max()


def run_norm(x, res, post, gate, act, scale, pre, **kw):
    y, h = ops.residual_norm(x, res, post_norm=post, gate=gate, gate_act=act, scale=scale, pre_norm=pre, **kw)
    yw, dy, hw, dh = L.residual_norm(x, res, post, gate, act, scale, pre)
    check_norm(y, yw, dy, res.dtype)
    if pre is None:
        assert h is None
    else:
        check_norm(h, hw, dh, x.dtype)
    return y, h


def row_norm(C, seed, dtype, kind):
    if kind == "bare":
        return ops.RowNorm(eps=1e-5)
    w, b = 1 + 0.3 * randn((C,), seed, F32), 0.2 * randn((C,), seed + 1, F32)
    if kind == "layer":
        return ops.RowNorm(w.to(dtype), b.to(dtype), 1e-5, centered=True)
    if kind == "offset":
        return ops.RowNorm((w - 1).to(dtype), eps=1e-6, offset=1.0)
    return ops.RowNorm(w.to(dtype), eps=1e-6)


@pytest.mark.parametrize("dtype,rdtype", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32), (F16, F32),
                                          (F32, BF16), (BF16, F16)])
@pytest.mark.parametrize("n,C,post,gate,act,pre", [
    (1, 1, "rms", "full", "none", "rms"), (3, 7, "layer", "token", "sigmoid", "layer"),
    (5, 64, "rms", "channel", "none", "rms"), (9, 250, None, "full", "tanh", "layer"),
    (6, 512, "offset", None, "none", "bare"), (301, 1024, "rms", "full", "sigmoid", "rms"),
    (2, 1032, "layer", "channel", "none", None), (303, 2050, "layer", "full", "sigmoid", "layer"),
    (16, 5120, "rms", None, "none", "rms"), (299, 5120, "rms", "one", "tanh", "offset"),
    (4, 8200, "rms", None, "none", "layer"), (2, 16392, "layer", "full", "none", "rms"),
    (300, 4097, None, None, "none", "rms"), (1, 32768, "layer", "channel", "tanh", "layer"),
    (300, 32767, "rms", "full", "none", None)])
def test_residual_norm_matches_plain_form(n, C, post, gate, act, pre, dtype, rdtype):
    if n * C > 3_000_000 and rdtype == F16:
        n = 150                                            # the oracle's time
    x, res = randn((n, C), 1, dtype, 5), (3 * randn((n, C), 2, F32, 7)).to(rdtype)
    shape = dict(full=(n, C), channel=(C,), token=(n, 1), one=(1,)).get(gate)
    g = None if shape is None else randn(shape, 3, dtype)
    run_norm(x, res, post and row_norm(C, 4, dtype, post), g, act, 0.5 if gate == "channel" else 1.0,
             pre and row_norm(C, 8, F32 if rdtype == F32 else dtype, pre))


def test_residual_norm_views_in_place_and_broadcasts():
    """Slices of a wider buffer, transposed batches, other strides of the last dim, results into views;
    residual and x as their own results; every chunk width of the kernel."""
    post, pre = row_norm(96, 1, BF16, "rms"), row_norm(96, 2, F32, "layer")
    wide = randn((2, 5, 3 * 96 + 3), 3)
    for off in (0, 1, 2, 8):
        x, res = wide[..., off: off + 96], wide[..., 96 + off: 192 + off]
        run_norm(x, res, post, wide[:, :1, 192: 288], "sigmoid", 2.0, pre)
    t = randn((5, 2, 96), 4).transpose(0, 1)               # (B, T, C) of (T, B, C) memory
    run_norm(t, randn((2, 5, 96), 5, F32), post, None, "none", 1.0, pre)
    cols = randn((96, 7), 6).t()
    run_norm(cols, randn((7, 96), 7), post, randn((96, 7), 8).t(), "tanh", 1.0, pre)
    run_norm(randn((96,), 9), randn((96,), 10), post, None, "none", 1.0, pre)
    run_norm(randn((2, 3, 2, 96), 9), randn((2, 3, 2, 96), 10), None, randn((2, 1, 2, 1), 11), "none", 1.0, pre)
    same = randn((1, 96), 12).expand(6, 96)                # one block output for all rows
    run_norm(same, randn((6, 96), 13), post, None, "none", 1.0, pre)
    x, res, gate = randn((9, 96), 14), randn((9, 96), 15, F32), randn((9, 96), 16)
    y, h = run_norm(x, res, post, gate, "none", 1.0, pre)
    x2, res2 = x.clone(), res.clone()
    a, b = ops.residual_norm(x2, res2, post, gate, "none", 1.0, pre, residual_out=res2, out=x2)
    assert a is res2 and b is x2 and torch.equal(a, y) and torch.equal(b, h)
    buf = torch.zeros((9, 300), dtype=BF16, device=DEV)
    ops.residual_norm(x, res, post, gate, "none", 1.0, pre, residual_out=res2, out=buf[:, 101: 197])
    # chunks of other widths sum in another order: a last bit at most
    ref = b.float()
    assert (buf[:, 101: 197].float() - ref).abs().max() <= 2.0 ** -7 * ref.abs().max()
    assert (buf[:, :101] == 0).all() and (buf[:, 197:] == 0).all()
    e, f = ops.residual_norm(x[:0], res[:0], post, gate[:0], "none", 1.0, pre)
    assert e.shape == f.shape == (0, 96)


def test_residual_norm_extremes():
    """A zero row stays zero (eps > 0); NaN and infinity keep to their own row; a result does not
    depend on the rows around it, nor on when it is computed."""
    post = ops.RowNorm(eps=1e-5)
    x, res = randn((400, 1500), 1, F32), randn((400, 1500), 2, F32)
    x[0], res[0] = 0, 0
    x[1, 3], x[2, 4] = float("nan"), float("inf")
    res[3, 5] = float("-inf")
    y, h = ops.residual_norm(x, res, post, None, "none", 1.0, post)
    assert (y[0] == 0).all() and (h[0] == 0).all()
    assert y[1].isnan().all() and y[2].isnan().any() and y[3].isinf().sum() == 1 and h[3].isnan().any()
    rows = torch.tensor([r for r in range(400) if r not in (1, 2, 3)], device=DEV)
    assert y[rows].isfinite().all() and h[rows].isfinite().all()
    again = ops.residual_norm(x, res, post, None, "none", 1.0, post)
    assert torch.equal(again[0][rows], y[rows]) and torch.equal(again[1][rows], h[rows])
    some = ops.residual_norm(x[rows[:350]], res[rows[:350]], post, None, "none", 1.0, post)
    assert torch.equal(some[0], y[rows[:350]]) and torch.equal(some[1], h[rows[:350]])


def test_residual_norm_captured_and_on_another_stream():
    norm = row_norm(640, 1, BF16, "rms")
    x, res, gate = randn((33, 640), 2), randn((33, 640), 3, F32), randn((33, 1), 4)
    want = ops.residual_norm(x, res, norm, gate, "sigmoid", 1.0, norm)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.residual_norm(x, res, norm, gate, "sigmoid", 1.0, norm)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    live = x.clone(), res.clone(), gate.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.residual_norm(live[0], live[1], norm, live[2], "sigmoid", 1.0, norm)
    for seed in (5, 9):
        for i, t in enumerate(live):
            t.copy_(randn(t.shape, seed + i, F32))
        want = ops.residual_norm(live[0], live[1], norm, live[2], "sigmoid", 1.0, norm)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("n,C", [(20011, 64), (2003, 1026), (1201, 4096), (601, 8192)])
@pytest.mark.parametrize("gate", [None, "full"])
def test_residual_norm_in_place_over_many_rows(n, C, gate):
    """Rows that are on their way while earlier ones are written over: the same bits as into
    other memory, and the first and last rows those of a call of their own."""
    post, pre = row_norm(C, 1, BF16, "rms"), row_norm(C, 2, BF16, "layer")
    x, res = randn((n, C), 3), randn((n, C), 4, F32)
    g = randn((n, C), 5) if gate else None
    y, h = ops.residual_norm(x, res, post, g, "none", 1.0, pre)
    for at in (slice(0, 3), slice(n - 3, n)):
        a, b = run_norm(x[at], res[at], post, g if g is None else g[at], "none", 1.0, pre)
        assert torch.equal(a, y[at]) and torch.equal(b, h[at])
    ops.residual_norm(x, res, post, g, "none", 1.0, pre, residual_out=res, out=x)
    assert torch.equal(res, y) and torch.equal(x, h)


@pytest.mark.parametrize("kind", ["rms", "layer", "bare"])
@pytest.mark.parametrize("gdtype", [BF16, F16, F32, None])
@pytest.mark.parametrize("n,C,extra", [(5, 64, 0), (7, 1024, 0), (3, 1000, 1), (4, 2050, 0), (3, 4096, 0), (3, 4096, 1),
                                       (3, 4096, 2), (3, 5128, 0), (2, 8192, 0), (3, 8200, 0), (3, 4097, 0), (2, 20000, 0)])
def test_residual_norm_of_one_row_is_the_row_of_a_batch(n, C, extra, gdtype, kind):
    """Rows called one by one give the bits that the batch gives, whatever the gate is a row of (a gate of
    its own per element, the channels', one number) and its type, and for slices of wider buffers."""
    dtype = F16 if gdtype == F16 else BF16
    post, pre = row_norm(C, 1, dtype, kind), row_norm(C, 2, F32, kind)
    x, res = (randn((n, C + extra), i, d)[:, :C] for i, d in ((3, dtype), (4, F32)))
    gates = [None] if gdtype is None else [2 * randn(s, 5, gdtype) for s in ((n, C), (C,), (1, C), (n, 1), (1,))]
    for gate in gates:
        y, h = ops.residual_norm(x, res, post, gate, "sigmoid" if gate is not None else "none", 0.7, pre)
        for i in range(n):
            at = slice(i, i + 1)
            g = gate[at] if gate is not None and gate.shape[0] == n and gate.dim() == 2 else gate
            a, b = ops.residual_norm(x[at], res[at], post, g, "sigmoid" if g is not None else "none", 0.7, pre)
            assert torch.equal(a, y[at]) and torch.equal(b, h[at]), (gate is not None and gate.shape, i)


def test_residual_norm_of_one_sequence_is_that_of_a_batch():
    """(B, T, C) with gates (B, 1, C): a sequence by itself, and a token of it."""
    B, T, C = 3, 4, 1032
    post, pre = row_norm(C, 1, BF16, "layer"), row_norm(C, 2, F32, "rms")
    x, res = randn((B, T, C), 3), randn((B, T, C), 4, F32)
    for gdtype in (BF16, F32):
        gate = randn((B, 1, C), 5, gdtype)
        y, h = ops.residual_norm(x, res, post, gate, "tanh", 0.7, pre)
        for b in range(B):
            for t in (slice(0, T), slice(2, 3)):
                one = ops.residual_norm(x[b: b + 1, t], res[b: b + 1, t], post, gate[b: b + 1], "tanh", 0.7, pre)
                assert torch.equal(one[0], y[b: b + 1, t]) and torch.equal(one[1], h[b: b + 1, t])


def test_paged_attention_with_norms_and_no_rotation_takes_positions():
    """A model whose layers partly have no rotation passes positions always: a layer with head norms alone
    does not look at them."""
    from bhaskera_col_b200.inference.vllm_turboquant import TurboQuantPagedAttention, VLLMBatch
    D, Hq, H, n = 128, 4, 2, 135
    norms = [ops.HeadNorm(1 + 0.1 * randn((D,), i, F32)) for i in range(2)]
    bt = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    batch = VLLMBatch(torch.tensor([0, 130, n], dtype=torch.int32, device=DEV),
                      torch.tensor([130, 5], dtype=torch.int32, device=DEV), bt, n, 130)
    q, k, v = (randn((n + 2, h, D), 10 + h) for h in (Hq, H, H + 2))
    v = v[:, :H]
    outs = []
    for pos in (None, torch.arange(n + 2, device=DEV), torch.full((3, n + 2), -1, device=DEV)):
        for kw in (dict(q_norm=norms[0], k_norm=norms[1]), dict(q_norm=norms[0]), dict(k_norm=norms[1])):
            layer = TurboQuantPagedAttention(3, 32, Hq, H, D, num_blocks=8, block_size=64, device=DEV)
            layer.pool.zero_()
            outs.append((layer.forward(q, k, v, batch, positions=pos, **kw)[:n],
                         layer.paged(layer.stream_table(bt)).pool))
    for i in range(3, 9):
        assert all(torch.equal(a, b) for a, b in zip(outs[i], outs[i % 3]))
    assert ok_status() == 0


def gates_over_the_range(dtype, n=4096):
    """Gates over the type's whole range, both signs, beside the places where the function's parts end."""
    top = float(torch.finfo(dtype).max)
    x = torch.cat([torch.linspace(-20, 20, n // 2, dtype=torch.float64),
                   torch.logspace(-30, np.log10(top) - 1e-6, n // 4, dtype=torch.float64)])
    x = torch.cat([x, -x[n // 2:]]).clamp(-top, top)
    edges = [0.0, -0.0, top, -top, float("inf"), -float("inf"), 1e-8, -1e-8]
    edges += [s * (c + d) for c in (87.0, 87.33655, 87.5, 88.72284, 89.0, 126.0, 127.0) for d in (-1e-5, 0.0, 1e-5)
              for s in (-1.0, 1.0) if c < top]
    x[: len(edges)] = torch.tensor(edges, dtype=torch.float64).clamp(-top, top) * 1.0
    x[4], x[5] = float("inf"), -float("inf")
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["channel", "element", "row"])
def test_gate_functions_over_their_range(kind, dtype, act):
    """y = act(gate) alone (x = 1, residual 0, fp32).  sigmoid = 1 / (1 + e^-g): e^-g is off, relatively,
    by the exponential's 2^-22 and three roundings of 2^-24 at most, the sum by one more, the quotient by
    2 ulp (2^-22): 2^-21 + 2^-22 in all; below 2^-126 results may be flushed.  tanh: 2 ulp (2^-22) and a
    rounding.  Infinite gates give the limits, NaN gives NaN in its own place."""
    g = gates_over_the_range(dtype)
    C = g.numel()
    want = g.double()
    want = torch.tanh(want) if act == "tanh" else torch.where(want >= 0, 1 / (1 + (-want).exp()),
                                                               want.exp() / (1 + want.exp()))
    one, zero = torch.ones((3, C), device=DEV), torch.zeros((3, C), device=DEV)
    gate = {"channel": g, "element": torch.stack([g.roll(i) for i in range(3)]), "row": g[:, None]}[kind]
    if kind == "row":
        one, zero, want = torch.ones((C, 8), device=DEV), torch.zeros((C, 8), device=DEV), want[:, None].expand(C, 8)
    elif kind == "element":
        want = torch.stack([want.roll(i) for i in range(3)])
    y, _ = ops.residual_norm(one, zero, gate=gate, gate_act=act)
    err = (y.double() - want).abs()
    assert (err <= (2.0 ** -21 + 2.0 ** -22) * want.abs() + 2.0 ** -126).all(), (err / want.abs()).nan_to_num().max()
    assert (y.abs() <= 1).all()
    bad = gate.clone()
    bad.view(-1)[7] = float("nan")
    y2, _ = ops.residual_norm(one, zero, gate=bad, gate_act=act)
    hit = bad.isnan().expand(y2.shape)
    assert hit.any() and y2[hit].isnan().all() and torch.equal(y2[~hit], y[~hit])
