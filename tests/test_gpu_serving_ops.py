"""The serving operators on ragged batches (qk_rope, append_ragged, dequantize_ragged,
attend_ragged) against their plain forms in 64 bits.

Tolerances (u = 2^-24; half_ulp(t) = eps(t) / 2):
  * qk_rope: one rounding to the output type, half_ulp |y|, plus the fp32 arithmetic
    (serving_oracle.rope_slack); fp16 results below 2^-14 are off by at most 2^-25;
  * append_ragged codes: an fp32 dot product of unit vectors is off by at most D u <= 7.6e-6 and the
    normed, rotated input by 16 u of its largest entry, so a code may differ from the 64-bit one
    only where the rotated value lies within 1e-5 of a boundary; norms: fp16 half ulp plus 32 u;
  * dequantize_ragged: half_ulp |x| plus 2^-16 n sum_j |c_j R_ji| (D = 128 fp32 terms: 2^-17); bf16
    results of the tensor-core form take c in fp16, off by 2^-11 |c_j| in each term: 2^-11 of the
    same sum more;
  * attend_ragged: the bar of the prefill tests for fp16 tensor-core operands, cosine >= 0.9999
    and max-abs within 4e-3 max|o| plus half an ulp of the output type.
"""
import numpy as np
import pytest
import torch

import serving_oracle as S
from bhaskera_col_b200 import _lib
from bhaskera_col_b200.inference import ops
from test_gpu_parity import DEV, cosine, make_tables

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def randn(shape, seed, dtype=BF16, outlier=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if outlier:
        x[..., outlier % shape[-1]] *= 8
    return x.to(dtype).to(DEV)


def int32(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


def make_batch(lens, lead=0):
    """lens: (new tokens, tokens in the cache) per request; the first row is `lead`."""
    start = np.concatenate([[0], np.cumsum([a for a, _ in lens])]) + lead
    seq = [b for _, b in lens]
    return (ops.RaggedBatch(int32(start), int32(seq), max([a for a, _ in lens] + [0])),
            start.tolist(), seq)


def make_paged(tables, streams, tokens, seed=0):
    """An empty pool in shuffled order behind a block table, and the table."""
    P = max(-(-tokens // 64), 1)
    pb = ops.page_bytes(tables.head_dim, tables.key_bits, tables.value_bits, False)
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(streams * P + 3, generator=g)[: streams * P].to(torch.int32).view(streams, P)
    pool = torch.zeros((streams * P + 3, pb), dtype=torch.uint8, device=DEV)
    return ops.PagedPages(pool, perm.to(DEV))


def contiguous(pages):
    return pages.pool[pages.block_table.long()] if isinstance(pages, ops.PagedPages) else pages


def fill(tables, pages, R, H, tokens, seed):
    """Every request's tokens [0, tokens) stored through tq_append."""
    k, v = (randn((R, H, tokens, tables.head_dim), seed + i, outlier=5 + i) for i in range(2))
    ops.append(tables, pages, k, v, 0)


def ok_status():
    torch.cuda.synchronize()
    return ops.device_status(DEV)


# ------------------------------------------------------------------------------------- qk_rope
def check_rope(got, x, table, pos, norm):
    w = norm.weight if norm else None
    eps, off = (norm.eps, norm.offset) if norm else (0.0, 0.0)
    cs = table.cos_sin if table else None
    want = S.rope(x, cs, pos, table.interleaved if table else False, w, eps, off)
    tol = S.half_ulp(x.dtype) * np.abs(want) + S.rope_slack(x, w, eps, off)
    if x.dtype == F16:
        tol = tol + 2.0 ** -25
    err = np.abs(got.detach().cpu().double().numpy() - want)
    assert (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,hq,hkv,D,rot,norm", [
    (1, 1, 1, 128, 128, False), (5, 8, 2, 128, 128, True), (131, 5, 1, 64, 64, True),
    (33, 4, 4, 128, 64, False), (17, 3, 3, 96, 32, True), (9, 2, 1, 256, 256, True),
    (7, 2, 2, 80, 48, True), (3, 1, 1, 2, 2, False), (64, 40, 8, 128, 128, True)])
def test_qk_rope_matches_plain_form(n, hq, hkv, D, rot, norm, dtype, interleaved):
    table = ops.RopeTable.build(rot, 5000, interleaved=interleaved, device=DEV)
    pos = torch.randint(0, 5000, (n,), generator=torch.Generator().manual_seed(n))
    pos[0], pos[-1] = 0, 4999
    norms = [ops.HeadNorm(randn((D,), 7 + i, dtype if i else F32), 1e-6, float(i))
             if norm else None for i in range(2)]
    q, k = randn((n, hq, D), 1, dtype, 3), randn((n, hkv, D), 2, dtype)
    for bits in (torch.int32, torch.int64):
        qo, ko = ops.qk_rope(q, k, table, pos.to(DEV, bits), *norms)
        assert qo.dtype == dtype and qo.shape == q.shape
        check_rope(qo, q, table, pos.numpy(), norms[0])
        check_rope(ko, k, table, pos.numpy(), norms[1])
    assert ok_status() == 0


def test_qk_rope_views_in_place_and_one_side():
    """Slices of one fused projection, rotated in place; HF's (B, H, T, D) transposed layout;
    broadcast positions and broadcast inputs; rows a multiple of nothing."""
    table = ops.RopeTable.build(128, 300, device=DEV)
    n, hq, hkv, D = 19, 6, 2, 128
    fused = randn((n, (hq + 2 * hkv) * D), 3)
    keep = fused.clone()
    q = fused[:, : hq * D].view(n, hq, D)
    k = fused[:, hq * D: (hq + hkv) * D].view(n, hkv, D)
    pos = torch.arange(n, device=DEV) * 7
    qk = q.clone(), k.clone()
    ops.qk_rope(q, k, table, pos, q_out=q, k_out=k)
    check_rope(q, qk[0], table, pos.cpu().numpy(), None)
    check_rope(k, qk[1], table, pos.cpu().numpy(), None)
    assert torch.equal(fused[:, (hq + hkv) * D:], keep[:, (hq + hkv) * D:])      # v untouched
    # (B, H, T, D) views of (B, T, H, D) memory, odd element offset, positions (T,) and (B, T)
    B, T = 2, 13
    raw = randn((B * T * hq * D + 1,), 4)
    x = raw[1:].view(B, T, hq, D).transpose(1, 2)
    for p in (torch.arange(T, device=DEV), torch.arange(B * T, device=DEV).view(B, T).flip(0)):
        y, none = ops.qk_rope(x, None, table, p)
        assert none is None
        pp = p.expand(B, T).cpu().numpy()
        for b in range(B):
            check_rope(y[b].transpose(0, 1), x[b].transpose(0, 1), table, pp[b], None)
    # one head read by all (stride 0), and a reversed head dim order through strides
    one = randn((n, 1, D), 5).expand(n, 4, D)
    y, _ = ops.qk_rope(one, None, table, pos)
    check_rope(y, one.contiguous(), table, pos.cpu().numpy(), None)
    z = randn((n, D, 3), 6).transpose(1, 2)
    _, y = ops.qk_rope(None, z, table, pos)
    check_rope(y, z.contiguous(), table, pos.cpu().numpy(), None)
    # only a norm
    norm = ops.HeadNorm(randn((D,), 8), 1e-5)
    y, _ = ops.qk_rope(z, None, None, None, q_norm=norm)
    check_rope(y, z.contiguous(), None, None, norm)
    # no rows
    e, _ = ops.qk_rope(z[:0], None, table, pos[:0])
    assert e.shape == (0, 3, D) and ok_status() == 0


def test_qk_rope_extremes():
    """Zero rows stay zero under the norm, huge and tiny rows keep their direction, NaN and inf
    stay in their own head; a position outside the table is flagged and turns by row 0."""
    table = ops.RopeTable.build(64, 100, device=DEV)
    x = randn((6, 2, 64), 1, F32)
    x[0] = 0
    x[1] *= 1e18
    x[2] *= 1e-18
    x[3, 0, 5] = float("nan")
    x[4, 1, 6] = float("inf")
    norm = ops.HeadNorm(torch.ones(64, device=DEV), 1e-6)
    pos = torch.tensor([1, 2, 3, 4, 5, 6], device=DEV)
    y, _ = ops.qk_rope(x, None, table, pos, q_norm=norm)
    assert (y[0] == 0).all()
    want = S.rope(x, table.cos_sin, pos.cpu().numpy(), False, norm.weight, 1e-6)
    ok = [(1, 0), (1, 1), (2, 0), (2, 1), (3, 1), (4, 0), (5, 0), (5, 1)]
    for r, h in ok:
        w = want[r, h]
        assert np.abs(y[r, h].cpu().double().numpy() - w).max() <= 40 * 2.0 ** -24 * np.abs(w).max()
    assert y[3, 0].isnan().any() and y[4, 1].isnan().any()
    assert ok_status() == 0
    bad = torch.tensor([100, -1, 0, 99, 1 << 40, 5], device=DEV)
    y, _ = ops.qk_rope(x[5:].expand(6, 2, 64).contiguous(), None, table, bad)
    assert ok_status() == _lib.DEV_BAD_POSITION
    assert torch.equal(y[0], y[2]) and torch.equal(y[1], y[2]) and torch.equal(y[4], y[2])


def test_rope_table_far_positions():
    """Angles come from 64 bits: at position 10^6 the table is the rounding of the exact values."""
    t = ops.RopeTable.build(32, 1_000_001, base=500000.0, scale=1.25, device=DEV)
    f = 500000.0 ** (-np.arange(0, 32, 2) / 32)
    a = 1_000_000 * f
    want = 1.25 * np.concatenate([np.cos(a), np.sin(a)])
    # 64-bit angle off by 2^-53 * 1e6 at most (2e-10), then one rounding to fp32
    assert np.abs(t.cos_sin[1_000_000].cpu().double().numpy() - want).max() <= 1.25 * 2.0 ** -24 + 1e-9


# --------------------------------------------------------------- append_ragged, dequantize_ragged
LENS = {
    "decode": [(1, 1), (1, 64), (1, 65), (1, 200)],
    "prompts": [(70, 70), (128, 128), (1, 1), (63, 63)],
    "mixed": [(5, 130), (1, 77), (0, 50), (64, 64), (129, 300), (3, 3)],
    "one": [(1, 1)],
}


def check_stored(tables, pages, k, v, start, seq, R, H, kx):
    """Codes and norms of every new token against 64 bits; kx: the transformed keys in 64 bits."""
    D = tables.head_dim
    tokens = contiguous(pages).shape[1] * 64
    f = S.parse(tables, contiguous(pages), tokens)
    Rm = tables.rot.cpu().double().numpy()
    r, pos = S.positions(start, seq, k.shape[0])
    rows = np.nonzero(r >= 0)[0]
    for name, x, bnd in (("k", kx, tables.k_boundaries), ("v", v.cpu().double().numpy(), tables.v_boundaries)):
        b = bnd.cpu().double().numpy()
        idx = f[f"{name}_idx"].reshape(R, H, tokens, D)[r[rows], :, pos[rows]]
        nrm = f[f"{name}_norm"].reshape(R, H, tokens)[r[rows], :, pos[rows]].astype(np.float64)
        xs = x[rows]
        n = np.linalg.norm(xs, axis=-1)
        y = (xs / np.maximum(n, 1e-8)[..., None]) @ Rm.T
        want = (y[..., None] > b).sum(-1)
        off = idx != want
        assert off.mean() <= 1e-4
        near = np.abs(y[..., None] - b).min(-1)
        assert (near[off] <= 1e-5).all()
        assert (np.abs(idx - want) <= 1).all()
        assert (np.abs(nrm - n) <= n * (2.0 ** -11 + 32 * 2.0 ** -24) + 2.0 ** -25).all()


def check_read(tables, pages, batch, start, seq, n, H, dtype):
    D = tables.head_dim
    tokens = contiguous(pages).shape[1] * 64
    kd, vd = S.dense(tables, contiguous(pages), tokens)
    f = S.parse(tables, contiguous(pages), tokens)
    aR = np.abs(tables.rot.cpu().double().numpy())
    r, pos = S.positions(start, seq, n)
    outs = [torch.full((n, H, D), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    ops.dequantize_ragged(tables, pages, batch, *outs)
    for name, out, x, c in (("k", outs[0], kd, tables.k_centroids), ("v", outs[1], vd, tables.v_centroids)):
        got = out.cpu().double().numpy()
        ac = np.abs(c.cpu().double().numpy())[f[f"{name}_idx"]] @ aR
        slack = (ac * f[f"{name}_norm"].astype(np.float64)[..., None]).reshape(-1, H, tokens, D)
        x = x.reshape(-1, H, tokens, D)
        for i in range(n):
            if r[i] < 0:
                assert (got[i] == 7.0).all()
                continue
            want = x[r[i], :, pos[i]]
            rel = 2.0 ** -16 + (2.0 ** -11 if dtype == BF16 else 0.0)
            tol = S.half_ulp(dtype) * np.abs(want) + rel * slack[r[i], :, pos[i]] + 2.0 ** -25
            assert (np.abs(got[i] - want) <= tol).all()
    only = torch.full((n, H, D), 7.0, dtype=dtype, device=DEV)
    ops.dequantize_ragged(tables, pages, batch, None, only)
    assert torch.equal(only, outs[1])


@pytest.mark.parametrize("D,kb,vb,H,dtype,xform", [
    (128, 4, 2, 2, BF16, "rope"), (128, 4, 4, 8, BF16, "norm+rope"), (128, 3, 3, 1, F16, "norm"),
    (128, 8, 1, 3, F32, "interleaved"), (64, 3, 3, 4, F16, "rope"), (64, 4, 2, 5, BF16, "none"),
    (64, 6, 5, 2, F32, "interleaved"), (96, 5, 7, 1, BF16, "norm+rope"),
    (32, 2, 2, 2, BF16, "rope"), (128, 2, 3, 5, BF16, "interleaved"), (128, 6, 6, 2, BF16, "none")])
@pytest.mark.parametrize("lens", sorted(LENS))
def test_append_ragged_and_read_back(D, kb, vb, H, dtype, xform, lens):
    tables = make_tables(D, kb, vb, False)
    lens = LENS[lens]
    R = len(lens)
    batch, start, seq = make_batch(lens, lead=2)
    n = start[-1] + 3                                     # rows before and behind the batch
    pages = make_paged(tables, R * H, max(seq))
    before = pages.pool.clone()
    k, v = randn((n, H, D), 1, dtype, 9), randn((n, H, D), 2, dtype, 11)
    rope = None if xform in ("none", "norm") else \
        ops.RopeTable.build(D if xform != "interleaved" else D // 2, 400,
                            interleaved=xform == "interleaved", device=DEV)
    norm = ops.HeadNorm(1 + 0.2 * randn((D,), 3, F32), 1e-6) if "norm" in xform else None
    ops.append_ragged(tables, pages, k, v, batch, rope=rope, k_norm=norm)
    assert ok_status() == 0
    r, pos = S.positions(start, seq, n)
    kx = S.rope(k, rope.cos_sin if rope else None, np.maximum(pos, 0), xform == "interleaved",
                norm.weight if norm else None, 1e-6)
    check_stored(tables, pages, k, v, start, seq, R, H, kx)
    # nothing but the new tokens changed: blank them and compare with the pool before
    geom_rows = {(int(pages.block_table[r[i] * H + h, pos[i] // 64]), int(pos[i] % 64))
                 for i in range(n) if r[i] >= 0 for h in range(H)}
    after = pages.pool.clone()
    kr, vr = D * kb // 8, D * vb // 8
    for pg, sl in geom_rows:
        for off, row in ((0, kr), (64 * kr, vr), (64 * (kr + vr), 2), (64 * (kr + vr) + 128, 2)):
            after[pg, off + sl * row: off + (sl + 1) * row] = 0
    assert torch.equal(after, before)
    for t in (dtype, BF16):
        check_read(tables, pages, batch, start, seq, n, H, t)
    assert ok_status() == 0


def test_append_ragged_equals_append_and_takes_strides():
    """Without a transform the codes are tq_append's; k and v may be slices of one projection;
    rotation positions may be given; contiguous pages work like paged ones."""
    D, H, R = 128, 2, 3
    tables = make_tables(D, 4, 2, False)
    lens = [(40, 40), (33, 33), (1, 1)]
    batch, start, seq = make_batch(lens)
    n = start[-1]
    fused = randn((n, 3 * H * D), 5)
    k, v = fused[:, H * D: 2 * H * D].view(n, H, D), fused[:, 2 * H * D:].view(n, H, D)
    pb = ops.page_bytes(D, 4, 2, False)
    pages = torch.zeros((R * H, 1, pb), dtype=torch.uint8, device=DEV)
    ops.append_ragged(tables, pages, k, v, batch)
    ref = torch.zeros_like(pages)
    for r, (m, _) in enumerate(lens):
        rows = slice(start[r], start[r + 1])
        ops.append(tables, ref[r * H: (r + 1) * H], k[rows].transpose(0, 1).unsqueeze(0),
                   v[rows].transpose(0, 1).unsqueeze(0), 0)
    a, b = S.parse(tables, pages, 64), S.parse(tables, ref, 64)
    for name in ("k_idx", "v_idx"):
        assert (a[name] != b[name]).mean() <= 1e-4
    for name in ("k_norm", "v_norm"):
        assert (a[name] != b[name]).mean() <= 1e-3
    # rotation positions other than the places in the request
    rope = ops.RopeTable.build(D, 5000, device=DEV)
    pos = torch.randint(0, 5000, (n,), generator=torch.Generator().manual_seed(1)).to(DEV)
    for p in (pos, pos.to(torch.int32), pos.repeat_interleave(2)[::2]):
        pages.zero_()
        ops.append_ragged(tables, pages, k, v, batch, rope=rope, positions=p)
        check_stored(tables, pages, k, v, start, seq, R, H,
                     S.rope(k, rope.cos_sin, pos.cpu().numpy()))
    assert ok_status() == 0


def test_append_ragged_bad_places():
    """Tokens beyond the pages or before the start are dropped and flagged, pages outside the pool
    neither written nor read; the others are stored; read-back zeroes what has no place."""
    D, H = 128, 2
    tables = make_tables(D, 4, 4, False)
    batch, start, seq = make_batch([(3, 66), (4, 2), (2, 2), (2, 2)])
    n = start[-1]
    pages = make_paged(tables, 4 * H, 64)                 # room for 64 tokens a request
    pages.block_table[2 * H] = -1
    pages.block_table[2 * H + 1] = pages.pool.shape[0]
    k, v = randn((n, H, D), 1), randn((n, H, D), 2)
    ops.append_ragged(tables, pages, k, v, batch)
    assert ok_status() == _lib.DEV_BAD_POSITION | _lib.DEV_BAD_BLOCK
    out = torch.full((n, H, D), 7.0, dtype=BF16, device=DEV)
    ops.dequantize_ragged(tables, pages, batch, out, None)
    assert ok_status() == _lib.DEV_BAD_POSITION | _lib.DEV_BAD_BLOCK
    stored = (out.float() * k.float()).sum((1, 2)) > 0.9 * k.float().square().sum((1, 2))
    # request 0: positions 63 (stored), 64, 65 (outside); request 1: -2, -1 (outside), 0, 1
    assert stored[:7].tolist() == [True, False, False, False, False, True, True]
    assert (out[[1, 2, 3, 4]] == 0).all() and (out[7:9] == 0).all()
    assert stored[9:].all()


def test_append_ragged_zero_and_extreme_rows():
    """A zero vector stores norm 0 and reads back as 0; norms of 1e-7 and 6e4 stay exact to fp16;
    NaN keeps to its own vector."""
    D, H = 128, 1
    tables = make_tables(D, 4, 4, False)
    batch, start, seq = make_batch([(5, 5)])
    k = randn((5, H, D), 1, F32)
    k /= k.norm(dim=-1, keepdim=True)
    k[0] = 0
    k[1] *= 1e-7
    k[2] *= 6e4
    k[3, 0, 7] = float("nan")
    pages = make_paged(tables, H, 64)
    ops.append_ragged(tables, pages, k, k, batch)
    out = torch.empty((5, H, D), dtype=F32, device=DEV)
    ops.dequantize_ragged(tables, pages, batch, out, None)
    assert (out[0] == 0).all()
    for i in (1, 2, 4):
        n = k[i].norm().item()
        assert abs(out[i].norm().item() / n - 1) < 0.1 if i != 1 else out[i].norm().item() < 2e-7
        assert cosine(out[i].cpu(), k[i].cpu()) > 0.98 or i == 1
    assert out[[0, 2, 4]].isfinite().all()
    assert ok_status() == 0


# ------------------------------------------------------------------------------- attend_ragged
def check_attend(out, want, dtype, rows=None):
    got = out.detach().cpu().double().numpy()
    inside = ~np.isnan(want).any((1, 2))
    g, w = got[inside], want[inside]
    assert np.isfinite(g).all()
    top = np.abs(w).max()
    assert (g[np.abs(w).max((1, 2)) == 0] == 0).all()
    assert cosine(g, w) >= 0.9999
    assert np.abs(g - w).max() <= 4e-3 * top + S.half_ulp(dtype) * top


ATTEND = {
    "tokens": ([(1, 1), (1, 64), (1, 65), (1, 513)], True),
    "drafts": ([(3, 5), (8, 700), (1, 129), (5, 64)], True),
    "chunks": ([(130, 130), (65, 400), (1, 90), (0, 33), (257, 257)], True),
    "empty rows": ([(6, 2), (3, 0), (2, 2), (0, 0)], True),
    "cross": ([(1, 300), (7, 1), (40, 129), (3, 0), (5, 64)], False),
    "split": ([(3, 5000)], True),
    "split cross": ([(2, 3000), (1, 10)], False),
}
GEOM = [(128, 4, 2, 8, 2), (128, 4, 4, 5, 1), (128, 3, 2, 20, 1), (64, 4, 3, 9, 3),
        (128, 3, 3, 6, 2), (128, 2, 2, 2, 2),
        (128, 6, 4, 8, 1), (128, 8, 8, 4, 2), (64, 4, 4, 4, 4), (64, 3, 3, 12, 4)]


@pytest.mark.parametrize("case", sorted(ATTEND))
@pytest.mark.parametrize("D,kb,vb,Hq,H", GEOM)
def test_attend_ragged_matches_plain_form(D, kb, vb, Hq, H, case):
    lens, causal = ATTEND[case]
    tables = make_tables(D, kb, vb, False)
    R = len(lens)
    batch, start, seq = make_batch(lens, lead=1)
    n = start[-1] + 2
    pages = make_paged(tables, R * H, max(max(seq), 1))
    fill(tables, pages, R, H, pages.shape[1] * 64, 3)
    kd, vd = (x.reshape(R, H, -1, D) for x in S.dense(tables, contiguous(pages), pages.shape[1] * 64))
    ws = ops.DecodeWorkspace()
    engines = [0, 1] + ([2] if D == 128 and kb < 8 else []) + ([3] if kb <= 4 else [])
    for dtype in (BF16, F32):
        q = randn((n, Hq, D), 4, dtype)
        want = S.attend(q, kd, vd, start, seq, S.default_scale(D), causal)
        for engine in engines if dtype == BF16 else [0]:
            out = torch.full_like(q, 7.0)
            got = ops.attend_ragged(tables, pages, q, batch, causal=causal, out=out, workspace=ws,
                                    engine=engine)
            assert got is out and ok_status() == 0
            outside = np.isnan(want).any((1, 2))
            assert (out[torch.from_numpy(outside).to(DEV)] == 7.0).all()
            check_attend(out, want, dtype)
            again = ops.attend_ragged(tables, pages, q, batch, causal=causal, engine=engine)
            inside = torch.from_numpy(~outside).to(DEV)
            assert torch.equal(again[inside], out[inside])       # joined in a fixed order
    assert ws.status() == 0


def test_attend_ragged_views_scale_and_max_q_len():
    """q a slice of one projection, out transposed memory, a scale; a larger max_q_len than needed
    changes nothing beyond rounding; contiguous pages."""
    D, Hq, H, R = 128, 4, 2, 3
    tables = make_tables(D, 4, 4, False)
    batch, start, seq = make_batch([(4, 200), (9, 9), (1, 64)])
    n = start[-1]
    pb = ops.page_bytes(D, 4, 4, False)
    pages = torch.zeros((R * H, 4, pb), dtype=torch.uint8, device=DEV)
    fill(tables, pages, R, H, 256, 8)
    kd, vd = (x.reshape(R, H, -1, D) for x in S.dense(tables, pages, 256))
    q = randn((n, (Hq + 2) * D + 1), 1, F16)[:, 1: 1 + Hq * D].view(n, Hq, D)
    want = S.attend(q, kd, vd, start, seq, 0.05, True)
    out = torch.empty((Hq, n, D), dtype=F16, device=DEV).transpose(0, 1)
    ops.attend_ragged(tables, pages, q, batch, scale=0.05, out=out)
    check_attend(out, want, F16)
    wide = ops.RaggedBatch(batch.q_start, batch.seq_lens, 5000)
    check_attend(ops.attend_ragged(tables, pages, q, wide, scale=0.05), want, F16)
    one = ops.RaggedBatch(batch.q_start, batch.seq_lens, 0)          # a wrong bound is only slower
    check_attend(ops.attend_ragged(tables, pages, q, one, scale=0.05), want, F16)
    assert ok_status() == 0


@pytest.mark.parametrize("engine", [1, 2, 3])
def test_attend_ragged_infinite_and_nan_norms(engine):
    """A key or value whose stored norm is inf or NaN makes NaN of the rows that see it and of no
    other: earlier rows of the chunk and other requests stay as they were."""
    D, Hq, H = 128, 2, 1
    tables = make_tables(D, 4, 4, False)
    batch, start, seq = make_batch([(70, 70), (5, 900)])
    n = start[-1]
    pages = make_paged(tables, 2 * H, 900)
    fill(tables, pages, 2, H, pages.shape[1] * 64, 1)
    q = randn((n, Hq, D), 2)
    clean = ops.attend_ragged(tables, pages, q, batch, engine=engine)
    kr = D * 4 // 8
    norms = 64 * 2 * kr
    for what in (0, 128):                                  # K norms, V norms
        for bad in (float("inf"), float("nan")):
            pool = pages.pool.clone()
            pg = int(pages.block_table[0, 0])
            at = norms + what + 2 * 40                     # token 40 of request 0
            pool[pg, at: at + 2] = torch.tensor([bad], dtype=F16).view(torch.uint8).to(DEV)
            # beyond the end of request 1 (page of tokens 896..959), nothing looks there
            pg1 = int(pages.block_table[1, 14])
            at1 = norms + what + 2 * 10
            pool[pg1, at1: at1 + 2] = torch.tensor([bad], dtype=F16).view(torch.uint8).to(DEV)
            out = ops.attend_ragged(tables, ops.PagedPages(pool, pages.block_table), q, batch,
                                    engine=engine)
            assert torch.equal(out[:40], clean[:40]) and torch.equal(out[70:], clean[70:])
            assert out[40:70].isnan().all()
    assert ok_status() == 0


def test_attend_ragged_bad_pages_and_batches():
    """Block-table entries outside the pool are flagged and never read; offsets that do not ascend
    run nothing and are flagged."""
    D, H = 128, 1
    tables = make_tables(D, 4, 2, False)
    batch, start, seq = make_batch([(2, 100), (2, 100)])
    pages = make_paged(tables, 2, 128)
    fill(tables, pages, 2, H, 128, 1)
    q = randn((4, 2, D), 2)
    clean = ops.attend_ragged(tables, pages, q, batch)
    pages.block_table[1, 0] = -1
    pages.block_table[1, 1] = pages.pool.shape[0]
    for engine in (1, 2, 3):
        out = ops.attend_ragged(tables, pages, q, batch, engine=engine)
        assert ok_status() == _lib.DEV_BAD_BLOCK
        assert (out[:2].float() - clean[:2].float()).abs().max() < 0.02 and out.isfinite().all()
    huge = ops.RaggedBatch(int32([0, 4] * 40 + [4]), int32([100] * 80), 4)
    many = make_paged(tables, 80, 128)
    ops.attend_ragged(tables, many, q, huge)
    assert ok_status() in (0, _lib.DEV_BAD_BATCH)
    wild = ops.RaggedBatch(int32([-5, 90, 1 << 30]), int32([1 << 30, -7]), 4)
    ops.attend_ragged(tables, pages, q, wild)
    ops.append_ragged(tables, pages, q[:, :1].contiguous(), q[:, :1].contiguous(), wild)
    torch.cuda.synchronize()
    ops.device_status(DEV)


# ---------------------------------------------------------------------------------- together
def test_serving_step_together_captured_and_on_another_stream():
    """rope -> append -> attend as a serving step runs them, eager, on a side stream and replayed
    from a graph after the inputs and lengths changed in place: the same bits each time."""
    D, Hq, H, R = 128, 8, 2, 4
    tables = make_tables(D, 4, 2, False)
    rope = ops.RopeTable.build(D, 1000, device=DEV)
    norms = [ops.HeadNorm(1 + 0.1 * randn((D,), i, F32)) for i in range(2)]
    lens = [[(1, 100), (4, 260), (1, 65), (2, 2)], [(2, 102), (1, 261), (3, 68), (2, 4)]]
    pages = make_paged(tables, R * H, 320)
    fill(tables, pages, R, H, 320, 1)
    pool0 = pages.pool.clone()
    ws = ops.DecodeWorkspace()
    n = 8
    data = [tuple(randn((n, h, D), 10 * i + j) for j, h in enumerate((Hq, H, H))) for i in range(2)]

    def step(q, k, v, batch, pos, w):
        qr, _ = ops.qk_rope(q, None, rope, pos, q_norm=norms[0])
        ops.append_ragged(tables, pages, k, v, batch, rope=rope, k_norm=norms[1])
        return ops.attend_ragged(tables, pages, qr, batch, workspace=w)

    def args(i):
        batch, start, seq = make_batch(lens[i])
        _, pos = S.positions(start, seq, n)
        return (*data[i], batch, int32(pos))

    eager = []
    for i in range(2):
        pages.pool.copy_(pool0)
        eager.append((step(*args(i), ws), pages.pool.clone()))
        start, seq = args(i)[3].q_start.tolist(), args(i)[3].seq_lens.tolist()
        kd, vd = (x.reshape(R, H, -1, D) for x in S.dense(tables, contiguous(pages), 320))
        qx = torch.from_numpy(S.rope(data[i][0], rope.cos_sin, args(i)[4].cpu().numpy(), False,
                                     norms[0].weight, 1e-6))
        want = S.attend(qx, kd, vd, start, seq, S.default_scale(D), True)
        want[start[-1]:] = np.nan
        check_attend(eager[i][0], want, BF16)
    side = torch.cuda.Stream()
    pages.pool.copy_(pool0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        out = step(*args(1), ops.DecodeWorkspace())
    side.synchronize()
    m = int(args(1)[3].q_start[-1])
    assert torch.equal(out[:m], eager[1][0][:m]) and torch.equal(pages.pool, eager[1][1])
    # one graph, replayed on both sets of inputs
    live = [x if isinstance(x, ops.RaggedBatch) else x.clone() for x in args(0)]
    graph_ws = ops.DecodeWorkspace()
    pages.pool.copy_(pool0)
    step(*live, graph_ws)                                  # workspace in place before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*live, graph_ws)
    for i in (0, 1, 0):
        pages.pool.copy_(pool0)
        for dst, src in zip(live, args(i)):
            if isinstance(dst, ops.RaggedBatch):
                dst.q_start.copy_(src.q_start)
                dst.seq_lens.copy_(src.seq_lens)
            else:
                dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        m = int(args(i)[3].q_start[-1])
        assert torch.equal(out[:m], eager[i][0][:m]) and torch.equal(pages.pool, eager[i][1])
    assert ok_status() == 0


def test_decode_and_ragged_forms_agree():
    """One new token a request: append_ragged + attend_ragged give what the fused decode step
    gives (same pages up to boundary codes, outputs within the fp16 operands' bar)."""
    D, Hq, H, R = 128, 8, 2, 3
    tables = make_tables(D, 4, 2, False)
    seq = [65, 200, 1]
    pages = make_paged(tables, R * H, 256)
    fill(tables, pages, R, H, 256, 1)
    pool0 = pages.pool.clone()
    q, k, v = randn((R, Hq, D), 1), randn((R, H, D), 2), randn((R, H, D), 3)
    want = ops.decode_step(tables, pages, k.unsqueeze(2), v.unsqueeze(2), 255, q.unsqueeze(2),
                           seq_lens=int32(seq))[:, :, 0]
    pool1 = pages.pool.clone()
    pages.pool.copy_(pool0)
    batch, _, _ = make_batch([(1, s) for s in seq])
    ops.append_ragged(tables, pages, k, v, batch)
    assert (pages.pool != pool1).float().mean() < 1e-4
    pages.pool.copy_(pool1)
    got = ops.attend_ragged(tables, pages, q, batch)
    assert cosine(got.float().cpu(), want.float().cpu()) >= 0.9999
    assert (got.float() - want.float()).abs().max() <= 8e-3 * want.float().abs().max() + 2.0 ** -8
    assert ok_status() == 0


def test_no_rows():
    """A batch without rows (and requests without new tokens) runs every operator and writes nothing."""
    D, H = 128, 2
    tables = make_tables(D, 4, 2, False)
    pages = make_paged(tables, 2 * H, 64)
    batch, _, _ = make_batch([(0, 0), (0, 30)])
    x = torch.empty((0, H, D), dtype=BF16, device=DEV)
    rope = ops.RopeTable.build(D, 10, device=DEV)
    ops.append_ragged(tables, pages, x, x, batch, rope=rope)
    ops.dequantize_ragged(tables, pages, batch, x, x)
    assert ops.attend_ragged(tables, pages, x, batch).shape == (0, H, D)
    y = torch.full((3, H, D), 7.0, dtype=BF16, device=DEV)          # rows of no request
    ops.append_ragged(tables, pages, y, y, batch)
    ops.dequantize_ragged(tables, pages, batch, y, None)
    ops.attend_ragged(tables, pages, y.clone(), batch, out=y)
    assert (y == 7).all() and (pages.pool == 0).all() and ok_status() == 0


# ------------------------------------------------------------------- through the public classes
def test_paged_attention_layer_with_rope_matches_rotated_heads():
    """TurboQuantPagedAttention.forward(rope=...) over a served schedule (prompts, mixed and
    decode-only steps, padding rows behind the batch) against the 64-bit form on what it stored; the
    pages against append of the rotated keys; read() gives the pages' tokens."""
    from bhaskera_col_b200.inference.vllm_turboquant import TurboQuantPagedAttention, VLLMBatch
    D, Hq, H = 128, 8, 2
    layer = TurboQuantPagedAttention(5, 32, Hq, H, D, num_blocks=40, block_size=64, key_bits=4,
                                     value_bits=2, device=DEV)
    rope = ops.RopeTable.build(D, 1000, interleaved=True, device=DEV)
    qn, kn = (ops.HeadNorm(1 + 0.1 * randn((D,), i, F32)) for i in range(2))
    free = torch.randperm(40, generator=torch.Generator().manual_seed(3)).tolist()
    blocks, length, stored = {}, {}, {}
    steps = [[("A", 130), ("B", 64), ("C", 1)], [("A", 1), ("B", 3), ("C", 70)],
             [("C", 1), ("A", 1), ("B", 1)], [("B", 129), ("A", 1)]]
    for i, work in enumerate(steps):
        start, seq = [0], []
        for r, n in work:
            blocks.setdefault(r, [])
            length[r] = length.get(r, 0) + n
            while len(blocks[r]) * 64 < length[r]:
                blocks[r].append(free.pop())
            start.append(start[-1] + n)
            seq.append(length[r])
        N = start[-1]
        bt = torch.zeros((len(work), max(len(blocks[r]) for r, _ in work) + 1), dtype=torch.int32)
        for j, (r, _) in enumerate(work):
            bt[j, : len(blocks[r])] = torch.tensor(blocks[r], dtype=torch.int32)
        batch = VLLMBatch(int32(start), int32(seq), bt.to(DEV), N, max(n for _, n in work))
        q, k, v = (randn((N + 2, h, D), 10 * i + j, BF16, 7) for j, h in enumerate((Hq, H, H)))
        out = torch.full_like(q, 7.0)
        got = layer.forward(q, k, v, batch, out=out, rope=rope, q_norm=qn, k_norm=kn)
        assert got is out and (out[N:] == 7.0).all() and ok_status() == 0
        assert batch.query_start_loc_cpu is None and batch.seq_lens_cpu is None     # no host copies
        req, pos = S.positions(start, seq, N)
        assert batch.positions().tolist() == pos.tolist()
        pages = layer.paged(layer.stream_table(batch.block_table))
        kx = S.rope(k[:N], rope.cos_sin, pos, True, kn.weight, 1e-6)
        check_stored(layer.tables, pages, k[:N], v[:N], start, seq, len(work), H, kx)
        tokens = pages.shape[1] * 64
        kd, vd = (x.reshape(len(work), H, -1, D) for x in S.dense(layer.tables, contiguous(pages), tokens))
        qx = torch.from_numpy(S.rope(q[:N], rope.cos_sin, pos, True, qn.weight, 1e-6))
        check_attend(out[:N], S.attend(qx, kd, vd, start, seq, layer.scale, True), BF16)
        rk, rv = layer.read(batch)
        for t, x in ((rk, kd), (rv, vd)):
            want = x[req, :, pos]
            assert np.abs(t.double().cpu().numpy() - want).max() <= 2.0 ** -7 * np.abs(want).max()
    assert layer.tokens_stored == sum(n for w in steps for _, n in w)
    with pytest.raises(ValueError, match="rope"):
        layer.forward(q, k, v, batch, positions=batch.positions())


def test_cache_with_rope_matches_rotated_heads():
    """TurboQuantKVCache.prefill / decode(rope=...) store and attend exactly what they do for heads
    rotated by qk_rope beforehand, at the cache's own positions or given ones."""
    from bhaskera_col_b200.inference import TurboQuantKVCache
    B, Hq, H, D, T = 2, 4, 2, 128, 37
    rope = ops.RopeTable.build(D, 500, device=DEV)
    qn, kn = (ops.HeadNorm(1 + 0.1 * randn((D,), i, F32)) for i in range(2))

    def cache():
        return TurboQuantKVCache(1, B, H, D, residual_window=0, protected_layers=0, device=DEV,
                                 max_seq_len=128)

    a, b = cache(), cache()
    pads = torch.tensor([[5], [0]], device=DEV)
    for i, n in enumerate((T, 1, 1)):
        q, k, v = (randn((B, h, n, D), 5 * i + j) for j, h in enumerate((Hq, H, H)))
        at = torch.arange(n, device=DEV) + (0 if i == 0 else T + i - 1)
        given = (at[None] - pads).clamp_min(0) if i == 2 else None
        call = (a.prefill, b.prefill) if n > 1 else (a.decode, b.decode)
        qr, kr = ops.qk_rope(q, k, rope, at if given is None else given, qn, kn)
        want = call[1](qr, kr, v, 0)
        got = call[0](q, k, v, 0, rope=rope, positions=given, q_norm=qn, k_norm=kn)
        assert torch.equal(got, want)
    assert torch.equal(a._stores[0]._pages, b._stores[0]._pages) and ok_status() == 0
    # only one norm: the other heads pass through
    q, k, v = (randn((B, h, 1, D), 50 + j) for j, h in enumerate((Hq, H, H)))
    kr = ops.qk_rope(None, k, None, k_norm=kn)[1]
    assert torch.equal(a.decode(q, k, v, 0, k_norm=kn), b.decode(q, kr, v, 0))


def test_inputs_of_a_backward_pass_and_mixed_devices_are_refused():
    x = randn((3, 2, 128), 1, F32).requires_grad_()
    table = ops.RopeTable.build(128, 10, device=DEV)
    pos = torch.arange(3, device=DEV)
    with pytest.raises(RuntimeError, match="no backward pass"):
        ops.qk_rope(x, None, table, pos)
    with torch.no_grad():
        ops.qk_rope(x, None, table, pos)
    ops.qk_rope(x.detach(), None, table, pos)
    with pytest.raises(ValueError, match="tensors on"):
        ops.qk_rope(x.detach(), None, table, pos.cpu())
    with pytest.raises(ValueError, match="positions"):
        ops.qk_rope(x.detach(), None, table, pos[:2])
    with pytest.raises(ValueError, match="weights"):
        ops.qk_rope(x.detach(), None, None, q_norm=ops.HeadNorm(torch.ones(64, device=DEV)))
    batch, _, _ = make_batch([(3, 3)])
    tables = make_tables(128, 4, 2, False)
    pages = make_paged(tables, 2, 64)
    for call in (lambda: ops.append_ragged(tables, pages, x, x, batch),
                 lambda: ops.attend_ragged(tables, pages, x, batch)):
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
    with pytest.raises(_lib.TqError, match="overlaps"):
        buf = randn((4, 2, 128), 2)
        ops.qk_rope(buf[:3], None, table, pos, q_out=buf[1:])


@pytest.mark.parametrize("D,kb,vb,dtype,pairs,norm", [
    (64, 3, 3, F16, "interleaved", False), (64, 4, 2, F32, "half", True),
    (128, 4, 4, BF16, "half", True), (128, 5, 1, F16, "part", True), (128, 6, 4, BF16, "none", False)])
def test_append_ragged_codes_are_those_of_exact_arithmetic(D, kb, vb, dtype, pairs, norm):
    """A million coordinates: about one of 32-bit arithmetic's codes in a million is off by one;
    none is here.  Coordinates within 64-bit rounding (1e-12) of a boundary may go either way."""
    tables = make_tables(D, kb, vb, False)
    H, n = 4, (1 << 20) // (4 * D) - 5
    batch, start, seq = make_batch([(n - 700, n - 700), (700, 900)])
    pages = make_paged(tables, 2 * H, max(seq))
    k, v = randn((n, H, D), 21, dtype), randn((n, H, D), 22, dtype, 7)
    rope = None if pairs == "none" else \
        ops.RopeTable.build(D // 2 if pairs == "part" else D, n,
                            interleaved=pairs == "interleaved", device=DEV)
    w = ops.HeadNorm(0.2 * randn((D,), 23, F32), 1e-6, 1.0) if norm else None
    ops.append_ragged(tables, pages, k, v, batch, rope=rope, k_norm=w)
    got = S.parse(tables, contiguous(pages), max(seq))
    r, pos = S.positions(start, seq, n)
    kx = S.rope(k, rope.cos_sin if rope else None, pos, pairs == "interleaved",
                w.weight if w else None, 1e-6, 1.0)
    R = tables.rot.double().cpu().numpy()
    for name, x, bnd in (("k_idx", kx, tables.k_boundaries), ("v_idx", v, tables.v_boundaries)):
        x = np.asarray(x.double().cpu().numpy() if torch.is_tensor(x) else x, dtype=np.float64)
        y = (x / np.linalg.norm(x, axis=-1, keepdims=True)) @ R.T
        b = bnd.double().cpu().numpy()[: (1 << (kb if name[0] == "k" else vb)) - 1]
        at = np.searchsorted(b, y, side="left")
        gap = np.abs(y[..., None] - b[np.clip(np.stack([at - 1, at], -1), 0, len(b) - 1)]).min(-1)
        have = got[name].reshape(2, H, -1, D)[r, :, pos]
        assert not ((have != at) & (gap > 1e-12)).any()
    assert ok_status() == 0


@pytest.mark.parametrize("engine", [0, 1, 3])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,kb,vb,Hq,H", [(128, 4, 2, 8, 2), (128, 3, 3, 20, 1), (64, 2, 2, 4, 4),
                                          (64, 3, 4, 6, 2), (64, 6, 6, 4, 2), (128, 2, 4, 6, 2)])
def test_attend_ragged_fp16_and_fp32_results_are_exact_to_their_type(D, kb, vb, Hq, H, dtype, engine):
    """Operands of 22 bits: a score is off by at most 2^-20 |scale q k| (three products of two
    values that are each off by 2^-22, and the sums), so is its exponential, relatively; P and V add
    3 x 2^-22 and the sums of fp32 less than 2^-18."""
    codes = (kb, vb)
    if engine == 3 and max(codes) > 4 or engine == 1 and codes in ((3, 4), (2, 4)):
        pytest.skip("no such kernel")
    tables = make_tables(D, kb, vb, False)
    lens = [(3, 700), (200, 300), (1, 1), (2, 0), (40, 1500)]
    batch, start, seq = make_batch(lens)
    pages = make_paged(tables, len(lens) * H, 1500)
    fill(tables, pages, len(lens), H, pages.shape[1] * 64, 31)
    kd, vd = (x.reshape(len(lens), H, -1, D) for x in S.dense(tables, contiguous(pages), pages.shape[1] * 64))
    q = randn((start[-1], Hq, D), 32, dtype)
    want = S.attend(q, kd, vd, start, seq, D ** -0.5, True)
    got = ops.attend_ragged(tables, pages, q, batch, engine=engine).double().cpu().numpy()
    most = D ** -0.5 * np.linalg.norm(q.double().cpu().numpy(), axis=-1).max() * \
        np.linalg.norm(kd, axis=-1).max()
    top = np.abs(vd).max()
    tol = (2 * most * 2.0 ** -20 + 2.0 ** -18) * top
    assert (np.abs(got - want) <= tol + S.half_ulp(dtype) * np.abs(want) + 2.0 ** -25).all()
    out = q.clone()                                       # in place
    ops.attend_ragged(tables, pages, out, batch, out=out, engine=engine)
    assert np.array_equal(out.double().cpu().numpy(), got)
    assert ok_status() == 0


@pytest.mark.parametrize("engine", [1, 2, 3])
def test_attend_ragged_in_place(engine):
    """out may be q: every CTA of a cut tile has read its queries before the last one writes."""
    tables = make_tables(128, 4, 2, False)
    lens = [(5, 4000), (150, 3000), (1, 64)]
    batch, start, seq = make_batch(lens)
    pages = make_paged(tables, len(lens) * 2, 4000)
    fill(tables, pages, len(lens), 2, pages.shape[1] * 64, 33)
    q = randn((start[-1], 8, 128), 34, BF16)
    want = ops.attend_ragged(tables, pages, q, batch, engine=engine)
    for _ in range(5):
        out = q.clone()
        ops.attend_ragged(tables, pages, out, batch, out=out, engine=engine)
        assert torch.equal(out, want)
    assert ok_status() == 0


def test_paged_attention_layer_with_rope_replays_with_new_lengths():
    """A captured forward of a batch that an eager one has used takes its positions from the
    lengths at replay."""
    from bhaskera_col_b200.inference.vllm_turboquant import TurboQuantPagedAttention, VLLMBatch
    D, Hq, H, R = 128, 4, 2, 3
    rope = ops.RopeTable.build(D, 300, device=DEV)
    q, k, v = (randn((R, h, D), 41 + j, BF16) for j, h in enumerate((Hq, H, H)))
    table = torch.arange(2 * R, dtype=torch.int32, device=DEV).view(R, 2)
    outs = []
    for graph in (False, True):
        layer = TurboQuantPagedAttention(5, 32, Hq, H, D, num_blocks=2 * R, block_size=64,
                                         key_bits=4, value_bits=2, device=DEV)
        batch = VLLMBatch(int32([0, 1, 2, 3]), int32([10, 64, 1]), table, R, 1)
        out = torch.empty_like(q)
        layer.forward(q, k, v, batch, out=out, rope=rope)
        first = out.clone()
        if graph:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                layer.forward(q, k, v, batch, out=out, rope=rope)
        batch.seq_lens.add_(1)
        if graph:
            g.replay()
        else:
            layer.forward(q, k, v, batch, out=out, rope=rope)
        outs.append((first, out.clone(), layer.pool.clone()))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert ok_status() == 0


def test_captured_layer_replays_after_its_workspace_grew():
    """A decode step is captured, a larger eager prompt follows (the workspace grows), other tensors
    take whatever memory was given back, and the graph is replayed: they stay as they were and the
    replay gives what an eager step gives."""
    from bhaskera_col_b200.inference.vllm_turboquant import TurboQuantPagedAttention, VLLMBatch
    D, Hq, H, R, T = 128, 8, 2, 4, 700
    rope = ops.RopeTable.build(D, 2000, device=DEV)
    layer = TurboQuantPagedAttention(5, 32, Hq, H, D, num_blocks=24 * R, block_size=64, key_bits=4,
                                     value_bits=2, device=DEV)
    table = torch.arange(24 * R, dtype=torch.int32, device=DEV).view(R, 24)
    heads = lambda n, s: [randn((n, h, D), s + j) for j, h in enumerate((Hq, H, H))]  # noqa: E731
    decode = VLLMBatch(int32(range(R + 1)), int32([10, 64, 1, 33]), table, R, 1)
    step = heads(R, 51)
    out = torch.empty_like(step[0])
    layer.forward(*step, decode, out=out, rope=rope)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(*step, decode, out=out, rope=rope)
    held = layer.ragged_workspace.buf
    prompts = VLLMBatch(int32([T * i for i in range(R + 1)]), int32([T] * R), table, T * R, T)
    layer.forward(*heads(T * R, 61), prompts, rope=rope)
    assert layer.ragged_workspace.buf.numel() > held.numel()
    at, size = held.data_ptr(), held.numel()
    del held
    fill = [torch.full((size,), 7, dtype=torch.uint8, device=DEV) for _ in range(4)]
    assert all(x.data_ptr() + size <= at or at + size <= x.data_ptr() for x in fill)
    decode.seq_lens.copy_(int32([T + 1] * R))
    pool = layer.pool.clone()
    graph.replay()
    torch.cuda.synchronize()
    assert all((x == 7).all() for x in fill)
    got, stored = out.clone(), layer.pool.clone()
    layer.pool.copy_(pool)
    layer.forward(*step, decode, out=out, rope=rope)
    assert torch.equal(out, got) and torch.equal(layer.pool, stored) and ok_status() == 0


@pytest.mark.parametrize("rope", ["half", "interleaved", "none"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,hq,hkv,D", [(3, 8, 2, 128), (7, 5, 1, 64), (1, 4, 4, 128), (5, 2, 3, 256),
                                        (9, 1, 1, 32), (2, 9, 5, 80)])
def test_qk_rope_norm_of_one_side(n, hq, hkv, D, dtype, rope):
    """Only the queries or only the keys are normed, in one call for both: heads of either side lie
    beside each other in a warp."""
    table = None if rope == "none" else ops.RopeTable.build(D, 50, interleaved=rope == "interleaved",
                                                            device=DEV)
    pos = torch.arange(n) * 5
    q, k = randn((n, hq, D), 1, dtype, 3), randn((n, hkv, D), 2, dtype)
    norm = ops.HeadNorm(1 + 0.2 * randn((D,), 7, F32), 1e-6)
    for norms in ((norm, None), (None, norm)):
        if table is None:
            with pytest.raises(_lib.TqError, match="neither a rotation nor a norm"):
                ops.qk_rope(q, k, None, None, *norms)
            continue
        qo, ko = ops.qk_rope(q, k, table, pos.to(DEV), *norms)
        check_rope(qo, q, table, pos.numpy(), norms[0])
        check_rope(ko, k, table, pos.numpy(), norms[1])
    assert ok_status() == 0


@pytest.mark.parametrize("engine", [0, 1, 2, 3])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_ragged_runs_what_it_accepts(D, engine):
    """Every pair of code widths and every result type: the call is refused before anything runs, or
    gives the right result; few and many rows.  A refusal leaves nothing behind for the next call."""
    H, Hq = 1, 4
    batch, start, seq = make_batch([(2, 40), (70, 100)])
    ran = set()
    for kb in range(1, 9):
        for vb in range(1, 9):
            tables = make_tables(D, kb, vb, False)
            pages = make_paged(tables, 2 * H, 100)
            fill(tables, pages, 2, H, 128, 3)
            kd, vd = (x.reshape(2, H, -1, D) for x in S.dense(tables, contiguous(pages), 128))
            for dtype in (BF16, F16, F32):
                q = randn((start[-1], Hq, D), 4, dtype)
                try:
                    got = ops.attend_ragged(tables, pages, q, batch, engine=engine)
                except _lib.TqError as e:
                    assert "no kernel for" in str(e) and "workspace_bytes" in str(e)
                    continue
                ran.add((kb, vb, dtype))
                check_attend(got, S.attend(q, kd, vd, start, seq, S.default_scale(D), True), dtype)
    assert ok_status() == 0
    pairs = {t: {(k, v) for k, v, u in ran if u == t} for t in (BF16, F16, F32)}
    assert pairs[F16] == pairs[F32]
    if engine == 0:      # what bf16 models run, fp16 ones do too: protected layers' widths among them
        assert pairs[BF16] == pairs[F32] and {(6, 4), (6, 6), (5, 5), (4, 4)} <= pairs[F32]
        assert D == 64 or (5, 4) in pairs[F32]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("engine,dtype", [(0, BF16), (1, BF16), (2, BF16), (3, BF16), (0, F32), (1, F32)])
def test_attend_ragged_requests_longer_than_their_pages(engine, dtype, causal):
    """Rows keep the positions that the lengths give them; they see the tokens that the pages hold."""
    D, Hq, H = 128, 8, 2
    tables = make_tables(D, 4, 2, False)
    lens = [(40, 150), (3, 129), (2, 128), (5, 400), (150, 150), (1, (1 << 31) - 1)]
    batch, start, seq = make_batch(lens)
    pages = make_paged(tables, len(lens) * H, 128)
    fill(tables, pages, len(lens), H, 128, 3)
    kd, vd = (x.reshape(len(lens), H, -1, D) for x in S.dense(tables, contiguous(pages), 128))
    q = randn((start[-1], Hq, D), 4, dtype)
    got = ops.attend_ragged(tables, pages, q, batch, causal=causal, engine=engine)
    assert ok_status() == _lib.DEV_BAD_POSITION
    check_attend(got, S.attend(q, kd, vd, start, seq, S.default_scale(D), causal), dtype)
    fits, _, _ = make_batch([(2, 128), (3, 60), (0, 1 << 20)])       # a request without rows is not run
    ops.attend_ragged(tables, ops.PagedPages(pages.pool, pages.block_table[: 3 * H]), q[:5], fits,
                      causal=causal, engine=engine)
    assert ok_status() == 0


def value_norms(tables, pool):
    """The fp16 value norms in a pool's pages (a view)."""
    at = pool.shape[1] - 128
    return pool[:, at:].view(F16)


SMALL = [(3, 700), (130, 300), (1, 1), (40, 1500), (2, 5000)]


@pytest.mark.parametrize("engine,dtype", [(3, BF16), (3, F32), (0, F32), (1, BF16), (1, F32), (2, BF16),
                                          (2, F32), (0, BF16)])
@pytest.mark.parametrize("D,kb,vb,Hq,H", [(128, 4, 2, 8, 2), (128, 3, 3, 20, 1), (64, 2, 4, 3, 3),
                                          (64, 6, 6, 4, 2)])
def test_attend_ragged_scales_with_the_value_norms(D, kb, vb, Hq, H, engine, dtype):
    """Value norms times a power of two (all of them normal halves before and after) give the result
    times that power, to the bit: no product ends at fp16's smallest values."""
    if engine == 3 and kb > 4 or engine == 1 and (kb, vb) == (2, 4) or engine == 2 and D != 128:
        pytest.skip("no such kernel")
    tables = make_tables(D, kb, vb, False)
    batch, start, _ = make_batch(SMALL)
    pages = make_paged(tables, len(SMALL) * H, 5000)
    fill(tables, pages, len(SMALL), H, pages.shape[1] * 64, 71)
    q = randn((start[-1], Hq, D), 72, dtype)
    want = ops.attend_ragged(tables, pages, q, batch, engine=engine)
    norms = value_norms(tables, pages.pool)
    kept = norms.clone()
    assert kept[kept > 0].min() >= 4 and kept.max() < 2 ** 7
    for e in (-16, -9, 5, 9):
        norms.copy_(kept * 2.0 ** e)
        got = ops.attend_ragged(tables, pages, q, batch, engine=engine)
        assert torch.equal(got, want * 2.0 ** e), e
    assert ok_status() == 0


@pytest.mark.parametrize("engine", [0, 1, 3])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,kb,vb,Hq,H", [(128, 4, 2, 8, 2), (128, 3, 3, 20, 1), (64, 2, 4, 3, 3),
                                          (128, 6, 6, 4, 2), (64, 5, 5, 4, 2)])
def test_attend_ragged_results_of_small_and_mixed_value_norms(D, kb, vb, Hq, H, dtype, engine):
    """fp16 and fp32 results with the bounds of 22-bit operands (2 most 2^-20 + 2^-18, see above)
    taken of the very terms of each sum, W_i = sum_j |R_ji| sum_t p_t n_t |c_tj|, where the norms of
    all or some tokens are far below 1 or above it."""
    if engine == 3 and kb > 4 or engine == 1 and (kb, vb) == (2, 4):
        pytest.skip("no such kernel")
    tables = make_tables(D, kb, vb, False)
    batch, start, seq = make_batch(SMALL[:4])
    R = len(seq)
    pages = make_paged(tables, R * H, 1500)
    fill(tables, pages, R, H, pages.shape[1] * 64, 73)
    tokens = pages.shape[1] * 64
    q = randn((start[-1], Hq, D), 74, dtype)
    norms = value_norms(tables, pages.pool)
    kept = norms.clone()
    aR = np.abs(tables.rot.cpu().double().numpy())
    for name, e in (("small", [-13]), ("large", [8]), ("mixed", [-9, 3, -15, -4, -9]), ("zeros", [-30, -10])):
        e = torch.tensor(e, device=DEV).repeat(64)[:64]
        norms.copy_(kept * 2.0 ** e)
        kd, vd = (x.reshape(R, H, -1, D) for x in S.dense(tables, contiguous(pages), tokens))
        f = S.parse(tables, contiguous(pages), tokens)
        w = np.abs(tables.v_centroids.cpu().double().numpy())[f["v_idx"]] * f["v_norm"].astype(np.float64)[..., None]
        want = S.attend(q, kd, vd, start, seq, D ** -0.5, True)
        terms = S.attend(q, kd, w.reshape(R, H, -1, D), start, seq, D ** -0.5, True) @ aR
        got = ops.attend_ragged(tables, pages, q, batch, engine=engine).double().cpu().numpy()
        most = D ** -0.5 * np.linalg.norm(q.double().cpu().numpy(), axis=-1).max() * \
            np.linalg.norm(kd, axis=-1).max()
        tol = (2 * most * 2.0 ** -20 + 2.0 ** -18) * terms + S.half_ulp(dtype) * np.abs(want)
        if dtype == F16:
            tol = tol + 2.0 ** -25
        assert (np.abs(got - want) <= tol).all(), (name, (np.abs(got - want) / tol).max())
    assert ok_status() == 0


@pytest.mark.parametrize("start", [
    [0, 4, 2, 6], [0, 5, 5, 4], [-1, 2, 3, 6], [0, 2, 3, 9], [3, 2, 1, 0], [-5, 90, 1 << 30, -(1 << 31)],
    [0, 1] * 300 + [6], [0, 4] * 750 + [6], list(range(0, 7)) + [6] * 1200 + [7]])
@pytest.mark.parametrize("D,kb,vb", [(128, 4, 2), (96, 4, 4)])
def test_offsets_that_do_not_ascend_run_nothing(D, kb, vb, start):
    """Descending, negative and too large offsets, in batches of few and of many requests: flagged by
    every operator, and nothing is stored or written."""
    R, H, n = len(start) - 1, 1, 6
    tables = make_tables(D, kb, vb, False)
    batch = ops.RaggedBatch(int32(start), int32([64] * R), 4)
    pages = make_paged(tables, R * H, 64)
    fill(tables, pages, R, H, 64, 1)
    kept = pages.pool.clone()
    x = randn((n, H, D), 2)
    ops.append_ragged(tables, pages, x, x, batch)
    assert ok_status() == _lib.DEV_BAD_BATCH and torch.equal(pages.pool, kept)
    out = [torch.full((n, H, D), 7.0, dtype=BF16, device=DEV) for _ in range(2)]
    ops.dequantize_ragged(tables, pages, batch, *out)
    assert ok_status() == _lib.DEV_BAD_BATCH and all((o == 7).all() for o in out)
    if D != 96:
        for engine in (0, 1, 2, 3):
            ops.attend_ragged(tables, pages, x, batch, out=out[0], engine=engine)
            assert ok_status() == _lib.DEV_BAD_BATCH and (out[0] == 7).all()
    good = ops.RaggedBatch(int32([0] * R + [n]), int32([64] * R), n)
    ops.append_ragged(tables, pages, x, x, good)
    assert ok_status() == 0 and not torch.equal(pages.pool, kept)


def test_layers_share_a_workspace():
    """Layers of one stream with one workspace between them give what layers with their own do, eager
    and in one captured graph of both."""
    from bhaskera_col_b200.inference.vllm_turboquant import TurboQuantPagedAttention, VLLMBatch
    D, Hq, H, R = 128, 8, 2, 3
    rope = ops.RopeTable.build(D, 300, device=DEV)
    table = torch.arange(4 * R, dtype=torch.int32, device=DEV).view(R, 4)
    shared = ops.DecodeWorkspace()

    def layers(**kw):
        return [TurboQuantPagedAttention(i, 32, Hq, H, D, num_blocks=4 * R, block_size=64, key_bits=4,
                                         value_bits=2, device=DEV, **kw) for i in (1, 7)]

    steps = [([0, 70, 200, 201], [70, 130, 1]), ([0, 1, 2, 3], [71, 131, 2])]
    results = []
    for ls, graph in ((layers(), False), (layers(ragged_workspace=shared), False),
                      (layers(ragged_workspace=shared), True)):
        for j, (start, seq) in enumerate(steps):
            n = start[-1]
            batch = VLLMBatch(int32(start), int32(seq), table, n, max(b - a for a, b in zip(start, start[1:])))
            q, k, v = (randn((n, h, D), 80 + 3 * j + i) for i, h in enumerate((Hq, H, H)))
            outs = [torch.empty_like(q) for _ in ls]
            step = lambda: [l.forward(x, k, v, batch, out=o, rope=rope)  # noqa: E731
                            for l, x, o in zip(ls, (q, outs[0]), outs)]
            step()
            if graph:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    step()
                g.replay()
            results.append([o.clone() for o in outs] + [l.pool.clone() for l in ls])
    for a, b, c in zip(results[:2], results[2:4], results[4:]):
        assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))
    assert shared.buf is not None and ok_status() == 0


@pytest.mark.parametrize("engine,dtype", [(0, BF16), (0, F32), (1, BF16), (1, F32), (2, BF16), (3, BF16), (3, F32)])
def test_attend_ragged_norms_of_either_sign(engine, dtype):
    """Norms are stored as they are given: a page written by hand may hold negative ones and -0."""
    D, Hq, H = 128, 8, 2
    tables = make_tables(D, 4, 4, False)
    lens = [(3, 300), (70, 130), (1, 1)]
    batch, start, seq = make_batch(lens)
    pages = make_paged(tables, len(lens) * H, 320)
    fill(tables, pages, len(lens), H, 320, 91)
    q = randn((start[-1], Hq, D), 92, dtype)
    for first in (0, 128):                                 # value norms, both
        norms = pages.pool[:, pages.pool.shape[1] - 128 - first:].view(F16)
        norms *= torch.tensor([-1, 1, -1, -0.0, -1], device=DEV).repeat(norms.shape[1])[: norms.shape[1]]
        kd, vd = (x.reshape(len(lens), H, -1, D) for x in S.dense(tables, contiguous(pages), 320))
        got = ops.attend_ragged(tables, pages, q, batch, engine=engine)
        check_attend(got, S.attend(q, kd, vd, start, seq, S.default_scale(D), True), dtype)
    pages.pool[:, pages.pool.shape[1] - 128:].view(F16).abs_().neg_()      # nothing but negative ones
    kd, vd = (x.reshape(len(lens), H, -1, D) for x in S.dense(tables, contiguous(pages), 320))
    got = ops.attend_ragged(tables, pages, q, batch, engine=engine)
    check_attend(got, S.attend(q, kd, vd, start, seq, S.default_scale(D), True), dtype)
    assert ok_status() == 0


def test_paged_attention_read_of_a_padded_batch_is_zero_there():
    """Rows of a padded batch that belong to no request come back as 0."""
    from bhaskera_col_b200.inference.vllm_turboquant import TurboQuantPagedAttention, VLLMBatch
    D, H = 128, 2
    layer = TurboQuantPagedAttention(5, 32, 4, H, D, num_blocks=4, block_size=64, device=DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
    batch = VLLMBatch(int32([1, 3, 4]), int32([2, 1]), table, 7, 2)
    q, k, v = (randn((7, h, D), 5 + j) for j, h in enumerate((4, H, H)))
    layer.forward(q, k, v, batch, rope=ops.RopeTable.build(D, 10, device=DEV))
    junk = [torch.full((7, H, D), 9.0, dtype=BF16, device=DEV) for _ in range(8)]
    del junk                                               # memory that an allocation may get
    rk, rv = layer.read(batch)
    for x in (rk, rv):
        assert (x[[0, 4, 5, 6]] == 0).all() and (x[1:4].abs().sum((1, 2)) > 0).all()
    assert ok_status() == 0


@pytest.mark.parametrize("engine", [1, 2])
def test_attend_ragged_large_norms_far_into_long_segments(engine):
    """Segments of more than 256 pages with a few pages of far larger value norms anywhere in them: as
    the few-row kernel's 22-bit operands have it, within the bar of fp16 operands."""
    D, Hq, H, T = 128, 8, 1, 1 << 17
    tables = make_tables(D, 4, 2, False)
    batch, start, _ = make_batch([(1500, T)])
    pages = make_paged(tables, H, T)
    fill(tables, pages, 1, H, T, 95)
    norms = value_norms(tables, pages.pool)
    norms *= 2.0 ** -9
    far = torch.randperm(T // 64, generator=torch.Generator().manual_seed(4))[:12].to(DEV)
    norms[pages.block_table[0, far].long()] *= 2.0 ** 12
    q = 3 * randn((start[-1], Hq, D), 96, F32)
    want = ops.attend_ragged(tables, pages, q, batch, engine=3).double().cpu().numpy()
    got = ops.attend_ragged(tables, pages, q, batch, engine=engine)
    check_attend(got, want, F32)
    assert ok_status() == 0
