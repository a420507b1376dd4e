"""Differential attention off the packed pages (diff_attend_ragged) against its plain form in 64 bits.

Tolerances.  A weight p of a map is off, relatively, by twice its score's error (its own and the sum's);
scores: q' and the decoded key, fp16 operands of bf16 results, are off by 2^-11 each and the key by its
norm's product once more, so 3 x 2^-11 of at most `most` = scale max|q| max|k|; the exponential's argument
in fp16 makes 2^-7 at worst, P, V, its norm's product and the sums 2^-9.  Operands of 22 bits (fp16 and fp32
results): 2^-20 `most` and 2^-18, as for attend_ragged.  Of both maps' sum of p |v| (mag), through the norm
(gain); then half an ulp of the result's type.  bf16 results also keep a cosine of 0.9999."""
import numpy as np
import pytest
import torch

import layer_oracle as L
import serving_oracle as S
from bhaskera_col_b200 import _lib
from bhaskera_col_b200.inference import ops
from test_gpu_parity import DEV, cosine, make_tables
from test_gpu_serving_ops import (BF16, F16, F32, contiguous, fill, make_batch, make_paged, ok_status, randn,
                                  value_norms)

pytestmark = pytest.mark.gpu


def make_pair(n, H, W, seed, keys, pairs, norm=True, rows=False, out_scale=0.4):
    g = torch.Generator().manual_seed(seed)
    lam = (0.2 + 0.6 * torch.rand((n, H) if rows else (H,), generator=g)).to(DEV)
    w = ops.HeadNorm(1 + 0.2 * randn((W,), seed + 1, F32), 1e-5) if norm else None
    return ops.DiffHeads(lam, keys, pairs, w, out_scale)


def want_diff(tables, pages, q, pair, start, seq, causal, H, scale=None):
    tokens = pages.shape[1] * 64
    kd, vd = (x.reshape(-1, H, tokens, tables.head_dim) for x in S.dense(tables, contiguous(pages), tokens))
    D = tables.head_dim
    scale = D ** -0.5 if scale is None else scale
    most = scale * np.linalg.norm(L.arr(q), axis=-1).max() * np.linalg.norm(kd, axis=-1).max()
    n = pair.norm
    return (*L.diff_attend(q, kd, vd, pair.lam, start, seq, scale, causal, pair.keys == "shared",
                           pair.pairs == "halves", n.weight if n else None, n.eps if n else 0.0,
                           n.offset if n else 0.0, pair.out_scale), most)


def check_diff(out, want, precise, cos=True):
    w, mag, gain, most = want
    dtype = out.dtype
    inside = ~np.isnan(w).any((1, 2))
    g, w, mag, gain = L.arr(out)[inside], w[inside], mag[inside], np.broadcast_to(gain, want[0].shape)[inside]
    rel = 2 * most * 2.0 ** -20 + 2.0 ** -18 if precise else 2 * most * 3 * 2.0 ** -11 + 2.0 ** -7 + 2.0 ** -9
    top = mag.max(-1, keepdims=True)                       # the norm's sum takes every column's error
    tol = rel * top * gain + S.half_ulp(dtype) * np.abs(w) + (2.0 ** -25 if dtype == F16 else 0)
    assert np.isfinite(g).all()
    assert (g[mag.max((1, 2)) == 0] == 0).all()
    assert (np.abs(g - w) <= tol).all(), (np.abs(g - w) - tol).max()
    if cos and not precise and mag.any():
        assert cosine(g, w) >= 0.9999
    if cos and precise and dtype == F32 and mag.any():     # far below what fp16 operands leave
        assert np.abs(g - w).max() <= 2e-5 * np.abs(w).max()


DIFF = {
    "tokens": ([(1, 1), (1, 64), (1, 65), (1, 513)], True),
    "drafts": ([(3, 5), (8, 700), (1, 129), (5, 64)], True),
    "chunks": ([(130, 130), (65, 300), (1, 90), (0, 33), (140, 140)], True),
    "empty rows": ([(6, 2), (3, 0), (2, 2), (0, 0)], True),
    "cross": ([(1, 300), (7, 1), (40, 129), (3, 0), (5, 64)], False),
    "split": ([(3, 4000)], True),
}
# D, kb, vb, pairs of query heads, KV heads, keys, pairs
GEOM = [(128, 4, 2, 4, 4, "own", "adjacent"), (128, 4, 4, 3, 2, "own", "halves"),
        (128, 3, 3, 8, 2, "own", "adjacent"), (128, 2, 2, 2, 4, "own", "halves"),
        (64, 4, 3, 5, 2, "own", "adjacent"), (64, 3, 3, 4, 4, "own", "halves"),
        (128, 6, 4, 2, 2, "own", "adjacent"), (64, 8, 8, 2, 2, "own", "adjacent"),
        (128, 4, 2, 4, 2, "shared", "adjacent"), (128, 3, 3, 3, 1, "shared", "adjacent"),
        (64, 4, 4, 4, 4, "shared", "adjacent"), (64, 2, 2, 5, 1, "shared", "adjacent"),
        (128, 8, 8, 2, 2, "shared", "adjacent")]


@pytest.mark.parametrize("case", sorted(DIFF))
@pytest.mark.parametrize("D,kb,vb,H,Hkv,keys,pairs", GEOM)
def test_diff_attend_matches_plain_form(D, kb, vb, H, Hkv, keys, pairs, case):
    lens, causal = DIFF[case]
    tables = make_tables(D, kb, vb, False)
    R = len(lens)
    batch, start, seq = make_batch(lens, lead=1)
    n = start[-1] + 2
    pages = make_paged(tables, R * Hkv, max(max(seq), 1))
    fill(tables, pages, R, Hkv, pages.shape[1] * 64, 3)
    ws = ops.DecodeWorkspace()
    W = 2 * D if keys == "own" else D
    for dtype, norm in ((BF16, True), (BF16, False), (F32, True), (F16, False)):
        q = randn((n, 2 * H, D), 4, dtype)
        pair = make_pair(n, H, W, 5, keys, pairs, norm, rows=case in ("drafts", "cross"))
        want = want_diff(tables, pages, q, pair, start, seq, causal, Hkv)
        outside = np.isnan(want[0]).any((1, 2))
        inside = torch.from_numpy(~outside).to(DEV)
        ran = 0
        for engine in (0, 1, 2, 3):
            out = torch.full((n, H, W), 7.0, dtype=dtype, device=DEV)
            try:
                got = ops.diff_attend_ragged(tables, pages, q, batch, pair, causal=causal, out=out,
                                             workspace=ws, engine=engine)
            except _lib.TqError as e:
                assert engine > 1 and "no kernel" in str(e)
                continue
            ran += 1
            assert got is out and ok_status() == 0
            assert (out[~inside] == 7.0).all()
            check_diff(out, want, dtype != BF16 and engine != 2)
            again = ops.diff_attend_ragged(tables, pages, q, batch, pair, causal=causal, engine=engine)
            assert torch.equal(again[inside], out[inside])       # joined in a fixed order
        assert ran >= 2
    assert ws.status() == 0


@pytest.mark.parametrize("case", ["tokens", "chunks", "cross", "split"])
@pytest.mark.parametrize("D,kb,vb,H,Hkv,keys,pairs", GEOM)
def test_diff_attend_bf16_results_row_by_row(D, kb, vb, H, Hkv, keys, pairs, case):
    """bf16 results where the maps do not cancel (no norm, lam below 0.3), every row and pair by itself: the
    root of the mean square of the error beside that of the row.  The result's rounding is 2^-8 at worst and
    0.43 x 2^-8 over mantissas alike likely (their step over sqrt(12), root of the mean of 1 / m^2 0.735).
    Operands: a score's 2^-12 roundings of q', key and norm are independent over the dims, at most
    sqrt(3 / D) `most` 2^-11 of them, seldom more than 2^-10; P and V 2^-11 each: together below 2^-9.
    So 2^-8 + 2^-9 for the worst row and sqrt(0.43^2 + 0.5^2) 2^-8 = 2.6e-3 over all."""
    lens, causal = DIFF[case]
    tables = make_tables(D, kb, vb, False)
    R = len(lens)
    batch, start, seq = make_batch(lens)
    n = start[-1]
    pages = make_paged(tables, R * Hkv, max(max(seq), 1))
    fill(tables, pages, R, Hkv, pages.shape[1] * 64, 3)
    q = randn((n, 2 * H, D), 4, BF16)
    lam = (0.3 * torch.rand((H,), generator=torch.Generator().manual_seed(5))).to(DEV)
    pair = ops.DiffHeads(lam, keys, pairs)
    want = want_diff(tables, pages, q, pair, start, seq, causal, Hkv)[0]
    for engine in (0, 1, 2, 3):
        try:
            out = L.arr(ops.diff_attend_ragged(tables, pages, q, batch, pair, causal=causal, engine=engine))
        except _lib.TqError as e:
            assert engine > 1 and "no kernel" in str(e)
            continue
        keys_seen = ~(want == 0).all(-1)
        err, size = ((x * x).mean(-1)[keys_seen] ** 0.5 for x in (out - want, want))
        assert (err <= (2.0 ** -8 + 2.0 ** -9) * size).all(), (engine, (err / size).max())
        assert (((err / size) ** 2).mean() ** 0.5) <= 2.6e-3, engine
        assert (out[~keys_seen] == 0).all()
    assert ok_status() == 0


def skip_without_kernel(keys, engine):
    """Own keys have no kernel of 256 rows (engine 2)."""
    if keys == "own" and engine in NO_OWN:
        pytest.skip("no such kernel")


NO_OWN = (2,)


def setup_case(lens, D=128, kb=4, vb=4, H=4, Hkv=4, keys="own", pairs="adjacent", seed=3, norm=True, lead=0):
    tables = make_tables(D, kb, vb, False)
    batch, start, seq = make_batch(lens, lead)
    pages = make_paged(tables, len(lens) * Hkv, max(max(seq), 1))
    fill(tables, pages, len(lens), Hkv, pages.shape[1] * 64, seed)
    pair = make_pair(start[-1], H, 2 * D if keys == "own" else D, seed + 7, keys, pairs, norm)
    return tables, batch, start, seq, pages, pair


@pytest.mark.parametrize("keys", ["own", "shared"])
def test_diff_attend_views_scale_types_and_lam_shapes(keys):
    """q a slice of one projection at an odd offset, out in transposed memory and of another type, a
    scale; lam of one number, of pairs, of rows, strided; contiguous pages; other bounds of max_q_len."""
    D, H, Hkv = 128, 4, 4
    tables = make_tables(D, 4, 4, False)
    batch, start, seq = make_batch([(4, 200), (9, 9), (140, 200), (1, 64)])
    n, W = start[-1], 2 * D if keys == "own" else D
    pages = torch.zeros((4 * Hkv, 4, ops.page_bytes(D, 4, 4, False)), dtype=torch.uint8, device=DEV)
    fill(tables, pages, 4, Hkv, 256, 8)
    q = randn((n, (2 * H + 2) * D + 1), 1)[:, 1: 1 + 2 * H * D].view(n, 2 * H, D)
    rows = 0.1 + 0.8 * torch.rand((n, 2 * H), generator=torch.Generator().manual_seed(2)).to(DEV)
    w = ops.HeadNorm(0.2 * randn((W,), 9), 1e-6, 1.0)
    for lam in (rows[0, :1], rows[0, :H], rows[:, :H], rows[:, ::2], rows[:, :1]):
        pair = ops.DiffHeads(lam, keys, "adjacent", w, 0.7)
        want = want_diff(tables, pages, q, pair, start, seq, True, Hkv, 0.05)
        out = torch.empty((H, n, W + 3), dtype=F32, device=DEV)[..., 1: W + 1].transpose(0, 1)
        ops.diff_attend_ragged(tables, pages, q, batch, pair, scale=0.05, out=out)
        check_diff(out, want, True)
        check_diff(ops.diff_attend_ragged(tables, pages, q, batch, pair, scale=0.05), want, False)
    for bound in (5000, 0):
        other = ops.RaggedBatch(batch.q_start, batch.seq_lens, bound)
        check_diff(ops.diff_attend_ragged(tables, pages, q, other, pair, scale=0.05), want, False)
    e = ops.diff_attend_ragged(tables, pages, q[:0], make_batch([(0, 5)] * 4)[0], ops.DiffHeads(
        torch.ones(1, device=DEV), keys))
    assert e.shape == (0, H, W) and ok_status() == 0


@pytest.mark.parametrize("keys", ["own", "shared"])
def test_diff_attend_follows_from_both_maps(keys):
    """With lam 0 the result is the first map's; shared keys: lam times the second map's attention off the
    first's, to fp32's rounding; the same query twice with lam 1 leaves nothing, whatever the norm."""
    lens = [(3, 700), (1, 64), (150, 300)]
    tables, batch, start, seq, pages, pair = setup_case(lens, keys=keys, norm=False)
    n, H, D = start[-1], 4, 128
    q = randn((n, 2 * H, D), 6, F32)
    pair = ops.DiffHeads(pair.lam, keys)
    got = ops.diff_attend_ragged(tables, pages, q, batch, pair)
    if keys == "shared":
        both = ops.attend_ragged(tables, pages, q, batch)
        want = both[:, 0::2] - pair.lam[:, None] * both[:, 1::2]
        assert (got - want).abs().max() <= 4 * 2.0 ** -24 * both.abs().max()
        twice = q[:, 0::2].repeat_interleave(2, 1).contiguous()
        one = ops.DiffHeads(torch.ones(1, device=DEV), keys, norm=ops.HeadNorm(torch.ones(D, device=DEV), 0.0))
        assert (ops.diff_attend_ragged(tables, pages, twice, batch, one) == 0).all()
    zero = ops.DiffHeads(torch.zeros(H, device=DEV), keys)
    first = ops.diff_attend_ragged(tables, pages, q, batch, zero)
    other = q.clone()
    other[:, 1::2] = randn((n, H, D), 8, F32)
    assert torch.equal(ops.diff_attend_ragged(tables, pages, other, batch, zero), first)
    assert ok_status() == 0


@pytest.mark.parametrize("engine", [0, 1, 2, 3])
@pytest.mark.parametrize("keys", ["own", "shared"])
def test_diff_attend_infinite_and_nan_norms(keys, engine):
    """A key or value of either head whose stored norm is not finite makes NaN of the pairs' rows that see
    it and of no other row or pair."""
    skip_without_kernel(keys, engine)
    lens = [(150, 150), (3, 200)]
    tables, batch, start, seq, pages, pair = setup_case(lens, keys=keys)
    n, H, D, Hkv = start[-1], 4, 128, 4
    q = randn((n, 2 * H, D), 6)
    want = ops.diff_attend_ragged(tables, pages, q, batch, pair, engine=engine)
    off = pages.pool.shape[1] - 256
    for head in (0, 1):
        for at in (0, 128):                                # key norms, value norms
            for bad in (float("inf"), float("nan")):
                keep = pages.pool.clone()
                page = int(pages.block_table[head, 70 // 64])
                pages.pool[page, off + at: off + at + 128].view(F16)[70 % 64] = bad
                got = ops.diff_attend_ragged(tables, pages, q, batch, pair, engine=engine)
                hit = [h for h in range(H) if (h // (H // Hkv) == head if keys == "shared" else
                                               h // (H // (Hkv // 2)) == 0)]
                seen = torch.zeros((n, H), dtype=torch.bool, device=DEV)
                seen[70:150, hit] = True
                assert got[seen].isnan().all() and torch.equal(got[~seen], want[~seen])
                pages.pool.copy_(keep)
    assert ok_status() == 0


@pytest.mark.parametrize("kb,vb,engine", [(4, 4, 0), (4, 4, 1), (4, 4, 3), (6, 6, 0), (8, 8, 0), (6, 4, 1)])
@pytest.mark.parametrize("keys,pairs", [("own", "adjacent"), ("own", "halves"), ("shared", "adjacent")])
def test_diff_attend_rows_that_see_a_norm_that_is_not_finite_are_nan_whole(keys, pairs, kb, vb, engine):
    """Without a norm behind the difference, which would carry NaN over the row: every column of the rows
    that see the token, and nothing else, on every kernel."""
    lens = [(150, 150), (3, 200)]
    tables, batch, start, seq, pages, pair = setup_case(lens, kb=kb, vb=vb, keys=keys, pairs=pairs, norm=False)
    if keys == "shared" and engine == 3 and kb > 4:
        pytest.skip("no such kernel")
    n, H, D, Hkv = start[-1], 4, 128, 4
    off = pages.pool.shape[1] - 256
    for dtype in (BF16, F32):
        q = randn((n, 2 * H, D), 6, dtype)
        want = ops.diff_attend_ragged(tables, pages, q, batch, pair, engine=engine)
        for head in (0, 1, 3):
            for at in (0, 128):                            # key norms, value norms
                for bad in (float("inf"), float("-inf"), float("nan")):
                    page = int(pages.block_table[head, 70 // 64])
                    place = pages.pool[page, off + at: off + at + 128].view(F16)
                    keep = place[70 % 64].clone()
                    place[70 % 64] = bad
                    got = ops.diff_attend_ragged(tables, pages, q, batch, pair, engine=engine)
                    hit = [h for h in range(H) if (h == head if keys == "shared" else
                                                   h // 2 == (head // 2 if pairs == "adjacent" else head % 2))]
                    seen = torch.zeros((n, H), dtype=torch.bool, device=DEV)
                    seen[70:150, hit] = True
                    assert got[seen].isnan().all() and torch.equal(got[~seen], want[~seen]), (head, at, bad)
                    place[70 % 64] = keep
    assert ok_status() == 0


@pytest.mark.parametrize("engine,dtype", [(0, BF16), (1, BF16), (2, BF16), (3, BF16), (0, F32)])
@pytest.mark.parametrize("keys", ["own", "shared"])
def test_diff_attend_small_value_norms_and_long_requests(keys, engine, dtype):
    """Norms far below fp16's range keep their digits; a request longer than its pages keeps its rows'
    places and is flagged."""
    skip_without_kernel(keys, engine)
    lens = [(40, 150), (3, 129), (150, 150), (5, 400), (1, 1 << 30)]
    tables, batch, start, seq, pages, pair = setup_case([(a, min(b, 128)) for a, b in lens], keys=keys,
                                                        norm=False)
    batch, start, seq = make_batch(lens)
    value_norms(tables, pages.pool).mul_(0.004)
    q = randn((start[-1], 8, 128), 6, dtype)
    want = want_diff(tables, pages, q, pair, start, seq, True, 4)
    got = ops.diff_attend_ragged(tables, pages, q, batch, pair, engine=engine)
    assert ok_status() == _lib.DEV_BAD_POSITION
    check_diff(got, want, dtype != BF16)


@pytest.mark.parametrize("keys", ["own", "shared"])
def test_diff_attend_bad_pages_and_batches(keys):
    """Pages outside the pool are flagged and leave other requests alone; offsets that do not ascend run
    nothing."""
    lens = [(3, 100), (2, 130), (140, 200)]
    tables, batch, start, seq, pages, pair = setup_case(lens, keys=keys)
    q = randn((start[-1], 8, 128), 6)
    for dtype in (BF16, F32):
        want = ops.diff_attend_ragged(tables, pages, q.to(dtype), batch, pair)
        bad = ops.PagedPages(pages.pool, pages.block_table.clone())
        bad.block_table[1, 0], bad.block_table[2, 1] = -5, pages.pool.shape[0]
        got = ops.diff_attend_ragged(tables, bad, q.to(dtype), batch, pair)
        assert ok_status() == _lib.DEV_BAD_BLOCK and torch.equal(got[3:], want[3:])
    for offsets in ([0, 3, 2, 145], [-1, 3, 5, 145], [0, 3, 5, 146], [5, 3, 5, 145]):
        wrong = ops.RaggedBatch(torch.tensor(offsets, dtype=torch.int32, device=DEV), batch.seq_lens, 145)
        for dtype in (BF16, F32):
            out = torch.full((start[-1], 4, 256 if keys == "own" else 128), 7.0, dtype=dtype, device=DEV)
            ops.diff_attend_ragged(tables, pages, q.to(dtype), wrong, pair, out=out)
            assert ok_status() == _lib.DEV_BAD_BATCH and (out == 7.0).all()


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("keys", ["own", "shared"])
def test_diff_attend_runs_what_it_accepts(D, keys):
    """Every pair of code widths and result type is refused before anything runs, or right: few and many
    rows."""
    batch, start, seq = make_batch([(2, 40), (70, 100)])
    ran = set()
    for kb in range(1, 9):
        for vb in range(1, 9):
            tables = make_tables(D, kb, vb, False)
            pages = make_paged(tables, 4, 100)
            fill(tables, pages, 2, 2, 128, 3)
            for dtype in (BF16, F16):
                pair = make_pair(start[-1], 2, 2 * D if keys == "own" else D, 3, keys, "adjacent")
                q = randn((start[-1], 4, D), 4, dtype)
                try:
                    got = ops.diff_attend_ragged(tables, pages, q, batch, pair)
                except _lib.TqError as e:
                    assert "no kernel for" in str(e)
                    continue
                ran.add((kb, vb, dtype))
                check_diff(got, want_diff(tables, pages, q, pair, start, seq, True, 2), dtype != BF16)
    assert ok_status() == 0
    for t in (BF16, F16):     # a cache's usual codes and those of its protected layers
        assert {(4, 2), (4, 4), (3, 3), (2, 2), (6, 4), (6, 6), (5, 5)} <= {(k, v) for k, v, u in ran if u == t}


def test_diff_attend_captured_on_another_stream_and_with_a_shared_workspace():
    """Eager, on a side stream and replayed with lengths, lam and inputs changed in place: the same bits;
    layers of both forms share a workspace."""
    D, H, Hkv, R = 128, 4, 4, 4
    tables = make_tables(D, 4, 2, False)
    pages = make_paged(tables, R * Hkv, 320)
    fill(tables, pages, R, Hkv, 320, 1)
    lens = [[(1, 100), (4, 260), (1, 65), (140, 200)], [(2, 102), (141, 261), (3, 68), (0, 4)]]
    n = 146
    ws = ops.DecodeWorkspace()
    norm = ops.HeadNorm(1 + 0.1 * randn((2 * D,), 3, F32))

    def layer(q, batch, lam, w):
        own = ops.diff_attend_ragged(tables, pages, q, batch, ops.DiffHeads(lam, norm=norm), workspace=w)
        return own, ops.diff_attend_ragged(tables, pages, q, batch, ops.DiffHeads(lam, "shared"), workspace=w)

    def args(i):
        return randn((n, 2 * H, D), 10 + i), make_batch(lens[i])[0], torch.rand(
            (H,), generator=torch.Generator().manual_seed(i)).to(DEV)

    rows = [sum(a for a, _ in x) for x in lens]
    eager = [layer(*args(i), ws) for i in range(2)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = layer(*args(1), ops.DecodeWorkspace())
    side.synchronize()
    for a, b in zip(got, eager[1]):
        assert torch.equal(a[: rows[1]], b[: rows[1]])
    q, batch, lam = args(0)
    batch = ops.RaggedBatch(batch.q_start, batch.seq_lens, 141)
    keep = ops.DecodeWorkspace()
    layer(q, batch, lam, keep)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(q, batch, lam, keep)
    for i in (0, 1, 0):
        x = args(i)
        q.copy_(x[0])
        batch.q_start.copy_(x[1].q_start)
        batch.seq_lens.copy_(x[1].seq_lens)
        lam.copy_(x[2])
        graph.replay()
        torch.cuda.synchronize()
        again = layer(*(x[0], ops.RaggedBatch(x[1].q_start, x[1].seq_lens, 141), x[2]), ops.DecodeWorkspace())
        for a, b in zip(out, again):
            assert torch.equal(a[: rows[i]], b[: rows[i]])
    assert ok_status() == 0


def test_layer_runs_together():
    """A layer as it is served: the norm before it, heads normed and rotated by three axes, keys and values
    appended, differential attention, and the sum and norm behind it, against the same chain in 64 bits on
    the codes that were stored.  Chained roundings: each tensor handed on is compared by itself."""
    D, H, Hkv, R, C = 128, 4, 4, 3, 512
    tables = make_tables(D, 4, 4, False)
    lens = [(70, 170), (1, 200), (5, 5)]
    batch, start, seq = make_batch(lens)
    n = start[-1]
    pages = make_paged(tables, R * Hkv, 256)
    fill(tables, pages, R, Hkv, 256, 1)
    axes = ops.RopeTable.axis_of_pairs((24, 20, 20), True)
    rope = ops.RopeTable.build(D, 4000, device=DEV, axes=axes)
    pos = torch.randint(0, 4000, (3, n), generator=torch.Generator().manual_seed(4))
    norms = [ops.HeadNorm(1 + 0.1 * randn((D,), i, F32)) for i in range(2)]
    pre, post = ops.RowNorm(1 + 0.1 * randn((C,), 5, F32)), ops.RowNorm(1 + 0.1 * randn((C,), 6, F32))
    pair = make_pair(n, H, 2 * D, 7, "own", "adjacent")
    proj = [randn((C, w), 8 + i) / C ** 0.5 for i, w in enumerate((2 * H * D, Hkv * D, Hkv * D))]
    back = randn((H * 2 * D, C), 12) / (2 * H * D) ** 0.5
    stream, block = randn((n, C), 13, F32), randn((n, C), 14)
    mid, h = ops.residual_norm(block, stream, post, None, "none", 1.0, pre)
    q, k, v = ((h @ p).view(n, -1, D) for p in proj)
    qr, _ = ops.qk_rope(q, None, rope, pos.to(DEV), q_norm=norms[0])
    ops.append_ragged(tables, pages, k, v, batch, rope=rope, k_norm=norms[1], positions=pos.to(DEV))
    o = ops.diff_attend_ragged(tables, pages, qr, batch, pair)
    end, h2 = ops.residual_norm(o.flatten(1) @ back, mid, post, torch.full((C,), 0.3, device=DEV, dtype=BF16),
                                "sigmoid", 1.0, pre)
    assert ok_status() == 0
    ym, dm, hm, dh = L.residual_norm(block, stream, post, None, "none", 1.0, pre)
    assert (np.abs(L.arr(mid) - ym) <= dm + S.half_ulp(F32) * np.abs(ym)).all()
    qw = L.rope_axes(q, rope.cos_sin, pos.numpy(), axes, False, norms[0].weight, 1e-6)
    assert (np.abs(L.arr(qr) - qw) <= S.half_ulp(BF16) * np.abs(qw) + S.rope_slack(q, norms[0].weight, 1e-6)).all()
    from test_gpu_serving_ops import check_stored
    kw = L.rope_axes(k, rope.cos_sin, pos.numpy(), axes, False, norms[1].weight, 1e-6)
    check_stored(tables, pages, k, v, start, seq, R, Hkv, kw)
    check_diff(o, want_diff(tables, pages, qr, pair, start, seq, True, Hkv), False)
    ye, de, he, dhe = L.residual_norm(o.flatten(1) @ back, mid, post,
                                      torch.full((C,), 0.3, dtype=BF16), "sigmoid", 1.0, pre)
    assert (np.abs(L.arr(h2) - he) <= dhe * (1 + 2.0 ** -8) + S.half_ulp(BF16) * np.abs(he)).all()


def test_sum_and_norm_behind_differential_attention():
    """Both results of residual_norm on what differential attention and its projection leave, fp16 and bf16
    blocks on an fp32 stream: the sum that the next layer starts from, and its norm."""
    tables, batch, start, seq, pages, pair = setup_case([(70, 170), (1, 200), (5, 5)])
    n, H, D, C = start[-1], 4, 128, 512
    post, pre = ops.RowNorm(1 + 0.1 * randn((C,), 5, F32)), ops.RowNorm(1 + 0.1 * randn((C,), 6, F32), centered=True)
    stream = randn((n, C), 13, F32)
    for dtype in (BF16, F16):
        back = randn((H * 2 * D, C), 12, dtype) / (2 * H * D) ** 0.5
        o = ops.diff_attend_ragged(tables, pages, randn((n, 2 * H, D), 3, dtype), batch, pair).flatten(1) @ back
        for gate in (torch.full((C,), 0.3, device=DEV, dtype=dtype), randn((n, C), 4, F32), None):
            act = "none" if gate is None else "sigmoid"
            end, h = ops.residual_norm(o, stream, post, gate, act, 1.0, pre)
            ye, de, he, dh = L.residual_norm(o, stream, post, gate, act, 1.0, pre)
            assert (np.abs(L.arr(end) - ye) <= de + S.half_ulp(F32) * np.abs(ye)).all()
            assert (np.abs(L.arr(h) - he) <= dh * (1 + 2.0 ** -8) + S.half_ulp(dtype) * np.abs(he) + 2.0 ** -25).all()
    assert ok_status() == 0


@pytest.mark.parametrize("keys", ["own", "shared"])
def test_paged_attention_layer_with_axes_and_pairs(keys):
    """TurboQuantPagedAttention.forward with positions of three axes and differential heads over a served
    schedule, rows behind the batch: what the operators give for the same pages."""
    from bhaskera_col_b200.inference.vllm_turboquant import TurboQuantPagedAttention, VLLMBatch
    D, Hq, H = 128, 8, 2
    layer = TurboQuantPagedAttention(3, 32, Hq, H, D, num_blocks=12, block_size=64, device=DEV)
    axes = ops.RopeTable.axis_of_pairs((24, 20, 20), True)
    rope = ops.RopeTable.build(D, 500, device=DEV, axes=axes)
    qn, kn = (ops.HeadNorm(1 + 0.1 * randn((D,), i, F32)) for i in range(2))
    bt = torch.randperm(12, generator=torch.Generator().manual_seed(2))[:8].view(2, 4).to(torch.int32).to(DEV)
    length = [0, 0]
    for i, new in enumerate(([130, 5], [1, 1], [3, 100])):
        length = [a + b for a, b in zip(length, new)]
        start, N = [0, new[0], sum(new)], sum(new)
        batch = VLLMBatch(torch.tensor(start, dtype=torch.int32, device=DEV),
                          torch.tensor(length, dtype=torch.int32, device=DEV), bt, N, max(new))
        q, k, v = (randn((N + 2, h, D), 10 * i + j) for j, h in enumerate((Hq, H, H)))
        pos = torch.randint(0, 500, (3, N + 2), generator=torch.Generator().manual_seed(i)).to(DEV)
        pair = make_pair(N + 2, Hq // 2, 2 * D if keys == "own" else D, i, keys, "adjacent", rows=True)
        out = layer.forward(q, k, v, batch, rope=rope, q_norm=qn, k_norm=kn, positions=pos, pair=pair)
        pages = layer.paged(layer.stream_table(bt))
        req, at = S.positions(start, length, N)
        kx = L.rope_axes(k[:N], rope.cos_sin, pos[:, :N].cpu().numpy(), axes, False, kn.weight, 1e-6)
        from test_gpu_serving_ops import check_stored
        check_stored(layer.tables, pages, k[:N], v[:N], start, length, 2, H, kx)
        qr, _ = ops.qk_rope(q[:N], None, rope, pos[:, :N], q_norm=qn)
        short = ops.DiffHeads(pair.lam[:N], keys, "adjacent", pair.norm, pair.out_scale)
        want = ops.diff_attend_ragged(layer.tables, pages, qr, batch.ragged(), short, scale=layer.scale)
        assert torch.equal(out[:N], want) and ok_status() == 0
        check_diff(want, want_diff(layer.tables, pages, qr, short, start, length, True, H, layer.scale), False)
    with pytest.raises(ValueError, match="rope"):
        layer.forward(q, k, v, batch, positions=pos, pair=pair)


def test_cache_with_axes_matches_rotated_heads():
    """TurboQuantKVCache.prefill / decode with a rope of several axes: positions (axes, B, T)."""
    from bhaskera_col_b200.inference import TurboQuantKVCache
    B, Hq, H, D = 2, 4, 2, 128
    rope = ops.RopeTable.build(D, 500, device=DEV, axes=ops.RopeTable.axis_of_pairs((16, 24, 24)))
    a, b = (TurboQuantKVCache(1, B, H, D, residual_window=0, protected_layers=0, device=DEV, max_seq_len=128)
            for _ in range(2))
    for i, n in enumerate((37, 1)):
        q, k, v = (randn((B, h, n, D), 5 * i + j) for j, h in enumerate((Hq, H, H)))
        pos = torch.randint(0, 500, (3, B, n), generator=torch.Generator().manual_seed(i)).to(DEV)
        call = (a.prefill, b.prefill) if n > 1 else (a.decode, b.decode)
        qr, kr = ops.qk_rope(q, k, rope, pos)
        assert torch.equal(call[0](q, k, v, 0, rope=rope, positions=pos), call[1](qr, kr, v, 0))
    assert torch.equal(a._stores[0]._pages, b._stores[0]._pages) and ok_status() == 0


def test_inputs_of_a_backward_pass_and_mixed_devices_are_refused():
    tables, batch, start, seq, pages, pair = setup_case([(3, 3)])
    q = randn((3, 8, 128), 1)
    with pytest.raises(RuntimeError, match="no backward pass"):
        ops.diff_attend_ragged(tables, pages, q.float().requires_grad_(), batch, pair)
    with pytest.raises(RuntimeError, match="no backward pass"):
        ops.diff_attend_ragged(tables, pages, q, batch, ops.DiffHeads(pair.lam.clone().requires_grad_()))
    with pytest.raises(ValueError, match="tensors on"):
        ops.diff_attend_ragged(tables, pages, q, batch, ops.DiffHeads(pair.lam.cpu()))
    with pytest.raises(ValueError, match="lam must be"):
        ops.diff_attend_ragged(tables, pages, q, batch, ops.DiffHeads(torch.ones(3, device=DEV)))
    with pytest.raises(ValueError, match="weights"):
        ops.diff_attend_ragged(tables, pages, q, batch,
                               ops.DiffHeads(pair.lam, norm=ops.HeadNorm(torch.ones(128, device=DEV))))
    x = randn((3, 64), 2, F32)
    for kw in (dict(residual=x.clone().requires_grad_()), dict(gate=x.clone().requires_grad_()),
               dict(pre_norm=ops.RowNorm(torch.ones(64, device=DEV, requires_grad=True)))):
        with pytest.raises(RuntimeError, match="no backward pass"):
            ops.residual_norm(x, **{"residual": x.clone(), **kw})
    with pytest.raises(ValueError, match="tensors on"):
        ops.residual_norm(x, x.clone(), gate=torch.ones(64))
    with pytest.raises(ValueError, match="values for rows"):
        ops.residual_norm(x, x.clone(), post_norm=ops.RowNorm(torch.ones(32, device=DEV)))
