"""Plain 64-bit forms of the serving operators on ragged batches, for their tests."""
import math

import numpy as np
import torch

from oracle import tq_oracle as O


def rope(x, cos_sin, pos, interleaved=False, w=None, eps=0.0, offset=0.0):
    """(N, H, D) heads normed (w given) and rotated (cos_sin given) by positions pos (N,)."""
    y = x.detach().cpu().double().numpy().copy()
    if w is not None:
        with np.errstate(invalid="ignore"):
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * \
                (w.cpu().double().numpy() + offset)
    if cos_sin is None:
        return y
    t = cos_sin.cpu().double().numpy()[np.asarray(pos)]
    half = t.shape[1] // 2
    c, s = t[:, None, :half], t[:, None, half:]
    ia = np.arange(half) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    a, b = y[..., ia].copy(), y[..., ib].copy()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def rope_slack(x, w=None, eps=0.0, offset=0.0):
    """Bound of the fp32 arithmetic's error in rope(): the norm's sum of squares passes at most 13
    roundings (half of them survive the root), mean, eps, root, quotient, weight and two products at
    most 7 more, a rotated element 3 on |a| + |b| <= 2 max|row|: under 16 u of that, u = 2^-24."""
    y = rope(x, None, None, w=w, eps=eps, offset=offset)
    return 16 * 2.0 ** -24 * 2 * np.abs(y).max(-1, keepdims=True)


def positions(q_start, seq_lens, n):
    """(request, position) of every row; request -1 for a row outside the batch."""
    r, p = np.full(n, -1), np.zeros(n, np.int64)
    for i in range(len(seq_lens)):
        a, b = q_start[i], q_start[i + 1]
        r[a:b] = i
        p[a:b] = seq_lens[i] - (b - a) + np.arange(b - a)
    return r, p


def parse(tables, pages, tokens):
    """Codes and norms of (streams, pages, bytes) contiguous pages."""
    geom = O.PageGeom(tables.head_dim, tables.key_bits, tables.value_bits, False)
    return O.parse_pages(geom, pages.cpu().numpy(), tokens)


def dense(tables, pages, tokens):
    """Stored K and V of every stream, (streams, tokens, D) in 64 bits."""
    f = parse(tables, pages, tokens)
    R = tables.rot.cpu().double().numpy()
    out = []
    for i, n, c in (("k_idx", "k_norm", tables.k_centroids), ("v_idx", "v_norm", tables.v_centroids)):
        c = c.cpu().double().numpy()
        out.append((c[f[i]] @ R) * f[n].astype(np.float64)[..., None])
    return out


def attend(q, k, v, q_start, seq_lens, scale, causal):
    """q (N, Hq, D), k / v (R, Hkv, T, D): rows outside the batch are NaN, rows without keys 0."""
    n, hq, d = q.shape
    q = q.detach().cpu().double().numpy()
    g = hq // k.shape[1]
    r, pos = positions(q_start, seq_lens, n)
    out = np.full((n, hq, d), np.nan)
    for i in range(n):
        if r[i] < 0:
            continue
        m = seq_lens[r[i]]
        if causal:
            m = min(m, pos[i] + 1)
        if m <= 0:
            out[i] = 0
            continue
        for h in range(hq):
            s = k[r[i], h // g, :m] @ q[i, h] * scale
            p = np.exp(s - s.max())
            out[i, h] = p @ v[r[i], h // g, :m] / p.sum()
    return out


def half_ulp(t):
    return torch.finfo(t).eps / 2


def default_scale(d):
    return 1.0 / math.sqrt(d)
