"""Plain 64-bit forms of rotations with several axes, of differential attention off the packed pages
and of the norms around a block, for their tests."""
import numpy as np

import serving_oracle as S

U = 2.0 ** -24


def arr(x):
    return None if x is None else x.detach().cpu().double().numpy()


def rope_axes(x, cos_sin, pos, axes, interleaved=False, w=None, eps=0.0, offset=0.0):
    """S.rope with pair i at position pos[axes[i]], pos (axes, N): a table of a token's own, one row
    per token, picked pair by pair."""
    t = arr(cos_sin)
    half, pos = t.shape[1] // 2, np.asarray(pos)
    own = np.empty((pos.shape[1], 2 * half))
    for i, a in enumerate(axes):
        own[:, i], own[:, half + i] = t[pos[a], i], t[pos[a], half + i]

    class Own:
        def cpu(self):
            return self

        def double(self):
            return self

        def numpy(self):
            return own
    return S.rope(x, Own(), np.arange(pos.shape[1]), interleaved, w, eps, offset)


def _norm(y, dy, norm):
    """(norm(y), bound of the kernel's error), dy the bound of y's.  In units of u: a row's sum of C
    values passes at most 32 roundings in a thread, 5 in a warp and 32 across warps; half of those of
    the squares survive the root; mean, eps, root, quotient, two products, a sum: under 48 in all.  An
    error of y turns up once by itself and once through the sum of squares (at most max dy / rms);
    the mean's is 70 u mean |y|."""
    w, b = arr(norm.weight), arr(norm.bias)
    w = np.ones(y.shape[-1]) if w is None else w + norm.offset
    b = np.zeros(y.shape[-1]) if b is None else b
    top = np.broadcast_to(dy, y.shape).max(-1, keepdims=True)
    if norm.centered:
        mean = y.mean(-1, keepdims=True)
        top = 2 * top + 72 * U * np.abs(y).mean(-1, keepdims=True) + U * np.abs(y).max(-1, keepdims=True)
        y = y - mean
    with np.errstate(invalid="ignore", divide="ignore"):
        ms = (y * y).mean(-1, keepdims=True) + norm.eps
        r = 1 / np.sqrt(ms)
        z = y * r * w
        err = 48 * U * np.abs(z) + r * np.abs(w) * top + np.abs(z) * top * r + 2 * U * np.abs(b)
    return z + b, err


def residual_norm(x, residual, post=None, gate=None, act="none", scale=1.0, pre=None):
    """(y, its bound, h, its bound): bounds of the fp32 arithmetic before the rounding of the results.
    The gate's function is off by 8 u at most (two calls and a quotient)."""
    z, r = arr(x), arr(residual)
    dz = np.zeros_like(z)
    if post is not None:
        z, dz = _norm(z, dz, post)
    f = np.full(z.shape, float(scale))
    if gate is not None:
        g = np.broadcast_to(arr(gate), z.shape)
        f = f * {"none": lambda v: v, "sigmoid": lambda v: 1 / (1 + np.exp(-v)), "tanh": np.tanh}[act](g)
    y = r + f * z
    dy = np.abs(f) * dz + 12 * U * np.abs(f * z) + U * np.abs(y)
    if pre is None:
        return y, dy, None, None
    h, dh = _norm(y, dy, pre)
    return y, dy, h, dh


def diff_attend(q, k, v, lam, q_start, seq_lens, scale, causal, shared, halves, norm=None, eps=0.0,
                offset=0.0, out_scale=1.0):
    """q (N, 2H, D), k / v (R, Hkv, T, D) in 64 bits; lam (H,) or (N, H).  Returns (out, mag, gain) of
    (N, H, W): rows outside the batch are NaN, rows without keys 0.  mag = sum_t (p1 + |lam| p2) |v_t|:
    what errors of the weights and values are relative to, before the norm; gain: the bound of what the
    norm and out_scale make of such an error (by itself, and through the sum of squares)."""
    n, hq, d = q.shape
    H, hkv = hq // 2, k.shape[1]
    qs = arr(q)
    qs = np.stack([qs[:, :H], qs[:, H:]] if halves else [qs[:, 0::2], qs[:, 1::2]])
    lam = np.broadcast_to(arr(lam), (n, H))
    r, pos = S.positions(q_start, seq_lens, n)
    W = d if shared else 2 * d
    out, mag = np.full((n, H, W), np.nan), np.zeros((n, H, W))
    for i in range(n):
        if r[i] < 0:
            continue
        m = seq_lens[r[i]]
        if causal:
            m = min(m, pos[i] + 1)
        m = min(m, k.shape[2])
        out[i] = 0
        if m <= 0:
            continue
        for h in range(H):
            if shared:
                ks = [h // (H // hkv)] * 2
                val = v[r[i], ks[0], :m]
            else:
                p, P = h // (H // (hkv // 2)), hkv // 2
                ks = [p, P + p] if halves else [2 * p, 2 * p + 1]
                val = np.concatenate([v[r[i], s, :m] for s in ks], -1)
            for j, f in enumerate((1.0, -lam[i, h])):
                s = k[r[i], ks[j], :m] @ qs[j, i, h] * scale
                e = np.exp(s - s.max())
                out[i, h] += f * (e @ val) / e.sum()
                mag[i, h] += abs(f) * (e @ np.abs(val)) / e.sum()
    gain = np.full((n, H, 1), abs(out_scale))
    if norm is not None:
        w = np.abs(arr(norm) + offset) * abs(out_scale)
        with np.errstate(invalid="ignore", divide="ignore"):
            rms = np.sqrt((out * out).mean(-1, keepdims=True) + eps)
            y = out / rms * (arr(norm) + offset)
            gain = w * (1 + np.abs(out) / rms) / rms
        out = np.where(out == 0, 0, y)
    return out * out_scale, mag, gain
