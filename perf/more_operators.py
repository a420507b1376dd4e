"""Cases of the operators of a layer with several position axes and differential heads, on a
flattened batch of requests whose keys and values live in the packed pages.

  rope    norms of the query and key heads with a rotation whose pairs follow different position
          axes (time, height, width), in one pass
  store   a ragged append of such tokens: keys normed and rotated on the way into the pages, and what
          the pages then hold read back
  diff    differential attention straight off the packed pages: two softmax maps of a pair of heads,
          the second taken off with a learned weight, a norm over what is left.  "own": each map has
          keys of its own and the values of both KV heads side by side; "shared": both query heads
          of a pair attend the same KV head
  norm    a block's output through its norm and its gate onto the residual stream, and the next
          block's norm of the sum

Each case is run in its plain form (elementary torch operations) where ``own`` is false, and by the
calls that a user of the package makes where it is true.
"""
import math
import random

import torch

own = False

DEV = "cuda"
PAGE = 64                      # tokens of a page
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_POS = 1 << 16              # rows of the rotation table


# --------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 16 sequences that hold images: latency
        dict(name="rope decode 16", op="rope", n=16, hq=32, hkv=8, d=128, axes="16 24 24", mixed=0,
             pairs="half", norm=0, dtype="bf16", lens=1),
        # prompts of text and video frames, heads normed, the axes' pairs in turn
        dict(name="rope frames 16k", op="rope", n=16381, hq=40, hkv=8, d=128, axes="24 20 20",
             mixed=1, pairs="half", norm=1, dtype="bf16", lens=2),
        # the tokens of image encoders: height and width, all heads with keys of their own
        dict(name="rope patches d64", op="rope", n=4097, hq=16, hkv=16, d=64, axes="16 16", mixed=0,
             pairs="interleaved", norm=0, dtype="fp16", lens=3),
        # one new token for each of 64 requests
        dict(name="store decode 64", op="store", r=64, q_lo=1, q_hi=1, t_lo=256, t_hi=16384, hkv=8,
             d=128, kb=4, vb=2, axes="16 24 24", mixed=0, pairs="half", norm=0, dtype="bf16",
             lens=4),
        # a batch of whole prompts with images, heads normed
        dict(name="store frames 18k", op="store", r=8, q_lo=512, q_hi=4096, t_lo=0, t_hi=0, hkv=8,
             d=128, kb=4, vb=4, axes="24 20 20", mixed=1, pairs="half", norm=1, dtype="bf16",
             lens=5),
        # one short request: latency
        dict(name="diff one short", op="diff", keys="own", r=1, q_lo=1, q_hi=1, t_lo=500, t_hi=500,
             hq=32, hkv=8, d=128, kb=4, vb=2, norm=1, causal=1, dtype="bf16", lens=6),
        # a decode step of 64 requests of very different lengths
        dict(name="diff decode 64", op="diff", keys="own", r=64, q_lo=1, q_hi=1, t_lo=256, t_hi=16384,
             hq=32, hkv=8, d=128, kb=4, vb=2, norm=1, causal=1, dtype="bf16", lens=7),
        # a few draft tokens over one long context, both maps over the same keys
        dict(name="diff long shared", op="diff", keys="shared", r=1, q_lo=3, q_hi=3, t_lo=65001,
             t_hi=65001, hq=32, hkv=4, d=128, kb=3, vb=3, norm=0, causal=1, dtype="bf16", lens=8),
        # chunked prefill of a batch: compute-bound
        dict(name="diff chunks", op="diff", keys="own", r=16, q_lo=96, q_hi=2048, t_lo=64, t_hi=6000,
             hq=32, hkv=8, d=128, kb=4, vb=4, norm=1, causal=1, dtype="bf16", lens=9),
        # one decode step of 16 sequences: latency
        dict(name="norm decode 16", op="norm", n=16, c=5120, post=1, pre=1, gate="none", layer=0,
             dtype="bf16", rdtype="bf16", lens=10),
        # prompts through a block with a norm on both sides
        dict(name="norm prompts 16k", op="norm", n=16381, c=4096, post=1, pre=1, gate="channel",
             layer=0, dtype="bf16", rdtype="bf16", lens=11),
        # an odd width, the residual stream in fp32, a gate of every token's own, layer norms
        dict(name="norm odd gated", op="norm", n=2051, c=2050, post=1, pre=1, gate="full", layer=1,
             dtype="fp16", rdtype="fp32", lens=12),
    ]


def _log(rng, lo, hi):
    """An integer of lo..hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _sections(rng, pairs):
    """Pairs of each of two to four axes."""
    cut = sorted(rng.sample(range(1, pairs), rng.choice([1, 2, 2, 3])))
    return " ".join(str(b - a) for a, b in zip([0] + cut, cut + [pairs]))


def draw(rng):
    op = rng.choice(["rope", "store", "diff", "diff", "norm"])
    lens = rng.randrange(1 << 30)
    if op == "norm":
        post = rng.randrange(2)
        return dict(op=op, n=_log(rng, 1, 4096), c=_log(rng, 64, 12288), post=post,
                    pre=1 if not post else rng.randrange(2),
                    gate=rng.choice(["none", "channel", "token", "full"]), layer=rng.randrange(2),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    rdtype=rng.choice(["same", "same", "fp32"]), lens=lens)
    hkv = rng.choice([2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 5, 8])
    d = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("rope", "store"):
        rot = d if op == "store" else rng.choice([d, d, d // 2])
        turn = dict(axes=_sections(rng, rot // 2), mixed=rng.randrange(2),
                    pairs=rng.choice(["half", "interleaved"]), norm=rng.randrange(2))
    if op == "rope":
        return dict(op=op, n=_log(rng, 1, 5000), hq=hkv * g, hkv=hkv, d=d,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), lens=lens, **turn)
    kb, vb = rng.choice([(4, 2), (4, 4), (3, 3), (2, 2)])
    r = _log(rng, 1, 32)
    q_hi = _log(rng, 1, 9000 // r)
    q_lo = _log(rng, 1, q_hi)
    if op == "store":
        t_hi = _log(rng, 1, 8192)
        return dict(op=op, r=r, q_lo=q_lo, q_hi=q_hi, t_lo=_log(rng, 1, t_hi), t_hi=t_hi, hkv=hkv,
                    d=d, kb=kb, vb=vb, dtype=dtype, lens=lens, **turn)
    keys = rng.choice(["own", "own", "shared"])
    hq = hkv * g * (2 if keys == "shared" else 1)
    q_hi = min(q_hi, 1024 if dtype == "bf16" else 64, 4096 // r)
    q_lo = min(q_lo, q_hi)
    t_hi = _log(rng, 1, 60000 // r if q_hi * r <= 512 else 6000 // r)
    return dict(op=op, keys=keys, r=r, q_lo=q_lo, q_hi=q_hi, t_lo=_log(rng, 1, t_hi), t_hi=t_hi,
                hq=hq, hkv=hkv, d=d, kb=kb, vb=vb, norm=rng.randrange(2),
                causal=rng.choice([1, 1, 0]), dtype=dtype, lens=lens)


def _lens(c):
    """(new tokens, tokens in the cache with the new ones) of each request.  With t_hi = 0 the
    cache holds nothing but the new tokens; a full (not causal) attention's queries are not in
    the cache."""
    rng = random.Random(c["lens"])
    q = [_log(rng, c["q_lo"], c["q_hi"]) for _ in range(c["r"])]
    t = [_log(rng, c["t_lo"], c["t_hi"]) if c["t_hi"] else 0 for _ in range(c["r"])]
    return (q, [a + b for a, b in zip(q, t)]) if c.get("causal", 1) else (q, t)


def _sizes(c):
    """Pairs of each axis."""
    return [int(n) for n in c["axes"].split()]


def _axis_of_pair(c):
    """The axis that each pair follows: runs of pairs, or (mixed) one pair of each axis in turn as
    long as it has any left."""
    if not c["mixed"]:
        return [a for a, n in enumerate(_sizes(c)) for _ in range(n)]
    left, out = _sizes(c), []
    while any(left):
        for a, n in enumerate(left):
            if n:
                out.append(a)
                left[a] -= 1
    return out


# --------------------------------------------------------------------------------------------
# the packed page: codes of K rows in quad order, of V rows in octet order, low bits first, then
# the fp16 norms of both
# --------------------------------------------------------------------------------------------
def _orders(d):
    """Coordinate at each position of a K row and of a V row."""
    k = [16 * j + 2 * t + e for t in range(4) for j in range(d // 16) for e in (0, 1, 8, 9)]
    v = [g + 8 * c for g in range(8) for c in range(d // 8)]
    return k, v


def _page_bytes(d, kb, vb):
    return PAGE * (d * kb // 8 + d * vb // 8 + 4)


def _pack(codes, bits):
    """(..., d) codes in row order -> (..., d * bits / 8) bytes."""
    b = (codes.unsqueeze(-1) >> torch.arange(bits, device=codes.device, dtype=torch.uint8)) & 1
    b = b.reshape(*codes.shape[:-1], -1, 8)
    w = (1 << torch.arange(8, device=codes.device)).to(torch.uint8)
    return (b * w).sum(-1, dtype=torch.uint8)


def _unpack(rows, d, bits):
    """(..., d * bits / 8) bytes -> (..., d) codes in row order."""
    b = (rows.unsqueeze(-1) >> torch.arange(8, device=rows.device, dtype=torch.uint8)) & 1
    b = b.reshape(*rows.shape[:-1], d, bits)
    w = 1 << torch.arange(bits, device=rows.device)
    return (b * w).sum(-1)


def _codebook(d, bits):
    """Lloyd-Max centroids and boundaries of N(0, 1/d) by fixed-point iteration (conditional means
    in closed form)."""
    n = 1 << bits
    pdf = lambda x: math.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)  # noqa: E731
    cdf = lambda x: 0.5 * math.erfc(-x / math.sqrt(2))  # noqa: E731
    c = [4.0 * (2 * i + 1 - n) / n for i in range(n)]
    for _ in range(400):
        e = [-40.0] + [(a + b) / 2 for a, b in zip(c, c[1:])] + [40.0]
        c = [(pdf(a) - pdf(b)) / max(cdf(b) - cdf(a), 1e-300) for a, b in zip(e, e[1:])]
    c = torch.tensor(c, dtype=torch.float64) / math.sqrt(d)
    return c.float().to(DEV), ((c[1:] + c[:-1]) / 2).float().to(DEV)


# --------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------
def _randn(gen, shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _heads(gen, n, h, d, dtype):
    """(n, h, d) projections: N(0, 1) with two channels of 8 times the size, as attention inputs of
    language models have."""
    x = _randn(gen, (n, h, d))
    x[..., torch.randint(0, d, (2,), generator=gen, device=DEV)] *= 8
    return x.to(DTYPES[dtype])


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cos_sin(rot):
    """(positions, rot) fp32: cosines, then sines, of position * 10000^(-2i/rot); from 64 bits."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    a = torch.arange(MAX_POS, device=DEV, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], -1).float()


def _positions(gen, n, axes):
    """int64 (axes, n): stretches of 1,024 tokens, text first (all axes alike), then a frame of 32
    tokens a row (time stands, height and width count); each stretch starts anywhere."""
    i = torch.arange(n, device=DEV)
    first = torch.randint(0, MAX_POS - 1024, (1 + n // 1024,), generator=gen, device=DEV)[i // 1024]
    i = i % 1024
    p = (i - 256).clamp_min(0)
    frame = [torch.zeros_like(p), p // 32, p % 32, p // 64]
    order = [1, 2] if axes == 2 else list(range(axes))
    return torch.stack([first + torch.where(i < 256, i, 256 + frame[a]) for a in order])


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    if c["op"] == "norm":
        n, w, dt = c["n"], c["c"], DTYPES[c["dtype"]]
        rdt = dt if c["rdtype"] == "same" else DTYPES[c["rdtype"]]
        # a residual stream with a few large channels; a block's output of smaller size
        s["residual"] = _randn(gen, (n, w)) * (1 + 3 * _randn(gen, (w,)).abs())
        s["residual"][:, torch.randint(0, w, (2,), generator=gen, device=DEV)] *= 20
        s["residual"] = s["residual"].to(rdt)
        s["x"] = (0.3 * _randn(gen, (n, w)) + 0.1 * _randn(gen, (w,))).to(dt)
        s["weights"] = [(1 + 0.2 * _randn(gen, (w,))).to(dt) for _ in range(2)]
        s["biases"] = [(0.1 * _randn(gen, (w,))).to(dt) if c["layer"] else None for _ in range(2)]
        shape = dict(none=None, channel=(w,), token=(n, 1), full=(n, w))[c["gate"]]
        s["gate"] = None if shape is None else _randn(gen, shape).to(dt)
        s["scale"] = 0.5 if c["gate"] == "channel" else 1.0
    else:
        _prepare_heads(s, c, gen)
    if own:
        _handles(s)
    return s


def _prepare_heads(s, c, gen):
    d = c["d"]
    if c["op"] in ("rope", "store"):
        s["cos_sin"] = _cos_sin(2 * sum(_sizes(c)))
        s["axis"] = torch.tensor(_axis_of_pair(c), device=DEV)
        s["w"] = (1 + 0.2 * _randn(gen, (2, d))).to(DTYPES[c["dtype"]])
    if c["op"] == "rope":
        s["q"], s["k"] = (_heads(gen, c["n"], c[h], d, c["dtype"]) for h in ("hq", "hkv"))
        s["pos"] = _positions(gen, c["n"], len(_sizes(c)))
        return
    qlen, tlen = _lens(c)
    r, hkv = c["r"], c["hkv"]
    s["qlen"], s["tlen"] = qlen, tlen
    s["q_start"] = _int32([sum(qlen[:i]) for i in range(r + 1)])
    s["seq_lens"] = _int32(tlen)
    n, pages = sum(qlen), -(-max(tlen) // PAGE)
    s["n"] = n
    s["kc"], s["kbnd"] = _codebook(d, c["kb"])
    s["vc"], s["vbnd"] = _codebook(d, c["vb"])
    s["R"] = torch.linalg.qr(_randn(gen, (d, d)).double())[0].float().contiguous()
    # a pool of pages in any order; the pages of request b, head h are table[b * hkv + h]
    need = [-(-t // PAGE) for t in tlen]
    perm = torch.randperm(sum(need) * hkv, generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros((r, hkv, pages), dtype=torch.int32, device=DEV)
    at = 0
    for i, m in enumerate(need):
        table[i, :, :m] = perm[at: at + hkv * m].view(hkv, m)
        at += hkv * m
    s["table"] = table.view(r * hkv, pages)
    if c["op"] == "store":
        s["pool"] = torch.zeros((sum(need) * hkv, _page_bytes(d, c["kb"], c["vb"])),
                                dtype=torch.uint8, device=DEV)
        s["k"], s["v"] = (_heads(gen, n, hkv, d, c["dtype"]) for _ in range(2))
        s["pos"] = _positions(gen, n, len(_sizes(c)))
        return
    parts = []
    for bits, bnd in ((c["kb"], s["kbnd"]), (c["vb"], s["vbnd"])):
        y = _randn(gen, (sum(need) * hkv, PAGE, d))
        y /= y.square().sum(-1, keepdim=True).sqrt()
        code = torch.bucketize(y, bnd, out_int32=True).to(torch.uint8)
        del y
        parts.append(_pack(code, bits).reshape(sum(need) * hkv, -1))
        del code
    norms = math.sqrt(d) * (1 + 0.1 * _randn(gen, (sum(need) * hkv, 2 * PAGE)))
    s["pool"] = torch.cat(parts + [norms.half().view(torch.uint8)], -1).contiguous()
    # heads of a pair next to each other; scores spread as those of attention that picks keys out
    s["q"] = (2 * _randn(gen, (n, c["hq"], d))).to(DTYPES[c["dtype"]])
    s["lam"] = 0.2 + 0.6 * torch.rand((c["hq"] // 2,), generator=gen, device=DEV)
    width = 2 * d if c["keys"] == "own" else d
    s["w"] = (1 + 0.2 * _randn(gen, (width,))).to(DTYPES[c["dtype"]])


def _handles(s):
    """What a program that serves with the package keeps between calls: the norms, the layer's
    tables, the paged pool, the rotation table and the workspace; and a step's batch description,
    which all layers of the step share."""
    from bhaskera_col_b200.inference import ops
    c = s["case"]
    if c["op"] == "norm":
        s["norms"] = [ops.RowNorm(w, bias=b, eps=1e-5, centered=bool(c["layer"]))
                      for w, b in zip(s["weights"], s["biases"])]
        return
    if c["op"] in ("rope", "store"):
        s["rope"] = ops.RopeTable(s["cos_sin"], interleaved=c["pairs"] == "interleaved",
                                  axes=tuple(_axis_of_pair(c)))
        s["norms"] = [ops.HeadNorm(w, eps=1e-6) if c["norm"] else None for w in s["w"]]
    if c["op"] == "diff":
        s["pair"] = ops.DiffHeads(s["lam"], keys=c["keys"], out_scale=0.5,
                                  norm=ops.HeadNorm(s["w"], eps=1e-5) if c["norm"] else None)
    if c["op"] != "rope":
        s["tables"] = ops.LayerTables(c["d"], c["kb"], c["vb"], False, s["kc"], s["kbnd"], s["vc"],
                                      s["vbnd"], s["R"])
        s["pages"] = ops.PagedPages(s["pool"], s["table"])
        s["batch"] = ops.RaggedBatch(s["q_start"], s["seq_lens"], max(s["qlen"]))
        s["workspace"] = ops.DecodeWorkspace()


# --------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from bhaskera_col_b200.inference import ops
    c = s["case"]
    if c["op"] == "rope":
        q, k = ops.qk_rope(s["q"], s["k"], s["rope"], s["pos"], q_norm=s["norms"][0],
                           k_norm=s["norms"][1])
        return {"q": q, "k": k}
    if c["op"] == "store":
        ops.append_ragged(s["tables"], s["pages"], s["k"], s["v"], s["batch"], rope=s["rope"],
                          k_norm=s["norms"][1], positions=s["pos"])
        shape = (s["n"], c["hkv"], c["d"])
        k, v = (torch.empty(shape, dtype=DTYPES[c["dtype"]], device=DEV) for _ in range(2))
        ops.dequantize_ragged(s["tables"], s["pages"], s["batch"], k, v)
        return {"k": k, "v": v}
    if c["op"] == "diff":
        return {"out": ops.diff_attend_ragged(s["tables"], s["pages"], s["q"], s["batch"], s["pair"],
                                              causal=bool(c["causal"]), workspace=s["workspace"])}
    y, h = ops.residual_norm(s["x"], s["residual"], post_norm=s["norms"][0] if c["post"] else None,
                             gate=s["gate"], gate_act="sigmoid" if c["gate"] == "full" else "none",
                             scale=s["scale"], pre_norm=s["norms"][1] if c["pre"] else None)
    return {"residual": y} if h is None else {"residual": y, "h": h}


def _norm_rope(x, cos, sin, pairs, w):
    """RMS norm over the head (where w is given), then the rotation of its first dims."""
    if w is not None:
        x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    if pairs == "half":
        a, b = x[..., :half], x[..., half: 2 * half]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., 2 * half:]], -1)


def _angles(s):
    """(n, pairs) cosines and sines: pair i of token t from row pos[axis[i], t]."""
    rows = s["pos"][s["axis"]].T                           # (n, pairs)
    half = rows.shape[1]
    pair = torch.arange(half, device=DEV)
    return s["cos_sin"][rows, pair], s["cos_sin"][rows, half + pair]


def _stored(x, R, cent, bnd):
    """What the cache gives back for x: the codes' centroids of the rotated unit vector, rotated
    back, times the norm in fp16."""
    n = x.square().sum(-1, keepdim=True).sqrt()
    y = (x / n.clamp_min(1e-8)) @ R.T
    return (cent[torch.bucketize(y, bnd)] @ R) * n.half().to(x.dtype)


def _row_norm(x, w, b):
    """RMS norm, or layer norm where there is a bias."""
    if b is not None:
        x = x - x.mean(-1, keepdim=True)
    x = x * (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w.float()
    return x if b is None else x + b.float()


def _run_plain(s):
    c = s["case"]
    dtype = DTYPES[c["dtype"]]
    if c["op"] == "rope":
        cos, sin = _angles(s)
        return {x: _norm_rope(s[x].float(), cos, sin, c["pairs"],
                              s["w"][i].float() if c["norm"] else None).to(dtype)
                for i, x in enumerate(("q", "k"))}
    if c["op"] == "store":
        # in 64 bits: a code turns over where the rotated value lies next to a boundary
        cos, sin = _angles(s)
        k = _norm_rope(s["k"].double(), cos.double(), sin.double(), c["pairs"],
                       s["w"][1].double() if c["norm"] else None)
        R = s["R"].double()
        return {"k": _stored(k, R, s["kc"].double(), s["kbnd"].double()).to(dtype),
                "v": _stored(s["v"].double(), R, s["vc"].double(), s["vbnd"].double()).to(dtype)}
    if c["op"] == "norm":
        z = s["x"].float()
        if c["post"]:
            z = _row_norm(z, s["weights"][0], s["biases"][0])
        if s["gate"] is not None:
            gate = s["gate"].float()
            z = z * (1 / (1 + (-gate).exp()) if c["gate"] == "full" else gate)
        y = s["residual"].float() + s["scale"] * z
        out = {"residual": y.to(s["residual"].dtype)}
        if c["pre"]:
            out["h"] = _row_norm(y, s["weights"][1], s["biases"][1]).to(dtype)
        return out
    # request by request, pair of KV heads by pair
    h, d, hkv = c["hq"] // 2, c["d"], c["hkv"]
    own_keys = c["keys"] == "own"
    out = torch.empty((s["n"], h, 2 * d if own_keys else d), dtype=dtype, device=DEV)
    at = 0
    for i, (n, t) in enumerate(zip(s["qlen"], s["tlen"])):
        k, v = _dense(s, i, t)                             # (hkv, t, d)
        q = s["q"][at: at + n].float()
        if own_keys:
            k = k.view(hkv // 2, 2, t, d)
            v = torch.cat([v[0::2], v[1::2]], -1)          # (pairs, t, 2 d)
            q = q.view(n, hkv // 2, -1, 2, d).permute(3, 1, 2, 0, 4)
            x = torch.stack([_map(q[m], k[:, m], c, n, t) for m in (0, 1)])
        else:
            q = q.view(n, hkv, -1, 2, d).permute(3, 1, 2, 0, 4)
            x = torch.stack([_map(q[m], k, c, n, t) for m in (0, 1)])
        groups = x.shape[2]                                # (2, kv, g, n, t)
        lam = s["lam"].view(-1, groups, 1, 1)
        o = x[0].flatten(1, 2) @ v - lam.repeat(1, 1, n, 1).flatten(1, 2) * (x[1].flatten(1, 2) @ v)
        o = o.view(-1, groups, n, v.shape[-1])
        if c["norm"]:
            o = o * (o.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * s["w"].float()
        out[at: at + n] = (0.5 * o).permute(2, 0, 1, 3).reshape(n, h, -1).to(dtype)
        at += n
    return {"out": out}


def _map(q, k, c, n, t):
    """Softmax of q (kv, g, n, d) over keys k (kv, t, d); masked keys are -inf."""
    kv, g, _, d = q.shape
    x = (q.reshape(kv, g * n, d) @ k.transpose(-1, -2)).view(kv, g, n, t)
    x *= 1.0 / math.sqrt(d)
    if c["causal"]:
        key, last = torch.arange(t, device=DEV), torch.arange(t - n, t, device=DEV)
        x.masked_fill_(key[None] > last[:, None], float("-inf"))
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    x /= x.sum(-1, keepdim=True)
    return x


def _dense(s, i, t, dt=torch.float32):
    """Request i's first t keys and values, (hkv, t, d), from the packed pages."""
    c = s["case"]
    d, hkv = c["d"], c["hkv"]
    pg = s["pool"][s["table"].view(c["r"], hkv, -1)[i, :, : -(-t // PAGE)].long()]
    krow, vrow = d * c["kb"] // 8, d * c["vb"] // 8
    out = []
    for w, (off, row, bits, cent) in enumerate(((0, krow, c["kb"], s["kc"]),
                                                (PAGE * krow, vrow, c["vb"], s["vc"]))):
        code = _unpack(pg[..., off: off + PAGE * row].unflatten(-1, (PAGE, row)), d, bits)
        at = PAGE * (krow + vrow) + 2 * PAGE * w
        n = pg[..., at: at + 2 * PAGE].contiguous().view(torch.float16).to(dt)
        R = s["R"].to(dt)[_orders(d)[w]]                   # rows in the order of the codes
        out.append(((cent.to(dt)[code] @ R) * n.unsqueeze(-1)).reshape(hkv, -1, d)[:, :t])
    return out


# --------------------------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "rope":
        return {x: _exact_rope(s[x], s, c, s["w"][i]) for i, x in enumerate(("q", "k"))}
    if c["op"] == "store":
        out = {}
        for name, cent, bnd in (("k", s["kc"], s["kbnd"]), ("v", s["vc"], s["vbnd"])):
            x = _exact_rope(s["k"], s, c, s["w"][1]) if name == "k" else s["v"].double()
            n = torch.linalg.vector_norm(x, dim=-1)
            y = torch.einsum("nhi,ji->nhj", x / n.clamp_min(1e-8)[..., None], s["R"].double())
            val = torch.zeros_like(y) + cent[0].double()
            for j in range(len(bnd)):                      # the highest boundary below y
                val = torch.where(y > bnd[j].double(), cent[j + 1].double(), val)
            out[name] = torch.einsum("nhj,ji,nh->nhi", val, s["R"].double(), n.half().double())
        return out
    if c["op"] == "norm":
        return _exact_norm(s, c)
    return {"out": _exact_diff(s, c)}


def _exact_rope(x, s, c, w):
    """The rotation as a product of complex numbers, an axis at a time."""
    x = x.double()
    if c["norm"]:
        x = x / (torch.sum(x * x, -1, keepdim=True) / c["d"] + 1e-6).sqrt() * w.double()
    rot = s["cos_sin"].shape[1]
    axis = _axis_of_pair(c)
    y = x.clone()
    for a, pos in enumerate(s["pos"]):
        turn = torch.complex(*s["cos_sin"].double()[pos].split(rot // 2, -1))
        for i in (i for i in range(rot // 2) if axis[i] == a):
            lo, hi = (i, rot // 2 + i) if c["pairs"] == "half" else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., lo], x[..., hi]) * turn[:, i, None]
            y[..., lo], y[..., hi] = z.real, z.imag
    return y


def _exact_norm(s, c):
    def norm(x, i):
        w = s["weights"][i].double()
        if not c["layer"]:
            return x / (torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / c["c"] + 1e-5).sqrt() * w
        var, mean = torch.var_mean(x, dim=-1, keepdim=True, correction=0)
        return (x - mean) / (var + 1e-5).sqrt() * w + s["biases"][i].double()

    z = s["x"].double()
    if c["post"]:
        z = norm(z, 0)
    if s["gate"] is not None:
        gate = s["gate"].double()
        z = z * (torch.sigmoid(gate) if c["gate"] == "full" else gate)
    y = s["residual"].double() + s["scale"] * z
    return {"residual": y, "h": norm(y, 1)} if c["pre"] else {"residual": y}


def _exact_diff(s, c):
    """Head by head, the keys and values of a stream decoded bit by bit."""
    d, hkv, h = c["d"], c["hkv"], c["hq"] // 2
    own_keys = c["keys"] == "own"
    inv = [torch.tensor(o, device=DEV).argsort() for o in _orders(d)]
    krow, vrow = d * c["kb"] // 8, d * c["vb"] // 8
    outs = []
    for i, (n, t) in enumerate(zip(s["qlen"], s["tlen"])):
        pg = s["pool"][s["table"].view(c["r"], hkv, -1)[i, :, : -(-t // PAGE)].long()]
        kv = []
        for w, (off, row, bits, cent) in enumerate(((0, krow, c["kb"], s["kc"]),
                                                    (PAGE * krow, vrow, c["vb"], s["vc"]))):
            rows = pg[..., off: off + PAGE * row].reshape(hkv, -1, row).long()
            bit = torch.stack([(rows >> b) & 1 for b in range(8)], -1).reshape(*rows.shape[:2], -1)
            code = sum(bit[..., b::bits] << b for b in range(bits))[..., inv[w]]
            at = PAGE * (krow + vrow) + 2 * PAGE * w
            nrm = pg[..., at: at + 2 * PAGE].contiguous().view(torch.float16).reshape(hkv, -1)
            x = cent.double()[code] * nrm.double()[..., None]
            kv.append(torch.einsum("htj,ji->hti", x, s["R"].double())[:, :t])
        k, v = kv
        a = sum(s["qlen"][:i])
        q = s["q"][a: a + n].double()
        o = torch.empty((n, h, 2 * d if own_keys else d), dtype=torch.float64, device=DEV)
        for j in range(h):
            pair = j // (h // (hkv // 2)) if own_keys else j // (h // hkv)
            vj = torch.cat([v[2 * pair], v[2 * pair + 1]], -1) if own_keys else v[pair]
            maps = []
            for m in (0, 1):
                x = torch.einsum("nd,td->nt", q[:, 2 * j + m],
                                 k[2 * pair + m] if own_keys else k[pair]) / math.sqrt(d)
                if c["causal"]:
                    x = x + torch.full_like(x, float("-inf")).triu(t - n + 1)
                maps.append(torch.softmax(x, -1))
            o[:, j] = (maps[0] - s["lam"][j].double() * maps[1]) @ vj
        if c["norm"]:
            o = o / (torch.sum(o * o, -1, keepdim=True) / o.shape[-1] + 1e-5).sqrt() * s["w"].double()
        outs.append(o / 2)
    return torch.cat(outs)


# --------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------
def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "norm":
        n, w = c["n"], c["c"]
        rsize = size if c["rdtype"] == "same" else 4 if c["rdtype"] == "fp32" else 2
        gate = dict(none=0, channel=w, token=n, full=n * w)[c["gate"]]
        norms = (c["post"] + c["pre"]) * (2 if c["layer"] else 1)
        return {"bytes": n * w * (size * (1 + c["pre"]) + 2 * rsize) + (gate + norms * w) * size,
                "flops": n * w * (2 + 4 * (c["post"] + c["pre"]) + (c["gate"] != "none"))}
    d = c["d"]
    if c["op"] == "rope":
        rows, rot = c["n"] * (c["hq"] + c["hkv"]), 2 * sum(_sizes(c))
        # heads in and out, a pair's cosine and sine and the positions for each token
        return {"bytes": 2 * rows * d * size + c["n"] * (4 * rot + 8 * len(_sizes(c))),
                "flops": rows * (3 * rot + (4 * d if c["norm"] else 0))}
    qlen, tlen = _lens(c)
    n, hkv, r = sum(qlen), c["hkv"], c["r"]
    packed = d * (c["kb"] + c["vb"]) // 8 + 4               # bytes of one token of one head
    plan = 8 * r + 4 + sum(4 * hkv * -(-t // PAGE) for t in tlen)
    if c["op"] == "store":
        # packed and read back; K and V through the rotation on both ways
        once = n * hkv * (packed + 2 * d * size)
        return {"bytes": 2 * once + n * (4 * d + 8 * len(_sizes(c))) + plan,
                "flops": 2 * n * hkv * 2 * 2 * d * d}
    # both maps' scores, then their difference times the values
    width = 2 * d if c["keys"] == "own" else d
    seen = sum(a * b - (a * (a - 1) // 2 if c["causal"] else 0) for a, b in zip(qlen, tlen))
    h = c["hq"] // 2
    return {"bytes": sum(tlen) * hkv * packed + n * (c["hq"] * d + h * width) * size + plan + 4 * h,
            "flops": seen * h * (4 * d + 2 * width) + 2 * n * (c["hq"] + h * width // d) * d * d}
