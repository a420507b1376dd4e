"""Cases of the serving operators around the packed KV cache: what a serving step does between a
layer's q/k/v projections and its output projection, on a flattened batch of requests.

  rope    norms of the query and key heads with the position rotation, in one pass
  store   a ragged append: the new tokens' keys (normed and rotated on the way) and values are
          quantised into their requests' pages; what the pages then hold is read back
  read    a ragged read-back of stored tokens as dense keys and values
  attend  attention of every request's new tokens over its packed pages: causal (prompt chunks,
          draft verification, single tokens) or full (a decoder's cross attention over an encoder's
          states)

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
MAX_POS = 1 << 18              # rows of the rotation table


# --------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 16 sequences, 32 / 8 heads: latency
        dict(name="rope decode 16", op="rope", n=16, hq=32, hkv=8, d=128, rot=128, pairs="half",
             norm=0, dtype="bf16", lens=1),
        # prompt chunks of a batch, heads normed before the rotation
        dict(name="rope prompts 16k", op="rope", n=16381, hq=40, hkv=8, d=128, rot=128,
             pairs="half", norm=1, dtype="bf16", lens=2),
        # one new token for each of 64 requests
        dict(name="store decode 64", op="store", r=64, q_lo=1, q_hi=1, t_lo=256, t_hi=16384, hkv=8,
             d=128, kb=4, vb=2, pairs="half", norm=0, dtype="bf16", lens=3),
        # a batch of whole prompts, heads normed
        dict(name="store prompts 16k", op="store", r=8, q_lo=512, q_hi=4096, t_lo=0, t_hi=0, hkv=8,
             d=128, kb=4, vb=4, pairs="half", norm=1, dtype="bf16", lens=4),
        # odd chunks of small heads, interleaved pairs, 3-bit codes
        dict(name="store odd d64", op="store", r=13, q_lo=1, q_hi=700, t_lo=1, t_hi=3000, hkv=4,
             d=64, kb=3, vb=3, pairs="interleaved", norm=0, dtype="fp16", lens=5),
        # a short prefix handed to another attention
        dict(name="read prefix", op="read", r=3, q_lo=50, q_hi=200, t_lo=50, t_hi=200, hkv=8,
             d=128, kb=4, vb=2, dtype="bf16", lens=6),
        # whole contexts of a batch
        dict(name="read contexts 32k", op="read", r=8, q_lo=1024, q_hi=8192, t_lo=0, t_hi=0, hkv=8,
             d=128, kb=4, vb=4, dtype="bf16", lens=7),
        # one short request: latency
        dict(name="attend one short", op="attend", r=1, q_lo=4, q_hi=4, t_lo=500, t_hi=500, hq=32,
             hkv=8, d=128, kb=4, vb=2, causal=1, dtype="bf16", lens=8),
        # draft verification: a few tokens for each of 64 requests of very different lengths
        dict(name="attend drafts 64", op="attend", r=64, q_lo=2, q_hi=8, t_lo=256, t_hi=16384,
             hq=32, hkv=8, d=128, kb=4, vb=2, causal=1, dtype="bf16", lens=9),
        # a few tokens over one long context
        dict(name="attend long 128k", op="attend", r=1, q_lo=5, q_hi=5, t_lo=131001, t_hi=131001,
             hq=40, hkv=8, d=128, kb=3, vb=3, causal=1, dtype="bf16", lens=10),
        # chunked prefill of a batch: compute-bound
        dict(name="attend chunks", op="attend", r=16, q_lo=96, q_hi=2048, t_lo=64, t_hi=6000,
             hq=32, hkv=8, d=128, kb=4, vb=4, causal=1, dtype="bf16", lens=11),
        # cross attention of decoder tokens over encoder states of other lengths
        dict(name="attend encoder d64", op="attend", r=16, q_lo=1, q_hi=128, t_lo=300, t_hi=1500,
             hq=16, hkv=16, d=64, kb=4, vb=4, causal=0, dtype="bf16", lens=12),
    ]


def _log(rng, lo, hi):
    """An integer of lo..hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "store", "read", "attend", "attend"])
    lens = rng.randrange(1 << 30)
    hkv = rng.choice([1, 2, 4, 5, 8])
    g = rng.choice([1, 2, 3, 4, 5, 8])
    d = rng.choice([64, 128, 128])
    pairs = rng.choice(["half", "interleaved"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rope":
        return dict(op=op, n=_log(rng, 1, 5000), hq=hkv * g, hkv=hkv, d=d,
                    rot=rng.choice([d, d, d // 2]), pairs=pairs, norm=rng.randrange(2),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), lens=lens)
    kb, vb = rng.choice([(4, 2), (4, 4), (3, 3), (2, 2)])
    r = _log(rng, 1, 32)
    q_hi = _log(rng, 1, 9000 // r)
    q_lo = _log(rng, 1, q_hi)
    if op in ("store", "read"):
        t_hi = _log(rng, 1, 8192)
        return dict(op=op, r=r, q_lo=q_lo, q_hi=q_hi, t_lo=_log(rng, 1, t_hi), t_hi=t_hi, hkv=hkv,
                    d=d, kb=kb, vb=vb, dtype=dtype, lens=lens,
                    **(dict(pairs=pairs, norm=rng.randrange(2)) if op == "store" else {}))
    q_hi = min(q_hi, 1024, 4096 // r)
    q_lo = min(q_lo, q_hi)
    t_hi = _log(rng, 1, 60000 // r if q_hi * r <= 512 else 6000 // r)
    return dict(op=op, r=r, q_lo=q_lo, q_hi=q_hi, t_lo=_log(rng, 1, t_hi), t_hi=t_hi, hq=hkv * g,
                hkv=hkv, d=d, kb=kb, vb=vb, causal=rng.choice([1, 1, 0]), dtype="bf16", lens=lens)


def _lens(c):
    """(new tokens, tokens in the cache with the new ones) of each request.  With t_hi = 0 the
    cache holds nothing but the new tokens; a full (not causal) attention's queries are not in
    the cache."""
    rng = random.Random(c["lens"])
    q = [_log(rng, c["q_lo"], c["q_hi"]) for _ in range(c["r"])]
    t = [_log(rng, c["t_lo"], c["t_hi"]) if c["t_hi"] else 0 for _ in range(c["r"])]
    return (q, [a + b for a, b in zip(q, t)]) if c.get("causal", 1) else (q, t)


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


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    d = c["d"]
    if c["op"] in ("rope", "store"):
        s["cos_sin"] = _cos_sin(c.get("rot", d))
        s["w"] = 1 + 0.2 * _randn(gen, (2, d))
        s["w"] = s["w"].to(DTYPES[c["dtype"]])
    if c["op"] == "rope":
        n = c["n"]
        s["q"], s["k"] = (_heads(gen, n, c[h], d, c["dtype"]) for h in ("hq", "hkv"))
        # runs of consecutive positions, as flattened prompts and single tokens have
        first = torch.randint(0, MAX_POS - n, (1 + n // 512,), generator=gen, device=DEV)
        s["pos"] = first[torch.arange(n, device=DEV) // 512] + torch.arange(n, device=DEV) % 512
    else:
        qlen, tlen = _lens(c)
        r, hkv = c["r"], c["hkv"]
        s["q_start"] = _int32([sum(qlen[:i]) for i in range(r + 1)])
        s["seq_lens"] = _int32(tlen)
        s["max_q"], s["max_t"] = max(qlen), max(tlen)
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
        else:
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
            if c["op"] == "attend":
                s["q"] = _randn(gen, (n, c["hq"], d)).to(DTYPES[c["dtype"]])
    if own:
        _handles(s)
    return s


def _handles(s):
    """What a program that serves with the package keeps between calls: the layer's tables, the
    paged pool, the rotation table, the norms and the workspace; and a step's batch description,
    which all layers of the step share."""
    from bhaskera_col_b200.inference import ops
    c = s["case"]
    if "cos_sin" in s:
        s["rope"] = ops.RopeTable(s["cos_sin"], interleaved=c["pairs"] == "interleaved")
        s["norms"] = [ops.HeadNorm(w, eps=1e-6) if c["norm"] else None for w in s["w"]]
    if c["op"] != "rope":
        s["tables"] = ops.LayerTables(c["d"], c["kb"], c["vb"], False, s["kc"], s["kbnd"], s["vc"],
                                      s["vbnd"], s["R"])
        s["pages"] = ops.PagedPages(s["pool"], s["table"])
        s["batch"] = ops.RaggedBatch(s["q_start"], s["seq_lens"], s["max_q"])
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
                          k_norm=s["norms"][1])
    if c["op"] in ("store", "read"):
        shape = (s["n"], c["hkv"], c["d"])
        k, v = (torch.empty(shape, dtype=DTYPES[c["dtype"]], device=DEV) for _ in range(2))
        ops.dequantize_ragged(s["tables"], s["pages"], s["batch"], k, v)
        return {"k": k, "v": v}
    return {"out": ops.attend_ragged(s["tables"], s["pages"], s["q"], s["batch"],
                                     causal=bool(c["causal"]), workspace=s["workspace"])}


def _norm_rope(x, cos_sin, pairs, w):
    """RMS norm over the head (where w is given), then the rotation of its first dims."""
    if w is not None:
        x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
    half = cos_sin.shape[-1] // 2
    cos, sin = cos_sin[:, None, :half], cos_sin[:, None, half:]
    if pairs == "half":
        a, b = x[..., :half], x[..., half: 2 * half]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., 2 * half:]], -1)


def _tokens(s):
    """(request, position in it) of every flattened token; int64."""
    i = torch.arange(s["n"], device=DEV)
    r = (i[:, None] >= s["q_start"][None, 1:]).sum(-1)
    return r, i - s["q_start"][1:][r] + s["seq_lens"][r]


def _stored(x, R, cent, bnd):
    """What the cache gives back for x: the codes' centroids of the rotated unit vector, rotated
    back, times the norm in fp16."""
    n = x.square().sum(-1, keepdim=True).sqrt()
    y = (x / n.clamp_min(1e-8)) @ R.T
    return (cent[torch.bucketize(y, bnd)] @ R) * n.half().to(x.dtype)


def _run_plain(s):
    c = s["case"]
    dtype = DTYPES[c["dtype"]]
    if c["op"] == "rope":
        rows = s["cos_sin"][s["pos"]]
        return {x: _norm_rope(s[x].float(), rows, c["pairs"],
                              s["w"][i].float() if c["norm"] else None).to(dtype)
                for i, x in enumerate(("q", "k"))}
    if c["op"] == "store":
        # in 64 bits: a code turns over where the rotated value lies next to a boundary
        _, pos = _tokens(s)
        k = _norm_rope(s["k"].double(), s["cos_sin"][pos].double(), c["pairs"],
                       s["w"][1].double() if c["norm"] else None)
        R = s["R"].double()
        return {"k": _stored(k, R, s["kc"].double(), s["kbnd"].double()).to(dtype),
                "v": _stored(s["v"].double(), R, s["vc"].double(), s["vbnd"].double()).to(dtype)}
    k, v = _dense(s)
    if c["op"] == "read":
        r, pos = _tokens(s)
        return {"k": k[r, :, pos].to(dtype), "v": v[r, :, pos].to(dtype)}
    # queries padded to (r, hkv, g * max_q, d); scores of masked keys are -inf
    r, hkv, d, mq = c["r"], c["hkv"], c["d"], s["max_q"]
    g = c["hq"] // hkv
    req, pos = _tokens(s)
    slot = torch.arange(s["n"], device=DEV) - s["q_start"][req]
    q = torch.zeros((r, mq, hkv, g, d), device=DEV)
    q[req, slot] = s["q"].float().view(-1, hkv, g, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(r, hkv, g * mq, d)
    x = (q @ k.transpose(-1, -2)).view(r, hkv, g, mq, -1)
    x *= 1.0 / math.sqrt(d)
    key = torch.arange(k.shape[2], device=DEV)
    hide = key[None, None] >= s["seq_lens"][:, None, None]
    if c["causal"]:
        last = (s["seq_lens"] - s["q_start"].diff())[:, None] + torch.arange(mq, device=DEV)
        hide = hide | (key[None, None] > last[:, :, None])
    x.masked_fill_(hide[:, None, None], float("-inf"))
    x -= x.amax(-1, keepdim=True).clamp_min(-1e30)
    x.exp_()
    x /= x.sum(-1, keepdim=True).clamp_min(1e-30)
    o = (x.view(r, hkv, g * mq, -1) @ v).view(r, hkv, g, mq, d).permute(0, 3, 1, 2, 4)
    return {"out": o[req, slot].reshape(s["n"], c["hq"], d).to(dtype)}


def _dense(s, dt=torch.float32):
    """Every request's keys and values, (r, hkv, pages * 64, d), from the packed pages."""
    c = s["case"]
    d = c["d"]
    pg = s["pool"][s["table"].long()]                      # (r * hkv, pages, bytes)
    krow, vrow = d * c["kb"] // 8, d * c["vb"] // 8
    out = []
    for i, (off, row, bits, cent) in enumerate(((0, krow, c["kb"], s["kc"]),
                                                (PAGE * krow, vrow, c["vb"], s["vc"]))):
        code = _unpack(pg[..., off: off + PAGE * row].unflatten(-1, (PAGE, row)), d, bits)
        at = PAGE * (krow + vrow) + 2 * PAGE * i
        n = pg[..., at: at + 2 * PAGE].contiguous().view(torch.float16).to(dt)
        R = s["R"].to(dt)[_orders(d)[i]]                   # rows in the order of the codes
        x = (cent.to(dt)[code] @ R) * n.unsqueeze(-1)
        out.append(x.reshape(c["r"], c["hkv"], -1, d))
    return out


# --------------------------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    d = c["d"]
    if c["op"] == "rope":
        return {x: _exact_rope(s[x], s["cos_sin"], s["pos"], c, s["w"][i])
                for i, x in enumerate(("q", "k"))}
    qlen, tlen = _lens(c)
    if c["op"] == "store":
        pos = torch.cat([torch.arange(t - n, t, device=DEV) for n, t in zip(qlen, tlen)])
        out = {}
        for name, cent, bnd in (("k", s["kc"], s["kbnd"]), ("v", s["vc"], s["vbnd"])):
            x = s[name].double()
            if name == "k":
                x = _exact_rope(s["k"], s["cos_sin"], pos, c, s["w"][1])
            n = torch.linalg.vector_norm(x, dim=-1)
            y = torch.einsum("nhi,ji->nhj", x / n.clamp_min(1e-8)[..., None], s["R"].double())
            val = torch.zeros_like(y) + cent[0].double()
            for j in range(len(bnd)):                      # the highest boundary below y
                val = torch.where(y > bnd[j].double(), cent[j + 1].double(), val)
            out[name] = torch.einsum("nhj,ji,nh->nhi", val, s["R"].double(), n.half().double())
        return out
    ks, vs = [], []
    outs = []
    inv = [torch.tensor(o, device=DEV).argsort() for o in _orders(d)]
    krow, vrow = d * c["kb"] // 8, d * c["vb"] // 8
    for i, (n, t) in enumerate(zip(qlen, tlen)):
        pg = s["pool"][s["table"].view(c["r"], c["hkv"], -1)[i, :, : -(-t // PAGE)].long()]
        kv = []
        for w, (off, row, bits, cent) in enumerate(((0, krow, c["kb"], s["kc"]),
                                                    (PAGE * krow, vrow, c["vb"], s["vc"]))):
            rows = pg[..., off: off + PAGE * row].reshape(c["hkv"], -1, row).long()
            bit = torch.stack([(rows >> b) & 1 for b in range(8)], -1).reshape(*rows.shape[:2], -1)
            code = sum(bit[..., b::bits] << b for b in range(bits))[..., inv[w]]
            at = PAGE * (krow + vrow) + 2 * PAGE * w
            nrm = pg[..., at: at + 2 * PAGE].contiguous().view(torch.float16).reshape(c["hkv"], -1)
            x = cent.double()[code] * nrm.double()[..., None]
            kv.append(torch.einsum("htj,ji->hti", x, s["R"].double())[:, :t])
        k, v = kv
        if c["op"] == "read":
            ks.append(k[:, t - n:].transpose(0, 1))
            vs.append(v[:, t - n:].transpose(0, 1))
            continue
        a = sum(qlen[:i])
        q = s["q"][a: a + n].double()
        g = c["hq"] // c["hkv"]
        o = torch.empty_like(q)
        for h in range(c["hq"]):
            x = torch.einsum("nd,td->nt", q[:, h], k[h // g]) / math.sqrt(d)
            if c["causal"]:
                x = x + torch.full_like(x, float("-inf")).triu(t - n + 1)
            o[:, h] = torch.softmax(x, -1) @ v[h // g]
        outs.append(o)
    return {"out": torch.cat(outs)} if outs else {"k": torch.cat(ks), "v": torch.cat(vs)}


def _exact_rope(x, cos_sin, pos, c, w):
    """The rotation as a product of complex numbers."""
    x = x.double()
    if c["norm"]:
        x = x / (torch.sum(x * x, -1, keepdim=True) / c["d"] + 1e-6).sqrt() * w.double()
    rot = cos_sin.shape[1]
    turn = torch.complex(*cos_sin.double()[pos].split(rot // 2, -1))[:, None]
    y = x.clone()
    if c["pairs"] == "half":
        z = torch.complex(x[..., : rot // 2], x[..., rot // 2: rot]) * turn
        y[..., : rot // 2], y[..., rot // 2: rot] = z.real, z.imag
    else:
        z = torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous()) * turn
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


# --------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------
def work(case):
    c = case
    d, size = c["d"], 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "rope":
        rows, rot = c["n"] * (c["hq"] + c["hkv"]), c["rot"]
        # heads in and out, a table row and a position for each token
        return {"bytes": 2 * rows * d * size + c["n"] * (4 * rot + 8),
                "flops": rows * (3 * rot + (4 * d if c["norm"] else 0))}
    qlen, tlen = _lens(c)
    n, hkv, r = sum(qlen), c["hkv"], c["r"]
    packed = d * (c["kb"] + c["vb"]) // 8 + 4               # bytes of one token of one head
    plan = 8 * r + 4 + sum(4 * hkv * -(-t // PAGE) for t in tlen)
    if c["op"] in ("store", "read"):
        once = n * hkv * (packed + 2 * d * size)            # packed on one side, dense on the other
        turn = n * hkv * 2 * 2 * d * d                      # K and V through the rotation
        if c["op"] == "read":
            return {"bytes": once + plan, "flops": turn}
        return {"bytes": 2 * once + n * 4 * d + plan, "flops": 2 * turn}
    g = c["hq"] // hkv
    seen = sum(a * b - (a * (a - 1) // 2 if c["causal"] else 0) for a, b in zip(qlen, tlen))
    return {"bytes": sum(tlen) * hkv * packed + 2 * n * c["hq"] * d * size + plan,
            "flops": 4 * d * seen * g * hkv + 4 * n * c["hq"] * d * d}
