"""Cases for three operators of attention layers: what they compute in plain torch, and what has to be moved for it.

* ``qk_norm_rope`` - RMS norm of every query and key head and the rotation of its positions, in one pass
  (norm after or before the rotation, interleaved or half layout, whole heads or a part), forward and backward.
* ``append``       - new keys and values quantised into a paged cache of 8-bit integers with one magnitude for
  each block of tokens and head, and read back from its pages.
* ``attend``       - causal attention of one or a few new tokens over such a cache.

``own`` false runs the plain forms, true the calls that a user makes.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a small serving batch: four rows, where only latency counts
        _rope("rope decode 4", rows=4, seq=0, hq=16, hkv=4, d=128, rot=128, layout="interleaved", norm="after"),
        # a prefill of 4 x 512 tokens at head size 64, half layout on half of each head
        _rope("rope prefill 2048", rows=2048, seq=512, hq=24, hkv=4, d=64, rot=32, layout="half", norm="before"),
        # the training step's 4 x 2048 tokens, forward and backward
        _rope("rope train 8192", rows=8192, seq=2048, hq=16, hkv=4, d=128, rot=128, layout="interleaved", norm="after",
              train=True),
        # an odd packed batch in 32 bits with as many key heads as query heads
        _rope("rope train 3003 fp32", rows=3003, seq=1001, hq=12, hkv=12, d=96, rot=64, layout="half", norm="before",
              train=True, dtype="fp32"),
        # one new token for each of 32 running requests, at lengths of their own
        _append("append decode 32", batch=32, new=1, start=3000, hkv=4, d=128, page=128, block=32, ragged=True),
        # a 512-token prefill behind a shared prefix, then the whole prefix read for the prefill attention
        _append("append prefill 4x512", batch=4, new=512, start=1536, hkv=4, d=128, page=128, block=32, ragged=False),
        # odd lengths that start inside a block and leave some rows shorter than others
        _append("append odd 5x77", batch=5, new=77, start=333, hkv=2, d=64, page=64, block=16, ragged=True, dtype="fp16"),
        # a single short conversation: latency
        _attend("attend 1x200", batch=1, new=1, length=200, hq=16, hkv=4, d=128, page=128, block=32, ragged=False),
        # a serving batch of 32 requests of 4096 tokens
        _attend("attend 32x4096", batch=32, new=1, length=4096, hq=16, hkv=4, d=128, page=128, block=32, ragged=False),
        # requests of very different lengths at head size 64, small pages
        _attend("attend 24 ragged", batch=24, new=1, length=16000, hq=24, hkv=4, d=64, page=64, block=16, ragged=True),
        # four proposed tokens verified at once for each of 8 requests
        _attend("attend 8x4 verify", batch=8, new=4, length=8191, hq=16, hkv=4, d=128, page=128, block=64, ragged=True),
        # four long documents
        _attend("attend 4x131072", batch=4, new=1, length=131072, hq=16, hkv=4, d=128, page=128, block=32, ragged=False),
    ]


def _rope(name, rows, seq, hq, hkv, d, rot, layout, norm, train=False, dtype="bf16"):
    return {"name": name, "op": "rope", "rows": rows, "seq": seq, "hq": hq, "hkv": hkv, "d": d, "rot": rot,
            "layout": layout, "norm": norm, "train": train, "dtype": dtype}


def _append(name, batch, new, start, hkv, d, page, block, ragged, dtype="bf16"):
    return {"name": name, "op": "append", "batch": batch, "new": new, "start": start, "hkv": hkv, "d": d, "page": page,
            "block": block, "ragged": ragged, "dtype": dtype}


def _attend(name, batch, new, length, hq, hkv, d, page, block, ragged, dtype="bf16"):
    return {"name": name, "op": "attend", "batch": batch, "new": new, "length": length, "hq": hq, "hkv": hkv, "d": d,
            "page": page, "block": block, "ragged": ragged, "dtype": dtype}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend"])
    if op == "rope":
        hq, hkv = rng.choice([(16, 4), (24, 4), (12, 12), (8, 1), (32, 8), (7, 7)])
        d = rng.choice([64, 96, 128, 192, 256])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        rows = _log(rng, 1, max(1, 8192 * 20 * 128 * 2 // ((hq + hkv) * d * _BYTES[dtype])))
        c = _rope("", rows=rows, seq=rng.choice([0, rng.randint(1, rows)]), hq=hq, hkv=hkv, d=d,
                  rot=rng.choice([d, d, d // 2, d // 2 + 16]), layout=rng.choice(["interleaved", "half"]),
                  norm=rng.choice(["after", "before", "none"]), train=rng.random() < 0.5, dtype=dtype)
    elif op == "append":
        page, block = rng.choice([(128, 32), (64, 16), (64, 64), (128, 128), (192, 64), (16, 16)])
        batch, new = _log(rng, 1, 64), _log(rng, 1, 1024)
        batch = max(1, min(batch, 4096 // new))
        c = _append("", batch=batch, new=new, start=_log(rng, 1, max(1, min(8192, 16384 // batch))) - 1,
                    hkv=rng.choice([1, 2, 4, 8]), d=rng.choice([64, 128]), page=page, block=block,
                    ragged=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    else:
        page, block = rng.choice([(128, 32), (64, 16), (64, 64), (128, 128), (192, 64), (16, 16)])
        hq, hkv = rng.choice([(16, 4), (24, 4), (8, 8), (8, 1), (32, 8), (32, 2), (7, 1)])
        d = rng.choice([64, 128])
        batch = _log(rng, 1, 64)
        most = 4 * 131072 * 4 * 128 // (batch * hkv * d)
        new = rng.choice([1, 1, 1, rng.randint(2, 8)])
        c = _attend("", batch=batch, new=new, length=_log(rng, new, min(131072, most)), hq=hq, hkv=hkv, d=d, page=page,
                    block=block, ragged=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _starts(case):
    """Cached tokens of each row before the call and after it. Ragged rows are spread evenly over the lengths up to
    the case's, in an order that looks like none, and appends of ragged rows leave the last ones shorter."""
    n, new = case["batch"], case["new"]
    top = case["start"] if case["op"] == "append" else case["length"] - new
    if not case["ragged"]:
        return [top] * n, [top + new] * n
    at = [(i * 7 + 3) % n if math.gcd(7, n) == 1 else (i * 11 + 3) % n if math.gcd(11, n) == 1 else i for i in range(n)]
    starts = [top * (a + 1) // n for a in at]
    if case["op"] == "append":
        return starts, [s + max(0, new - (i % 3)) for i, s in enumerate(starts)]
    return starts, [s + new for s in starts]


def _dequant(q, absmax, block):
    return q * (absmax / 127).repeat_interleave(block, dim=2)[..., None]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "rope":
        rows, d, h = case["rows"], case["d"], case["hq"] + case["hkv"]
        # projections of a normalised hidden state: unit scale with a spread of its own for each head
        x = _randn(g, rows, h, d) * torch.exp(0.3 * _randn(g, h, 1))
        width = h * d if case["train"] else (h + case["hkv"]) * d  # serving has the values behind the keys
        s["x"] = torch.zeros(rows, width, device="cuda", dtype=dt)
        s["x"][:, : h * d] = x.reshape(rows, -1).to(dt)
        s["wq"], s["wk"] = ((1 + 0.1 * _randn(g, d)).to(dt) for _ in range(2))
        top = max(4096, case["rows"])
        half = torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64)
        angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (-2 * half / case["rot"])
        s["table"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        if case["seq"]:  # rows of whole sequences from position 0
            s["pos"] = (torch.arange(rows, device="cuda") % case["seq"]).int()
        else:            # one token of each request
            s["pos"] = torch.randint(0, top, (rows,), device="cuda", generator=g).int()
        if case["train"]:
            s["dy"] = (_randn(g, rows, h * d) * 0.1).to(dt)
            for k in ("x", "wq", "wk"):
                s[k].requires_grad_()
        return s
    starts, lens = _starts(case)
    page, block, hkv, d = case["page"], case["block"], case["hkv"], case["d"]
    per = [max(1, -(-(a + case["new"]) // page)) for a in starts]
    n_pages, width = sum(per) + 3, max(per)
    for name in ("k", "v"):  # cached tokens: some channels of the keys are much larger than others
        spread = torch.exp((0.8 if name == "k" else 0.3) * _randn(g, hkv, 1, d))
        x = _randn(g, n_pages, hkv, page, d).mul_(spread).to(dt).float()
        a = x.view(n_pages, hkv, page // block, block * d).abs().amax(-1)
        x.view(n_pages, hkv, page // block, block, d).mul_((127 / a)[..., None, None]).round_()
        s[name + "c"], s[name + "a"] = x.to(torch.int8), a
    order = torch.randperm(n_pages, device="cuda", generator=g).int()  # a pool that has been in use for a while
    table = torch.full((case["batch"], width), -1, dtype=torch.int32)
    s["table"] = table.cuda()
    at = 0
    for i, n in enumerate(per):
        s["table"][i, :n] = order[at: at + n]
        at += n
    s["starts"] = torch.tensor(starts, dtype=torch.int32).cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
    s["longest"] = max(lens)
    if case["op"] == "append":
        buf = _randn(g, case["batch"], case["new"], 3, hkv, d)  # the projection's output: queries, keys, values
        buf[:, :, 1] *= torch.exp(0.8 * _randn(g, hkv, d))
        buf = buf.to(dt)
        s["k"], s["v"] = buf[:, :, 1], buf[:, :, 2]
        # read back: the touched blocks after a decode step, everything after a prefill chunk
        if case["new"] == 1:
            s["first"], s["count"] = (s["starts"] // block * block).int(), block
        else:
            s["first"], s["count"] = torch.zeros_like(s["starts"]), max(lens)
    else:
        s["q"] = _randn(g, case["batch"], case["new"], case["hq"], d).to(dt)
    return s


# ------------------------------------------------------------------------------------------ the plain forms
def _norm(x, w, eps=1e-6):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w


def _turn(x, table, pos, rot, layout):
    cs = table[pos.long()][:, None]
    c, s = cs[..., 0], cs[..., 1]
    part = x[..., :rot]
    if layout == "half":
        a, b = part[..., : rot // 2], part[..., rot // 2:]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rope(s):
    h, d = s["hq"] + s["hkv"], s["d"]
    x = s["x"][:, : h * d].float().view(-1, h, d)
    w = torch.cat([s["wq"].float().expand(s["hq"], d), s["wk"].float().expand(s["hkv"], d)])
    if s["norm"] == "before":
        x = _norm(x, w)
    x = _turn(x, s["table"], s["pos"], s["rot"], s["layout"])
    if s["norm"] == "after":
        x = _norm(x, w)
    return x.reshape(-1, h * d).to(s["x"].dtype)


def _plain_append_one(cache, absmax, new, s):
    """Every block that a row touches: its live tokens and the new ones under the larger magnitude."""
    block, page, n = s["block"], s["page"], s["new"]
    starts, lens = s["starts"].long(), s["lens"].long()
    first = starts // block
    blocks = first[:, None] + torch.arange((n - 1 + block - 1) // block + 1, device="cuda")
    pos = (blocks[..., None] * block + torch.arange(block, device="cuda")).flatten(1)
    where = blocks * block // page
    pages = s["table"].long().gather(1, where.clamp(max=s["table"].shape[1] - 1))
    ok = (pages >= 0) & (where < s["table"].shape[1]) & (blocks * block < lens[:, None]) & (lens > starts)[:, None]
    p, inside = pages.clamp(min=0), blocks % (page // block)
    old = cache.unflatten(2, (-1, block))[p, :, inside].float()       # [B, blocks, Hkv, block, D]
    was = absmax[p, :, inside]                                        # [B, blocks, Hkv]
    pos = pos.unflatten(1, (-1, block))
    live = (pos < starts[:, None, None])[:, :, None, :, None]
    fresh = ((pos >= starts[:, None, None]) & (pos < lens[:, None, None]))[:, :, None, :, None]
    take = (pos - starts[:, None, None]).clamp(0, n - 1)
    x = new.float()[torch.arange(len(starts), device="cuda")[:, None, None], take].transpose(2, 3)
    x = x.masked_fill(~fresh, 0)
    was = torch.where(blocks[:, :, None] * block < starts[:, None, None], was, 0)
    now = torch.maximum(was, x.abs().amax((-1, -2)))
    by = torch.where(now > 0, now, 1)[..., None, None]
    q = torch.where(live, torch.round(old * was[..., None, None] / by), torch.round(x * 127 / by)).clamp(-127, 127)
    q = torch.where(live | fresh, q, old).to(torch.int8)
    # a block past the row's end repeats the row's first one; a row without new tokens rewrites a block of its own as it is
    ok, some = ok[..., None], ok[:, :1]
    p0 = torch.where(some, p[:, :1], s["table"][:, :1].long())
    i0 = torch.where(some, inside[:, :1], 0)
    q0 = torch.where(some[..., None, None, None], q[:, :1], cache.unflatten(2, (-1, block))[p0, :, i0])
    a0 = torch.where(some[..., None], now[:, :1], absmax[p0, :, i0])
    p, inside = torch.where(ok[..., 0], p, p0), torch.where(ok[..., 0], inside, i0)
    cache.unflatten(2, (-1, block))[p, :, inside] = torch.where(ok[..., None, None], q, q0)
    absmax[p, :, inside] = torch.where(ok, now, a0)


def _plain_gather_one(cache, absmax, s):
    pos = s["first"].long()[:, None] + torch.arange(s["count"], device="cuda")
    where = pos // s["page"]
    pages = s["table"].long().gather(1, where.clamp(max=s["table"].shape[1] - 1))
    ok = (pages >= 0) & (where < s["table"].shape[1]) & (pos < s["lens"].long()[:, None])
    p, inside = pages.clamp(min=0), pos % s["page"]
    x = cache[p, :, inside].float() * (absmax[p, :, inside // s["block"]] / 127)[..., None]
    return x.masked_fill(~ok[..., None, None], 0).to(s["k"].dtype)


def _plain_attend(s):
    b, n, hq, d = s["q"].shape
    hkv, page = s["hkv"], s["page"]
    p = s["table"].long().clamp(min=0)
    k = _dequant(s["kc"].float(), s["ka"], s["block"])[p].transpose(1, 2).flatten(2, 3)  # [B, Hkv, tokens, D]
    q = s["q"].float().view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)              # [B, Hkv, G, S, D]
    score = q.flatten(2, 3) @ k.transpose(-1, -2) / math.sqrt(d)
    del k
    key = torch.arange(p.shape[1] * page, device="cuda")
    last = s["starts"].long()[:, None] + torch.arange(n, device="cuda")                  # each query's own position
    hidden = (key > last[..., None]).repeat(1, hq // hkv, 1)[:, None]
    weight = torch.exp(score.masked_fill(hidden, -math.inf) - score.masked_fill(hidden, -math.inf).amax(-1, True))
    v = _dequant(s["vc"].float(), s["va"], s["block"])[p].transpose(1, 2).flatten(2, 3)
    out = weight @ v / weight.sum(-1, keepdim=True)
    return out.unflatten(2, (-1, n)).permute(0, 3, 1, 2, 4).reshape(b, n, hq, d).to(s["q"].dtype)


def run(s):
    if s["op"] == "rope":
        if own:
            from astrai_b200.ops.qk_norm import qk_norm_rope

            w = (None, None) if s["norm"] == "none" else (s["wq"], s["wk"])
            y = qk_norm_rope(s["x"], s["hq"], s["hkv"], s["d"], s["table"], *w, positions=s["pos"], eps=1e-6,
                             layout=s["layout"], norm=s["norm"], rot_dim=s["rot"])
        else:
            y = _plain_rope(s)
        if not s["train"]:
            return {"y": y}
        wrt = (s["x"],) if s["norm"] == "none" else (s["x"], s["wq"], s["wk"])
        return dict(zip(("y", "dx", "dwq", "dwk"), (y.detach(),) + torch.autograd.grad(y, wrt, s["dy"])))
    if s["op"] == "append":
        if own:
            from astrai_b200.ops.kv8 import KV8, kv8_append, kv8_gather

            cache = KV8(s["kc"], s["vc"], s["ka"], s["va"])
            kv8_append(cache, s["k"], s["v"], s["table"], s["starts"], s["lens"])
            k, v = kv8_gather(cache, s["table"], s["lens"], s["count"], starts=s["first"], dtype=s["k"].dtype)
        else:
            _plain_append_one(s["kc"], s["ka"], s["k"], s)
            _plain_append_one(s["vc"], s["va"], s["v"], s)
            k, v = _plain_gather_one(s["kc"], s["ka"], s), _plain_gather_one(s["vc"], s["va"], s)
        return {"k": k, "v": v, "k_absmax": s["ka"], "v_absmax": s["va"]}
    if own:
        from astrai_b200.ops.kv8 import KV8, kv8_attention

        return {"o": kv8_attention(s["q"], KV8(s["kc"], s["vc"], s["ka"], s["va"]), s["table"], s["lens"])}
    return {"o": _plain_attend(s)}


# ------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
    if case["op"] == "rope":
        d, b = case["d"], _BYTES[case["dtype"]]
        heads = case["rows"] * (case["hq"] + case["hkv"])
        cs = min(case["rows"], case["seq"] or case["rows"]) * case["rot"] * 4  # each (cos, sin) row that is used, once
        moved = heads * d * b * 2 + cs + case["rows"] * 4 + 2 * d * b
        flops = heads * (3 * case["rot"] + (0 if case["norm"] == "none" else 4 * d))
        if case["train"]:  # backward: the gradient and the input in, the input's gradient out
            moved += heads * d * b * 3 + cs + 4 * d * b
            flops += heads * (3 * case["rot"] + (0 if case["norm"] == "none" else 10 * d))
        return {"bytes": moved, "flops": flops}
    starts, lens = _starts(case)
    hkv, d, block = case["hkv"], case["d"], case["block"]
    if case["op"] == "append":
        new = sum(e - a for a, e in zip(starts, lens))
        touched = sum(-(-e // block) - a // block for a, e in zip(starts, lens) if e > a)
        read = sum(min(e, a // block * block + block) - a // block * block if case["new"] == 1 else e
                   for a, e in zip(starts, lens))
        rows = len(starts) * (block if case["new"] == 1 else max(lens))
        # new tokens in and quantised; the cache read back and written out in the input's type; the magnitudes
        moved = new * d * 2 * (2 + 1) + read * d * 2 + rows * d * 2 * 2 + touched * 2 * 8
        return {"bytes": hkv * moved, "flops": hkv * d * 2 * (3 * new + read)}
    tokens, rows = sum(lens), case["batch"] * case["new"] * case["hq"]
    blocks = sum(-(-e // block) for e in lens)
    seen = sum(e - case["new"] + (case["new"] + 1) / 2 for e in lens)  # keys that a query sees, on average
    return {"bytes": hkv * (tokens * 2 * d + blocks * 8) + rows * d * 4,
            "flops": int(4 * seen * case["new"] * case["hq"] * d)}


# ------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rope": _exact_rope, "append": _exact_append, "attend": _exact_attend}[case["op"]](s)


def _exact_rope(s):
    """The rotation as a complex product, and the gradients from the formulas."""
    hq, h, d, rot = s["hq"], s["hq"] + s["hkv"], s["d"], s["rot"]
    angle = torch.complex(*s["table"][s["pos"].long()].double().unbind(-1))[:, None]

    def rotate(t, by):
        part = t[..., :rot]
        z = (torch.complex(part[..., : rot // 2].contiguous(), part[..., rot // 2:].contiguous()) if s["layout"] == "half"
             else torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous())) * by
        back = torch.cat([z.real, z.imag], -1) if s["layout"] == "half" else torch.view_as_real(z).flatten(-2)
        return torch.cat([back, t[..., rot:]], -1)

    x = s["x"].detach()[:, : h * d].double().view(-1, h, d)
    w = torch.empty(h, d, dtype=torch.float64, device=x.device)
    w[:hq], w[hq:] = s["wq"].detach().double(), s["wk"].detach().double()
    inner = x if s["norm"] == "before" else rotate(x, angle)  # what the norm sees
    r = (inner.square().sum(-1, keepdim=True) / d + 1e-6) ** -0.5
    y = {"none": inner, "after": inner * r * w, "before": rotate(inner * r * w, angle)}[s["norm"]]
    out = {"y": y.reshape(-1, h * d)}
    if not s["train"]:
        return out
    g = s["dy"].double().view(-1, h, d)
    if s["norm"] == "none":
        return {**out, "dx": rotate(g, angle.conj()).reshape(-1, h * d)}
    if s["norm"] == "before":
        g = rotate(g, angle.conj())
    unit = inner * r
    dw = (g * unit).sum(0)
    g = g * w
    dx = (g - unit * (g * unit).sum(-1, keepdim=True) / d) * r
    if s["norm"] == "after":
        dx = rotate(dx, angle.conj())
    return {**out, "dx": dx.reshape(-1, h * d), "dwq": dw[:hq].sum(0), "dwk": dw[hq:].sum(0)}


def _exact_append(s):
    """Row by row, block by block, as the definition says it."""
    page, block = s["page"], s["block"]
    table, starts, lens, first = (s[n].tolist() for n in ("table", "starts", "lens", "first"))
    out = {}
    for name in ("k", "v"):
        cache, absmax, new = s[name + "c"].double(), s[name + "a"].double(), s[name].double()
        got = torch.zeros(len(starts), s["count"], s["hkv"], s["d"], dtype=torch.float64, device=new.device)
        for b, (a, e) in enumerate(zip(starts, lens)):
            for at in range(a // block * block, e if e > a else 0, block):
                p, o, i = table[b][at // page], at % page, at % page // block
                kept, end = max(0, a - at), min(e - at, block)
                x = new[b, at + kept - a: at + end - a].transpose(0, 1)  # [Hkv, tokens, D]
                most = x.abs().amax((1, 2))
                was = absmax[p, :, i].clone() if kept else torch.zeros_like(most)
                now = torch.maximum(was, most)
                by = torch.where(now > 0, now, 1)[:, None, None]
                cache[p, :, o: o + kept] = torch.round(cache[p, :, o: o + kept] * was[:, None, None] / by)
                cache[p, :, o + kept: o + end] = torch.round(127 * x / by)
                absmax[p, :, i] = now
            for at in range(first[b], min(e, first[b] + s["count"]), block):
                p, o, end = table[b][at // page], at % page, min(block, e - at, first[b] + s["count"] - at)
                value = cache[p, :, o: o + end] * absmax[p, :, o // block, None, None] / 127
                got[b, at - first[b]: at - first[b] + end] = value.transpose(0, 1)
        out[name], out[name + "_absmax"] = got, absmax
    return out


def _exact_attend(s):
    page, block, d = s["page"], s["block"], s["d"]
    b, n, hq, _ = s["q"].shape
    out = torch.zeros(b, n, hq, d, dtype=torch.float64, device=s["q"].device)
    for i, e in enumerate(s["lens"].tolist()):
        pages = s["table"][i, : -(-e // page)].long()
        k, v = (s[c][pages].double().unflatten(2, (-1, block)) * s[a][pages].double()[..., None, None] / 127
                for c, a in (("kc", "ka"), ("vc", "va")))
        k, v = (t.flatten(2, 3).transpose(0, 1).flatten(1, 2)[:, :e] for t in (k, v))  # [Hkv, tokens, D]
        for j in range(n):
            m = e - n + j + 1  # keys that this query sees
            q = s["q"][i, j].double().view(s["hkv"], -1, d)
            p = torch.softmax(q @ k[:, :m].transpose(1, 2) / d ** 0.5, -1)
            out[i, j] = (p @ v[:, :m]).reshape(hq, d)
    return {"o": out}
