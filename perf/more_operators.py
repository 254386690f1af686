"""Cases for three operators over rows of logits: what they compute in plain torch, and what has to be moved for it.

* ``distill`` - the distillation loss of a student's logits against a teacher's top logits (and the mass that it
  leaves to all other tokens), with a share of the hard labels' cross entropy, and the gradient of the logits.
* ``top``     - a teacher's top logits in order, and the log-sum-exp of all others.
* ``sample``  - one token per row from a given uniform number, under temperature, top-k, top-p and min-p.

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
        # the answer of one short example: sixteen rows, where latency counts
        _distill("distill 16", rows=16, vocab=32000, k=16, temperature=1.0, hard=0.0, rest=False, ignored=0),
        # the training step's 4 x 2048 tokens, softened, with half of the hard labels' cross entropy
        _distill("distill train 8192", rows=8192, vocab=32000, k=64, temperature=2.0, hard=0.5, rest=True, ignored=0),
        # packed prompts and answers, the prompts ignored, an odd vocabulary
        _distill("distill answers 1003 fp16", rows=1003, vocab=50021, k=37, temperature=1.0, hard=0.0, rest=False,
                 ignored=301, dtype="fp16"),
        # a large vocabulary with logits in 32 bits
        _distill("distill 768x131072 fp32", rows=768, vocab=131072, k=128, temperature=1.5, hard=0.1, rest=True,
                 ignored=8, dtype="fp32"),
        # the loss of a validation batch: no gradient
        _distill("distill validation 4096", rows=4096, vocab=32000, k=64, temperature=1.0, hard=0.0, rest=True,
                 ignored=0, train=False),
        # the teacher's rows of one short example
        _top("top 16", rows=16, vocab=32000, k=16),
        # the teacher's rows of the training step
        _top("top 8192", rows=8192, vocab=32000, k=64, temperature=2.0),
        # an odd vocabulary in 32 bits with a long tail kept
        _top("top 999x50021 fp32", rows=999, vocab=50021, k=200, dtype="fp32"),
        # one conversation: latency
        _sample("sample 1", rows=1, vocab=32000),
        # a serving batch whose requests have settings of their own
        _sample("sample 64", rows=64, vocab=32000),
        # rollouts in a large vocabulary
        _sample("sample 512x131072", rows=512, vocab=131072),
        # an odd vocabulary in 32 bits
        _sample("sample 129x50021 fp32", rows=129, vocab=50021, dtype="fp32"),
    ]


def _distill(name, rows, vocab, k, temperature, hard, rest, ignored, dtype="bf16", train=True):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "k": k, "temperature": temperature,
            "hard": hard, "rest": rest, "ignored": ignored, "dtype": dtype, "train": train}


def _top(name, rows, vocab, k, temperature=1.0, dtype="bf16"):
    return {"name": name, "op": "top", "rows": rows, "vocab": vocab, "k": k, "temperature": temperature, "dtype": dtype}


def _sample(name, rows, vocab, dtype="bf16"):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype}


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["distill", "distill", "top", "sample", "sample"])
    vocab = rng.choice([_spread(rng, 1000, 131072), _spread(rng, 1000, 131072) // 8 * 8])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "sample":
        return _drawn(_sample("", _spread(rng, 1, min(512, 2 ** 26 // vocab)), vocab, dtype))
    most = 2 ** 27 // vocab  # half of the largest listed
    rows = _spread(rng, 1, min(8192, most))
    if op == "top":
        return _drawn(_top("", rows, vocab, _spread(rng, 1, 256), rng.choice([1.0, 0.7, 2.0]), dtype))
    return _drawn(_distill("", rows, vocab, _spread(rng, 1, 256), rng.choice([1.0, 1.0, 2.0, 1.3]),
                           rng.choice([0.0, 0.0, 0.3]), rng.random() < 0.5,
                           rng.choice([0, rows // 3]), dtype, rng.random() < 0.75))


def _drawn(case):
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------ inputs
def _logits(case, gen):
    """Rows from nearly flat (an untrained model) to peaked ones (a trained model)."""
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=gen, device="cuda")
    return x * (1 + 3.5 * torch.rand(rows, 1, generator=gen, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype, rows, vocab = _DTYPES[case["dtype"]], case["rows"], case["vocab"]
    s = dict(case)
    x = _logits(case, gen)
    if case["op"] == "top":
        s["logits"] = x.to(dtype)
    elif case["op"] == "sample":
        x[:, torch.randint(vocab, (3,), generator=gen, device="cuda")] = -math.inf  # tokens that are not allowed
        s["logits"] = x.to(dtype)

        def pick(values, kind=torch.float32):
            at = torch.randint(len(values), (rows,), generator=gen, device="cuda")
            return torch.tensor(values, device="cuda", dtype=kind)[at]

        s["uniform"] = torch.rand(rows, generator=gen, device="cuda")
        s["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3])
        s["top_k"] = pick([0, 0, 20, 50, 200], torch.int32)
        s["top_p"] = pick([1.0, 0.9, 0.95, 0.98])
        s["min_p"] = pick([0.0, 0.0, 0.02, 0.1])
    else:
        # a teacher that agrees with the student in part
        t = 0.7 * x + torch.randn(rows, vocab, generator=gen, device="cuda")
        t = t.to(dtype).float()
        values, ids = t.topk(case["k"], -1)
        s["values"], s["ids"] = values.to(dtype), ids.to(torch.int32)
        t.scatter_(1, ids, -math.inf)
        s["rest"] = torch.logsumexp(t / case["temperature"], -1) if case["rest"] else None
        s["target"] = torch.randint(vocab, (rows,), generator=gen, device="cuda")
        s["target"][torch.randperm(rows, generator=gen, device="cuda")[: case["ignored"]]] = -100
        s["logits"] = x.to(dtype).requires_grad_(case["train"])
        # the loss scale that keeps a mean's gradients inside the range of 16-bit floats
        s["scale"] = 2.0 ** round(math.log2(64 * rows)) if case["dtype"] == "fp16" else 1.0
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    if not own:
        with torch.no_grad():
            return {"distill": _plain_distill, "top": _plain_top, "sample": _plain_sample}[state["op"]](state)
    if state["op"] == "sample":
        from astrai_b200.inference.sample import sample_given

        token, logprob = sample_given(state["logits"], state["uniform"], temperature=state["temperature"],
                                      top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"],
                                      return_logprobs=True)
        return {"token": token, "logprob": logprob}
    from astrai_b200.ops.distill import TopLogits, distill_loss, top_logits

    if state["op"] == "top":
        top = top_logits(state["logits"], state["k"], temperature=state["temperature"])
        return {"ids": top.ids, "values": top.values, "rest": top.rest}
    scale = state["scale"]
    loss = distill_loss(state["logits"], TopLogits(state["ids"], state["values"], state["rest"]),
                        temperature=state["temperature"], target=state["target"], hard_weight=state["hard"],
                        expected_grad=scale)
    if not state["train"]:
        return {"loss": loss}
    grad = torch.autograd.grad(loss * scale if scale != 1 else loss, state["logits"])[0]
    return {"loss": loss.detach(), "dlogits": grad}


def _plain_distill(s):
    tau, hard = s["temperature"], s["hard"]
    ids, target = s["ids"].long(), s["target"]
    counted = target != -100
    n = counted.sum().clamp(min=1).float()
    label = torch.where(counted, target, 0)[:, None]
    x = s["logits"].float()
    z = x / tau
    z = z - z.amax(-1, keepdim=True)
    e = z.exp()
    total = e.sum(-1, keepdim=True)
    t = s["values"].float() / tau
    if s["rest"] is not None:
        t = torch.cat([t, s["rest"][:, None]], -1)
    t = t - t.amax(-1, keepdim=True)
    p = t.exp()
    mass = p.sum(-1, keepdim=True)
    logp, p = t - mass.log(), p / mass
    logq = z.gather(1, ids) - total.log()
    if s["rest"] is not None:
        others = e.scatter(1, ids, 0.0).sum(-1, keepdim=True)
        logq = torch.cat([logq, others.log() - total.log()], -1)
    row = (1 - hard) * tau ** 2 * (p * (logp - logq)).sum(-1)
    if hard:
        y = x - x.amax(-1, keepdim=True)
        f = y.exp()
        ftotal = f.sum(-1, keepdim=True)
        row = row + hard * (ftotal.log() - y.gather(1, label))[:, 0]
    loss = torch.where(counted, row, 0.0).sum() / n
    if not s["train"]:
        return {"loss": loss}
    scale = torch.where(counted, s["scale"] / n, 0.0)[:, None]
    k = s["k"]
    d = e * ((1 - p[:, k:] * total / others) / total) if s["rest"] is not None else e / total
    d.scatter_(1, ids, e.gather(1, ids) / total - p[:, :k])
    d.mul_((1 - hard) * tau)
    if hard:
        d.add_(f / ftotal, alpha=hard).scatter_add_(1, label, torch.full_like(scale, -hard))
    return {"loss": loss, "dlogits": d.mul_(scale).to(s["logits"].dtype)}


def _plain_top(s):
    x = s["logits"].float()
    values, ids = torch.sort(x, dim=-1, descending=True, stable=True)  # of equal logits, the lowest id first
    k = s["k"]
    most = values[:, k: k + 1].double() / s["temperature"]
    rest = most + (values[:, k:].double() / s["temperature"] - most).exp().sum(-1, keepdim=True).log()
    return {"ids": ids[:, :k].int(), "values": values[:, :k].to(s["logits"].dtype), "rest": rest[:, 0].float()}


def _plain_sample(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    greedy = s["temperature"] == 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    most = x.amax(-1, keepdim=True)
    w = ((x.double() - most.double()) / t).exp()  # 64 bits: a token's border may lie anywhere near the given number
    order = x.sort(-1, descending=True).values
    # top-k: not below the k-th largest value
    k = torch.where((s["top_k"] <= 0) | (s["top_k"] > vocab), vocab, s["top_k"]).long()[:, None]
    low = order.gather(1, k - 1)
    # top-p: the mass of all larger values, of what top-k kept, is not above p
    kept = torch.where(order >= low, ((order.double() - most.double()) / t).exp(), 0.0)
    before = torch.cat([torch.zeros_like(t), kept.cumsum(-1)], -1)
    first = torch.searchsorted(-order, -order)  # where this value begins
    p = torch.where(s["top_p"] >= 1, math.inf, s["top_p"].double())[:, None]
    inside = (before.gather(1, first) <= p * before[:, -1:]) & (order >= low)
    low = order.gather(1, inside.sum(-1, keepdim=True) - 1)
    # min-p: not below this share of the largest probability
    keep = (x >= low) & (w >= s["min_p"].double()[:, None])
    keep = keep & ~greedy[:, None]
    w = torch.where(greedy[:, None] | keep, w, 0.0)
    sums = w.cumsum(-1)
    z = sums[:, -1:]
    token = torch.searchsorted(sums, s["uniform"].double()[:, None] * z, right=True)
    best = (x == most).int().argmax(-1, keepdim=True)
    token = torch.where(greedy[:, None], best, token.clamp(max=vocab - 1))
    return {"token": token[:, 0], "logprob": (w.gather(1, token) / z).log()[:, 0].float()}


# ------------------------------------------------------------------------------------------ work
def work(case):
    rows, vocab, size = case["rows"], case["vocab"], _BYTES[case["dtype"]]
    if case["op"] == "sample":
        return {"bytes": rows * (vocab * size + 5 * 4 + 8 + 4), "flops": 4 * rows * vocab}
    if case["op"] == "top":
        return {"bytes": rows * (vocab * size + case["k"] * (4 + size) + 4), "flops": 4 * rows * vocab}
    counted = rows - case["ignored"]
    moved = counted * (vocab * size + case["k"] * (4 + size) + (4 if case["rest"] else 0)) + rows * 8 + 4
    terms = 8 if case["hard"] and case["temperature"] != 1 else 4
    if case["train"]:
        return {"bytes": moved + rows * vocab * size, "flops": 2 * terms * counted * vocab}
    return {"bytes": moved, "flops": terms * counted * vocab}


# ------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"distill": _exact_distill, "top": _exact_top, "sample": _exact_sample}[case["op"]](s)


def _exact_distill(s):
    """The loss as its definition says it, a few rows at a time, and autograd's gradient of it."""
    tau, counted = s["temperature"], s["target"] != -100
    n = max(1, int(counted.sum()))
    loss, grads = 0.0, []
    step = max(1, 2 ** 24 // s["vocab"])
    for a in range(0, s["rows"], step):
        rows = slice(a, a + step)
        x = s["logits"][rows].detach().double().requires_grad_(s["train"])
        ids, use = s["ids"][rows].long(), counted[rows].double()
        logq = torch.log_softmax(x / tau, -1)
        teacher, student = s["values"][rows].double() / tau, logq.gather(1, ids)
        if s["rest"] is not None:
            others = torch.ones_like(x, dtype=torch.bool).scatter(1, ids, False)
            teacher = torch.cat([teacher, s["rest"][rows].double()[:, None]], -1)
            student = torch.cat([student, logq.masked_fill(~others, -math.inf).logsumexp(-1, keepdim=True)], -1)
        logp = torch.log_softmax(teacher, -1)
        part = (1 - s["hard"]) * tau ** 2 * (logp.exp() * (logp - student)).sum(-1)
        if s["hard"]:
            label = s["target"][rows].clamp(min=0)[:, None]
            part = part - s["hard"] * torch.log_softmax(x, -1).gather(1, label)[:, 0]
        part = (part * use).sum() / n
        if s["train"]:
            grads += torch.autograd.grad(part * s["scale"], x)
        loss += part.detach()
    return {"loss": loss, "dlogits": torch.cat(grads)} if s["train"] else {"loss": loss}


def _exact_top(s):
    """One row after another: the largest taken by value, of equal ones the lowest id first."""
    ids, values, rest = [], [], []
    for row in s["logits"].double():
        bound = row.topk(s["k"]).values[-1]
        more = (row > bound).nonzero()[:, 0]
        more = more[row[more].argsort(descending=True, stable=True)]
        at = torch.cat([more, (row == bound).nonzero()[:, 0]])[: s["k"]]
        others = torch.ones_like(row, dtype=torch.bool)
        others[at] = False
        ids.append(at)
        values.append(row[at])
        rest.append(torch.logsumexp(row[others] / s["temperature"], 0))
    return {"ids": torch.stack(ids).int(), "values": torch.stack(values), "rest": torch.stack(rest)}


def _exact_sample(s):
    """One row after another, over its distinct values."""
    tokens, logprobs = [], []
    settings = zip(*(s[n].tolist() for n in ("uniform", "temperature", "top_k", "top_p", "min_p")))
    for row, (u, t, k, p, m) in zip(s["logits"].double(), settings):
        if t == 0:
            at = int((row == row.max()).nonzero()[0])
            tokens.append(at)
            logprobs.append(row[at] - torch.logsumexp(row, 0))
            continue
        value, count = torch.unique(row, return_counts=True)
        value, count = value.flip(0), count.flip(0)
        prob = torch.exp((value - value[0]) / t)
        if k > 0:
            prob = torch.where(count.cumsum(0) - count < k, prob, 0.0)
        mass = prob * count
        if p < 1:
            prob = torch.where(mass.cumsum(0) - mass <= p * mass.sum(), prob, 0.0)
        prob = torch.where(prob >= m, prob, 0.0)
        low = value[prob > 0][-1]
        at = (row >= low).nonzero()[:, 0]
        w = torch.exp((row[at] - value[0]) / t)
        sums = w.cumsum(0)
        i = min(int((sums <= u * sums[-1]).sum()), at.numel() - 1)
        tokens.append(int(at[i]))
        logprobs.append((w[i] / sums[-1]).log())
    return {"token": torch.tensor(tokens, device="cuda"), "logprob": torch.stack(logprobs)}
