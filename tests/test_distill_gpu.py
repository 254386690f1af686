"""The distillation kernel against its formulas in 64 bits.

Tolerances. A weight 2^t with t from one fp32 fused multiply-add is off by at most |t| 2^-24 ln 2 from the rounding of
the factor, as much from that of the result, and 2^-22 from the exponential: below 2^-16 for all |t| <= 126, beyond
which it is zero. A sum over a row has terms of one sign and adds at most 64 of them in a thread, 16 over the CTA and 16
over a cluster: 2^-17 of it. Half of 2^-15 covers both, and 2^-15 of the magnitudes that a gradient is the difference of
covers a quotient of two. The result is rounded once to its type: half a spacing, at least that of its subnormals. The
logarithms in the loss turn those relative errors into absolute ones, so its magnitudes count one for each.
"""

import math

import pytest
import torch

from tests.distill_oracle import oracle

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: (2.0 ** -8, 2.0 ** -126), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.float32: (2.0 ** -24, 2.0 ** -126)}


@pytest.fixture(autouse=True)
def _clean_error_word():
    from astrai_b200.ops._ext import native

    native().read_error()
    yield
    torch.cuda.synchronize()
    assert native().read_error() == 0


def _inputs(rows, V, K, dtype=torch.bfloat16, tau=1.0, rest=True, labels=True, seed=0, sigma=3.0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = (torch.randn(rows, V, generator=g, device="cuda") * sigma).to(dtype)
    t = (0.7 * x.float() + torch.randn(rows, V, generator=g, device="cuda")).to(dtype)
    values, ids = t.float().topk(K, -1)
    r = torch.logsumexp(t.float().scatter(1, ids, -math.inf) / tau, -1) if rest else None
    y = torch.randint(V, (rows,), generator=g, device="cuda") if labels else None
    return x, ids.int(), values.to(dtype), r, y


def _check(x, ids, values, rest, tau=1.0, target=None, hard=0.0, upstream=1.0, expected=1.0, got=None):
    from astrai_b200.ops.distill import TopLogits, distill_loss

    if got is None:
        leaf = x.detach().requires_grad_()
        loss = distill_loss(leaf, TopLogits(ids, values, rest), tau, target, hard, expected_grad=expected)
        (dx,) = torch.autograd.grad(loss, leaf, torch.full_like(loss, upstream))
        got = loss.detach(), dx
    want, want_dx, size, dsize = oracle(x, ids, values, rest, tau, target, hard, upstream=upstream)
    assert got[0].dtype == torch.float32 and got[0].dim() == 0 and got[1].dtype == x.dtype and got[1].shape == x.shape
    assert abs(float(got[0]) - want) <= 2.0 ** -15 * size + 2.0 ** -24 * abs(want), (float(got[0]), want)
    half, least = HALF[x.dtype]
    error = (got[1].double().cpu() - want_dx).abs()
    worst = (error - 2.0 ** -15 * dsize - half * want_dx.abs() - least).max()
    assert worst <= 0, float(worst)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,V,K", [(1, 1, 1), (2, 7, 3), (3, 8, 8), (5, 100, 100), (4, 1000, 1), (3, 4097, 16),
                                      (2, 8193, 513), (3, 16385, 64), (2, 32000, 1024), (2, 33000, 37), (1, 70001, 256),
                                      (1, 131072, 64)])
def test_sizes(dtype, rows, V, K):
    up = 64.0 if dtype == torch.float16 else 1.0
    _check(*_inputs(rows, V, K, dtype, rest=K < V)[:4], upstream=up, expected=up)


@pytest.mark.parametrize("tau", [0.5, 1.0, 2.0, 3.7])
@pytest.mark.parametrize("hard", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("rest", [False, True])
def test_options(tau, hard, rest):
    for V in (1001, 40000):
        x, ids, values, r, y = _inputs(4, V, 20, tau=tau, rest=rest, seed=3)
        y[1] = -100
        y[2] = ids[2, 5]  # a label among the teacher's tokens
        _check(x, ids, values, r, tau, y, hard)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1003, 33333])
def test_masked_and_repeated_entries(dtype, V):
    x, ids, values, rest, y = _inputs(12, V, 12, dtype, rest=True, seed=5)
    x[:, -7:] = -math.inf                # the student's padding of the vocabulary
    y = y % (V - 7)
    ids[0, 3] = -1                       # no entry
    ids[1, 4:] = V + 5
    ids[2] = -1                          # only the rest
    ids[3] = -1
    rest[3] = -math.inf                  # nothing at all
    values[4, 2:5] = -math.inf           # entries without mass
    ids[5, 1] = ids[5, 0]                # the same id twice
    ids[6, :] = ids[6, 0]                # always the same
    ids[7, 0] = V - 1                    # a masked token of the student: no mass of the teacher there
    values[7, 0] = -math.inf
    rest[8] = -math.inf                  # all of the teacher's mass is on its entries
    x[9].fill_(-math.inf)                # the student allows only the teacher's tokens
    x[9, ids[9].long()] = 1.5
    rest[9] = -math.inf
    y[9] = ids[9, 0]
    x[10] = 0                            # a flat student
    x[11] *= 20                          # a peaked one
    for hard in (0.0, 0.25):
        for tau in (1.0, 2.0):
            _check(x, ids.long() if tau == 2 else ids, values, rest, tau, y, hard)


def test_teacher_on_a_masked_token_costs_infinity():
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, _ = _inputs(2, 500, 4)
    x[1, ids[1, 2].long()] = -math.inf
    leaf = x.requires_grad_()
    loss = distill_loss(leaf, TopLogits(ids, values, rest))
    (dx,) = torch.autograd.grad(loss, leaf)
    assert loss == math.inf and torch.isfinite(dx.float()).all()


@pytest.mark.parametrize("where", ["student", "teacher", "rest"])
def test_nan_reaches_the_loss(where):
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, _ = _inputs(3, 9000, 4)
    {"student": x[1], "teacher": values[1], "rest": rest[1:2]}[where][0] = math.nan
    leaf = x.requires_grad_()
    loss = distill_loss(leaf, TopLogits(ids, values, rest))
    (dx,) = torch.autograd.grad(loss, leaf)
    assert loss.isnan() and dx[1].isnan().any() and torch.isfinite(dx[[0, 2]].float()).all()


def test_far_masses_do_not_overflow():
    """The teacher's tokens hundreds above or below all others, at either temperature."""
    for shift in (300.0, -300.0):
        for V in (600, 50000):
            x, ids, values, rest, y = _inputs(2, V, 6, torch.float32, tau=2.0)
            x.scatter_add_(1, ids.long(), torch.full(ids.shape, shift, device="cuda"))
            y[0] = ids[0, 0]
            _check(x, ids, values, rest, 2.0, y, 0.5)
            _check(x, ids, values, None, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_and_offset_logits(dtype):
    x, ids, values, rest, y = _inputs(6, 1001, 9, dtype)
    for pad, off in ((3, 0), (7, 5), (23, 1)):
        wide = torch.full((6, 1001 + pad + off), math.nan, dtype=dtype, device="cuda")
        view = wide[:, off: off + 1001]
        view.copy_(x)
        _, dx = _check(view, ids, values, rest, 1.0, y, 0.2)
    # every second row, a transposed layout, one row for all
    double = x.repeat_interleave(2, 0)
    _check(double[::2], ids, values, rest, 1.0, y, 0.2)
    _check(x.t().contiguous().t(), ids, values, rest, 1.0, y, 0.2)
    one = x[:1].expand(6, -1)
    _check(one, ids, values, rest, 1.0, y, 0.2)
    # the teacher's tensors too
    _check(x, ids.t().contiguous().t(), values.repeat_interleave(2, 1)[:, ::2], rest.repeat_interleave(2)[::2], 1.0,
           y.repeat_interleave(2)[::2].int(), 0.2)


def test_batch_dimensions():
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, y = _inputs(12, 777, 5)
    shaped = x.view(3, 4, 777).detach().requires_grad_()
    loss = distill_loss(shaped, TopLogits(ids.view(3, 4, 5), values.view(3, 4, 5), rest.view(3, 4)), 1.0, y.view(3, 4), 0.5)
    (dx,) = torch.autograd.grad(loss, shaped)
    assert dx.shape == shaped.shape
    _check(x, ids, values, rest, 1.0, y, 0.5, got=(loss.detach(), dx.view(12, 777)))
    # the positions but the last of each sequence, as a next-token loss takes them
    part = shaped[:, :-1]
    loss = distill_loss(part, TopLogits(ids.view(3, 4, 5)[:, :-1], values.view(3, 4, 5)[:, :-1], rest.view(3, 4)[:, :-1]))
    (dx,) = torch.autograd.grad(loss, shaped)
    assert (dx[:, -1] == 0).all()
    keep = torch.arange(12, device="cuda").view(3, 4)[:, :-1].flatten()
    _check(x[keep], ids[keep], values[keep], rest[keep], got=(loss.detach(), dx[:, :-1].reshape(9, 777)))
    one = x[0].detach().requires_grad_()
    loss = distill_loss(one, TopLogits(ids[0], values[0], rest[0]))
    (dx,) = torch.autograd.grad(loss, one)
    _check(x[:1], ids[:1], values[:1], rest[:1], got=(loss.detach(), dx[None]))


def test_no_position_counts():
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, y = _inputs(3, 200, 4)
    leaf = x.requires_grad_()
    loss = distill_loss(leaf, TopLogits(ids, values, rest), target=torch.full_like(y, -100))
    (dx,) = torch.autograd.grad(loss, leaf)
    assert loss == 0 and (dx == 0).all()
    none = x.detach()[:0].requires_grad_()
    loss = distill_loss(none, TopLogits(ids[:0], values[:0], rest[:0]))
    (dx,) = torch.autograd.grad(loss, none)
    assert loss == 0 and dx.shape == (0, 200)


@pytest.mark.parametrize("upstream,expected", [(1.0, 1.0), (0.25, 0.25), (1 / 3, 1 / 3), (0.7, 1.0), (-2.0, 1.0), (0.0, 1.0)])
def test_upstream_gradients(upstream, expected):
    for V in (3001, 40001):
        x, ids, values, rest, y = _inputs(4, V, 7, seed=9)
        _check(x, ids, values, rest, 1.5, y, 0.1, upstream, expected)


def test_retained_graph_and_accumulation():
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, y = _inputs(4, 2000, 7, torch.float32)
    leaf = x.requires_grad_()
    loss = distill_loss(leaf, TopLogits(ids, values, rest))
    (a,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    kept = a.clone()
    a.zero_()  # the gradient is its receiver's
    (b,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (c,) = torch.autograd.grad(3 * loss, leaf)
    assert torch.equal(kept, b) and (c - 3 * b).abs().max() <= 2.0 ** -22 * (3 * b).abs().max()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, leaf)
    first, second = (distill_loss(leaf, TopLogits(ids, values, r)) for r in (rest, None))
    (first + second).backward()
    (d,) = torch.autograd.grad(distill_loss(leaf, TopLogits(ids, values, None)), leaf)
    assert (leaf.grad - (b + d)).abs().max() <= 2.0 ** -23 * (b.abs() + d.abs()).max()


def test_without_gradient_and_deterministic():
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, y = _inputs(64, 32000, 50)
    ids[:, 7] = ids[:, 3]
    top = TopLogits(ids, values, rest)
    plain = distill_loss(x, top, 2.0, y, 0.4)
    assert not plain.requires_grad
    leaf = x.detach().requires_grad_()
    with torch.no_grad():
        assert torch.equal(distill_loss(leaf, top, 2.0, y, 0.4), plain)
    seen = []
    for _ in range(5):
        loss = distill_loss(leaf, top, 2.0, y, 0.4)
        seen.append((loss.detach(), torch.autograd.grad(loss, leaf)[0]))
    assert all(torch.equal(loss, plain) and torch.equal(dx, seen[0][1]) for loss, dx in seen)


def test_changed_inputs_are_noticed():
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, _ = _inputs(3, 300, 4)
    leaf = x.requires_grad_()
    y = leaf * 1
    loss = distill_loss(y, TopLogits(ids, values, rest))
    y.data.zero_()  # not seen by autograd: the gradient of the forward's values stays right
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()


def test_second_derivative_and_tangents_are_refused():
    from torch.autograd import forward_ad

    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, _ = _inputs(3, 300, 4)
    leaf = x.requires_grad_()
    top = TopLogits(ids, values, rest)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(distill_loss(leaf, top), leaf, create_graph=True)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            distill_loss(forward_ad.make_dual(x.detach(), torch.ones_like(x)), top)
    with pytest.raises(RuntimeError, match="gradient of the teacher"):
        distill_loss(leaf, TopLogits(ids, values.detach().requires_grad_(), rest))


def test_captured_forward_and_backward():
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, y = _inputs(5, 5000, 9)
    other = _inputs(5, 5000, 9, seed=1)
    static = [t.clone() for t in (x, ids, values, rest, y)]
    side = torch.cuda.Stream()

    def step(expected):
        leaf = static[0].detach().requires_grad_()
        loss = distill_loss(leaf, TopLogits(*static[1:4]), 2.0, static[4], 0.5, expected_grad=expected)
        return loss.detach(), torch.autograd.grad(0.5 * loss, leaf)[0]

    graphs = []
    for expected in (0.5, 1.0):  # handed out, and computed again
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(expected)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(expected)
        graphs.append((g, out))
    for inputs in ((x, ids, values, rest, y), other):
        for t, new in zip(static, inputs):
            t.copy_(new)
        for g, out in graphs:
            g.replay()
            _check(*inputs[:4], 2.0, inputs[4], 0.5, 0.5, got=out)


def test_on_another_stream():
    side = torch.cuda.Stream()
    x, ids, values, rest, y = _inputs(8, 40000, 9)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _check(x, ids, values, rest, 2.0, y, 0.5)
    side.synchronize()
    _check(x, ids, values, rest, 2.0, y, 0.5, got=got)


def test_refusals():
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, y = _inputs(3, 300, 4)
    ok = TopLogits(ids, values, rest)
    for bad in (dict(teacher=TopLogits(ids[:2], values[:2], rest)), dict(teacher=TopLogits(ids, values[:, :3], rest)),
                dict(teacher=TopLogits(ids, values, rest[:2])), dict(temperature=0.0), dict(temperature=-1.0),
                dict(temperature=math.inf), dict(hard_weight=0.5), dict(hard_weight=1.5, target=y),
                dict(target=y[:2]), dict(teacher=TopLogits(ids.repeat(1, 300), values.repeat(1, 300), rest))):
        with pytest.raises(ValueError):
            distill_loss(**{"logits": x, "teacher": ok, **bad})
    for bad in (dict(logits=x.double()), dict(teacher=TopLogits(ids.float(), values, rest)),
                dict(teacher=TopLogits(ids, values.double(), rest)), dict(teacher=TopLogits(ids, values, rest.half())),
                dict(teacher=TopLogits(ids.cpu(), values, rest)), dict(target=y.float()), dict(target=y.cpu())):
        with pytest.raises(RuntimeError):
            distill_loss(**{"logits": x, "teacher": ok, **bad})
    big = torch.zeros(1, 300000, device="cuda")
    with pytest.raises(ValueError, match="too large"):
        distill_loss(big, TopLogits(ids[:1], values[:1], rest[:1]))


# The largest distance in base-2 exponents that a weight is taken at is 126, beyond it the weight is zero. Where the exponent
# comes from a subtraction and a product with a rounded factor, it is off by three roundings: 3 * 126 * ln 2 * 2^-24 + 2^-22 =
# 1.59e-5 of a weight, and a sum of at most 100 terms one after another by 100 * 2^-24 = 6e-6 more: 2^-15 = 3.05e-5 still
# covers both together.
@pytest.mark.parametrize("V,dtype,parts", [(50000, torch.float32, 4), (131072, torch.bfloat16, 4), (40000, torch.bfloat16, 2)])
@pytest.mark.parametrize("low", [-60.0, -100.0, -1e4, "least"])
def test_parts_of_a_row_far_below_the_others(V, dtype, parts, low):
    """Each part of a row in turn masked with a large finite number: all that one CTA of a cluster has."""
    value = torch.finfo(dtype).min if low == "least" else low
    x, ids, values, _, y = _inputs(4, V, 24, dtype, labels=True, seed=11)
    size = V // parts
    for r in range(4):
        at = r % parts * size
        masked = slice(max(at - 16, 0), min(at + size + 16, V))  # the parts end on a vector
        other = (r + 1) % parts * size + 100
        if low == "least":
            x[r, masked] = value
        else:
            x[r, masked] += value
        ids[r, :4] = torch.arange(4, device="cuda") + at     # of the teacher's tokens, some lie there
        ids[r, 4:] = torch.arange(20, device="cuda") + other  # and some parts have none
        if low == "least":
            values[r, :4] = -math.inf  # with mass there the loss would be 1e38
            y[r] = ids[r, 5] + 100 * (r % 2)
    rest = torch.randn(4, device="cuda")
    for tau, hard in ((1.0, 0.0), (2.0, 0.3), (0.5, 0.3), (1.0, 0.3)):
        _check(x, ids, values, rest, tau, y, hard)
        _check(x, ids, values, None, tau, y, hard)


@pytest.mark.parametrize("high", [150.0, 1e4])
def test_parts_of_a_row_far_above_the_others(high):
    x, ids, values, rest, y = _inputs(8, 50000, 24, torch.float32, seed=12)
    for r in range(8):
        x[r, r * 6250: (r + 1) * 6250] += high
    for tau in (1.0, 2.0):
        _check(x, ids, values, rest, tau, y, 0.4)


@pytest.mark.parametrize("V,dtype", [(600, torch.float32), (9000, torch.bfloat16), (50000, torch.float32)])
@pytest.mark.parametrize("low", [-1e3, -1e5, "least"])
def test_all_others_far_below_the_teachers_tokens(V, dtype, low):
    """Every token but the teacher's masked with a large finite number: the label's part is the difference of two logits near
    each other, whatever lies between them and the others."""
    x, ids, values, _, y = _inputs(3, V, 24, dtype, seed=13)
    x = torch.full_like(x, torch.finfo(dtype).min if low == "least" else low).scatter_(1, ids.long(), values)
    y[:] = ids[:, 3].long()
    rest = torch.full((3,), -20.0, device="cuda")
    rest[1] = -math.inf
    for tau, hard in ((1.0, 0.0), (2.0, 0.3), (1.0, 0.5), (2.0, 1.0)):
        _check(x, ids, values, rest, tau, y, hard)
        _check(x, ids, values, None, tau, y, hard)


@pytest.mark.parametrize("V,dtype", [(600, torch.float32), (9000, torch.bfloat16), (50000, torch.float32)])
def test_teachers_tokens_far_below_all_others(V, dtype):
    x, ids, values, rest, y = _inputs(3, V, 24, dtype, seed=14)
    x.scatter_add_(1, ids.long(), torch.full(ids.shape, -1e5, device="cuda", dtype=dtype))
    y[0] = ids[0, 3]
    for tau, hard in ((1.0, 0.0), (2.0, 0.3), (1.0, 0.5)):
        _check(x, ids, values, rest, tau, y, hard)


@pytest.mark.parametrize("rows,V,part", [(4096, 17500, 128), (256, 130000, 16)])
def test_many_rows_in_turn_on_clusters(rows, V, part):
    """Rows that follow each other on a cluster give what they give in calls in which each cluster has one."""
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, y = _inputs(rows, V, 2, torch.float32, seed=15)
    y[::8] = -100  # as many in each part, so that the means' factors are the same numbers

    def gradient(at, upstream):
        leaf = x[at].detach().requires_grad_()
        loss = distill_loss(leaf, TopLogits(ids[at], values[at], rest[at]), 1.0, y[at], expected_grad=upstream)
        return torch.autograd.grad(loss, leaf, torch.full_like(loss, upstream))[0]

    for _ in range(3):
        together = gradient(slice(0, rows), 1.0)
        for i in range(0, rows, part):
            assert torch.equal(together[i: i + part], gradient(slice(i, i + part), part / rows))


def test_forward_and_backward_on_two_sides_of_a_capture():
    """The gradient that the forward leaves belongs to its own run: a captured backward writes its gradient at every replay,
    and an eager backward does not take what a captured forward has yet to write."""
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, rest, y = _inputs(5, 5000, 9)
    top = TopLogits(ids, values, rest)
    base = x.detach().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        logits = base * 1
        one = torch.ones((), device="cuda")
        loss = distill_loss(logits, top, 2.0, y, 0.5)
        other = distill_loss(logits, top, 2.0, y, 0.5)
        torch.autograd.grad(other, logits, one, retain_graph=True)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            (dx,) = torch.autograd.grad(loss, logits, one, retain_graph=True)
        for _ in range(2):
            dx.zero_()
            g.replay()
            _check(x, ids, values, rest, 2.0, y, 0.5, got=(loss.detach(), dx))
        later = torch.cuda.CUDAGraph()
        with torch.cuda.graph(later, stream=side):
            captured = distill_loss(logits, top, 2.0, y, 0.5)
        (dx,) = torch.autograd.grad(captured, logits, one)
        later.replay()
        _check(x, ids, values, rest, 2.0, y, 0.5, got=(captured.detach(), dx))
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("V,dtype", [(139300, torch.float32), (278524, torch.float32), (278523, torch.float32),
                                     (300001, torch.bfloat16), (557048, torch.float16), (557047, torch.bfloat16)])
def test_longest_rows(V, dtype):
    """Up to the largest vocabulary of each type, on the largest clusters."""
    up = 64.0 if dtype == torch.float16 else 1.0
    x, ids, values, rest, y = _inputs(2, V, 64, dtype, tau=2.0, seed=16)
    y[0] = ids[0, 7]
    _check(x, ids, values, rest, 2.0, y, 0.3, upstream=up, expected=up)
    _check(x, ids, values, None, upstream=up, expected=1.0)


@pytest.mark.parametrize("tau", [1.0, 1.3, 2.0])
@pytest.mark.parametrize("V,dtype", [(1000, torch.float32), (33000, torch.bfloat16), (50000, torch.float32)])
def test_a_small_divergence_keeps_its_digits(V, dtype, tau):
    """One token of the teacher and the rest, within 1e-3 of the student's: a divergence of 1e-7 between logarithms of up to 12.

    The token's own weights are one exactly. The sum outside is off by at most 2^-15 of itself, the factors between the two
    masses by less; being in both distributions' sums, that counts as |p_0 - q_0| of it. The logarithms of the two ratios
    and what they are multiplied by are fp32: 2^-22 of them."""
    from astrai_b200.ops.distill import TopLogits, distill_loss

    g = torch.Generator().manual_seed(V)
    for i in range(24):
        x = (3 * torch.randn(1, V, generator=g)).to(dtype)
        j = int(x.argmax()) if i % 2 else int(torch.randint(V, (1,), generator=g))
        if i % 3 == 0:
            x[0, j] = 9.0 + i / 8
        z = x[0].double() / tau
        q = torch.softmax(z, -1)
        q0 = float(1 - q[j]) if q[j] < 0.5 else float(torch.cat([q[:j], q[j + 1:]]).sum())
        rest = (torch.cat([z[:j], z[j + 1:]]).logsumexp(0) + 1e-3 * torch.randn((), generator=g)).float()
        value = x[:, j: j + 1].clone()
        log_p = torch.log_softmax(torch.stack([value[0, 0].double() / tau, rest.double()]), 0)
        log_q = torch.tensor([q[j], q0]).double().log()
        want = float((log_p.exp() * (log_p - log_q)).sum()) * tau ** 2
        top = TopLogits(torch.tensor([[j]], device="cuda"), value.cuda(), rest[None].cuda())
        bound = 2.0 ** -15 * abs(float(log_p[1].exp()) - q0) + 2.0 ** -22 * float((log_p - log_q).abs().sum()) + 2.0 ** -48
        assert abs(float(distill_loss(x.cuda(), top, tau)) - want) <= tau ** 2 * bound, (i, float(distill_loss(x.cuda(), top, tau)), want, bound)


@pytest.mark.parametrize("V,dtype,tau", [(17500, torch.bfloat16, 1.3), (50001, torch.bfloat16, 2.0), (17500, torch.float32, 1.3),
                                         (3000, torch.float16, 2.0)])
def test_the_loss_is_the_same_with_and_without_a_gradient(V, dtype, tau):
    """Row by row: in a mean a last bit is lost."""
    from astrai_b200.ops.distill import TopLogits, distill_loss

    x, ids, values, _, y = _inputs(3000, V, 2, dtype, tau, seed=17, sigma=0.01)
    rest = 10 * torch.randn(3000, device="cuda")
    leaf = x.detach().requires_grad_()
    differ = torch.zeros((), device="cuda")
    for r in range(3000):
        top = TopLogits(ids[r], values[r], rest[r])
        differ += distill_loss(leaf[r], top, tau, y[r], 0.3).detach() != distill_loss(x[r], top, tau, y[r], 0.3)
    assert differ == 0
