"""The k largest logits and the rest's log-sum-exp, against torch's stable sort and 64 bits.

Ids and values are compared for equality. Tolerance of `rest`: a weight 2^t with t from one fp32 fused multiply-add is off
by at most 2^-16 for all |t| <= 126 and zero beyond, a sum of terms of one sign by 2^-17 more: 2^-15 of the sum, so of its
logarithm too; and the result and the maximum over the temperature are rounded to fp32.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_error_word():
    from astrai_b200.ops._ext import native

    native().read_error()
    yield
    torch.cuda.synchronize()
    assert native().read_error() == 0


def _check(x, k, tau=1.0, got=None):
    from astrai_b200.ops.distill import top_logits

    top = got or top_logits(x, k, tau)
    values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    assert top.ids.dtype == torch.int32 and top.values.dtype == x.dtype and top.rest.dtype == torch.float32
    assert torch.equal(top.ids.long(), ids[..., :k])
    assert torch.equal(torch.nan_to_num(top.values, 7.0), torch.nan_to_num(values[..., :k], 7.0))
    want = torch.logsumexp(values[..., k:].double() / tau, -1)
    error = torch.where(want == top.rest, 0.0, (top.rest.double() - want).abs())
    size = values.double().masked_fill(~torch.isfinite(values), 0).abs().amax(-1) / tau
    nan = want.isnan()
    assert torch.equal(top.rest.isnan(), nan)
    assert (error <= 2.0 ** -15 + 2.0 ** -22 * (size + 12))[~nan].all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (2, 9, 4), (5, 100, 100), (4, 256, 256), (4, 257, 256),
                                      (3, 1000, 64), (3, 1000, 1), (7, 4097, 16), (2, 8193, 200), (5, 32000, 64),
                                      (3, 32003, 255), (2, 33001, 33), (2, 50021, 256), (3, 100003, 7), (1, 131072, 128),
                                      (2, 300001, 200)])
def test_sizes(dtype, rows, V, k):
    g = torch.Generator("cuda").manual_seed(V + k)
    for sigma in (0.05, 1.0, 4.0):
        _check((torch.randn(rows, V, generator=g, device="cuda") * sigma).to(dtype), k, 1.0 if sigma == 1 else 1.7)


@pytest.mark.parametrize("V", [300, 5000, 32000, 70000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_and_special_values(dtype, V):
    g = torch.Generator("cuda").manual_seed(V)
    x = torch.randn(16, V, generator=g, device="cuda").to(dtype)
    x[0] = 0.5                                       # all equal
    x[1] = -math.inf                                 # nothing allowed
    x[2, 5:] = -math.inf                             # fewer allowed than k
    x[3] = torch.where(x[3] > 0, 1.0, -1.0)          # two values
    x[4, ::3] = 9.0                                  # a third at the top
    x[5] = torch.where(x[5] > 0, 0.0, -0.0)          # zeros of both signs are equal
    x[6, 17] = math.nan
    x[7, 3::7] = math.nan                            # more than k
    x[8, [4, 9]] = math.inf
    x[9] = torch.arange(V, device="cuda").to(dtype)  # ascending: all of the largest in one place
    x[10] = -torch.arange(V, device="cuda").to(dtype)
    x[11] *= 1e30 if dtype != torch.float16 else 1e4
    x[12, :40] = 60.0                                # the k far above the rest
    x[13, 1] = 300.0
    x[14] = x[14].round()
    x[15, V // 2:] = x[15, : V - V // 2].clone()
    for k in (1, 2, 40, 41, 200):
        _check(x, k)
        _check(x, k, 0.5)


def test_more_infinities_than_k():
    from astrai_b200.ops.distill import top_logits

    x = torch.randn(2, 4000, device="cuda")
    x[:, 5:30] = math.inf
    top = top_logits(x, 10)
    assert torch.equal(top.ids, torch.arange(5, 15, device="cuda", dtype=torch.int32).expand(2, -1))
    assert (top.rest == math.inf).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_dimensions(dtype):
    from astrai_b200.ops.distill import top_logits

    x = torch.randn(6, 5003, device="cuda").to(dtype)
    for pad, off in ((3, 0), (7, 5), (23, 1)):
        wide = torch.full((6, 5003 + pad + off), math.inf, dtype=dtype, device="cuda")
        wide[:, off: off + 5003] = x
        _check(wide[:, off: off + 5003], 50)
    _check(x.repeat_interleave(2, 0)[::2], 50)
    _check(x.t().contiguous().t(), 50)
    _check(x[:1].expand(6, -1), 50)
    shaped = x.view(2, 3, 5003)
    top = top_logits(shaped, 9)
    assert top.ids.shape == (2, 3, 9) and top.rest.shape == (2, 3)
    _check(shaped, 9, got=top)
    _check(shaped[:, 1:], 9)
    _check(x[0], 9)
    none = top_logits(x[:0], 5)
    assert none.ids.shape == (0, 5) and none.rest.shape == (0,)


def test_many_rows_same_each_time():
    x = torch.randn(3000, 2049, device="cuda").bfloat16()
    from astrai_b200.ops.distill import top_logits

    first = top_logits(x, 64, 2.0)
    for _ in range(5):
        again = top_logits(x, 64, 2.0)
        assert torch.equal(first.ids, again.ids) and torch.equal(first.rest, again.rest)
    _check(x, 64, 2.0, got=first)


@pytest.mark.parametrize("rows,V,dtype", [(1500, 300, torch.bfloat16), (1300, 9001, torch.float16), (700, 33000, torch.bfloat16),
                                          (400, 70000, torch.float32)])
def test_more_rows_than_run_at_a_time(rows, V, dtype):
    x = (torch.randn(rows, V, device="cuda") * 3).to(dtype)
    x[rows // 2] = 1.0
    _check(x, 33, 0.7)


def test_captured_and_on_another_stream():
    from astrai_b200.ops.distill import top_logits

    x = torch.randn(5, 40000, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = top_logits(x, 20)
    side.synchronize()
    _check(x, 20, got=got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = top_logits(x, 20)
    for seed in range(2):
        x.copy_(torch.randn(5, 40000, device="cuda"))
        if seed:
            x[2] = 1.0  # now with ties
        g.replay()
        _check(x, 20, got=out)


def test_refusals():
    from astrai_b200.ops.distill import top_logits

    x = torch.randn(2, 300, device="cuda")
    for bad in (dict(k=0), dict(k=301), dict(k=257), dict(k=5, temperature=0.0), dict(k=5, temperature=-1.0)):
        with pytest.raises(ValueError):
            top_logits(x, **bad)
    with pytest.raises(RuntimeError):
        top_logits(x.double(), 5)
    with pytest.raises(RuntimeError, match="no gradient"):
        top_logits(x.requires_grad_(), 5)
    with torch.no_grad():
        _check(x, 5)


def test_with_the_loss():
    """A teacher's rows into the student's loss: the same teacher as its student costs what its rest cannot tell apart."""
    from astrai_b200.ops.distill import distill_loss, top_logits

    teacher = (3 * torch.randn(9, 32003, device="cuda")).bfloat16()
    for tau in (1.0, 2.0):
        student = teacher.clone().requires_grad_()
        loss = distill_loss(student, top_logits(teacher, 64, tau), tau)
        (dx,) = torch.autograd.grad(loss, student)
        # equal distributions: zero but for the arithmetic, logarithms of up to 20 within 2^-15
        assert abs(float(loss.detach())) <= tau ** 2 * 2.0 ** -15 * 40
        assert dx.abs().max() <= tau / 9 * 2.0 ** -14


@pytest.mark.parametrize("rows,V,dtype", [(700, 4096, torch.bfloat16), (700, 8001, torch.float32), (1300, 32000, torch.float16)])
def test_largest_k_of_many_rows(rows, V, dtype):
    """The bound from a small CTA's 256 numbers lets more candidates through than their list holds."""
    g = torch.Generator("cuda").manual_seed(V)
    x = (torch.randn(rows, V, generator=g, device="cuda") * 3).to(dtype)
    for k in (240, 250, 256):
        _check(x, k, 0.7)
