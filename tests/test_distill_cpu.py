"""The plain path of the distillation loss: its formulas in 64 bits, its gradient by differences, its refusals."""

import math

import pytest
import torch

from astrai_b200.ops.distill import TopLogits, distill_loss
from tests.distill_oracle import oracle


def _inputs(rows=6, V=50, K=5, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = 3 * torch.randn(rows, V, generator=g)
    values, ids = (0.7 * x + torch.randn(rows, V, generator=g)).topk(K, -1)
    return x, ids, values, torch.randn(rows, generator=g), torch.randint(V, (rows,), generator=g)


@pytest.mark.parametrize("tau", [1.0, 2.0])
@pytest.mark.parametrize("hard", [0.0, 0.3])
@pytest.mark.parametrize("with_rest", [False, True])
def test_against_the_formulas(tau, hard, with_rest):
    x, ids, values, rest, y = _inputs()
    ids[0, 1] = -1
    ids[1] = 50
    ids[2, 1] = ids[2, 0]
    values[3, 1] = -math.inf
    rest[4] = -math.inf
    y[5] = -100
    rest = rest if with_rest else None
    leaf = x.clone().requires_grad_()
    loss = distill_loss(leaf, TopLogits(ids, values, rest), tau, y, hard)
    loss.backward()
    want, dx, size, dsize = oracle(x, ids, values, rest, tau, y, hard)
    # a few fp32 operations and sums of 50 terms: 2^-18 of the magnitudes
    assert abs(float(loss.detach()) - want) <= 2.0 ** -18 * size
    assert ((leaf.grad.double() - dx).abs() <= 2.0 ** -18 * dsize + 1e-30).all()


def test_oracle_gradient_by_differences():
    x, ids, values, rest, y = _inputs(2, 12, 3)
    ids[1, 2] = ids[1, 0]
    for hard, tau in ((0.0, 1.0), (0.4, 2.0)):
        _, dx, _, _ = oracle(x, ids, values, rest, tau, y, hard)
        for r in range(2):
            for v in range(12):
                up, down = x.double().clone(), x.double().clone()
                up[r, v] += 1e-4
                down[r, v] -= 1e-4
                slope = (oracle(up, ids, values, rest, tau, y, hard)[0] - oracle(down, ids, values, rest, tau, y, hard)[0]) / 2e-4
                # the third derivative is below 10 here: 1e-8 of truncation, 1e-11 of rounding
                assert abs(slope - float(dx[r, v])) < 2e-7


def test_nothing_counts():
    x, ids, values, rest, y = _inputs()
    leaf = x.requires_grad_()
    loss = distill_loss(leaf, TopLogits(ids, values, rest), target=torch.full_like(y, -100))
    loss.backward()
    assert loss == 0 and (leaf.grad == 0).all()
    leaf.grad = None
    empty = TopLogits(torch.full_like(ids, -1), values, None)
    loss = distill_loss(leaf, empty)
    loss.backward()
    assert loss == 0 and (leaf.grad == 0).all()


def test_refusals():
    x, ids, values, rest, y = _inputs()
    ok = TopLogits(ids, values, rest)
    for bad in (dict(teacher=TopLogits(ids[:2], values[:2], rest)), dict(teacher=TopLogits(ids, values[:, :3], rest)),
                dict(teacher=TopLogits(ids, values, rest[:2])), dict(temperature=0.0), dict(temperature=math.inf),
                dict(hard_weight=0.5), dict(hard_weight=1.5, target=y), dict(target=y[:2])):
        with pytest.raises(ValueError):
            distill_loss(**{"logits": x, "teacher": ok, **bad})
    with pytest.raises(RuntimeError, match="gradient of the teacher"):
        distill_loss(x, TopLogits(ids, values.requires_grad_(), rest))


def test_top_logits():
    from astrai_b200.ops.distill import top_logits

    x = torch.tensor([[1.0, 3.0, 3.0, -math.inf, 2.0], [0.0, 0.0, 0.0, 0.0, 0.0]])
    top = top_logits(x, 2, 2.0)
    assert top.ids.tolist() == [[1, 2], [0, 1]] and top.values.tolist() == [[3.0, 3.0], [0.0, 0.0]]
    want = torch.tensor([math.log(math.exp(0.5) + math.exp(1.0)), math.log(3.0)])
    assert (top.rest - want).abs().max() < 1e-6
    assert (top_logits(x, 5).rest == -math.inf).all()
    for k, tau in ((0, 1.0), (6, 1.0), (1, 0.0)):
        with pytest.raises(ValueError):
            top_logits(x, k, tau)
    with pytest.raises(RuntimeError, match="no gradient"):
        top_logits(x.requires_grad_(), 2)
