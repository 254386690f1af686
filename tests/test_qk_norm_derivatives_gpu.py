"""qk_norm_rope and derivatives that its kernels do not give: refused, not dropped; and what its backward keeps."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(rows=6, hq=2, hkv=1, d=64):
    from astrai_b200.ops.rope import rope_table

    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(rows, (hq + hkv) * d, device="cuda", generator=g).to(torch.bfloat16)
    w = [(1 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(torch.bfloat16) for _ in range(2)]
    return x, w[0], w[1], rope_table(d, rows, device="cuda")


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", ["x", "q_weight", "k_weight", "table"])
@pytest.mark.parametrize("in_place", [False, True])
def test_tangents_are_refused(which, grad_mode, in_place):
    """A dual number made of a plain tensor does not require a gradient."""
    from torch.autograd import forward_ad

    from astrai_b200.ops.qk_norm import qk_norm_rope, qk_norm_rope_

    x, wq, wk, t = _inputs()
    kw = dict(x=x, table=t, q_weight=wq, k_weight=wk)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        kw[which] = forward_ad.make_dual(kw[which].clone(), torch.ones_like(kw[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            (qk_norm_rope_ if in_place else qk_norm_rope)(n_heads=2, n_kv_heads=1, head_dim=64, seq_len=6, **kw)


def test_a_table_that_requires_a_gradient_is_refused():
    from astrai_b200.ops.qk_norm import qk_norm_rope, qk_norm_rope_

    x, wq, wk, t = _inputs()
    t = t.requires_grad_()
    for fn in (qk_norm_rope, qk_norm_rope_):
        with pytest.raises(RuntimeError, match="table"):
            fn(x, 2, 1, 64, t, wq, wk, seq_len=6)
    with torch.no_grad():
        qk_norm_rope(x, 2, 1, 64, t, wq, wk, seq_len=6)


def test_a_tangent_in_the_backward_is_refused():
    from torch.autograd import forward_ad

    from astrai_b200.ops.qk_norm import qk_norm_rope

    x, wq, wk, t = _inputs()
    leaf = x.clone().requires_grad_()
    y = qk_norm_rope(leaf, 2, 1, 64, t, wq, wk, seq_len=6)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize("which", ["q_weight", "k_weight"])
def test_in_place_refuses_weights_that_require_a_gradient(which):
    from astrai_b200.ops.qk_norm import qk_norm_rope_

    x, wq, wk, t = _inputs()
    kw = dict(table=t, q_weight=wq, k_weight=wk)
    kw[which] = kw[which].clone().requires_grad_()
    before = x.clone()
    with pytest.raises(RuntimeError, match="no gradient"):
        qk_norm_rope_(x, 2, 1, 64, seq_len=6, **kw)
    assert torch.equal(x, before)
    qk_norm_rope_(x.clone(), 2, 1, 64, seq_len=6, norm="none", **kw)  # the weight has no part in it
    with torch.no_grad():
        assert qk_norm_rope_(x, 2, 1, 64, seq_len=6, **kw) is x


def test_a_rotation_alone_keeps_no_input():
    """Its backward is the transposed rotation of the gradient: x may change before it, and is not kept alive."""
    from astrai_b200.ops.qk_norm import qk_norm_rope

    x, _, _, t = _inputs()
    dy = torch.randn(6, 192, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    leaf = x.clone().requires_grad_()
    want = torch.autograd.grad(qk_norm_rope(leaf, 2, 1, 64, t, norm="none", seq_len=6), leaf, dy)[0]
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda v: kept.append(v.shape) or v, lambda v: v):
        y = qk_norm_rope(leaf, 2, 1, 64, t, norm="none", seq_len=6)
    assert leaf.shape not in kept
    with torch.no_grad():
        leaf.mul_(2)
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], want)
