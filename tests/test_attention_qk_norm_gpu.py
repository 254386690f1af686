"""Attention with QK-norm and rotation on the fused projection: what its autograd function does not give is refused."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_second_derivative_is_refused():
    from astrai_b200.ops.attention import attention_qk_norm
    from astrai_b200.ops.qk_norm import QKRotary
    from astrai_b200.ops.rope import rope_table

    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn(128, 4 * 128, device="cuda", generator=g).bfloat16().requires_grad_()
    w = torch.ones(128, device="cuda", dtype=torch.bfloat16)
    rotary = QKRotary(rope_table(128, 128, device="cuda"), w, w)
    o = attention_qk_norm(qkv, rotary, 1, 128, 2, 1)
    first = torch.autograd.grad(o.float().square().sum(), qkv, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.float().sum().backward()
