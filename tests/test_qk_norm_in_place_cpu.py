"""The in-place norm + rotation on the CPU: refuses what it has no gradient of."""

import pytest
import torch

from astrai_b200.ops.qk_norm import qk_norm_rope_
from astrai_b200.ops.rope import rope_table


@pytest.mark.parametrize("which", ["q_weight", "k_weight", "table"])
def test_refuses_inputs_that_require_a_gradient(which):
    torch.manual_seed(0)
    x, kw = torch.randn(3, 48), dict(table=rope_table(16, 3), q_weight=torch.ones(16), k_weight=torch.ones(16))
    kw[which].requires_grad_()
    before = x.clone()
    with pytest.raises(RuntimeError, match="no gradient"):
        qk_norm_rope_(x, 2, 1, 16, seq_len=3, **kw)
    assert torch.equal(x, before) and not x.requires_grad
    with torch.no_grad():
        assert qk_norm_rope_(x, 2, 1, 16, seq_len=3, **kw) is x and not x.requires_grad
    if which != "table":  # a weight has no part in a rotation alone
        qk_norm_rope_(x, 2, 1, 16, seq_len=3, norm="none", **kw)
