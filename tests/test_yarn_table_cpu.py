"""YaRN tables: the pairs between the two corrected ones, which turn neither fast nor slow."""

import math

import pytest
import torch

from astrai_b200.ops.rope import scaled_rope_table


# the pair that turns 32 times over the trained positions, rounded down, and the one that turns once, rounded up:
# dim ln(L / (2 pi turns)) / (2 ln base) is 20.94 and 45.03, 23.60 and 39.65, 8.06 and 20.11, 45.03 and 69.11, -7.95 and 16.13
@pytest.mark.parametrize("base,dim,length,factor,low,high", [
    (1e4, 128, 4096, 4.0, 20, 46), (1e6, 128, 32768, 4.0, 23, 40), (1e4, 64, 2048, 16.0, 8, 21),
    (1e4, 128, 131072, 2.0, 45, 70), (1e4, 128, 64, 8.0, 0, 17)])
def test_mixed_pairs_ramp_over_the_index(base, dim, length, factor, low, high):
    """Angles of position 1 are below pi, so they can be read back from the table: fp32 cosines and sines, 2^-22."""
    t = scaled_rope_table(dim, 2, base, "yarn", factor, length).double()
    for i in range(dim // 2):
        keep = 1 - min(max((i - low) / (high - low), 0.0), 1.0)
        want = base ** (-2 * i / dim) * (keep + (1 - keep) / factor)
        got = math.atan2(t[1, i, 1], t[1, i, 0])
        assert abs(got - want) <= 2.0 ** -22 * want + 1e-12, i
        assert abs(t[1, i].norm().item() - (0.1 * math.log(factor) + 1)) < 1e-6


def test_refusals():
    for kw in (dict(base=1.0), dict(original_max_len=-4), dict(beta_slow=0.0), dict(beta_slow=64.0)):
        with pytest.raises(ValueError):
            scaled_rope_table(32, 8, **{**dict(base=1e4, method="yarn", factor=4.0, original_max_len=64), **kw})
    assert torch.isfinite(scaled_rope_table(32, 8, 1e4, "yarn", 4.0, 1)).all()  # all pairs slower than one turn
