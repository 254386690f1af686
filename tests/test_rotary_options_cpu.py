"""Model options of the one-pass norm and rotation that no kernel takes are refused with the
configuration."""

import pytest

from astrai_b200.models.components import AttnFactory


@pytest.mark.parametrize("dim,kw", [
    (256, dict(rope_fraction=0.3125)), (256, dict(rope_fraction=0.03125)),     # 20 and 2 of 64 channels
    (80, dict(fused_qk_norm=True)), (80, dict(rope_layout="half")), (80, dict(qk_norm_first=True)),  # heads of 20
    (80, dict(rope_fraction=0.4)), (2048, dict(fused_qk_norm=True)),           # 8 of 20; heads of 512
])
def test_sizes_that_the_kernels_do_not_take(dim, kw):
    with pytest.raises(ValueError, match="multiple of 8|at most 256"):
        AttnFactory.create("gqa", dim=dim, n_heads=4, n_kv_heads=2, use_qk_norm=True, **kw)


def test_sizes_that_they_take_and_layers_without_the_options():
    for dim, kw in ((256, dict(rope_fraction=0.375)), (96, dict(fused_qk_norm=True)), (1024, dict(rope_layout="half")),
                    (256, dict(rope_fraction=1.0)), (80, dict()), (80, dict(rope_fraction=1.0)), (2048, dict())):
        AttnFactory.create("gqa", dim=dim, n_heads=4, n_kv_heads=2, use_qk_norm=True, **kw)
