"""Model options of the one-pass norm and rotation that no kernel takes, or that an attention type does not have, are
refused with the configuration."""

import pytest
import torch

from astrai_b200.config import AutoRegressiveLMConfig
from astrai_b200.models import AutoRegressiveLM
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


def _mla(**kw):
    torch.manual_seed(0)
    return AutoRegressiveLM(AutoRegressiveLMConfig(
        vocab_size=50, hidden_size=64, num_hidden_layers=1, rms_norm_eps=1e-5, intermediate_size=64,
        tie_word_embeddings=False, max_position_embeddings=64, rope_theta=1e4, num_attention_heads=4, num_key_value_heads=4,
        attn_type="mla", kv_lora_rank=16, qk_nope_head_dim=8, qk_rope_head_dim=8, use_qk_norm=True, **kw))


@pytest.mark.parametrize("kw", [dict(rope_layout="half"), dict(rope_fraction=0.5), dict(qk_norm_first=True),
                                dict(fused_qk_norm=True)])
def test_mla_refuses_what_it_does_not_have(kw):
    with pytest.raises(ValueError, match=next(iter(kw))):
        _mla(**kw)


def test_mla_takes_defaults_and_scaled_tables():
    _mla(rope_layout="interleaved", rope_fraction=1.0, qk_norm_first=False, fused_qk_norm=False)
    m = _mla(rope_scaling_method="linear", rope_scaling=dict(factor=2.0))
    plain = _mla()
    assert torch.allclose(m.rotary_embedding.table()[2], plain.rotary_embedding.table()[1], atol=1e-6)


@pytest.mark.parametrize("shape", [(1, 9), (3, 9)])
def test_one_pass_takes_the_positions_that_the_separate_path_takes(shape):
    """One row of positions for the whole batch."""
    def model(**kw):
        torch.manual_seed(0)
        return AutoRegressiveLM(AutoRegressiveLMConfig(
            vocab_size=50, hidden_size=64, num_hidden_layers=2, rms_norm_eps=1e-5, intermediate_size=64,
            tie_word_embeddings=False, max_position_embeddings=64, rope_theta=1e4, num_attention_heads=4,
            num_key_value_heads=2, use_qk_norm=True, **kw)).eval()

    ids = torch.arange(27).view(3, 9)
    pos = (torch.arange(9) + 4).expand(*shape)
    mask = torch.ones(3, 9, 9, dtype=torch.bool).tril()
    for kw in ({}, dict(input_mask=mask)):
        a, b = (model(fused_qk_norm=f)(ids, position_ids=pos, **kw)["logits"] for f in (False, True))
        assert torch.allclose(a, b, atol=1e-5)
