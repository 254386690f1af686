"""Attention over the 8-bit cache has no gradient on CUDA: it says so instead of returning a result without one."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _call(q):
    from astrai_b200.ops.kv8 import KV8, kv8_attention

    c = KV8.allocate(2, 2, 32, 64, 16, "cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    return kv8_attention(q, c, torch.tensor([[0, 1]], **i32), torch.tensor([40], **i32))


def test_a_query_that_requires_a_gradient_is_refused():
    q = torch.randn(1, 1, 4, 64, device="cuda").bfloat16().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        _call(q)
    with torch.no_grad():
        assert _call(q).shape == q.shape
    assert _call(q.detach()).shape == q.shape


@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents_are_refused(grad_mode):
    from torch.autograd import forward_ad

    q = torch.randn(1, 1, 4, 64, device="cuda").bfloat16()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        with pytest.raises(RuntimeError, match="forward-mode"):
            _call(forward_ad.make_dual(q, torch.ones_like(q)))


@pytest.mark.parametrize("kw", [{}, dict(use_qk_norm=True), dict(use_qk_norm=True, fused_qk_norm=True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_models_decode_from_the_cache_outside_no_grad(kw, dtype):
    """Attention over a cache has no gradient; a forward outside no_grad() gives what it gives inside."""
    from astrai_b200.config import AutoRegressiveLMConfig
    from astrai_b200.inference import PageCache
    from astrai_b200.models import AutoRegressiveLM

    torch.manual_seed(0)
    cfg = AutoRegressiveLMConfig(vocab_size=128, hidden_size=256, num_hidden_layers=1, rms_norm_eps=1e-5,
                                 intermediate_size=256, tie_word_embeddings=False, max_position_embeddings=256,
                                 rope_theta=10000.0, num_attention_heads=2, num_key_value_heads=1, **kw)
    model = AutoRegressiveLM(cfg).to("cuda", dtype).eval()
    outs = []
    for grad in (True, False):
        cache = PageCache(1, 8, 64, 1, 128, "cuda", dtype, "int8")
        assert cache.task_alloc("a", list(range(20))) and cache.task_extend("a", 20)
        with torch.set_grad_enabled(grad):
            model(torch.arange(20, device="cuda")[None], position_ids=torch.arange(20, device="cuda")[None],
                  paged_cache=cache.bind(["a"], [20], 20, "cuda", uniform_start=0), logits_to_keep=1)
            outs.append(model(torch.tensor([[5]], device="cuda"), position_ids=torch.tensor([[20]], device="cuda"),
                              paged_cache=cache.bind(["a"], [21], 1, "cuda"), logits_to_keep=1)["logits"].detach())
    assert torch.equal(*outs)
