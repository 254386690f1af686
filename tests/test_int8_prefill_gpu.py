"""A prompt behind cached tokens of the int8 cache: in place up to INT8_ROWS query rows of a KV head, gathered for the
prefill kernel past that. Both are compared with the prompt's own prefill from its start; the bound is that of the decode
tests, half a step of 1/127 of a block's magnitude in k and v and the 16-bit roundings of both sides."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("over", [-1, 0, 1, 107])
def test_both_sides_of_the_threshold(over, dtype, monkeypatch):
    from astrai_b200.config import AutoRegressiveLMConfig
    from astrai_b200.inference import Int8Storage, PageCache
    from astrai_b200.inference.core.cache import INT8_ROWS
    from astrai_b200.models import AutoRegressiveLM

    torch.manual_seed(0)
    cfg = AutoRegressiveLMConfig(vocab_size=512, hidden_size=512, num_hidden_layers=2, rms_norm_eps=1e-5,
                                 intermediate_size=512, tie_word_embeddings=False, max_position_embeddings=1024,
                                 rope_theta=1e4, num_attention_heads=4, num_key_value_heads=2)
    model = AutoRegressiveLM(cfg).to("cuda", dtype).eval()
    gathers, in_place = [], []
    gather_rows, attend_rows = Int8Storage.gather_rows, Int8Storage.attend_rows
    monkeypatch.setattr(Int8Storage, "gather_rows", lambda self, *a: gathers.append(1) or gather_rows(self, *a))
    monkeypatch.setattr(Int8Storage, "attend_rows", lambda self, *a: in_place.append(1) or attend_rows(self, *a))
    n = INT8_ROWS // 2 + over  # two query heads to a KV head
    ids = torch.randint(0, 512, (128 + n,), generator=torch.Generator().manual_seed(5)).tolist()

    def run(cache, name, first):
        new = torch.tensor([ids[first:]], device="cuda")
        view = cache.bind([name], [len(ids)], len(ids) - first, "cuda", uniform_start=first)
        return model(new, paged_cache=view, position_ids=torch.arange(first, len(ids), device="cuda")[None])["logits"]

    with torch.inference_mode():
        cache = PageCache(2, 20, 64, 2, 128, "cuda", dtype, "int8")
        assert cache.task_alloc("a", ids)
        full = run(cache, "a", 0)
        assert not gathers and not in_place
        cache.task_record_hashes("a", ids[:128])
        assert cache.task_alloc("b", ids) and cache.task_cached("b") == 128
        rest = run(cache, "b", 128)
    assert (len(gathers), len(in_place)) == ((2, 0) if over > 0 else (0, 2))
    a, b = rest.float(), full[:, 128:].float()
    assert ((a - b).norm() / b.norm()).item() < 0.03
