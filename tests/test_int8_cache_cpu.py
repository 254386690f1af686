"""The int8 KV cache behind the cache API, the engine and the model options of the one-pass QK-norm, on the CPU."""

import copy

import pytest
import torch

from astrai_b200.config import AutoRegressiveLMConfig
from astrai_b200.inference import ContiguousCache, InferenceEngine, InferenceScheduler, Int8Storage, PageCache
from astrai_b200.models import AutoRegressiveLM


def _cfg(**kw):
    base = dict(vocab_size=200, hidden_size=64, num_hidden_layers=2, rms_norm_eps=1e-5, intermediate_size=96,
                tie_word_embeddings=False, max_position_embeddings=256, rope_theta=10000.0, num_attention_heads=4,
                num_key_value_heads=2)
    base.update(kw)
    return AutoRegressiveLMConfig(**base)


def _model(**kw):
    torch.manual_seed(0)
    return AutoRegressiveLM(_cfg(**kw)).eval()


def _decode(model, cache, prompts, steps, dev="cpu"):
    """Decode of the same given tokens through cache views; -> logits of each step."""
    tids = [f"t{i}" for i in range(len(prompts))]
    out = []
    with torch.inference_mode():
        for tid, ids in zip(tids, prompts):
            assert cache.task_alloc(tid, ids)
            view = cache.bind([tid], [len(ids)], len(ids), dev, uniform_start=0)
            model(torch.tensor([ids]), paged_cache=view, position_ids=torch.arange(len(ids))[None], logits_to_keep=1)
        lens = [len(p) for p in prompts]
        tok = torch.tensor([[7]] * len(prompts))
        for step in range(steps):
            for tid, n in zip(tids, lens):
                assert cache.task_extend(tid, n)
            view = cache.bind(tids, [n + 1 for n in lens], 1, dev)
            logits = model(tok, paged_cache=view, position_ids=torch.tensor(lens)[:, None], logits_to_keep=1)["logits"]
            out.append(logits[:, -1])
            tok = torch.tensor([[(17 * step + 31 * i) % 200] for i in range(len(prompts))])
            lens = [n + 1 for n in lens]
    return torch.stack(out)


def _caches(cfg, kv_dtype, block=16):
    hd = cfg.hidden_size // cfg.num_attention_heads
    yield PageCache(cfg.num_hidden_layers, 32, 32, cfg.num_key_value_heads, hd, "cpu", torch.float32, kv_dtype, block)
    yield ContiguousCache(cfg.num_hidden_layers, 4, 128, cfg.num_key_value_heads, hd, "cpu", torch.float32, kv_dtype, block)


@pytest.mark.parametrize("kw", [{}, dict(use_qk_norm=True), dict(use_qk_norm=True, fused_qk_norm=True),
                                dict(use_qk_norm=True, qk_norm_first=True, rope_layout="half", rope_fraction=0.5)])
def test_int8_decode_stays_near_the_exact_cache(kw):
    model = _model(**kw)
    prompts = [list(range(3, 40)), list(range(90, 95)), [11]]
    plain = [_decode(model, c, prompts, 8) for c in _caches(model.config, None)]
    assert torch.allclose(plain[0], plain[1], atol=1e-5)
    for cache in _caches(model.config, "int8"):
        assert isinstance(cache.storage, Int8Storage)
        got = _decode(model, cache, prompts, 8)
        # half a step of 1/127 of the largest magnitude per value, through two layers
        assert ((got - plain[0]).norm() / plain[0].norm()) < 0.02


def test_prefix_pages_are_shared_and_prefill_behind_them_reads_the_cache():
    model = _model()
    cache = next(_caches(model.config, "int8"))
    ids = list(range(10, 80))
    with torch.inference_mode():
        assert cache.task_alloc("a", ids) and cache.task_cached("a") == 0
        view = cache.bind(["a"], [70], 70, "cpu", uniform_start=0)
        full = model(torch.tensor([ids]), paged_cache=view, position_ids=torch.arange(70)[None], logits_to_keep=1)["logits"]
        cache.task_record_hashes("a", ids)
        assert cache.task_alloc("b", ids) and cache.task_cached("b") == 64
        view = cache.bind(["b"], [70], 6, "cpu", uniform_start=64)
        rest = model(torch.tensor([ids[64:]]), paged_cache=view, position_ids=torch.arange(64, 70)[None],
                     logits_to_keep=1)["logits"]
    assert ((full - rest).norm() / full.norm()) < 0.02


def test_scheduler_and_refusals():
    model = _model()
    prompts = [[1, 2, 3, 4], [9, 8, 7]]
    runs = []
    for kv in (None, "int8"):
        sched = InferenceScheduler(model, None, max_batch_size=2, max_seq_len=64, kv_cache_dtype=kv)
        assert isinstance(sched.cache.storage, Int8Storage) == (kv == "int8")
        runs.append(sched.cache.storage)
    with pytest.raises(ValueError):
        PageCache(1, 2, 32, 1, 64, "cpu", torch.float32, "int4")
    with pytest.raises(ValueError):
        PageCache(1, 2, 48, 1, 64, "cpu", torch.float32, "int8", 32)
    with pytest.raises(RuntimeError):
        runs[1].write_slots(0, torch.zeros(1, dtype=torch.int32), torch.zeros(1, 32), torch.zeros(1, 32))
    with pytest.raises(ValueError):
        InferenceEngine(model, None, cache=next(_caches(model.config, None)), kv_cache_dtype="int8")
    with pytest.raises(ValueError):
        Int8Storage(1, 2, 64, 1, 96, "cuda", torch.bfloat16)
    with pytest.raises(ValueError):
        Int8Storage(1, 2, 64, 1, 64, "cuda", torch.float32)


def test_fused_options_leave_other_models_alone_and_match_the_separate_path():
    sep, one = _model(use_qk_norm=True), _model(use_qk_norm=True, fused_qk_norm=True)
    assert not sep.layers[0].attention.one_pass and one.layers[0].attention.one_pass
    assert not _model().layers[0].attention.one_pass
    with torch.no_grad():
        for m in (sep, one):
            for layer in m.layers:
                layer.attention.q_norm.weight.copy_(torch.linspace(0.5, 1.5, 16))
    ids = torch.randint(0, 200, (2, 33), generator=torch.Generator().manual_seed(1))
    seg = torch.tensor([[0] * 20 + [1] * 13, [0] * 33])
    for kw in ({}, dict(seg_ids=seg), dict(position_ids=torch.arange(33).expand(2, -1) + 5),
               dict(input_mask=torch.ones(2, 33, 33, dtype=torch.bool).tril())):
        a, b = sep.train()(ids, **kw)["logits"], one.train()(ids, **kw)["logits"]
        assert torch.allclose(a, b, atol=1e-5)
        for m, y in ((sep, a), (one, b)):
            m.zero_grad()
            y.square().mean().backward()
        for p, q in zip(sep.parameters(), one.parameters()):
            assert torch.allclose(p.grad, q.grad, atol=1e-6)


def test_config_options():
    cfg = _cfg(rope_fraction=0.5, rope_layout="half", rope_scaling_method="yarn",
               rope_scaling=dict(factor=4.0, original_max_position_embeddings=64))
    again = AutoRegressiveLMConfig.from_dict(cfg.to_dict())
    m = AutoRegressiveLM(again)
    assert m.rotary_embedding.table().shape == (256, 4, 2)
    assert m.rotary_embedding.table()[3].norm(dim=-1).min() > 1.1  # the scaled table's gain
    half = copy.deepcopy(m).to(torch.bfloat16)
    assert torch.equal(half.rotary_embedding.table(), m.rotary_embedding.table())
    m.rotary_embedding.freqs_cis.zero_()
    m.rotary_embedding.reset_buffers()
    assert torch.equal(half.rotary_embedding.table(), m.rotary_embedding.table())
    for bad in (dict(rope_layout="other"), dict(rope_fraction=0.0), dict(rope_fraction=0.3)):
        with pytest.raises(ValueError):
            _model(**bad)
    with pytest.raises(ValueError):
        _model(rope_scaling_method="other", rope_scaling=dict(factor=2.0))


def test_command_line_flags(monkeypatch, tmp_path):
    from astrai_b200.cli import server
    from astrai_b200.inference.api import server as api

    seen = {}
    monkeypatch.setattr(api, "run_server", lambda path, **kw: seen.update(kw))
    server.main(["--param_path", str(tmp_path)])
    assert "kv_cache_dtype" not in seen
    server.main(["--param_path", str(tmp_path), "--n_pages", "8", "--kv_cache_dtype", "int8", "--kv_block", "64"])
    assert seen["kv_cache_dtype"] == "int8" and seen["kv_block"] == 64 and seen["n_pages"] == 8
    with pytest.raises(SystemExit):
        server.main(["--param_path", str(tmp_path), "--kv_cache_dtype", "int4"])
