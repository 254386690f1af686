"""Models with the one-pass QK-norm and the int8 KV cache on the GPU: against the CPU's fp32 model, the bfloat16
cache and the eager decode step."""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_error_word():
    from astrai_b200.ops._ext import native

    native().read_error()
    yield
    torch.cuda.synchronize()
    assert native().read_error() == 0


def _cfg(**kw):
    from astrai_b200.config import AutoRegressiveLMConfig

    base = dict(vocab_size=512, hidden_size=512, num_hidden_layers=2, rms_norm_eps=1e-5, intermediate_size=512,
                tie_word_embeddings=False, max_position_embeddings=1024, rope_theta=10000.0, num_attention_heads=4,
                num_key_value_heads=2)
    base.update(kw)
    return AutoRegressiveLMConfig(**base)


def _models(**kw):
    from astrai_b200.models import AutoRegressiveLM

    torch.manual_seed(0)
    cpu = AutoRegressiveLM(_cfg(**kw))
    with torch.no_grad():
        for p in cpu.parameters():
            p.copy_(p.to(torch.bfloat16).float())
    return cpu, copy.deepcopy(cpu).to("cuda", torch.bfloat16)


def _rel(a, b):
    a, b = a.float().cpu(), b.float().cpu()
    return ((a - b).norm() / b.norm().clamp_min(1e-12)).item()


OPTIONS = {
    "fused": dict(use_qk_norm=True, fused_qk_norm=True),
    "first_half": dict(use_qk_norm=True, qk_norm_first=True, rope_layout="half"),
    "part_no_norm": dict(rope_layout="half", rope_fraction=0.5),
    "yarn": dict(use_qk_norm=True, fused_qk_norm=True, rope_scaling_method="yarn",
                 rope_scaling=dict(factor=4.0, original_max_position_embeddings=256)),
    "heads_of_64": dict(use_qk_norm=True, fused_qk_norm=True, num_attention_heads=8, num_key_value_heads=2),
}


@pytest.mark.parametrize("name", list(OPTIONS))
def test_forward_and_backward_match_the_cpu(name):
    """Bounds as for the framework's other models on the GPU: activations are rounded to bfloat16 (2^-8) some ten
    times a layer."""
    cpu, gpu = _models(**OPTIONS[name])
    ids = torch.randint(0, 512, (2, 200), generator=torch.Generator().manual_seed(1))
    seg = torch.zeros(2, 200, dtype=torch.int32)
    seg[0, 90:] = 1
    a = cpu(ids, seg_ids=seg)["logits"]
    b = gpu(ids.cuda(), seg_ids=seg.cuda())["logits"]
    assert _rel(b, a) < 0.02
    w = torch.randn(a.shape, generator=torch.Generator().manual_seed(2))
    (a * w).sum().backward()
    (b.float() * w.cuda()).sum().backward()
    for (n, p), q in zip(cpu.named_parameters(), gpu.parameters()):
        assert _rel(q.grad, p.grad) < 0.05, n


def test_one_pass_is_nearer_to_the_cpu_than_the_separate_path():
    ids = torch.randint(0, 512, (2, 300), generator=torch.Generator().manual_seed(1))
    off = {}
    for fused in (False, True):
        cpu, gpu = _models(use_qk_norm=True, fused_qk_norm=fused)
        with torch.no_grad():
            off[fused] = _rel(gpu(ids.cuda())["logits"], cpu(ids)["logits"])
    assert off[True] <= off[False] * 1.1  # a rounding less; 10 % for chance


def _steps(model, cache, prompts, steps, tokens):
    dev = "cuda"
    tids = [f"t{i}" for i in range(len(prompts))]
    out, lens = [], [len(p) for p in prompts]
    with torch.inference_mode():
        for tid, ids in zip(tids, prompts):
            assert cache.task_alloc(tid, ids)
            view = cache.bind([tid], [len(ids)], len(ids), dev, uniform_start=0)
            model(torch.tensor([ids], device=dev), paged_cache=view,
                  position_ids=torch.arange(len(ids), device=dev)[None], logits_to_keep=1)
        for s in range(steps):
            for tid, n in zip(tids, lens):
                assert cache.task_extend(tid, n)
            view = cache.bind(tids, [n + 1 for n in lens], 1, dev)
            out.append(model(tokens[s], paged_cache=view, position_ids=torch.tensor(lens, device=dev)[:, None],
                             logits_to_keep=1)["logits"][:, -1])
            lens = [n + 1 for n in lens]
    return torch.stack(out)


@pytest.mark.parametrize("name", ["fused", "first_half", "heads_of_64", "plain", "fp16"])
def test_int8_decode_stays_near_the_unrounded_cache(name):
    """Half a step of 1/127 of a block's largest magnitude: about 0.2 - 0.4 % of k and v in norm, which the random
    model's logits pass on; the bound is the one of the CPU test plus the 16-bit roundings of both sides."""
    from astrai_b200.inference import ContiguousCache, PageCache

    _, model = _models(**OPTIONS.get(name, {}))
    model = model.eval()
    if name == "fp16":
        model = model.to(torch.float16)
    cfg, dt = model.config, next(model.parameters()).dtype
    hd = cfg.hidden_size // cfg.num_attention_heads
    prompts = [list(range(3, 150)), list(range(90, 95)), [11], list(range(200, 400))]
    tokens = torch.randint(0, 512, (6, 4, 1), generator=torch.Generator().manual_seed(3)).cuda()

    def caches(kv):
        yield PageCache(2, 40, 64, cfg.num_key_value_heads, hd, "cuda", dt, kv)
        yield ContiguousCache(2, 4, 400, cfg.num_key_value_heads, hd, "cuda", dt, kv)

    for plain, int8 in zip(caches(None), caches("int8")):
        a, b = _steps(model, plain, prompts, 6, tokens), _steps(model, int8, prompts, 6, tokens)
        assert _rel(b, a) < 0.03


def test_prefill_behind_shared_pages_and_rows_of_several_tokens():
    from astrai_b200.inference import PageCache

    _, model = _models()
    model, cfg = model.eval(), model.config
    ids = torch.randint(0, 512, (300,), generator=torch.Generator().manual_seed(5)).tolist()
    cache = PageCache(2, 20, 64, 2, 128, "cuda", torch.bfloat16, "int8")
    with torch.inference_mode():
        assert cache.task_alloc("a", ids)
        full = model(torch.tensor([ids], device="cuda"), paged_cache=cache.bind(["a"], [300], 300, "cuda", uniform_start=0),
                     position_ids=torch.arange(300, device="cuda")[None])["logits"]
        cache.task_record_hashes("a", ids)
        assert cache.task_alloc("b", ids) and cache.task_cached("b") == 256
        for n in (44, 20):  # gathered for the prefill kernel; in place
            view = cache.bind(["b"], [256 + n], n, "cuda", uniform_start=256)
            rest = model(torch.tensor([ids[256: 256 + n]], device="cuda"), paged_cache=view,
                         position_ids=torch.arange(256, 256 + n, device="cuda")[None])["logits"]
            assert _rel(rest, full[:, 256: 256 + n]) < 0.03
        # rows of different lengths, several new tokens each
        assert cache.task_alloc("c", ids[:100])
        model(torch.tensor([ids[:96]], device="cuda"), paged_cache=cache.bind(["c"], [96], 96, "cuda", uniform_start=0),
              position_ids=torch.arange(96, device="cuda")[None], logits_to_keep=1)
        view = cache.bind(["b", "c"], [260, 100], 4, "cuda")
        pos = torch.tensor([[256, 257, 258, 259], [96, 97, 98, 99]], device="cuda")
        new = torch.tensor([ids[256:260], ids[96:100]], device="cuda")
        both = model(new, paged_cache=view, position_ids=pos)["logits"]
    assert _rel(both[0], full[0, 256:260]) < 0.03 and _rel(both[1], full[0, 96:100]) < 0.03


@pytest.mark.parametrize("kv_dtype", [None, "int8"])
def test_one_pass_over_a_cache_outside_no_grad(kv_dtype):
    """A forward over a cache has no gradient and needs no no_grad() around it."""
    from astrai_b200.inference import PageCache

    _, model = _models(**OPTIONS["fused"])
    model = model.eval()
    ids, outs = list(range(7, 60)), []
    for grad in (True, False):
        cache = PageCache(2, 8, 64, 2, 128, "cuda", torch.bfloat16, kv_dtype)
        assert cache.task_alloc("a", ids)
        with torch.set_grad_enabled(grad):
            outs.append(model(torch.tensor([ids], device="cuda"), position_ids=torch.arange(53, device="cuda")[None],
                              paged_cache=cache.bind(["a"], [53], 53, "cuda", uniform_start=0))["logits"].detach())
    assert torch.equal(*outs)


def test_rows_shorter_than_the_step():
    """Four tokens a row of which one row has two: its first two have no position and are not kept."""
    from astrai_b200.inference import PageCache
    from astrai_b200.ops._ext import native

    _, model = _models()
    model = model.eval()
    ids = torch.randint(0, 512, (2, 4), generator=torch.Generator().manual_seed(3))
    cache = PageCache(2, 8, 64, 2, 128, "cuda", torch.bfloat16, "int8")
    with torch.inference_mode():
        for name, n in (("a", 4), ("b", 2), ("c", 2)):
            assert cache.task_alloc(name, [1] * n)
        pos = torch.tensor([[0, 1, 2, 3], [0, 0, 0, 1]], device="cuda")
        both = model(ids.cuda(), paged_cache=cache.bind(["a", "b"], [4, 2], 4, "cuda"), position_ids=pos)["logits"]
        alone = model(ids[1:, 2:].cuda(), paged_cache=cache.bind(["c"], [2], 2, "cuda"),
                      position_ids=torch.arange(2, device="cuda")[None])["logits"]
    torch.cuda.synchronize()
    native().read_error()  # the rotation records positions before 0
    assert _rel(both[1, 2:], alone[0]) < 0.03


@pytest.mark.parametrize("paged", [False, True])
def test_graph_decode_equals_eager_decode(paged):
    from astrai_b200.inference import ContiguousCache, PageCache
    from astrai_b200.inference.core.executor import Executor
    from astrai_b200.inference.core.task import Task

    _, model = _models(**OPTIONS["fused"])
    model = model.eval()
    outs = []
    for graph in (False, True):
        cache = PageCache(2, 40, 64, 2, 128, "cuda", torch.bfloat16, "int8") if paged else \
            ContiguousCache(2, 4, 300, 2, 128, "cuda", torch.bfloat16, "int8")
        ex = Executor(model, None, cache, use_cuda_graph=graph, max_batch_size=4, max_seq_len=300, seed=0)
        tasks = [Task(f"t{i}", list(range(5 + i, 40 + 30 * i)), 12, temperature=0.0, top_p=1.0, top_k=0) for i in range(3)]
        for t in tasks:
            assert cache.task_alloc(t.task_id, t.prompt_ids)
            assert cache.task_extend(t.task_id, 290)
            ex.execute_prefill([t], len(t.prompt_ids), 0)
        for _ in range(8):
            ex.execute_decode(tasks)
        outs.append([t.output_ids for t in tasks])
    assert outs[0] == outs[1]


def test_engine_serves_from_an_int8_cache(test_tokenizer):
    from astrai_b200.inference import InferenceEngine
    from astrai_b200.models import AutoRegressiveLM

    torch.manual_seed(0)
    model = AutoRegressiveLM(_cfg(vocab_size=len(test_tokenizer), **OPTIONS["first_half"])).to("cuda", torch.bfloat16).eval()
    for kw in (dict(n_pages=64, page_size=64), {}):
        with InferenceEngine(model, test_tokenizer, max_batch_size=4, max_seq_len=256, kv_cache_dtype="int8", **kw) as eng:
            out = eng.generate(["hello world", "abc"], max_tokens=12, temperature=0.0)
            assert len(out) == 2 and out == eng.generate(["hello world", "abc"], max_tokens=12, temperature=0.0)


def test_training_micro_step_replays_from_a_graph():
    """The one-pass layer inside a captured forward + backward."""
    _, model = _models(**OPTIONS["fused"])
    ids = torch.randint(0, 512, (2, 128), device="cuda")

    def step():
        for p in model.parameters():
            if p.grad is not None:
                p.grad.zero_()
        model(ids)["logits"].float().square().mean().backward()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    want = [p.grad.clone() for p in model.parameters()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for p in model.parameters():
        p.grad.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    for p, w in zip(model.parameters(), want):
        assert _rel(p.grad, w) < 1e-2
