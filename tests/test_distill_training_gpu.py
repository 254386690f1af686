"""The operators over rows of logits as the framework's own paths call them: the distill strategy, eager and from a CUDA
graph, and the executor's mixed batches."""

import copy
import types

import pytest
import torch

from tests.test_graph_step_gpu import _model

pytestmark = pytest.mark.gpu


def _strategy(model, teacher, accum):
    from astrai_b200.trainer.strategy import StrategyFactory

    return StrategyFactory.create("distill", model=model, device="cuda", teacher_model=teacher,
                                  executor=types.SimpleNamespace(grad_accum_steps=accum), distill_top_k=32,
                                  distill_temperature=2.0, distill_hard_weight=0.25)


def test_strategy_against_the_operators_in_their_order():
    """Teacher's rows -> tokens drawn from the student -> loss -> gradients, as one training step has them."""
    from astrai_b200.inference.sample import sample_given
    from astrai_b200.ops.distill import distill_loss, top_logits

    student, teacher = _model(), _model()
    with torch.no_grad():
        for p in teacher.parameters():
            p.add_(0.05 * torch.randn_like(p))
    ids = torch.randint(0, 512, (3, 65), device="cuda")
    with torch.no_grad():
        top = top_logits(teacher(input_ids=ids[:, :-1])["logits"], 32, 2.0)
    logits = student(input_ids=ids[:, :-1])["logits"]
    drawn = sample_given(logits.detach().flatten(0, 1), torch.rand(3 * 64, device="cuda"), top_k=50, min_p=0.01).view(3, 64)
    want = distill_loss(logits, top, 2.0, drawn, 0.25)
    loss = _strategy(student, teacher, 1)({"input_ids": ids[:, :-1], "target_ids": drawn})
    assert torch.equal(loss, want)
    grads = []
    for x in (loss, want):
        student.zero_grad(set_to_none=True)
        x.backward()
        grads.append([p.grad.clone() for p in student.parameters()])
    assert all(torch.equal(a, b) and torch.isfinite(a.float()).all() for a, b in zip(*grads))


def test_graphed_micro_step_matches_eager():
    from astrai_b200.optim import FusedAdamW
    from astrai_b200.trainer.graph_step import GraphedMicroStep

    teacher = _model().requires_grad_(False).eval()
    with torch.no_grad():
        for p in teacher.parameters():
            p.add_(0.05 * torch.randn_like(p))
    ma = _model()
    mb = copy.deepcopy(ma)
    accum = 2
    oa, ob = FusedAdamW(ma.parameters(), lr=1e-3), FusedAdamW(mb.parameters(), lr=1e-3)
    fa = _strategy(ma, teacher, accum)
    step = GraphedMicroStep(_strategy(mb, teacher, accum), mb, torch.device("cuda"), scale=1.0 / accum, eager_calls=accum)
    g = torch.Generator().manual_seed(1)
    data = torch.randint(0, 512, (4, accum, 2, 129), generator=g).pin_memory()
    for s in range(4):
        for mi in range(accum):
            x = data[s, mi]
            batch = {"input_ids": x[:, :-1], "target_ids": x[:, 1:], "loss_mask": x[:, 1:] > 100}
            loss = fa(batch)
            (loss / accum).backward()
            got = step(batch)
            # the same kernels on weights that the optimizer keeps within bf16 rounding of each other
            assert abs(float(got) - float(loss.detach())) <= 1e-3 * abs(float(loss.detach()))
        for o in (oa, ob):
            o.step()
            o.zero_grad(set_to_none=False)
    torch.cuda.synchronize()
    assert step.disabled_reason is None and step.replays == 4 * accum - accum - 1
    for pa, pb in zip(ma.parameters(), mb.parameters()):
        assert torch.allclose(pa.float(), pb.float(), rtol=1e-2, atol=1e-3)


def test_executor_samples_mixed_batches():
    from astrai_b200.inference.core.executor import Executor
    from astrai_b200.inference.core.task import Task
    from astrai_b200.inference.sample import sample_given

    ex = Executor(_model().eval(), None, None, seed=0)
    logits = (2 * torch.randn(5, 512, device="cuda")).bfloat16()
    tasks = [Task("a", [1], 4, temperature=0.8, top_k=0, seed=3), Task("b", [1], 4, temperature=0.0),
             Task("c", [1], 4, top_k=7, min_p=0.2, seed=4), Task("d", [1], 4, top_k=1),
             Task("e", [1], 4, top_k=0, frequency_penalty=0.5)]
    toks, lps = ex._sample(logits, tasks)
    for i in (0, 2):
        t = tasks[i]
        want, lp = sample_given(logits[i: i + 1], torch.tensor([t.uniform()], dtype=torch.float64, device="cuda"),
                                temperature=t.temperature, top_k=t.top_k, top_p=t.top_p, min_p=t.min_p, return_logprobs=True)
        assert toks[i] == int(want) and lps[i] == float(lp)
    assert toks[1] == int(logits[1].float().argmax()) and toks[3] == int(logits[3].float().argmax())
    assert 0 <= toks[4] < 512
    alone, _ = ex._sample(logits[2:3], [tasks[2]])
    assert alone == [toks[2]]


def test_engine_with_seeds():
    from astrai_b200.inference.engine import InferenceEngine
    from tests.test_inference_gpu import _Tok, _gpu_model

    with InferenceEngine(_gpu_model(), _Tok(), max_batch_size=3, max_seq_len=128, use_cuda_graph=True) as eng:
        kw = dict(max_tokens=6, temperature=1.0, top_k=20)
        first = eng.generate("5 6 7 8", seed=11, **kw)
        assert eng.generate("5 6 7 8", seed=11, **kw) == first
        greedy = eng.generate("5 6 7 8", max_tokens=6, temperature=0.0)
        assert eng.generate("5 6 7 8", max_tokens=6, temperature=1.0, top_k=0, min_p=1.0) == greedy


def test_a_seeded_request_leaves_its_batch_on_the_decode_graph():
    from astrai_b200.inference.core.scheduler import InferenceScheduler
    from astrai_b200.inference.core.task import Task
    from tests.test_inference_gpu import _Tok, _gpu_model

    sch = InferenceScheduler(_gpu_model(), _Tok(), max_batch_size=4, max_seq_len=128, use_cuda_graph=True)
    replays, graphs = [], sch._executor._graphs
    run = graphs.run
    graphs.run = lambda tasks: replays.append(len(tasks)) or run(tasks)

    def generate(*settings):
        replays.clear()
        tasks = [Task(str(i), [5 + i, 6, 7 + i], 8, **{"top_k": 0, **s}) for i, s in enumerate(settings)]
        sch._run_wave(tasks)
        assert len(replays) == max(len(t.output_ids) for t in tasks) - 1
        return [(t.output_ids, t.output_logprobs) for t in tasks]

    greedy = dict(temperature=0.0)
    alone = generate(greedy, greedy, greedy)
    # min-p of one keeps the largest logit alone: drawn from this step's logits, or it would be another token
    mixed = generate(greedy, dict(min_p=1.0, seed=4), greedy)
    assert [ids for ids, _ in mixed] == [ids for ids, _ in alone] and mixed[0] == alone[0] and mixed[2] == alone[2]
    seeded = generate(dict(seed=11), greedy, dict(seed=12, min_p=0.02))
    assert seeded[1] == alone[1] and generate(dict(seed=11), greedy, dict(seed=12, min_p=0.02)) == seeded
    assert generate(dict(temperature=0.0, seed=11), greedy, greedy) == alone
    assert all(0 <= i < 2048 and lp <= 0.0 for ids, lps in seeded for i, lp in zip(ids, lps))
