"""Distillation through the trainer's own path, and seeded / min-p generation through the engine, on the CPU."""

import math

import pytest
import torch

from tests.conftest import TINY_CFG
from tests.test_inference_cpu import _Tok, _model
from tests.test_trainer_cpu import RandSeq, make_cfg


def _teacher():
    from astrai_b200.config import AutoRegressiveLMConfig
    from astrai_b200.models import AutoRegressiveLM

    torch.manual_seed(3)
    return AutoRegressiveLM(AutoRegressiveLMConfig(**TINY_CFG))


def test_trainer_distills(tmpdir_path):
    from astrai_b200.trainer import Trainer

    t = Trainer(make_cfg(RandSeq(8), tmpdir_path, strategy="distill", teacher_fn=_teacher,
                         extra_kwargs={"distill_top_k": 16, "distill_temperature": 2.0, "distill_hard_weight": 0.3}))
    t.train()
    ctx = t.last_context
    assert math.isfinite(ctx.loss) and ctx.optimizer_step == 2
    assert not any(p.requires_grad for p in ctx.strategy.teacher_model.parameters())


def test_strategy_against_the_operators():
    from astrai_b200.config import AutoRegressiveLMConfig
    from astrai_b200.models import AutoRegressiveLM
    from astrai_b200.ops.distill import TopLogits, distill_loss, top_logits
    from astrai_b200.trainer.strategy import StrategyFactory, doc_ids_from_positions

    torch.manual_seed(0)
    student, teacher = AutoRegressiveLM(AutoRegressiveLMConfig(**TINY_CFG)), _teacher()
    ids = torch.randint(0, 512, (2, 17))
    pos = torch.arange(16).repeat(2, 1)
    pos[:, 9:] -= 9
    mask = torch.rand(2, 16) < 0.7
    batch = {"input_ids": ids[:, :-1], "target_ids": ids[:, 1:], "position_ids": pos, "loss_mask": mask}
    kw = dict(distill_top_k=20, distill_temperature=1.5, distill_hard_weight=0.25)
    loss = StrategyFactory.create("distill", model=student, device="cpu", teacher_model=teacher, **kw)(batch)
    inputs = dict(input_ids=ids[:, :-1], position_ids=pos, seg_ids=doc_ids_from_positions(pos))
    with torch.no_grad():
        top = top_logits(teacher(**inputs)["logits"], 20, 1.5)
    want = distill_loss(student(**inputs)["logits"], top, 1.5, ids[:, 1:].masked_fill(~mask, -100), 0.25)
    assert torch.equal(loss, want)
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in student.parameters())
    # the teacher's rows with the batch
    stored = {**batch, "teacher_ids": top.ids, "teacher_logits": top.values, "teacher_rest": top.rest}
    again = StrategyFactory.create("distill", model=student, device="cpu", **kw)(stored)
    assert torch.equal(again, want)
    with pytest.raises(ValueError, match="teacher"):
        StrategyFactory.create("distill", model=student, device="cpu", **kw)(batch)
    assert isinstance(top, TopLogits)


def test_cli_builds_a_teacher(tmpdir_path):
    import os

    from astrai_b200.cli.train import build_config, parse_args
    from astrai_b200.dataset import DatasetFactory

    assert "distill" in DatasetFactory.list_registered()
    here = os.path.join(tmpdir_path, "m")
    _teacher().save_pretrained(here)
    args = parse_args(["--train_type", "distill", "--data_root_path", here, "--param_path", here])
    with pytest.raises(ValueError, match="teacher_path"):
        build_config(args)


def test_seeded_generation_repeats_in_any_batch():
    from astrai_b200.inference import InferenceEngine

    def run(prompts, **kw):
        with InferenceEngine(_model(), _Tok(), max_batch_size=3, max_seq_len=48) as eng:
            return eng.generate(prompts, max_tokens=8, temperature=1.0, top_k=0, **kw)

    alone = [run("1 2", seed=5), run("3 4 5", seed=6), run("1 2", seed=7)]
    assert run(["1 2", "3 4 5", "1 2"], seed=5) == alone
    assert alone[0] != alone[2]


def test_min_p_of_one_is_greedy_and_rows_may_differ():
    from astrai_b200.inference import InferenceEngine

    with InferenceEngine(_model(), _Tok(), max_batch_size=3, max_seq_len=48) as eng:
        greedy = eng.generate(["1 2", "3 4 5"], max_tokens=8, temperature=0.0)
        assert eng.generate(["1 2", "3 4 5"], max_tokens=8, temperature=1.0, top_k=0, min_p=1.0) == greedy
        # tokens only: the model's logits are rounded differently in batches of other sizes
        out = eng.scheduler.run_batch([[1, 2], [3, 4, 5], [6]], max_tokens=4, temperature=1.0, seeds=[1, 2, 3])
        again = eng.scheduler.run_batch([[6], [1, 2]], max_tokens=4, temperature=1.0, seeds=[3, 1])
        assert out[2] == again[0] and out[0] == again[1]
        with pytest.raises(ValueError, match="seeds"):
            eng.scheduler.run_batch([[1]], seeds=[1, 2])
        for bad in (dict(min_p=1.5), dict(seed=1.5), dict(seed=3, frequency_penalty=0.5), dict(min_p=0.1, frequency_penalty=0.5)):
            with pytest.raises(ValueError):
                eng.generate("1 2", max_tokens=2, **bad)


def test_mixed_batch_keeps_the_other_rows_sampler():
    """A seeded row does not change how the others are drawn."""
    from astrai_b200.inference.core.task import Task

    a, b = Task("a", [1], 4, seed=9), Task("b", [1], 4)
    assert a.given and not b.given and b.uniform() is None
    first = a.uniform()
    assert 0.0 <= first < 1.0 and first == Task("c", [2, 3], 9, seed=9).uniform()
    a.output_ids.append(5)
    assert a.uniform() != first
    with pytest.raises(ValueError, match="penalty"):
        Task("d", [1], 4, seed=9, frequency_penalty=0.2)
    spread = torch.tensor([Task("e", [1], 1, seed=s).uniform() for s in range(2000)])
    # the mean of 2000 even numbers is within five standard deviations, 0.2887 / sqrt(2000) = 0.0065 each
    assert abs(float(spread.mean()) - 0.5) < 5 * 0.0065


def test_server_takes_min_p_and_seed():
    from astrai_b200.inference.api.protocol import ProtocolHandler
    from astrai_b200.inference.api.server import ChatCompletionRequest, MessagesRequest

    class Engine:
        def generate_async(self, prompt, **kw):
            self.kw = kw

    def sent(cls, **kw):
        engine = Engine()
        message = {"role": "user", "content": "x"}
        ProtocolHandler(cls(messages=[message], **kw), engine, None)._agen("x")
        return engine.kw

    plain = sent(ChatCompletionRequest)
    assert "min_p" not in plain and "seed" not in plain
    assert sent(ChatCompletionRequest, seed=4)["seed"] == 4
    assert sent(ChatCompletionRequest, min_p=0.1)["min_p"] == 0.1
    assert sent(MessagesRequest, min_p=0.1)["min_p"] == 0.1
    assert "seed" not in sent(ChatCompletionRequest, seed=4, frequency_penalty=0.5)


def test_a_seed_at_temperature_0_draws_nothing():
    from astrai_b200.inference.core.task import Task

    assert not Task("a", [1], 4, temperature=0.0, seed=9).given and not Task("b", [1], 4, temperature=0.0, min_p=0.1).given
    assert Task("c", [1], 4, temperature=0.5, seed=9).given and Task("d", [1], 4, temperature=0.5, min_p=0.1).given
    with pytest.raises(ValueError, match="penalty"):
        Task("e", [1], 4, temperature=0.0, seed=9, frequency_penalty=0.2)


def test_teacher_with_a_larger_vocabulary_is_refused():
    from astrai_b200.config import AutoRegressiveLMConfig
    from astrai_b200.models import AutoRegressiveLM
    from astrai_b200.trainer.strategy import StrategyFactory

    student = AutoRegressiveLM(AutoRegressiveLMConfig(**TINY_CFG))
    ids = torch.randint(0, 400, (2, 9))
    batch = {"input_ids": ids[:, :-1], "target_ids": ids[:, 1:]}
    for more in (8, -8):
        teacher = AutoRegressiveLM(AutoRegressiveLMConfig(**{**TINY_CFG, "vocab_size": TINY_CFG["vocab_size"] + more}))
        strategy = StrategyFactory.create("distill", model=student, device="cpu", teacher_model=teacher)
        if more > 0:
            with pytest.raises(ValueError, match="vocabulary"):
                strategy(batch)
        else:
            assert torch.isfinite(strategy(batch))


def test_cli_trains_towards_a_saved_teacher(tmpdir_path):
    """The command's own configuration, on sft data, builds the saved teacher and runs steps towards it."""
    import os

    from astrai_b200.cli.train import build_config, parse_args
    from astrai_b200.serialization import save_bin
    from astrai_b200.trainer import Trainer

    student, there, data = (os.path.join(tmpdir_path, n) for n in ("student", "teacher", "data"))
    teacher = _teacher()
    teacher.save_pretrained(there)
    teacher.save_pretrained(student)
    g = torch.Generator().manual_seed(0)
    save_bin(data, {"sequence": [torch.randint(0, 512, (200,), generator=g) for _ in range(2)],
                    "loss_mask": [torch.randint(0, 2, (200,), generator=g) for _ in range(2)],
                    "position_ids": [torch.arange(200) % 50 for _ in range(2)]})
    cfg = build_config(parse_args([
        "--train_type", "distill", "--teacher_path", there, "--param_path", student, "--data_root_path", data,
        "--window_size", "32", "--batch_per_device", "2", "--grad_accum_steps", "1", "--n_epoch", "1", "--ckpt_dir",
        os.path.join(tmpdir_path, "ckpt"), "--log_dir", os.path.join(tmpdir_path, "logs"), "--device_type", "cpu",
        "--backend", "gloo", "--num_workers", "0", "--distill_top_k", "9", "--distill_temperature",
        "2.0", "--distill_hard_weight", "0.25"]))
    built = cfg.teacher_fn()
    assert all(p.dtype == torch.bfloat16 and torch.equal(p, q.bfloat16()) for p, q in zip(built.parameters(), teacher.parameters()))
    assert {k: v for k, v in cfg.extra_kwargs.items() if k.startswith("distill")} == {
        "distill_top_k": 9, "distill_temperature": 2.0, "distill_hard_weight": 0.25}
    batch = torch.utils.data.default_collate([cfg.dataset[i] for i in range(2)])
    assert batch["input_ids"].shape == (2, 32) and "loss_mask" in batch and "position_ids" in batch
    t = Trainer(cfg)
    t.train()
    ctx = t.last_context
    assert math.isfinite(ctx.loss) and ctx.optimizer_step > 0
    assert (ctx.strategy.top_k, ctx.strategy.temperature, ctx.strategy.hard_weight) == (9, 2.0, 0.25)
    assert not ctx.strategy.teacher_model.training
