"""8-bit paged KV cache on the CPU: the plain functions against their definitions. (The kernels are tested in
test_kv8_gpu.py, against oracles of their own.)"""

import math

import pytest
import torch

from astrai_b200.ops.kv8 import KV8, kv8_append, kv8_attention, kv8_gather


def _filled(B=3, width=3, H=2, page=32, D=64, block=16, lens=(70, 1, 33), seed=0):
    torch.manual_seed(seed)
    c = KV8.allocate(B * width + 1, H, page, D, block)
    table = torch.randperm(B * width + 1)[: B * width].view(B, width).int()
    S = max(lens)
    k, v = torch.randn(B, S, H, D), torch.randn(B, S, H, D)
    lens = torch.tensor(lens, dtype=torch.int32)
    kv8_append(c, k, v, table, torch.zeros(B, dtype=torch.int32), lens)
    return c, table, k, v, lens


def test_append_and_gather_round_to_half_a_step():
    c, table, k, v, lens = _filled()
    ko, vo = kv8_gather(c, table, lens, 80, dtype=torch.float32)
    for x, got in ((k, ko), (v, vo)):
        for b, n in enumerate(lens.tolist()):
            assert (got[b, n:] == 0).all()
            for at in range(0, n, 16):
                y = x[b, at: min(at + 16, n)]
                step = y.abs().amax((0, 2), keepdim=True) / 127
                assert ((got[b, at: at + y.shape[0]] - y).abs() <= step * (0.5 + 1e-5)).all()
    first, _ = kv8_gather(c, table, lens, 5, starts=torch.tensor([65, 0, 31]), dtype=torch.float32)
    assert torch.equal(first[0], ko[0, 65:70]) and torch.equal(first[2, :2], ko[2, 31:33]) and (first[2, 2:] == 0).all()
    assert c.block == 16 and c.page_size == 32


def test_append_behind_live_tokens_and_growth():
    c, table, k, v, lens = _filled()
    old = kv8_gather(c, table, lens, 70, dtype=torch.float32)[0]
    big = torch.full((3, 2, 2, 64), 50.0)
    new = lens + torch.tensor([2, 2, 0], dtype=torch.int32)
    kv8_append(c, big, big, table, lens, new)
    ko = kv8_gather(c, table, new, 72, dtype=torch.float32)[0]
    assert (ko[0, 70:72] == 50).all() and (ko[1, 1:3] == 50).all() and torch.equal(ko[2, :33], old[2, :33])
    assert torch.equal(ko[0, :64], old[0, :64])  # earlier blocks do not change
    assert ((ko[0, 64:70] - old[0, 64:70]).abs() <= 50 / 127 * 0.5 + 1e-5).all()
    # an append at an earlier position truncates: the block starts again under its own magnitude
    small = torch.full((3, 1, 2, 64), 0.25)
    kv8_append(c, small, small, table, torch.tensor([64, 0, 32]), torch.tensor([65, 1, 33]))
    got = kv8_gather(c, table, torch.tensor([65, 1, 33]), 65, dtype=torch.float32)[0]
    assert (got[0, 64] == 0.25).all() and (got[1, 0] == 0.25).all() and (got[2, 32] == 0.25).all()


def test_tokens_before_position_zero_are_dropped():
    torch.manual_seed(1)
    k, v = torch.randn(3, 40, 2, 64), torch.randn(3, 40, 2, 64)
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32)
    starts, lens = torch.tensor([-3, -40, -39]), torch.tensor([37, 0, 5])  # row 2 ends with the tokens that it has
    c, want = (KV8.allocate(6, 2, 32, 64, 16) for _ in range(2))
    kv8_append(c, k, v, table, starts, lens)
    for b, n in ((0, 37), (2, 1)):
        kv8_append(want, k[b: b + 1, 40 - n:], v[b: b + 1, 40 - n:], table[b: b + 1], torch.tensor([0]), torch.tensor([n]))
    assert all(torch.equal(x, y) for x, y in zip(c, want)) and c.k[0].any()


def test_non_finite_blocks_and_missing_pages():
    c = KV8.allocate(4, 1, 32, 64, 16)
    table = torch.tensor([[0, 1], [-1, 9]], dtype=torch.int32)
    k = torch.ones(2, 40, 1, 64)
    k[0, 3, 0, 0] = float("inf")
    kv8_append(c, k, k, table, torch.zeros(2, dtype=torch.int32), torch.tensor([40, 40]))
    ko, _ = kv8_gather(c, table, torch.tensor([40, 40]), 40, dtype=torch.float32)
    assert ko[0, :16].isnan().all() and (ko[0, 16:] == 1).all() and (ko[1] == 0).all()


@pytest.mark.parametrize("S", [1, 3])
def test_attention_is_softmax_over_the_read_back_values(S):
    c, table, _, _, lens = _filled()
    q = torch.randn(3, S, 4, 64)
    k, v = kv8_gather(c, table, lens, 96, dtype=torch.float32)
    o = kv8_attention(q, c, table, lens)
    for b, n in enumerate(lens.tolist()):
        for i in range(S):
            m = n - S + i + 1
            if m <= 0:
                assert (o[b, i] == 0).all()
                continue
            for h in range(4):
                p = torch.softmax(k[b, :m, h // 2] @ q[b, i, h] / math.sqrt(64), 0)
                assert torch.allclose(o[b, i, h], p @ v[b, :m, h // 2], atol=1e-5)
    padded = kv8_attention(q, c, table, lens, starts=lens - 1)
    assert (padded[:, 1:] == 0).all()
    assert torch.allclose(padded[:, 0], kv8_attention(q[:, :1], c, table, lens)[:, 0], atol=1e-6)


def test_allocation_refusals():
    for bad in (dict(block=48), dict(block=8), dict(page_size=48, block=32)):
        args = dict(n_pages=2, n_kv_heads=1, page_size=64, head_dim=64, block=32)
        args.update(bad)
        with pytest.raises(ValueError):
            KV8.allocate(**args)
