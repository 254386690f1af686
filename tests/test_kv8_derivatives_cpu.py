"""The 8-bit cache outside no_grad(): appends are updates of state and leave no graph behind."""

import torch

from astrai_b200.ops.kv8 import KV8, kv8_append, kv8_attention, kv8_gather


def test_append_leaves_no_graph():
    c, want = (KV8.allocate(2, 2, 32, 64, 16) for _ in range(2))
    table = torch.tensor([[0, 1]], dtype=torch.int32)
    torch.manual_seed(0)
    k, v = torch.randn(1, 20, 2, 64, requires_grad=True), torch.randn(1, 20, 2, 64, requires_grad=True)
    for first, end in ((0, 18), (18, 20)):
        args = (table, torch.tensor([first]), torch.tensor([end]))
        kv8_append(c, k[:, first:end], v[:, first:end], *args)
        kv8_append(want, k.detach()[:, first:end], v.detach()[:, first:end], *args)
    assert not any(t.requires_grad for t in c) and all(torch.equal(a, b) for a, b in zip(c, want))
    lens = torch.tensor([20])
    assert not any(t.requires_grad for t in kv8_gather(c, table, lens, 20, dtype=torch.float32))
    assert not kv8_attention(torch.randn(1, 1, 4, 64), c, table, lens).requires_grad
