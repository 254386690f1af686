"""The plain attention over the 8-bit cache: what a query does not see does not reach it."""

import torch

from astrai_b200.ops.kv8 import KV8, kv8_append, kv8_attention


def test_a_block_that_reads_as_nan_reaches_only_the_queries_that_see_it():
    torch.manual_seed(0)
    B, H, D, page, block, n, S = 2, 2, 64, 32, 16, 34, 4
    k, v = torch.randn(B, n, H, D), torch.randn(B, n, H, D)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    zero, lens = torch.zeros(B, dtype=torch.int32), torch.full((B,), n, dtype=torch.int32)
    clean, dirty = (KV8.allocate(4, H, page, D, block) for _ in range(2))
    kv8_append(clean, k, v, table, zero, lens)
    for x in (k, v):
        x[0, 33, 1] = float("nan")  # token 33 shares its block with token 32 alone
    kv8_append(dirty, k, v, table, zero, lens)
    q = torch.randn(B, S, 4, D)
    want, got = kv8_attention(q, clean, table, lens), kv8_attention(q, dirty, table, lens)
    bad = torch.zeros(B, S, 4, dtype=torch.bool)
    bad[0, 2:, 2:] = True  # tokens 32 and 33, the query heads of KV head 1
    assert torch.equal(got.isnan().all(-1), bad) and torch.equal(got.isnan().any(-1), bad)
    assert torch.equal(got[~bad], want[~bad])
