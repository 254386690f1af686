"""Attention over the 8-bit cache where one key outweighs a long tail: the tail's weights keep their bits.

Tolerance of an output: u |o| for its own rounding (u half the spacing of its type) and, times the sum over keys of
p_j |v_j|: 2^-22 for a weight held as two fp16 numbers, 2^-22 for each of two exp2, 2^-22 |log2 absmax| for a log2, at
most 2^-18 for fp32 sums over up to 64 tiles of a warp and the merges (together 2^-17), and the scores' own error: 16
fp32 sums of at most `reach` = 2 scale log2(e) absmax sum |q|, 2^-20 reach. What two fp16 numbers cannot hold of a
weight is below 2^-25; the largest weight is kept at 2^7 or more, so that is 2^-32 of the largest probability, per key,
times the largest value.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_SPACING = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(autouse=True)
def _clean_error_word():
    from astrai_b200.ops._ext import native

    native().read_error()
    yield
    torch.cuda.synchronize()
    assert native().read_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ahead", [9.3, 14.7, 17.6, 20.6])
@pytest.mark.parametrize("n,S,Hq,Hkv,D", [(200, 1, 4, 1, 64), (200, 1, 8, 2, 128), (3000, 1, 4, 1, 128), (900, 4, 16, 4, 128),
                                          (200, 4, 4, 1, 64)])
@pytest.mark.parametrize("at", [0, 1])
def test_a_tail_far_behind_one_key_keeps_its_bits(n, S, Hq, Hkv, D, ahead, dtype, at):
    """Key `at` (first or last) is 2^ahead ahead of all others and has the value 0: the output is the tail's alone."""
    from astrai_b200.ops.kv8 import KV8, kv8_attention

    page, block = 64, 32
    width = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(11)
    c = KV8.allocate(width, Hkv, page, D, block, "cuda")
    c.k_absmax.fill_(1.0)
    c.v_absmax.fill_(0.75)
    c.v.copy_(torch.randint(1, 128, c.v.shape, device="cuda", generator=g, dtype=torch.int8))
    table = torch.randperm(width, generator=torch.Generator().manual_seed(1)).int().view(1, -1).cuda()
    big = (n - S) * at  # seen by every query
    p, off = int(table[0, big // page]), big % page
    c.k[p, :, off, 0] = 127
    c.v[p, :, off] = 0
    scale = 1 / math.sqrt(D)
    q = torch.zeros(1, S, Hq, D, device="cuda", dtype=dtype)
    q[..., 0] = ahead / (scale * math.log2(math.e))
    got = kv8_attention(q, c, table, torch.tensor([n], dtype=torch.int32, device="cuda")).double()
    pages = table[0].long()
    k, v = (x[pages].transpose(0, 1).flatten(1, 2)[:, :n].double() * a / 127 for x, a in ((c.k, 1.0), (c.v, 0.75)))
    reach = 2 * scale * math.log2(math.e) * q.double().abs().sum(-1).max().item()
    for i in range(S):
        m = n - S + i + 1
        for h in range(Hq):
            prob = torch.softmax(k[h // (Hq // Hkv), :m] @ q[0, i, h].double() * scale, 0)
            want = prob @ v[h // (Hq // Hkv), :m]  # the values are positive: also the sum of p |v|
            tol = HALF_SPACING[dtype] * want + (2.0 ** -17 + 2.0 ** -20 * reach) * want \
                + m * 2.0 ** -32 * prob.max() * 0.75
            assert ((got[0, i, h] - want).abs() <= tol).all(), ((got[0, i, h] - want).abs() / tol).max().item()


def test_a_block_that_reads_as_nan_reaches_only_the_queries_that_see_it():
    from astrai_b200.ops.kv8 import KV8, kv8_append, kv8_attention

    B, H, D, page, block, n, S = 2, 2, 64, 32, 16, 34, 4
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(B, n, H, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    i32 = dict(dtype=torch.int32, device="cuda")
    table, zero, lens = torch.tensor([[0, 1], [2, 3]], **i32), torch.zeros(B, **i32), torch.full((B,), n, **i32)
    clean, dirty = (KV8.allocate(4, H, page, D, block, "cuda") for _ in range(2))
    kv8_append(clean, k, v, table, zero, lens)
    for x in (k, v):
        x[0, 33, 1] = float("nan")  # token 33 shares its block with token 32 alone
    kv8_append(dirty, k, v, table, zero, lens)
    for heads in (2, 4, 16):  # two, four and sixteen query rows of a KV head
        q = torch.randn(B, S, heads, D, device="cuda", generator=g).bfloat16()
        want, got = kv8_attention(q, clean, table, lens), kv8_attention(q, dirty, table, lens)
        bad = torch.zeros(B, S, heads, dtype=torch.bool, device="cuda")
        bad[0, 2:, heads // 2:] = True  # tokens 32 and 33, the query heads of KV head 1
        assert torch.equal(got.isnan().all(-1), bad) and torch.equal(got.isnan().any(-1), bad)
        assert torch.equal(got[~bad], want[~bad])
