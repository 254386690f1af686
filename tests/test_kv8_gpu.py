"""8-bit paged KV cache: append, read-back and attention kernels against 64-bit oracles.

What is stored is compared exactly: integers and magnitudes follow from 16-bit inputs without any rounding
that 64 bits would do differently. Read-back rounds once to its type. Attention: with u the half spacing of the
output's type, a result may be off by u |o| for its own rounding, and by the sum over keys of p_j |v_j| times
2^-11 (a weight held in fp16), 2^-12 (exp2, log2 and the running sums in fp32) and 2^-20 times the largest score
(scores are fp32 sums of exact products); weights below 2^-14 of the largest lose 2^-25 of it each.
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


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache(n_pages, Hkv, page, D, block, seed=0, spread=0.5):
    from astrai_b200.ops.kv8 import KV8

    g = _gen(seed)
    c = KV8.allocate(n_pages, Hkv, page, D, block, "cuda")
    for q, a in ((c.k, c.k_absmax), (c.v, c.v_absmax)):
        q.copy_(torch.randint(-127, 128, q.shape, device="cuda", generator=g, dtype=torch.int8))
        a.copy_(torch.exp(spread * torch.randn(a.shape, device="cuda", generator=g)).to(torch.bfloat16).float())
    return c


def _clone(c):
    return type(c)(*(t.clone() for t in c))


def _table(B, width, n_pages, seed=1):
    assert B * width <= n_pages
    p = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed))[: B * width]
    return p.view(B, width).int().cuda()


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _append_oracle(cache, k, v, table, starts, lens):
    """Token by token, block by block, in 64 bits on the CPU; -> the cache's tensors."""
    block, page = cache.block, cache.page_size
    kc, vc, ka, va = (t.cpu().clone() for t in cache)
    for b in range(k.shape[0]):
        s, e = int(starts[b]), int(lens[b])
        for base in range(s // block * block, e if e > s else 0, block):
            lp = base // page
            p = int(table[b, lp]) if lp < table.shape[1] else -1
            if p < 0 or p >= kc.shape[0]:
                continue
            for q, a, x in ((kc, ka, k), (vc, va, v)):
                for h in range(q.shape[1]):
                    new = {t: x[b, t - s, h].double().cpu() for t in range(max(base, s), min(base + block, e))}
                    most = max(float(t.abs().max()) for t in new.values())
                    was = float(a[p, h, base % page // block]) if base < s else 0.0
                    now = max(was, most)
                    for t in range(base, min(base + block, e)):
                        row = q[p, h, t % page]
                        if t >= s:
                            row.copy_(torch.round(new[t] * 127 / now) if now else torch.zeros_like(new[t]))
                        elif now > was:
                            row.copy_(torch.round(row.double() * was / now))
                    a[p, h, base % page // block] = now
    return kc, vc, ka, va


def _new(B, S, H, D, dtype, seed=2, scale=1.0):
    buf = (torch.randn(B, S, 3 * H, D, device="cuda", generator=_gen(seed)) * scale).to(dtype)
    return buf[:, :, H: 2 * H], buf[:, :, 2 * H:]  # strided: heads of one buffer


@pytest.mark.parametrize("page,block,D,H,S,starts,lens,dtype", [
    (16, 16, 64, 1, 1, [0, 5, 15, 16, 31], [1, 6, 16, 17, 32], torch.bfloat16),
    (64, 16, 128, 2, 1, [0, 1, 63, 64, 100], [1, 2, 64, 65, 100], torch.float16),
    (128, 32, 128, 3, 40, [0, 7, 31, 96, 120], [40, 47, 32, 136, 160], torch.bfloat16),
    (64, 64, 64, 2, 70, [0, 63, 64, 10, 0], [70, 100, 134, 10, 1], torch.bfloat16),
    (192, 64, 128, 1, 130, [0, 191, 100, 3, 254], [130, 321, 101, 133, 384], torch.float16),
    (128, 128, 128, 2, 129, [0, 127, 1, 128, 200], [129, 256, 2, 257, 329], torch.bfloat16),
    (128, 128, 64, 1, 300, [0, 5, 84, 84, 84], [300, 300, 384, 84, 85], torch.float16),
])
@pytest.mark.parametrize("scale", [0.3, 30.0])
def test_append_matches_the_definition(page, block, D, H, S, starts, lens, dtype, scale):
    """scale 0.3 mostly keeps the block magnitudes that the cache had, 30 grows them."""
    from astrai_b200.ops.kv8 import kv8_append

    width = -(-max(lens) // page)
    n_pages = len(starts) * width + 2
    cache = _cache(n_pages, H, page, D, block)
    table = _table(len(starts), width, n_pages)
    k, v = _new(len(starts), S, H, D, dtype, scale=scale)
    want = _append_oracle(cache, k, v, table.cpu(), starts, lens)
    kv8_append(cache, k, v, table, _i32(*starts), _i32(*lens))
    for got, ref in zip(cache, want):
        assert torch.equal(got.cpu(), ref)


def test_append_token_by_token_keeps_what_it_should():
    """Single-token appends through a block whose magnitude grows with every token: each integer is within half a step
    per growth, and tokens of other blocks and rows do not change."""
    from astrai_b200.ops.kv8 import kv8_append, kv8_gather

    B, H, D, page, block, n = 3, 2, 64, 64, 32, 50
    cache = _cache(B + 1, H, page, D, block)
    table = _table(B, 1, B + 1)
    k, v = _new(B, n, H, D, torch.bfloat16)
    k = k * torch.arange(1, n + 1, device="cuda").view(1, n, 1, 1).to(k.dtype) / 8
    for i in range(n):
        kv8_append(cache, k[:, i: i + 1], v[:, i: i + 1], table, _i32(*[i] * B), _i32(*[i + 1] * B))
    ko, vo = kv8_gather(cache, table, _i32(*[n] * B), n)
    for x, got, growths in ((k, ko, block), (v, vo, block)):
        top = torch.stack([x[:, i // block * block: i // block * block + block].float().abs().amax((1, 3))
                           for i in range(n)], 1)  # [B, n, H]
        assert ((x.float() - got.float()).abs().amax(-1) <= top / 127 * 0.5 * (1 + growths) + 2.0 ** -8 * top).all()
    spare = [p for p in range(B + 1) if p not in table.flatten().tolist()]
    assert torch.equal(cache.k[spare], _cache(B + 1, H, page, D, block).k[spare])


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_append_drops_tokens_before_position_zero(block):
    """k[b, i] has position starts[b] + i, also where that is negative for the first of them."""
    from astrai_b200.ops.kv8 import kv8_append

    H, D, page, S = 2, 64, 128, 150
    starts, lens = [-3, -150, -149, -1000, -70], [147, 0, 5, 20, 40]
    live = [(3, 147), (150, 0), (149, 1), (150, 0), (70, 40)]  # first token kept and their number
    c, want = _cache(12, H, page, D, block), _cache(12, H, page, D, block)
    table = _table(5, 2, 12)
    k, v = _new(5, S, H, D, torch.bfloat16)
    kv8_append(c, k, v, table, _i32(*starts), _i32(*lens))
    for b, (i, n) in enumerate(live):
        if n:
            kv8_append(want, k[b: b + 1, i: i + n], v[b: b + 1, i: i + n], table[b: b + 1], _i32(0), _i32(n))
    assert all(torch.equal(x, y) for x, y in zip(c, want))


def test_append_edges_missing_pages_zeros_and_non_finite():
    from astrai_b200.ops.kv8 import kv8_append, kv8_gather

    B, H, D, page, block, S = 6, 2, 128, 64, 32, 64
    cache = _cache(16, H, page, D, block)
    table = _table(B, 2, 16)
    table[0, 0], table[0, 1] = -1, 99  # missing, out of range
    k, v = (t.clone() for t in _new(B, S, H, D, torch.bfloat16))
    k[1] = 0                                   # a block of zeros
    k[2, 3, 0, 7], v[2, 40, 1, 0] = float("inf"), float("nan")
    k[3, 40:] = float("nan")                   # padding behind the row's end
    k[4, :, 0] = torch.finfo(torch.bfloat16).max
    k[4, 1, 0] = 1.0
    k[5] = 1e-40                               # below the smallest normal number
    before = _clone(cache)
    starts, lens = _i32(0, 0, 0, 0, 0, 0), _i32(64, 64, 64, 40, 64, 64)
    kv8_append(cache, k, v, table, starts, lens)
    touched = set(table[1:, 0].tolist())
    for p in range(16):
        if p not in touched:
            assert all(torch.equal(a[p], b[p]) for a, b in zip(cache, before))
    ko, vo = kv8_gather(cache, table, lens, 64)
    assert (ko[0] == 0).all() and (vo[0] == 0).all() and (ko[1] == 0).all()
    nan = torch.zeros(B, 64, H, dtype=torch.bool, device="cuda")
    nan[2, :32, 0] = True
    assert (ko.isnan().all(-1) == nan).all() and (ko.isnan().any(-1) == nan).all()
    assert vo[2, 32:, 1].isnan().all() and torch.isfinite(vo[2, :32]).all() and torch.isfinite(vo[2, :, 0]).all()
    assert (ko[3, 40:] == 0).all() and torch.isfinite(ko[3]).all()
    assert (ko[4, 0, 0] == torch.finfo(torch.bfloat16).max).all() and (ko[4, 1, 0] == 0).all()
    step = 1e-40 / 127
    assert ((ko[5].float() - 1e-40).abs() <= step + 1e-40 * 2.0 ** -3).all()  # subnormals keep few bits
    # a block that starts again forgets the NaN
    kv8_append(cache, torch.ones_like(k), torch.ones_like(v), table, starts, lens)
    ko, vo = kv8_gather(cache, table, lens, 64)
    assert (ko[2] == 1).all() and (vo[2] == 1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,block,D", [(16, 16, 64), (64, 32, 128), (192, 64, 64), (128, 128, 128)])
def test_gather(page, block, D, dtype):
    from astrai_b200.ops.kv8 import kv8_gather

    B, H, width = 4, 3, 3
    cache = _cache(B * width + 1, H, page, D, block)
    table = _table(B, width, B * width + 1)
    table[3, 1] = -1
    lens, starts = [0, 1, 2 * page + 5, 3 * page], [0, 0, page - 1, 7]
    total = 2 * page + 9
    for st in (None, starts):
        ko, vo = kv8_gather(cache, table, _i32(*lens), total, starts=None if st is None else _i32(*st), dtype=dtype)
        for out, q, a in ((ko, cache.k, cache.k_absmax), (vo, cache.v, cache.v_absmax)):
            assert out.shape == (B, total, H, D) and out.dtype == dtype
            want = torch.zeros(out.shape, dtype=torch.float64, device="cuda")
            for b in range(B):
                for i in range(total):
                    t = i + (st[b] if st else 0)
                    p = int(table[b, t // page]) if t < lens[b] else -1
                    if p >= 0:
                        want[b, i] = q[p, :, t % page].double() * a[p, :, t % page // block, None].double() / 127
            assert ((out.double() - want).abs() <= (HALF_SPACING[dtype] + 2.0 ** -22) * want.abs() + 1e-7).all()
    assert kv8_gather(cache, table, _i32(*lens), 0)[0].shape == (B, 0, H, D)


def _attend_oracle(q, cache, table, lens, starts, scale):
    """-> output, sum of p |v| for each output, largest |score|; rows without keys are zeros."""
    B, S, Hq, D = q.shape
    Hkv, page, block = cache.k.shape[1], cache.page_size, cache.block
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mag, top = torch.zeros_like(out), 0.0
    for b in range(B):
        n = int(lens[b])
        toks = [t for t in range(n) if 0 <= int(table[b, t // page]) < cache.k.shape[0]]
        if not toks:
            continue
        t = torch.tensor(toks, device="cuda")
        p, off = table[b].long()[t // page], t % page
        k, v = (c[p, :, off].double() * a[p, :, off // block].double()[..., None] / 127
                for c, a in ((cache.k, cache.k_absmax), (cache.v, cache.v_absmax)))
        for i in range(S):
            pos = (n - S if starts is None else int(starts[b])) + i
            seen = t <= pos
            if pos < 0 or pos >= n or not seen.any():
                continue
            for h in range(Hkv):
                g = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
                s = q[b, i, g].double() @ k[seen, h].T * scale
                w = torch.softmax(s, -1)
                out[b, i, g] = w @ v[seen, h]
                mag[b, i, g] = w @ v[seen, h].abs()
                top = max(top, s.abs().max().item())
    return out, mag, top


def _check_attention(q, cache, table, lens, starts=None, scale=None, got=None):
    from astrai_b200.ops.kv8 import kv8_attention

    if got is None:
        got = kv8_attention(q, cache, table, lens, starts=starts, scale=scale)
    want, mag, top = _attend_oracle(q, cache, table, lens, starts, scale or 1 / math.sqrt(q.shape[-1]))
    n = max(1, int(lens.max()))
    tol = HALF_SPACING[q.dtype] * want.abs() + (2.0 ** -11 + 2.0 ** -12 + 2.0 ** -20 * top + n * 2.0 ** -25) * mag
    tol = tol + n * 2.0 ** -25 * mag.amax(-1, keepdim=True) + 1e-30
    worst = ((got.double() - want).abs() / tol).max().item()
    assert got.dtype == q.dtype and worst <= 1.0, worst
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (16, 4), (6, 1), (7, 1), (24, 2), (16, 1)])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 32), (192, 64), (128, 128)])
def test_decode_attention(page, block, Hq, Hkv, D):
    lens = [0, 1, 15, 16, 17, 127, 128, 129, 300, 383]
    B, width = len(lens), -(-384 // page)
    cache = _cache(B * width + 1, Hkv, page, D, block)
    table = _table(B, width, B * width + 1)
    q = torch.randn(B, 1, Hq, D, device="cuda", generator=_gen(7)).to(torch.bfloat16)
    _check_attention(q, cache, table, _i32(*lens))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,Hq,Hkv,D", [(2, 16, 4, 128), (4, 16, 4, 64), (3, 7, 1, 128), (9, 4, 2, 128), (8, 16, 1, 64),
                                        (33, 3, 1, 128)])
def test_several_queries_are_causal(S, Hq, Hkv, D, dtype):
    lens = [S, S + 1, 1, 0, 130, 257]  # rows with fewer tokens than queries have queries before token 0
    B, page, block, width = len(lens), 64, 16, 5
    cache = _cache(B * width, Hkv, page, D, block)
    table = _table(B, width, B * width)
    buf = torch.randn(B, S, 2 * Hq, D, device="cuda", generator=_gen(8)).to(dtype)
    q = buf[:, :, Hq:]  # strided
    _check_attention(q, cache, table, _i32(*lens))
    # right-padded rows: the queries past the row's end give zeros
    starts = _i32(*[max(0, n - S + 1) for n in lens])
    got = _check_attention(q, cache, table, _i32(*lens), starts=starts, scale=0.3)
    for b, n in enumerate(lens):
        assert (got[b, max(0, n - int(starts[b])):] == 0).all()


def test_rows_split_over_many_ctas_and_ragged_batches():
    lens = [5000, 1, 0, 2049, 128, 4000, 17, 3333]
    B, page, block, Hq, Hkv, D = len(lens), 128, 32, 8, 2, 128
    width = -(-max(lens) // page)
    cache = _cache(B * width, Hkv, page, D, block, spread=0.1)
    table = _table(B, width, B * width)
    q = torch.randn(B, 1, Hq, D, device="cuda", generator=_gen(9)).to(torch.bfloat16) * 0.3
    first = _check_attention(q, cache, table, _i32(*lens))
    one = _check_attention(q[:1], cache, table[:1], _i32(lens[0]))  # the same row dealt out in other pieces
    assert ((one - first[:1]).abs() <= 2.0 ** -7 * first[:1].abs() + 1e-3).all()
    from astrai_b200.ops.kv8 import kv8_attention

    for _ in range(3):
        assert torch.equal(kv8_attention(q, cache, table, _i32(*lens)), first)


@pytest.mark.parametrize("S,Hq,Hkv,D,lens", [(4, 32, 8, 64, [4000, 3000, 2500, 1200]), (4, 16, 4, 128, [3500, 2100, 3333]),
                                             (1, 16, 1, 128, [4100, 2000, 3000, 700, 3900]), (11, 6, 2, 64, [3000, 4000])])
def test_wide_groups_in_several_pieces(S, Hq, Hkv, D, lens):
    """16 query rows at a time, rows long enough that a CTA's second piece fills the copy ring while its first is
    merged."""
    B, page, block = len(lens), 128, 32
    width = -(-max(lens) // page)
    cache = _cache(B * width, Hkv, page, D, block, spread=0.1)
    table = _table(B, width, B * width)
    q = torch.randn(B, S, Hq, D, device="cuda", generator=_gen(9)).to(torch.bfloat16) * 0.3
    first = _check_attention(q, cache, table, _i32(*lens))
    for _ in range(3):
        assert torch.equal(_check_attention(q, cache, table, _i32(*lens)), first)


@pytest.mark.parametrize("D", [64, 128])
def test_magnitudes_of_any_size(D):
    """Blocks whose values are 2^60 apart, a block of zeros, and queries far from 1."""
    lens, page, block, Hq, Hkv = [200, 140], 64, 16, 4, 2
    cache = _cache(10, Hkv, page, D, block, spread=0.0)
    cache.v_absmax.copy_((2.0 ** torch.randint(-30, 31, cache.v_absmax.shape, device="cuda", generator=_gen(3))))
    cache.v_absmax[3] = 0
    cache.k_absmax[5] = 0
    table = _table(2, 4, 10)
    for scale in (1.0, 2.0 ** -40, 2.0 ** 30):
        q = (torch.randn(2, 1, Hq, D, device="cuda", generator=_gen(4)) * scale).to(torch.bfloat16)
        _check_attention(q, cache, table, _i32(*lens), scale=0.05 / scale)
    q = torch.zeros(2, 1, Hq, D, device="cuda", dtype=torch.bfloat16)  # uniform weights
    _check_attention(q, cache, table, _i32(*lens))


def test_peaked_scores_and_one_dominant_key():
    page, block, D, Hq, Hkv, n = 128, 32, 128, 4, 1, 1000
    cache = _cache(8, Hkv, page, D, block)
    table = _table(1, 8, 8)
    q = (20 * torch.randn(1, 1, Hq, D, device="cuda", generator=_gen(4))).to(torch.bfloat16)
    _check_attention(q, cache, table, _i32(n))


def test_masked_places_may_hold_anything():
    from astrai_b200.ops.kv8 import kv8_attention

    lens, page, block, D, Hq, Hkv = [70, 0, 129], 64, 32, 128, 8, 2
    cache = _cache(16, Hkv, page, D, block)
    table = _table(3, 4, 15)
    table[table == 15] = 14
    table[0, 2:], table[1], table[2, 1] = -1, -1, 77  # unused, a row without pages, a page out of range
    q = torch.randn(3, 1, Hq, D, device="cuda", generator=_gen(4)).to(torch.bfloat16)
    want = _check_attention(q, cache, table, _i32(*lens))
    assert (want[1] == 0).all()
    dirty = _clone(cache)
    used = {(int(table[0, 0]), b) for b in range(2)} | {(int(table[0, 1]), 0)} | {(int(table[2, 0]), b) for b in range(2)} \
        | {(int(table[2, 2]), 0)}
    for p in range(16):
        for b in range(2):
            if (p, b) not in used:
                for a in (dirty.k_absmax, dirty.v_absmax):
                    a[p, :, b] = float("nan")
    for c in (dirty.k, dirty.v):  # slots of live blocks behind the row's end
        c[int(table[0, 1]), :, 70 - 64:] = 127
        c[int(table[2, 2]), :, 129 - 128:] = -127
    assert torch.equal(kv8_attention(q, dirty, table, _i32(*lens)), want)


def test_nan_reaches_its_own_rows_only():
    from astrai_b200.ops.kv8 import kv8_attention

    page, block, D, Hq, Hkv = 64, 32, 64, 8, 2
    for which in ("k_absmax", "v_absmax"):
        cache = _cache(4, Hkv, page, D, block)
        table = _table(2, 2, 4)
        getattr(cache, which)[int(table[0, 1]), 0, 0] = float("nan")
        q = torch.randn(2, 1, Hq, D, device="cuda", generator=_gen(4)).to(torch.bfloat16)
        o = kv8_attention(q, cache, table, _i32(100, 100))
        assert o[0, :, :4].isnan().all() and torch.isfinite(o[0, :, 4:]).all() and torch.isfinite(o[1]).all()
    cache = _cache(4, Hkv, page, D, block)
    q[0, 0, 1, 3], q[1, 0, 5, 0] = float("nan"), float("inf")
    o = kv8_attention(q, cache, table, _i32(100, 100))
    bad = torch.zeros(2, 1, Hq, dtype=torch.bool, device="cuda")
    bad[0, 0, 1] = bad[1, 0, 5] = True
    assert (torch.isfinite(o).all(-1) == ~bad).all()


def test_offsets_past_32_bits():
    """A cache of more than 2^31 values: pages at its far end."""
    from astrai_b200.ops.kv8 import KV8, kv8_append, kv8_gather

    page, block, D, Hkv = 128, 128, 128, 8
    n_pages = 2 ** 31 // (page * D * Hkv) + 40
    cache = KV8.allocate(n_pages, Hkv, page, D, block, "cuda")
    table = torch.arange(n_pages - 6, n_pages, device="cuda").flip(0).view(2, 3).int()
    k, v = _new(2, 300, Hkv, D, torch.bfloat16)
    starts, lens = _i32(0, 0), _i32(300, 290)
    kv8_append(cache, k, v, table, starts, lens)
    ko, vo = kv8_gather(cache, table, lens, 300)
    for x, got in ((k, ko), (v, vo)):
        assert ((x[:, :290].float() - got[:, :290].float()).abs() <= x.float().abs().max() / 127 * 0.51 + 0.02).all()
    assert not cache.k[: n_pages - 6].any()
    q = torch.randn(2, 1, 16, D, device="cuda", generator=_gen(4)).to(torch.bfloat16)
    _check_attention(q, cache, table, lens)


def test_other_streams_workspaces_and_graphs():
    from astrai_b200.ops.kv8 import kv8_append, kv8_attention, kv8_attention_workspace

    B, page, block, Hq, Hkv, D, width = 3, 64, 32, 8, 2, 128, 30
    cache = _cache(B * width, Hkv, page, D, block)
    table = _table(B, width, B * width)
    k, v = _new(B, 1, Hkv, D, torch.bfloat16)
    q = torch.randn(B, 1, Hq, D, device="cuda", generator=_gen(4)).to(torch.bfloat16)
    starts = _i32(1500, 77, 0)
    lens = starts + 1
    ref = _clone(cache)
    kv8_append(ref, k, v, table, starts, lens)
    want = kv8_attention(q, ref, table, lens)
    ws = torch.empty(kv8_attention_workspace(B, 1, Hq, cache, width), device="cuda")
    with pytest.raises(RuntimeError):
        kv8_attention(q, ref, table, lens, workspace=ws[:-1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv8_append(cache, k, v, table, starts, lens)
        got = kv8_attention(q, cache, table, lens, workspace=ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kv8_append(cache, k, v, table, starts, lens)
            replayed = kv8_attention(q, cache, table, lens, workspace=ws)
    side.synchronize()
    assert torch.equal(got, want)
    starts.copy_(_i32(1200, 1000, 3))
    lens.copy_(starts + 1)
    graph.replay()
    torch.cuda.synchronize()
    kv8_append(ref, k, v, table, starts, lens)
    assert torch.equal(replayed, kv8_attention(q, ref, table, lens))


def test_empty_calls():
    from astrai_b200.ops.kv8 import kv8_append, kv8_attention

    cache = _cache(2, 2, 64, 64, 32)
    before = _clone(cache)
    table = _table(1, 2, 2)
    k, v = _new(1, 0, 2, 64, torch.bfloat16)
    kv8_append(cache, k, v, table, _i32(3), _i32(3))
    k, v = _new(1, 4, 2, 64, torch.bfloat16)
    kv8_append(cache, k, v, table, _i32(9), _i32(9))
    kv8_append(cache, k[:0], v[:0], table[:0], _i32(), _i32())
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    q = torch.randn(1, 0, 4, 64, device="cuda").to(torch.bfloat16)
    assert kv8_attention(q, cache, table, _i32(9)).shape == q.shape
    assert kv8_attention(q[:0], cache, table[:0], _i32()).shape == (0, 0, 4, 64)


def test_refusals():
    from astrai_b200.ops.kv8 import KV8, kv8_append, kv8_attention, kv8_gather

    with pytest.raises(ValueError):
        KV8.allocate(2, 2, 64, 64, 48)
    with pytest.raises(ValueError):
        KV8.allocate(2, 2, 48, 64, 32)
    cache = _cache(4, 2, 64, 128, 32)
    table, lens, starts = _table(2, 2, 4), _i32(10, 20), _i32(9, 19)
    k, v = _new(2, 1, 2, 128, torch.bfloat16)
    q = torch.randn(2, 1, 8, 128, device="cuda").to(torch.bfloat16)
    kv8_append(cache, k, v, table, starts, lens)
    bad_appends = [(k.float(), v.float(), table, starts, lens), (k, v[:, :, :1], table, starts, lens),
                   (k[..., :64], v[..., :64], table, starts, lens), (k, v, table[:1], starts, lens),
                   (k, v, table, starts[:1], lens), (k, v, table, starts, lens[:1]), (k.cpu(), v.cpu(), table, starts, lens),
                   (k, v, table, starts.cpu(), lens), (k[0], v[0], table, starts, lens)]
    for a in bad_appends:
        with pytest.raises(RuntimeError):
            kv8_append(cache, *a)
    for qq in (q.float(), q[:, :, :3], q[..., :64], q[:1], q.cpu(), q[0]):
        with pytest.raises(RuntimeError):
            kv8_attention(qq, cache, table, lens)
    with pytest.raises(RuntimeError):
        kv8_attention(q, cache, table, lens, starts=starts[:1])
    with pytest.raises(RuntimeError):
        kv8_gather(cache, table, lens, 8, dtype=torch.float32)
    for c in (cache._replace(k=cache.k.float()), cache._replace(v=cache.v[:2]), cache._replace(v_absmax=cache.v_absmax[:2]),
              cache._replace(k=cache.k[..., :96].contiguous(), v=cache.v[..., :96].contiguous()),
              cache._replace(k_absmax=cache.k_absmax[..., :0], v_absmax=cache.v_absmax[..., :0]),
              cache._replace(k=cache.k.transpose(1, 2), v=cache.v.transpose(1, 2))):
        with pytest.raises((RuntimeError, ZeroDivisionError)):
            kv8_gather(c, table, lens, 8)


def test_caches_without_heads_or_pages():
    from astrai_b200.ops.kv8 import KV8, kv8_append, kv8_attention, kv8_gather

    table, lens, starts = _i32(0, 1).view(1, 2), _i32(20), _i32(0)
    q, k = torch.randn(1, 4, 4, 128, device="cuda").bfloat16(), torch.randn(1, 20, 2, 128, device="cuda").bfloat16()
    none = KV8.allocate(4, 0, 64, 128, 32, "cuda")
    for call in (lambda: kv8_attention(q, none, table, lens), lambda: kv8_gather(none, table, lens, 8),
                 lambda: kv8_append(none, k[:, :, :0], k[:, :, :0], table, starts, lens)):
        with pytest.raises(RuntimeError):
            call()
    empty = KV8.allocate(0, 2, 64, 128, 32, "cuda")  # no page to read
    kv8_append(empty, k, k, table, starts, lens)
    assert (kv8_attention(q, empty, table, lens) == 0).all() and (kv8_gather(empty, table, lens, 8)[0] == 0).all()


def test_more_rows_than_one_launch_takes():
    """1024 rows go in one launch: 1100 rows, split and whole ones, with and without a caller's workspace."""
    from astrai_b200.ops.kv8 import kv8_attention, kv8_attention_workspace

    for width in (1, 12):
        B, page, Hq, Hkv, D = 1100, 64, 4, 1, 64
        cache = _cache(40, Hkv, page, D, 32)
        table = (torch.arange(B * width, device="cuda") % 40).view(B, width).int()  # pages shared between rows
        lens = (torch.arange(B, device="cuda") * 7 % (width * page + 1)).int()
        q = torch.randn(B, 1, Hq, D, device="cuda", generator=_gen(4)).to(torch.bfloat16)
        got = kv8_attention(q, cache, table, lens)
        ws = torch.empty(max(1, kv8_attention_workspace(B, 1, Hq, cache, width)), device="cuda")
        assert torch.equal(kv8_attention(q, cache, table, lens, workspace=ws), got)
        pick = torch.tensor([0, 1, 5, 1023, 1024, 1025, 1099], device="cuda")
        _check_attention(q[pick], cache, table[pick], lens[pick], got=got[pick])
