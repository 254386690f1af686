"""Tokens drawn from given numbers, against extended precision.

Tokens are compared for equality wherever the given number is further than 1e-12 of the mass from a token's border: 64-bit
sums of 131072 terms, and the given number's product with them, are within 131072 * 2^-53 = 1.5e-11 of the mass in the worst
order and within 17 * 2^-53 = 2e-15 when added in a tree as here, behind an exponential within 2^-52. A log-probability is
the logarithm of a ratio whose sum, in 32 bits, is within 2^-20 of itself (an exponential within 2^-22, the rounding of its
argument |t| <= 17 on average over the mass, 17 * 1.3e-7 = 2^-18.8 at most), rounded to fp32: 2^-18 and 2^-23 of itself.
"""

import math

import numpy as np
import pytest
import torch

from tests.sample_oracle import kept_and_mass, oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_error_word():
    from astrai_b200.ops._ext import native

    native().read_error()
    yield
    torch.cuda.synchronize()
    assert native().read_error() == 0


def _check(x, u, t=1.0, k=0, p=1.0, m=0.0, got=None):
    from astrai_b200.inference.sample import sample_given

    rows = x.shape[0]
    if got is None:
        got = sample_given(x, u, temperature=t, top_k=k, top_p=p, min_p=m, return_logprobs=True)
    token, logprob = got
    assert token.dtype == torch.int64 and token.shape == (rows,) and logprob.dtype == torch.float32

    def rowwise(v):
        return (v.double() if torch.is_tensor(v) else torch.tensor(float(np.float32(v)) if isinstance(v, float) else v)
                ).expand(rows).tolist()

    xs, us = x.detach().double().cpu().numpy(), u.double().tolist()
    for r, (ur, tr, kr, pr, mr) in enumerate(zip(us, *(rowwise(v) for v in (t, k, p, m)))):
        want, lp, near = oracle(xs[r], ur, tr, int(kr), pr, mr)
        if near < 1e-12:
            continue
        assert int(token[r]) == want, (r, int(token[r]), want, near, tr, kr, pr, mr)
        assert abs(float(logprob[r]) - lp) <= 2.0 ** -18 + 2.0 ** -23 * abs(lp), (r, float(logprob[r]), lp)


def _logits(rows, V, dtype, seed, sigma=None):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(rows, V, generator=g, device="cuda")
    s = torch.tensor([0.3, 1.0, 2.0, 4.5], device="cuda").repeat(rows)[:rows, None] if sigma is None else sigma
    return (x * s).to(dtype), torch.rand(rows, generator=g, device="cuda")


SETTINGS = [dict(), dict(t=0.0), dict(t=0.7, k=50, p=0.95), dict(k=1), dict(k=40), dict(t=1.5, k=200, m=0.05), dict(k=256, p=0.5, m=0.1),
            dict(p=0.9), dict(t=0.6, p=0.98), dict(p=0.3, m=0.02), dict(m=0.1), dict(m=1e-6), dict(m=1.0), dict(p=0.0),
            dict(k=300), dict(t=2.0, k=3000, p=0.9, m=1e-4), dict(p=0.999999), dict(t=1e-9, k=5), dict(t=100.0, p=0.7)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 9, 100, 1000, 1025, 4097, 32000, 32003, 50021, 131072, 300001])
def test_sizes_and_settings(dtype, V):
    x, u = _logits(8, V, dtype, V)
    for s in SETTINGS if V < 40000 else SETTINGS[V % 3::3]:
        _check(x, u, **s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_settings_of_each_row(dtype):
    g = torch.Generator().manual_seed(1)
    x, u = _logits(60, 20001, dtype, 2)

    def pick(values, kind=torch.float32):
        return torch.tensor(values)[torch.randint(len(values), (60,), generator=g)].to(kind).cuda()

    _check(x, u, pick([0.0, 0.5, 1.0, 1.3]), pick([0, 5, 100, 400, 30000], torch.int32), pick([0.0, 0.4, 0.9, 1.0, 1.5]),
           pick([0.0, 0.01, 0.2, 1.0]))
    _check(x, u.double(), pick([0.9], torch.float64), pick([20, 0], torch.int64))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [700, 33000])
@pytest.mark.parametrize("s", [dict(), dict(p=0.9), dict(m=0.01), dict(k=60), dict(k=2000, p=0.8)])
def test_numbers_next_to_a_border(dtype, V, s):
    """The given number 1e-9 of the mass before and behind a token's border: 32-bit sums cannot tell."""
    x, _ = _logits(12, V, dtype, 3)
    xs = x.double().cpu().numpy()
    g = np.random.default_rng(0)
    for side in (-1e-9, 1e-9):
        u = []
        for row in xs:
            ids, w = kept_and_mass(row, 1.0, s.get("k", 0), float(np.float32(s.get("p", 1.0))), float(np.float32(s.get("m", 0.0))))
            sums = np.cumsum(w) / w.sum()
            u.append(float(sums[g.integers(max(1, ids.size - 1))]) + side)
        _check(x, torch.tensor(u, dtype=torch.float64, device="cuda"), **s)


@pytest.mark.parametrize("V", [40, 5000])
def test_top_p_next_to_a_border(V):
    x, u = _logits(16, V, torch.float32, 5)
    xs = x.double().cpu().numpy()
    for side in (-1e-7, 1e-7):
        p = []
        for r, row in enumerate(xs):
            w = np.sort(np.exp(row - row.max()))[::-1]
            p.append(float((np.cumsum(w) / w.sum())[min(3 + r * V // 60, V - 2)]) + side)
        _check(x, u, p=torch.tensor(p, device="cuda"))


def test_ends_of_the_unit_interval():
    for V in (5, 3000, 70000):
        x, _ = _logits(8, V, torch.bfloat16, 7)
        x[:, :2] = -math.inf
        x[:, -2:] = -math.inf
        for s in (dict(), dict(k=30), dict(p=0.8), dict(m=0.05)):
            _check(x, torch.zeros(8, device="cuda"), **s)
            _check(x, torch.full((8,), 1 - 2.0 ** -24, device="cuda"), **s)
            from astrai_b200.inference.sample import sample_given

            args = dict(top_k=s.get("k", 0), top_p=s.get("p", 1.0), min_p=s.get("m", 0.0))
            first, last = (sample_given(x, torch.full((8,), v, device="cuda"), **args) for v in (0.0, 1 - 2.0 ** -24))
            for v, same in ((-3.0, first), (math.nan, first), (1.0, last), (7.0, last)):
                assert torch.equal(sample_given(x, torch.full((8,), v, device="cuda", dtype=torch.float64), **args), same) \
                    or v >= 1  # the very end may lie one token behind 1 - 2^-24
            end = sample_given(x, torch.ones(8, device="cuda"), **args)
            for r in range(8):
                ids, w = kept_and_mass(x[r].double().cpu().numpy(), 1.0, s.get("k", 0), float(np.float32(s.get("p", 1.0))),
                                       float(np.float32(s.get("m", 0.0))))
                assert int(end[r]) == ids[np.nonzero(w > 0)[0][-1]]


@pytest.mark.parametrize("p", [0.9, 0.98, 0.999])
def test_top_p_of_many_equal_logits(p):
    """Few distinct logits, each the steps of several others apart: the bound may lie far from where their steps point."""
    x, u = _logits(48, 60000, torch.bfloat16, 21)
    _check((x.float() * 3).bfloat16(), u, p=p)
    _check((x.float() * 3).round().bfloat16(), u, p=p)


@pytest.mark.parametrize("V", [300, 5000, 40000])
def test_ties(V):
    """Equal logits are kept or dropped together; all of a flat row is drawn from."""
    x, u = _logits(6, V, torch.bfloat16, 9)
    x[0] = 0.25
    x[1] = x[1].round()
    x[2] = torch.where(x[2] > 0, 0.0, -0.0)
    x[3, ::2] = 3.0
    x[4, 10:] = -math.inf
    x[5] = -5e4
    for s in (dict(), dict(k=7), dict(k=300), dict(p=0.5), dict(m=0.3), dict(k=100, p=0.9, m=0.01), dict(p=0.0)):
        _check(x, u, **s)


@pytest.mark.parametrize("V", [50, 40000])
def test_rows_without_a_distribution(V):
    from astrai_b200.inference.sample import sample_given

    x, u = _logits(7, V, torch.float32, 11)
    x[0] = -math.inf
    x[1, 3] = math.nan
    x[2] = math.nan
    x[3, [V - 4, V - 2]] = math.inf
    x[4, 0] = math.nan
    x[4, 1:] = -math.inf
    best = x[1].nan_to_num(-1e9).argmax()
    for s in (dict(), dict(temperature=0.0), dict(top_k=5), dict(top_p=0.5), dict(min_p=0.5)):
        token, logprob = sample_given(x, u, return_logprobs=True, **s)
        assert token[:5].tolist() == [0, int(best), 0, V - 4, 1] and logprob[:5].isnan().all()
        assert torch.isfinite(logprob[5:]).all()


def test_huge_logits_and_temperatures():
    x, u = _logits(8, 3000, torch.float32, 13)
    _check(x * 1e30, u)
    _check(x * 1e30, u, t=3e30, p=0.9)
    _check(x + 1e6, u, k=20)
    _check(x, u, t=math.inf, k=100)
    _check(x, u, t=math.inf, m=1.0)
    _check(x * 1e-30, u, p=0.4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(dtype):
    x, u = _logits(6, 5003, dtype, 15)
    for pad, off in ((3, 0), (7, 5), (23, 1)):
        wide = torch.full((6, 5003 + pad + off), math.inf, dtype=dtype, device="cuda")
        wide[:, off: off + 5003] = x
        for s in (dict(), dict(k=30), dict(p=0.9)):
            _check(wide[:, off: off + 5003], u, **s)
    _check(x.repeat_interleave(2, 0)[::2], u.repeat_interleave(2)[::2], p=0.9)
    _check(x.t().contiguous().t(), u, p=0.9)
    _check(x[:1].expand(6, -1), u, p=0.9)
    _check(torch.stack([x, x], 1)[:, -1], u, k=9)  # the last position of each sequence


def test_same_each_time_and_in_any_batch():
    """A row's token depends on the row alone, not on its place in the batch."""
    from astrai_b200.inference.sample import sample_given

    x, u = _logits(200, 9000, torch.bfloat16, 17)
    for s in (dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.95), dict(min_p=0.02)):
        token, logprob = sample_given(x, u, return_logprobs=True, **s)
        for _ in range(3):
            again, lp = sample_given(x, u, return_logprobs=True, **s)
            assert torch.equal(token, again) and torch.equal(logprob, lp)
        order = torch.randperm(200, device="cuda")[:77]
        part, lp = sample_given(x[order], u[order], return_logprobs=True, **s)
        assert torch.equal(part, token[order]) and torch.equal(lp, logprob[order])


def test_frequencies_follow_the_distribution():
    """Evenly spread numbers give every token its probability to within one draw and the tokens' two borders."""
    from astrai_b200.inference.sample import sample_given

    n = 20000
    x = torch.randn(1, 50, device="cuda").expand(n, -1)
    u = (torch.arange(n, device="cuda", dtype=torch.float64) + 0.5) / n
    count = torch.bincount(sample_given(x, u, temperature=0.8), minlength=50)
    want = n * torch.softmax(x[0].double() / float(np.float32(0.8)), -1)
    assert (count - want).abs().max() <= 1.0


def test_captured_and_on_another_stream():
    from astrai_b200.inference.sample import sample_given

    x, u = _logits(9, 40000, torch.bfloat16, 19)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample_given(x, u, top_p=0.9, return_logprobs=True)
    side.synchronize()
    _check(x, u, p=0.9, got=got)
    p, k = torch.full((9,), 0.9, device="cuda"), torch.zeros(9, device="cuda", dtype=torch.int32)
    one, zero = torch.ones(9, device="cuda"), torch.zeros(9, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sample_given(x, u, one, k, p, zero, True)
    for seed in range(3):
        fresh, numbers = _logits(9, 40000, torch.bfloat16, seed)
        x.copy_(fresh)
        u.copy_(numbers)
        k.fill_(30 * seed)
        g.replay()
        _check(x, u, k=30 * seed, p=0.9, got=out)


def test_refusals():
    from astrai_b200.inference.sample import sample_given

    x, u = _logits(3, 100, torch.float32, 0)
    for bad in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=1.5), dict(top_p=math.nan), dict(min_p=-0.1),
                dict(uniform=u[:2]), dict(top_k=torch.zeros(2, device="cuda")), dict(logits=x[0]), dict(logits=x[None])):
        with pytest.raises(ValueError):
            sample_given(**{"logits": x, "uniform": u, **bad})
    for bad in (dict(logits=x.double()), dict(uniform=u.half()), dict(uniform=u.cpu())):
        with pytest.raises(RuntimeError):
            sample_given(**{"logits": x, "uniform": u, **bad})
    assert sample_given(x[:0], u[:0]).shape == (0,)
    assert not sample_given(x.requires_grad_(), u, return_logprobs=True)[1].requires_grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [5, 50, 3001, 40000, 70001])
def test_largest_number_beside_a_nan(dtype, V):
    """It may share a 16-byte vector with the NaN, at any place of the vector and of the row."""
    from astrai_b200.inference.sample import sample_given

    for off in (0, 3):
        wide = torch.full((24, V + 11), math.inf, dtype=dtype, device="cuda")
        x = wide[:, off: off + V]
        x.copy_(torch.randn(24, V, device="cuda"))
        want = []
        for r in range(24):
            best = (r * V // 24) if r % 2 else V - 1 - r * V // 48
            x[r, best] = 9.0 if r % 3 else math.inf
            x[r, best + 1 if best + 1 < V else best - 1] = math.nan
            if r % 5 == 0:
                x[r, max(best - 1, 0) if best + 1 < V else max(best - 2, 0)] = math.nan
            row = x[r].float().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
            want.append(int((row == row.max()).nonzero()[0]))
        for s in (dict(), dict(temperature=0.0), dict(top_k=5), dict(top_p=0.5), dict(min_p=0.5)):
            token, logprob = sample_given(x, torch.rand(24, device="cuda"), return_logprobs=True, **s)
            assert token.tolist() == want and logprob.isnan().all()
    # the rows of the CPU's test
    x = torch.zeros(4, 5, device="cuda", dtype=dtype)
    x[0] = -math.inf
    x[1, 0], x[1, 3] = math.nan, 2.0
    x[2] = math.nan
    x[3, 2] = math.inf
    token, logprob = sample_given(x, torch.rand(4, device="cuda"), return_logprobs=True)
    assert token.tolist() == [0, 3, 0, 2] and logprob.isnan().all()


@pytest.mark.parametrize("V", [2, 3000, 40000])
def test_min_p_whose_bound_lies_next_to_zero(V):
    """Logits near zero lie so close together that a search among the neighbours of max + T ln m alone may end below all that
    reach it. Apart from the largest each row has one token 0.02 T above the bound and one as far below."""
    top, t, m = [], [], []
    for temperature in (1.0, 0.7, 1.3):
        for share in (0.9, 0.5, 0.1, 0.02):
            tr, mr = float(np.float32(temperature)), float(np.float32(share))
            at = np.float32(-tr * math.log(mr))
            for step in (-2, -1, 0, 1, 2):
                value = at
                for _ in range(abs(step)):
                    value = np.nextafter(value, np.float32(math.inf if step > 0 else 0))
                top.append(float(value)), t.append(tr), m.append(mr)
    top.append(0.10536054521799088), t.append(1.0), m.append(float(np.float32(0.9)))
    rows = len(top)
    x = torch.full((rows, V), -30.0, device="cuda")
    t, m = torch.tensor(t, device="cuda"), torch.tensor(m, device="cuda")
    x[:, V - 1] = 0.02 * t
    if V > 2:
        x[:, V // 2] = -0.02 * t
    x[:, 0] = torch.tensor(top, device="cuda")
    for u in (0.001, 0.99):
        u = torch.full((rows,), u, device="cuda")
        for k, p in ((0, 1.0), (40, 1.0), (0, 0.9999), (V - 1, 1.0)):
            _check(x, u, t, k, p, m)


def _running(v, n):
    """Running sums of `n` numbers as a warp takes them by shuffles."""
    v = v.copy()
    o = 1
    while o < n:
        up = v[..., :-o].copy()
        v[..., o:] += up
        o *= 2
    return v


def _weights(steps, temperature):
    """2^(t / 16) of logits -0, -1, .. in 64 bits as the kernel computes it, where t is next to a multiple of 16."""
    from fractions import Fraction

    a = 0.6931471805599453 / 16.0
    terms = (a * a * a * a / 24.0, a * a * a / 6.0, a * a / 2.0, a, 1.0)
    out = []
    for n in range(steps):
        t = -float(n) * (16.0 * 1.4426950408889634 / temperature)
        whole = t + 6755399441055744.0 - 6755399441055744.0
        assert whole == -16 * n
        t, e = t - whole, a * a * a * a * a / 120.0
        for term in terms:
            e = float(Fraction(e) * Fraction(t) + Fraction(term))
        out.append(e * 2.0 ** -n)
    return np.array(out)


def test_numbers_between_two_roundings_of_a_border():
    """The sum up to a warp's end, taken by shuffles, and the sum before it and its own part may round differently. A number
    that falls between the two belongs to one of the tokens at the border, and not to none."""
    from astrai_b200.inference.sample import sample_given

    V, temperature = 32000, float(np.float32(1.4426950408889634))
    step = np.random.default_rng(0).integers(0, 12, (40, V))
    x = torch.from_numpy(-step.astype(np.float32)).cuda().bfloat16()  # rows start on the 16-byte grid
    weight = np.zeros((40, 16 * 256 * 8))
    weight[:, :V] = _weights(12, temperature)[step]
    weight = weight.reshape(40, 16, 8, 32, 8)  # warp, vector of a lane, lane, element
    vec = (weight[..., 0] + weight[..., 1]) + (weight[..., 2] + weight[..., 3])
    vec = vec + ((weight[..., 4] + weight[..., 5]) + (weight[..., 6] + weight[..., 7]))
    lane = np.zeros((40, 16, 32))
    for i in range(8):
        lane += vec[:, :, i]
    theirs = _running(lane, 32)[..., 31]
    padded = np.zeros((40, 32))
    padded[:, :16] = theirs
    upto = _running(padded, 32)
    rows, numbers, warps = [], [], []
    for r in range(40):
        total = upto[r, 31]
        for w in range(1, 15):
            if upto[r, w - 1] + theirs[r, w] < upto[r, w]:  # a number there is below neither's end, nor in the next warp's part
                border = upto[r, w - 1] + theirs[r, w]
                u = border / total
                for near in (u, np.nextafter(u, 0), np.nextafter(u, 1)):
                    if near * total == border:
                        rows.append(r), numbers.append(near), warps.append(w)
                        break
    assert len(rows) >= 20
    spoiled = torch.full((len(rows),), -7, device="cuda")
    del spoiled  # memory that the result may get
    token, logprob = sample_given(x[rows], torch.tensor(numbers, dtype=torch.float64, device="cuda"), temperature=temperature,
                                  return_logprobs=True)
    last = (torch.tensor(warps) + 1) * 2048 - 1
    away = token.cpu() - last
    assert ((away == 0) | (away == 1)).all(), away.tolist()
    want = torch.log_softmax(x[rows].double() / temperature, -1).gather(1, token[:, None])[:, 0]
    assert ((logprob - want).abs() <= 2.0 ** -18 + 2.0 ** -23 * want.abs()).all()


def test_top_k_beyond_32_bits_is_off():
    from astrai_b200.inference.sample import sample_given

    x, u = _logits(16, 2000, torch.float32, 23)
    off = sample_given(x, u)
    for k in (2 ** 31 + 1, 2 ** 32 + 1, 2 ** 40 + 3, -1, -2 ** 32 + 1):
        for n in (1, 16):
            assert torch.equal(sample_given(x, u, top_k=torch.full((n,), k, device="cuda")), off)


def test_numbers_beyond_the_unit_interval_count_as_its_ends():
    from astrai_b200.inference.sample import sample_given

    for V in (5, 3000, 70000):
        x, _ = _logits(8, V, torch.bfloat16, 25)
        for s in (dict(), dict(top_k=30), dict(top_p=0.8), dict(min_p=0.05)):
            first, last = (sample_given(x, torch.full((8,), v, device="cuda", dtype=torch.float64), **s) for v in (0.0, 1.0))
            for v, same in ((-3.0, first), (-math.inf, first), (math.nan, first), (7.0, last), (math.inf, last)):
                for kind in (torch.float32, torch.float64):
                    assert torch.equal(sample_given(x, torch.full((8,), v, device="cuda", dtype=kind), **s), same)


@pytest.mark.parametrize("V,dtype", [(2 ** 22, torch.bfloat16), (2 ** 22 - 3, torch.float32)])
def test_largest_vocabulary(V, dtype):
    from astrai_b200.inference.sample import sample_given

    x, u = _logits(2, V, dtype, 27, sigma=2.0)
    x[:, -1] = 12.0  # the last id among the candidates
    for s in (dict(), dict(k=200), dict(k=5000), dict(m=0.01), dict(p=0.5) if dtype == torch.bfloat16 else dict(k=50, p=0.9)):
        _check(x, u, **s)
    _check(x, torch.full((2,), 1.0, device="cuda"), k=40)
    with pytest.raises(ValueError, match="vocabulary"):
        sample_given(torch.zeros(1, 2 ** 22 + 1, device="cuda"), u[:1])
