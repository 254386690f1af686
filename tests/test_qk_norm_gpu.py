"""Per-head norm + rotation kernels against the formulas in 64 bits, forward and backward.

Tolerances: a result is the 64-bit one within one rounding to its type (half a spacing: 2^-8 of the value
for bfloat16, 2^-11 for float16, 2^-24 for float32) and the fp32 arithmetic before it. A head's values pass
through about 16 fp32 operations and a sum over its channels, each within 2^-24 of the largest magnitude
involved; 2^-19 of the row's largest magnitude covers them. Weight gradients add N products in fp32: their
error stays below (N / threads + 64) * 2^-24 of the sum of magnitudes, for which 2^-16 is ample here.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_SPACING = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def _clean_error_word():
    from astrai_b200.ops._ext import native

    native().read_error()
    yield
    torch.cuda.synchronize()
    assert native().read_error() == 0


def _table(rot, n, factor=1.0):
    inv = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    return (factor * torch.stack([a.cos(), a.sin()], -1)).float()


def _turn(x, cs, layout, rot, off, transpose=False):
    """64-bit rotation through a [rot, rot] matrix per token."""
    m = torch.zeros(x.shape[0], rot, rot, dtype=torch.float64, device=x.device)
    i = torch.arange(rot // 2, device=x.device)
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    c, s = cs[..., 0].double(), cs[..., 1].double()
    m[:, a, a], m[:, a, b], m[:, b, a], m[:, b, b] = c, -s, s, c
    if transpose:
        m = m.transpose(1, 2)
    y = x.clone()
    y[..., off: off + rot] = torch.einsum("tij,thj->thi", m, x[..., off: off + rot])
    return y


def _oracle(x, wq, wk, cs, hq, layout, norm, rot, off, eps, dy=None):
    x = x.double()
    h, d = x.shape[1], x.shape[2]
    w = torch.cat([wq.double().expand(hq, d), wk.double().expand(h - hq, d)])
    z = _turn(x, cs, layout, rot, off) if norm == "after" else x
    rms = (z.square().mean(-1, keepdim=True) + eps).sqrt()
    u = z / rms
    y = {"after": lambda: u * w, "before": lambda: _turn(u * w, cs, layout, rot, off),
         "none": lambda: _turn(x, cs, layout, rot, off)}[norm]()
    if dy is None:
        return y
    g = dy.double()
    if norm == "none":
        return y, _turn(g, cs, layout, rot, off, True), None, None
    if norm == "before":
        g = _turn(g, cs, layout, rot, off, True)
    gu = g * u
    dz = (g * w - u * (g * w * u).mean(-1, keepdim=True)) / rms
    dx = _turn(dz, cs, layout, rot, off, True) if norm == "after" else dz
    return y, dx, gu, rms


def _close(got, want, dtype, scale):
    """scale: the row's largest magnitude, broadcast against want."""
    tol = HALF_SPACING[dtype] * want.abs() + 2.0 ** -19 * scale + 1e-30
    worst = ((got.double() - want).abs() / tol).max().item()
    assert worst <= 1.0, worst


CASES = [
    # rows, seq, hq, hkv, D, rot, off, layout, norm, dtype
    (1, 1, 1, 1, 64, 64, 0, "interleaved", "after", torch.bfloat16),
    (7, 3, 16, 4, 128, 128, 0, "interleaved", "after", torch.bfloat16),
    (7, 3, 16, 4, 128, 128, 0, "half", "before", torch.bfloat16),
    (33, 33, 24, 4, 64, 32, 0, "half", "before", torch.float16),
    (33, 11, 5, 5, 96, 64, 16, "half", "after", torch.float32),
    (65, 13, 7, 1, 96, 48, 48, "interleaved", "before", torch.float32),
    (129, 129, 3, 3, 192, 64, 128, "interleaved", "after", torch.bfloat16),
    (130, 65, 2, 1, 256, 256, 0, "half", "after", torch.float16),
    (3, 3, 1, 0, 8, 8, 0, "half", "after", torch.float32),
    (61, 61, 9, 2, 72, 8, 0, "interleaved", "none", torch.bfloat16),
    (61, 61, 9, 2, 40, 24, 8, "half", "none", torch.float32),
    (2500, 1250, 12, 4, 128, 128, 0, "interleaved", "after", torch.bfloat16),
    (700, 350, 40, 8, 256, 128, 64, "half", "before", torch.float32),  # rows that take several launches
    (1301, 77, 31, 9, 96, 96, 0, "interleaved", "before", torch.float16),
]


def _inputs(rows, hq, hkv, d, dtype, seed=0, extra=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, hq + hkv, d, device="cuda", generator=g)
    x = x * torch.exp(torch.randn(rows, hq + hkv, 1, device="cuda", generator=g))  # heads of different scales
    buf = torch.full((rows, (hq + hkv) * d + extra), float("nan"), device="cuda", dtype=dtype)
    buf[:, : (hq + hkv) * d] = x.reshape(rows, -1).to(dtype)
    w = [(1 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(dtype) for _ in range(2)]
    dy = torch.randn(rows, (hq + hkv) * d, device="cuda", generator=g).to(dtype)
    return buf, w[0], w[1], dy


@pytest.mark.parametrize("rows,seq,hq,hkv,d,rot,off,layout,norm,dtype", CASES)
@pytest.mark.parametrize("factor", [1.0, 1.25])
def test_forward_and_backward_match_the_formulas(rows, seq, hq, hkv, d, rot, off, layout, norm, dtype, factor):
    from astrai_b200.ops.qk_norm import qk_norm_rope

    used, eps = (hq + hkv) * d, 1e-5
    buf, wq, wk, dy = _inputs(rows, hq, hkv, d, dtype)
    x = buf[:, :used].clone().requires_grad_()
    wq, wk = wq.requires_grad_(), wk.requires_grad_()
    table = _table(rot, seq + 5, factor)
    pos = (torch.arange(rows, device="cuda") % seq + 3).int()
    y = qk_norm_rope(x, hq, hkv, d, table, wq, wk, positions=pos, eps=eps, layout=layout, norm=norm, rot_dim=rot,
                     rot_off=off)
    xv, gv = x.detach().view(rows, -1, d), dy.view(rows, -1, d)
    want, dx, gu, rms = _oracle(xv, wq.detach(), wk.detach(), table[pos.long()], hq, layout, norm, rot, off, eps, gv)
    _close(y.detach().view_as(want), want, dtype, want.abs().amax(-1, keepdim=True))
    grads = torch.autograd.grad(y, (x,) if norm == "none" else (x, wq, wk), dy)
    spread = gv.double().abs().amax(-1, keepdim=True) * 2 * factor
    if rms is not None:
        spread = spread * (2 * max(wq.abs().max().item(), wk.abs().max().item())) / rms
    _close(grads[0].view_as(dx), dx, dtype, spread)
    if norm != "none":
        for got, part in zip(grads[1:], (gu[:, :hq], gu[:, hq:])):
            ref, mag = part.sum((0, 1)), part.abs().sum((0, 1))
            tol = HALF_SPACING[dtype] * ref.abs() + 2.0 ** -16 * mag + 1e-30
            assert ((got.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("norm", ["after", "before", "none"])
def test_gradient_matches_central_differences(layout, norm):
    from astrai_b200.ops.qk_norm import qk_norm_rope

    rows, hq, hkv, d, rot, off, eps = 2, 2, 1, 16, 8, 8, 1e-6
    buf, wq, wk, dy = _inputs(rows, hq, hkv, d, torch.float32, seed=3)
    table = _table(rot, rows)
    pos = torch.arange(rows, device="cuda").int()
    leaves = [t.clone().requires_grad_() for t in ((buf,) if norm == "none" else (buf, wq, wk))]
    y = qk_norm_rope(leaves[0], hq, hkv, d, table, *(leaves[1:] or (None, None)), positions=pos, eps=eps,
                     layout=layout, norm=norm, rot_dim=rot, rot_off=off)
    grads = torch.autograd.grad(y, leaves, dy)

    def loss(x, q, k):
        return (_oracle(x.view(rows, -1, d), q, k, table[pos.long()], hq, layout, norm, rot, off, eps).reshape(rows, -1)
                * dy.double()).sum()

    args = [buf.double(), wq.double(), wk.double()]
    for n, grad in enumerate(grads):
        flat = args[n].reshape(-1)
        num = torch.zeros_like(flat)
        for i in range(flat.numel()):
            step = 1e-5 * max(1.0, abs(flat[i].item()))
            for sign in (1, -1):
                moved = flat.clone()
                moved[i] += sign * step
                a = list(args)
                a[n] = moved.view_as(args[n])
                num[i] += sign * loss(*a) / (2 * step)
        # central differences: third derivatives times step^2 (about 1e-9 here), then the fp32 gradient itself
        scale = num.abs().max()
        assert (grad.double().reshape(-1) - num).abs().max() <= 2.0 ** -18 * scale + 1e-7


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_wide_buffer_in_place_and_row_positions(dtype, layout):
    """The value columns behind the keys hold NaN: they are neither read nor written."""
    from astrai_b200.ops.qk_norm import qk_norm_rope, qk_norm_rope_

    rows, seq, hq, hkv, d = 10, 5, 6, 2, 64
    used = (hq + hkv) * d
    buf, wq, wk, _ = _inputs(rows, hq, hkv, d, dtype, extra=hkv * d)
    table = _table(d, seq)
    want = _oracle(buf[:, :used].reshape(rows, -1, d), wq, wk, table[torch.arange(rows, device="cuda") % seq], hq, layout,
                   "after", d, 0, 1e-6)
    y = qk_norm_rope(buf, hq, hkv, d, table, wq, wk, seq_len=seq, layout=layout)
    assert y.shape == (rows, used)
    _close(y.view_as(want), want, dtype, want.abs().amax(-1, keepdim=True))
    before = buf[:, used:].clone()
    assert qk_norm_rope_(buf, hq, hkv, d, table, wq, wk, seq_len=seq, layout=layout) is buf
    assert torch.equal(buf[:, :used], y)
    assert torch.equal(buf[:, used:].isnan(), before.isnan())
    # a wide leaf gets a gradient of its own width, zero behind the keys
    wide = torch.nan_to_num(buf).requires_grad_()
    g = torch.autograd.grad(qk_norm_rope(wide, hq, hkv, d, table, wq, wk, seq_len=seq, layout=layout).sum(), wide)[0]
    assert g.shape == wide.shape and (g[:, used:] == 0).all() and torch.isfinite(g).all()


def test_rows_of_any_stride_other_streams_and_no_rows():
    from astrai_b200.ops.qk_norm import qk_norm_rope

    hq, hkv, d, rows = 4, 2, 64, 9
    buf, wq, wk, _ = _inputs(rows, hq, hkv, d, torch.bfloat16)
    table = _table(d, rows)
    want = qk_norm_rope(buf, hq, hkv, d, table, wq, wk, seq_len=rows)
    odd = torch.zeros(rows, buf.shape[1] + 3, device="cuda", dtype=buf.dtype)  # rows off the 16-byte grid
    odd[:, 1: 1 + buf.shape[1]] = buf
    assert torch.equal(qk_norm_rope(odd[:, 1: 1 + buf.shape[1]], hq, hkv, d, table, wq, wk, seq_len=rows), want)
    spaced = torch.zeros(rows * 2, buf.shape[1], device="cuda", dtype=buf.dtype)
    spaced[::2] = buf
    assert torch.equal(qk_norm_rope(spaced[::2], hq, hkv, d, table, wq, wk, seq_len=rows), want)
    assert torch.equal(qk_norm_rope(buf, hq, hkv, d, table, wq, wk, positions=torch.arange(rows, device="cuda")), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = qk_norm_rope(buf, hq, hkv, d, table, wq, wk, seq_len=rows)
    side.synchronize()
    assert torch.equal(got, want)
    empty = buf[:0].clone().requires_grad_()
    wq, wk = wq.requires_grad_(), wk.requires_grad_()
    y = qk_norm_rope(empty, hq, hkv, d, table, wq, wk, seq_len=rows)
    grads = torch.autograd.grad(y, (empty, wq, wk), y)
    assert y.shape == (0, (hq + hkv) * d) and grads[0].shape == empty.shape
    assert all((g == 0).all() for g in grads[1:])


def test_zero_rows_and_non_finite_values_stay_in_their_head():
    from astrai_b200.ops.qk_norm import qk_norm_rope

    hq, hkv, d, rows = 4, 2, 128, 6
    buf, wq, wk, dy = _inputs(rows, hq, hkv, d, torch.bfloat16, seed=5)
    buf[1, :d] = 0
    buf[2, d: 2 * d] = float("inf")
    buf[3, 3 * d + 5] = float("nan")
    table = _table(d, rows)
    x = buf.clone().requires_grad_()
    y = qk_norm_rope(x, hq, hkv, d, table, wq, wk, seq_len=rows)
    g = torch.autograd.grad(y, x, dy)[0]
    bad = torch.zeros(rows, hq + hkv, dtype=torch.bool, device="cuda")
    bad[2, 1] = bad[3, 3] = True
    for t in (y.detach(), g):
        t = t.view(rows, hq + hkv, d)
        assert (torch.isfinite(t).all(-1) == ~bad).all()
    assert (y.view(rows, -1, d)[1, 0] == 0).all()


def test_position_outside_the_table_sets_the_error_word():
    from astrai_b200.ops._ext import native
    from astrai_b200.ops.qk_norm import qk_norm_rope

    hq, hkv, d = 2, 1, 64
    buf, wq, wk, _ = _inputs(3, hq, hkv, d, torch.float32)
    table = _table(d, 4)
    y = qk_norm_rope(buf, hq, hkv, d, table, None, None, positions=torch.tensor([1, 4, -1], device="cuda").int(),
                     norm="none")
    assert native().read_error() == 6
    assert torch.equal(y[1:], buf[1:])


def test_refusals():
    from astrai_b200.ops.qk_norm import qk_norm_rope, qk_norm_rope_

    hq, hkv, d, rows = 2, 1, 64, 4
    buf, wq, wk, _ = _inputs(rows, hq, hkv, d, torch.bfloat16)
    t = _table(d, rows)

    def call(x=buf, h=hq, D=d, table=t, q=wq, k=wk, fn=qk_norm_rope, **kw):
        kw.setdefault("seq_len", rows)
        return fn(x, h, hkv, D, table, q, k, **kw)

    call()
    for kw in (dict(layout="other"), dict(norm="other"), dict(x=buf[:, :-8]), dict(x=buf[None]), dict(seq_len=None),
               dict(rot_dim=32), dict(rot_dim=d, rot_off=8), dict(q=None), dict(k=wk[:-8]),
               dict(positions=torch.zeros(rows + 1, device="cuda").int())):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(table=t.double()), dict(table=t.cpu()), dict(q=wq.float()), dict(q=wq.cpu()),
               dict(x=buf.to(torch.float64)),
               dict(table=_table(12, rows), rot_dim=12), dict(D=60, table=_table(56, rows), rot_dim=56, q=wq[:60], k=wk[:60])):
        with pytest.raises(RuntimeError):
            call(**kw)
    with pytest.raises(RuntimeError):
        call(x=buf.clone().requires_grad_(), fn=qk_norm_rope_)


def test_in_place_is_noticed_and_refuses_rows_that_overlap():
    from astrai_b200.ops.qk_norm import qk_norm_rope, qk_norm_rope_

    hq, hkv, d, rows = 2, 1, 64, 4
    buf, wq, wk, _ = _inputs(rows, hq, hkv, d, torch.bfloat16)
    t = _table(d, rows)
    w = torch.ones_like(buf).requires_grad_()
    out = buf * w  # saves buf
    qk_norm_rope_(buf, hq, hkv, d, t, wq, wk, seq_len=rows)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    same = buf[:1].expand(rows, -1)  # read, but not written
    y = qk_norm_rope(same, hq, hkv, d, t, wq, wk, seq_len=rows)
    assert torch.equal(y, qk_norm_rope(same.contiguous(), hq, hkv, d, t, wq, wk, seq_len=rows))
    with pytest.raises(RuntimeError):
        qk_norm_rope_(same, hq, hkv, d, t, wq, wk, seq_len=rows)
    with torch.inference_mode():
        x = buf.clone()
        assert torch.equal(qk_norm_rope_(x, hq, hkv, d, t, wq, wk, seq_len=rows),
                           qk_norm_rope(buf, hq, hkv, d, t, wq, wk, seq_len=rows))


def test_a_weight_of_any_shape_gets_a_gradient_of_it():
    from astrai_b200.ops.qk_norm import qk_norm_rope

    buf, wq, wk, dy = _inputs(6, 2, 1, 64, torch.bfloat16)
    t = _table(64, 6)
    flat = [w.clone().requires_grad_() for w in (wq, wk)]
    row = [w.view(1, 64).clone().requires_grad_() for w in (wq, wk)]
    a, b = (torch.autograd.grad(qk_norm_rope(buf, 2, 1, 64, t, *w, seq_len=6), w, dy) for w in (flat, row))
    assert all(y.shape == (1, 64) and torch.equal(x, y[0]) for x, y in zip(a, b))


def test_weight_gradients_are_the_same_every_time():
    from astrai_b200.ops.qk_norm import qk_norm_rope

    buf, wq, wk, dy = _inputs(5000, 8, 2, 128, torch.bfloat16)
    x, wq, wk = buf.requires_grad_(), wq.requires_grad_(), wk.requires_grad_()
    table = _table(128, 5000)
    runs = [torch.autograd.grad(qk_norm_rope(x, 8, 2, 128, table, wq, wk, seq_len=5000), (x, wq, wk), dy)
            for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_autograd_node():
    """What autograd asks of a node: saved-tensor hooks, one backward unless kept, no second derivative, no tangents,
    gradients for some of the inputs, a checkpointed region."""
    from torch.utils.checkpoint import checkpoint

    from astrai_b200.ops.qk_norm import qk_norm_rope

    buf, wq, wk, dy = _inputs(6, 2, 1, 64, torch.bfloat16)
    t, pos = _table(64, 6), torch.arange(6, device="cuda").int()
    x, wq, wk = buf.clone().requires_grad_(), wq.clone().requires_grad_(), wk.clone().requires_grad_()

    def run(a=x, b=wq, c=wk, **kw):
        return qk_norm_rope(a, 2, 1, 64, t, b, c, **(kw or dict(positions=pos)))

    y = run()
    assert y.grad_fn.name() == "QkNormRopeBackward" and not run(x.detach(), wq.detach(), wk.detach()).requires_grad
    want = torch.autograd.grad(y, (x, wq, wk), dy, retain_graph=True)
    again = torch.autograd.grad(y, (x, wq, wk), dy)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, x, dy)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda v: kept.append(v.shape) or v.cpu(), lambda v: v.cuda()):
        hooked = torch.autograd.grad(run(), (x, wq, wk), dy)
    remade = torch.autograd.grad(checkpoint(run, x, wq, wk, use_reentrant=False), (x, wq, wk), dy)
    assert len(kept) == 5
    for got in (again, hooked, remade):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(torch.autograd.grad(run(x, wq.detach(), wk.detach()), x, dy)[0], want[0])
    assert torch.equal(torch.autograd.grad(run(x.detach()), wk, dy)[0], want[2])
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(run(), x, dy, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            run(torch.autograd.forward_ad.make_dual(x, dy))
    y = run()
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)
    turned = qk_norm_rope(x, 2, 1, 64, t, norm="none", seq_len=6)
    turned.backward(dy)
    assert x.grad is not None and wq.grad is None
