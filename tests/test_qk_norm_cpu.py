"""Per-head norm + rotation on the CPU: the plain path against the framework's separate operations, its
gradient, the scaled tables and the refusals. (The kernels are tested in test_qk_norm_gpu.py.)"""

import math

import pytest
import torch
import torch.nn.functional as F

from astrai_b200.ops.qk_norm import qk_norm_rope, qk_norm_rope_
from astrai_b200.ops.rope import apply_rope_reference, rope_table, scaled_rope_table


def _inputs(rows=6, hq=4, hkv=2, d=16, dtype=torch.float32):
    torch.manual_seed(0)
    return (torch.randn(rows, (hq + hkv) * d).to(dtype), (1 + 0.2 * torch.randn(d)).to(dtype),
            (1 + 0.2 * torch.randn(d)).to(dtype))


def _separate(x, wq, wk, hq, hkv, d, table, pos, norm, eps):
    z = x.view(1, -1, hq + hkv, d)
    cs = table[pos].unsqueeze(0)

    def n(t):
        return torch.cat([F.rms_norm(t[:, :, :hq], (d,), wq, eps), F.rms_norm(t[:, :, hq:], (d,), wk, eps)], 2)

    if norm == "before":
        z = n(z)
    z = apply_rope_reference(z, cs)
    if norm == "after":
        z = n(z)
    return z.reshape(x.shape)


@pytest.mark.parametrize("norm", ["after", "before", "none"])
def test_matches_the_separate_operations(norm):
    hq, hkv, d = 4, 2, 16
    x, wq, wk = _inputs(6, hq, hkv, d)
    table = rope_table(d, 9)
    pos = torch.tensor([3, 0, 8, 1, 1, 5])
    y = qk_norm_rope(x, hq, hkv, d, table, wq, wk, positions=pos, eps=1e-5, norm=norm)
    assert torch.allclose(y, _separate(x, wq, wk, hq, hkv, d, table, pos, norm, 1e-5), atol=2e-6)


def test_half_layout_is_a_permutation_of_the_interleaved_one():
    hq, hkv, d, rot = 3, 1, 24, 16
    x, wq, wk = _inputs(5, hq, hkv, d)
    table = rope_table(rot, 5)
    off = 8
    order = torch.arange(d)
    order[off: off + rot] = off + torch.cat([torch.arange(0, rot, 2), torch.arange(1, rot, 2)])
    xp = x.view(5, -1, d)[..., order].reshape(x.shape)
    half = qk_norm_rope(xp, hq, hkv, d, table, wq[order], wk[order], seq_len=5, layout="half", rot_dim=rot, rot_off=off)
    inter = qk_norm_rope(x, hq, hkv, d, table, wq, wk, seq_len=5, rot_dim=rot, rot_off=off)
    assert torch.allclose(half.view(5, -1, d), inter.view(5, -1, d)[..., order], atol=1e-6)
    keep = [c for c in range(d) if not off <= c < off + rot]
    plain = qk_norm_rope(x, hq, hkv, d, table, norm="none", seq_len=5, rot_dim=rot, rot_off=off)
    assert torch.equal(plain.view(5, -1, d)[..., keep], x.view(5, -1, d)[..., keep])


@pytest.mark.parametrize("norm", ["after", "before", "none"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_gradient_and_in_place(norm, layout):
    hq, hkv, d = 2, 1, 8
    x, wq, wk = (t.double() for t in _inputs(3, hq, hkv, d))
    table = rope_table(d, 3)

    def f(x, wq, wk):
        return qk_norm_rope(x, hq, hkv, d, table, wq, wk, seq_len=3, norm=norm, layout=layout)

    assert torch.autograd.gradcheck(f, [t.clone().requires_grad_() for t in (x, wq, wk)])
    wide = torch.cat([x, torch.full((3, d), float("nan"), dtype=x.dtype)], 1)
    out = qk_norm_rope_(wide, hq, hkv, d, table, wq, wk, seq_len=3, norm=norm, layout=layout)
    assert out is wide and torch.equal(wide[:, : x.shape[1]], f(x, wq, wk)) and wide[:, x.shape[1]:].isnan().all()


def test_scaled_tables():
    d, n, base = 32, 64, 1e4
    plain = rope_table(d, n, base)
    assert torch.equal(scaled_rope_table(d, n, base, "linear", 1.0), plain) or torch.allclose(
        scaled_rope_table(d, n, base, "linear", 1.0), plain, atol=1e-5)
    assert torch.allclose(scaled_rope_table(d, 4 * n, base, "linear", 4.0)[::4], plain, atol=1e-5)
    t = scaled_rope_table(d, n, base, "yarn", 8.0, original_max_len=4096)
    gain = 0.1 * math.log(8.0) + 1
    assert torch.allclose(t.norm(dim=-1), torch.full((n, d // 2), gain), atol=1e-5)
    assert torch.allclose(t[:, 0], gain * plain[:, 0], atol=1e-4)  # fast pairs keep their angles
    slow = torch.atan2(t[1, -1, 1], t[1, -1, 0]).double()
    assert abs(slow - torch.atan2(plain[1, -1, 1], plain[1, -1, 0]).double() / 8) < 1e-8  # slow ones are interpolated
    assert torch.allclose(scaled_rope_table(d, n, base, "yarn", 8.0, original_max_len=4096, attention_factor=1.0).norm(dim=-1),
                          torch.ones(n, d // 2), atol=1e-5)
    assert torch.allclose(scaled_rope_table(d, n, base, "yarn", 1.0, original_max_len=4096), plain, atol=1e-5)
    for bad in (dict(method="other"), dict(factor=0.0), dict(method="yarn"),
                dict(method="yarn", original_max_len=64, beta_fast=1.0)):
        with pytest.raises(ValueError):
            scaled_rope_table(d, n, base, **bad)


def test_refusals():
    hq, hkv, d = 4, 2, 16
    x, wq, wk = _inputs(6, hq, hkv, d)
    t = rope_table(d, 6)
    for kw in (dict(layout="x"), dict(norm="x"), dict(seq_len=None), dict(rot_dim=8), dict(rot_dim=d, rot_off=2),
               dict(positions=torch.zeros(5)), dict(q_weight=None), dict(k_weight=wk[:8])):
        args = dict(q_weight=wq, k_weight=wk, seq_len=6)
        args.update(kw)
        with pytest.raises(ValueError):
            qk_norm_rope(x, hq, hkv, d, t, **args)
    with pytest.raises(ValueError):
        qk_norm_rope(x[:, 1:], hq, hkv, d, t, wq, wk, seq_len=6)
    with pytest.raises(RuntimeError):
        qk_norm_rope_(x.clone().requires_grad_(), hq, hkv, d, t, wq, wk, seq_len=6)
