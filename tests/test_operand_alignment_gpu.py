"""Operands off the 16-byte grid that the kernels read: copied, whether they are contiguous or not."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _off(t, by=1):
    """A contiguous tensor equal to t whose memory starts `by` elements behind a 16-byte boundary."""
    buf = torch.zeros(t.numel() + 16, device=t.device, dtype=t.dtype)
    out = buf[by: by + t.numel()].view(t.shape)
    out.copy_(t)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out


def _inputs(rows, hq, hkv, d, dtype):
    from astrai_b200.ops.rope import rope_table

    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(rows, (hq + hkv) * d, device="cuda", generator=g).to(dtype)
    w = [(1 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(dtype) for _ in range(2)]
    dy = torch.randn(rows, (hq + hkv) * d, device="cuda", generator=g).to(dtype)
    return x, w[0], w[1], rope_table(d, rows, device="cuda"), dy


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 7, 2000])
@pytest.mark.parametrize("norm", ["after", "before", "none"])
def test_qk_norm_rope_of_contiguous_rows_off_the_grid(rows, norm, dtype):
    from astrai_b200.ops.qk_norm import qk_norm_rope

    hq, hkv, d = 4, 2, 64
    used = (hq + hkv) * d
    x, wq, wk, t, dy = _inputs(rows, hq, hkv, d, dtype)

    def run(x, wq=wq, wk=wk, dy=dy):
        leaves = [v.detach().requires_grad_() for v in (x, wq, wk)]
        y = qk_norm_rope(leaves[0], hq, hkv, d, t, leaves[1], leaves[2], norm=norm, seq_len=rows)
        with torch.no_grad():
            again = qk_norm_rope(x, hq, hkv, d, t, wq, wk, norm=norm, seq_len=rows)
        assert torch.equal(again, y.detach())
        return (y.detach(),) + torch.autograd.grad(y, leaves[:1] if norm == "none" else leaves, dy)

    want = run(x)
    odd = torch.full((rows, used + 3), float("nan"), device="cuda", dtype=dtype)  # contiguous, rows off the grid
    odd[:, :used] = x
    pitched = torch.full((rows, used + 16), float("nan"), device="cuda", dtype=dtype)
    pitched[:, :used] = x
    for name, args in dict(start=(_off(x),), width=(odd,), view=(pitched[:, : used + 1],), one=(odd[:, :used],),
                           gradient=(x, wq, wk, _off(dy, 3)), weights=(x, _off(wq), _off(wk, 2))).items():
        got = run(*args)
        assert got[1].shape == args[0].shape, name
        assert torch.equal(got[0], want[0]) and torch.equal(got[1][:, :used], want[1]), name
        assert (got[1][:, used:] == 0).all(), name
        assert all(torch.equal(a, b) for a, b in zip(got[2:], want[2:])), name


def test_qk_norm_rope_gradient_through_a_concatenation():
    """Gradients of pieces of a flat tensor are contiguous and start anywhere."""
    from astrai_b200.ops.qk_norm import qk_norm_rope

    x, wq, wk, t, dy = _inputs(5, 4, 2, 64, torch.bfloat16)
    leaf = x.requires_grad_()
    want = torch.autograd.grad(qk_norm_rope(leaf, 4, 2, 64, t, wq, wk, seq_len=5), leaf, dy)[0]
    y = qk_norm_rope(leaf, 4, 2, 64, t, wq, wk, seq_len=5)
    flat = torch.cat([torch.zeros(3, device="cuda", dtype=x.dtype), y.flatten()])
    assert torch.equal(torch.autograd.grad(flat, leaf, torch.cat([flat.detach()[:3], dy.flatten()]))[0], want)


@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_kv8_operands_off_the_grid(dtype):
    from astrai_b200.ops.kv8 import KV8, kv8_append, kv8_attention

    g = torch.Generator(device="cuda").manual_seed(0)
    B, S, H, D, page, block = 2, 3, 2, 64, 32, 16
    k, v = (torch.randn(B, S, H, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    q = torch.randn(B, S, 4, D, device="cuda", generator=g).to(dtype)
    i32 = dict(dtype=torch.int32, device="cuda")
    table, starts, lens = torch.tensor([[0, 1], [2, 3]], **i32), torch.tensor([0, 0], **i32), torch.tensor([3, 2], **i32)
    want, got = (KV8.allocate(4, H, page, D, block, "cuda") for _ in range(2))
    kv8_append(want, k, v, table, starts, lens)
    kv8_append(got, _off(k), _off(v, 3), table, starts, lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and want.k.any()
    assert torch.equal(kv8_attention(_off(q), want, table, lens), kv8_attention(q, want, table, lens))
    one = torch.zeros(1, 1, 4 * D + 3, device="cuda", dtype=dtype)  # one token cut from a wider odd buffer
    one[..., 1: -2] = q[:1, :1].flatten(2)
    cut = one[..., 1: -2].unflatten(-1, (4, D))
    assert torch.equal(kv8_attention(cut, want, table[:1], lens[:1]), kv8_attention(q[:1, :1], want, table[:1], lens[:1]))
