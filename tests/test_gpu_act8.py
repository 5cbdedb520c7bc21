"""8-bit activation checkpoints: codes against a 64-bit restatement of their definition (exact), the weight gradient
against 64-bit products of the values the codes stand for, and the linear layer that uses them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def definition(x):
    """(codes, exps) of a float32 matrix, in numpy float64: every step is exact but the rounding."""
    x = x.double().cpu().numpy()
    n, f = x.shape
    stride, nb = (f + 15) // 16 * 16, (f + 31) // 32
    codes, exps = np.zeros((n, stride), np.int64), np.zeros((n, nb), np.int64)
    for b in range(nb):
        blk = x[:, 32 * b:32 * b + 32]
        for i in range(n):
            row = blk[i]
            if not np.isfinite(row).all():
                exps[i, b] = 255
                continue
            e = -126
            while np.abs(np.rint(row * 2.0 ** -e)).max() > 127:
                e += 1
            exps[i, b] = e + 127
            codes[i, 32 * b:32 * b + len(row)] = np.rint(row * 2.0 ** -e)
    return codes, exps


@pytest.mark.parametrize("n,f", [(1, 1), (3, 5), (17, 32), (40, 33), (9, 64), (21, 100), (64, 192), (5, 1023)])
def test_pack_and_unpack(cuda, n, f):
    from magic_amd.model.act8 import act8_pack, act8_unpack
    gen = torch.Generator().manual_seed(n * f)
    x = torch.randn(n, f, generator=gen) * torch.exp(4 * torch.randn(n, 1, generator=gen))
    if f > 2:
        x[0, :3] = torch.tensor([127.5, -127.5, 1.5])             # rounds to 128 at the smaller scale
        x[n // 2] = 0.0
        x[-1, 0] = 2.0 ** -140                                    # a subnormal
    a = act8_pack(x.to(cuda))
    codes, exps = definition(x)
    assert a.cols == f and np.array_equal(a.codes.cpu().numpy(), codes) and np.array_equal(a.exps.cpu().numpy(), exps)
    y = act8_unpack(a).cpu().double()
    want = torch.from_numpy(codes[:, :f] * 2.0 ** (np.repeat(exps, 32, 1)[:, :f] - 127.0))
    assert torch.equal(y, want)
    step = 2.0 ** (np.repeat(exps, 32, 1)[:, :f] - 127.0)
    assert (np.abs(y.numpy() - x.double().numpy()) <= step / 2).all()


def test_pack_strides_extremes_and_non_finite(cuda):
    from magic_amd.model.act8 import act8_pack, act8_unpack
    x = torch.randn(37, 96, device=cuda)
    want = act8_pack(x)
    wide = torch.zeros(37, 200, device=cuda)
    for off in (0, 4, 3):                                         # row stride, alignment
        wide[:, off:off + 96] = x
        got = act8_pack(wide[:, off:off + 96])
        assert torch.equal(got.codes, want.codes) and torch.equal(got.exps, want.exps)
    got = act8_pack(x.t().contiguous().t())
    assert torch.equal(got.codes, want.codes)
    big = torch.full((2, 32), torch.finfo(torch.float32).max, device=cuda)
    assert torch.equal(act8_unpack(act8_pack(torch.full((2, 32), 2.0 ** 127, device=cuda))),
                       torch.full((2, 32), 2.0 ** 127, device=cuda))
    # the largest float is half a step of its block away from 2^128: it reads back as an infinity of that size
    assert torch.isinf(act8_unpack(act8_pack(big))).all() or (act8_unpack(act8_pack(big)) / big - 1).abs().max() <= 2 ** -7
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[3, 40] = bad
        back = act8_unpack(act8_pack(y))
        assert torch.isnan(back[3, 32:64]).all()
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[3, 32:64] = False
        assert torch.equal(back[keep], act8_unpack(want)[keep])
    assert act8_unpack(act8_pack(x[:0])).shape == (0, 96)


@pytest.mark.parametrize("n,m,f", [(1, 1, 1), (15, 3, 5), (129, 64, 192), (300, 37, 69), (1000, 256, 256), (2001, 130, 100),
                                   (777, 320, 40), (4096, 8, 8), (0, 4, 8), (257, 129, 257)])
def test_weight_gradient(cuda, n, m, f):
    """|error| <= (n + 8) 2^-24 sum |dy| |xhat|: three exact planes of dy against one of xhat, float32 sums."""
    from magic_amd.model.act8 import act8_pack, act8_unpack, act8_weight_grad
    gen = torch.Generator(device=cuda).manual_seed(n + m)
    x = torch.randn(n, f, generator=gen, device=cuda) * torch.exp(torch.randn(n, 1, generator=gen, device=cuda))
    dy = torch.randn(n, m, generator=gen, device=cuda)
    a = act8_pack(x)
    xh = act8_unpack(a).double()
    want, mag = dy.double().t() @ xh, dy.double().abs().t() @ xh.abs()
    got = act8_weight_grad(dy, a)
    assert got.shape == (m, f)
    assert ((got.double() - want).abs() <= (n + 8) * 2.0 ** -24 * mag).all()
    assert torch.equal(got, act8_weight_grad(dy, a))
    wide = torch.zeros(n, m + 3, device=cuda)                     # a gradient that is a column block of a wider matrix
    wide[:, 1:m + 1] = dy
    assert ((act8_weight_grad(wide[:, 1:m + 1], a).double() - want).abs() <= (n + 8) * 2.0 ** -24 * mag).all()
    assert torch.equal(torch.ops.magic.act8_weight_grad(dy, a.codes, a.exps, f), got)


def test_weight_gradient_carries_nan(cuda):
    from magic_amd.model.act8 import act8_pack, act8_weight_grad
    x, dy = torch.randn(100, 64, device=cuda), torch.randn(100, 8, device=cuda)
    x[7, 40] = float("inf")
    dw = act8_weight_grad(dy, act8_pack(x))
    assert torch.isnan(dw[:, 32:]).all() and torch.isfinite(dw[:, :32]).all()


@pytest.mark.parametrize("n,f,m", [(1201, 69, 37), (3000, 192, 64), (1, 8, 8)])
def test_linear_with_8_bit_activations(cuda, n, f, m):
    """Forward value and input gradient are those of the float32 layer bit for bit; the weight gradient differs by at
    most half a step of every code: sum_n |dy| step / 2 (plus the float32 sum)."""
    from magic_amd.model.act8 import act8_pack
    from magic_amd.model.gat import linear_nobias
    gen = torch.Generator(device=cuda).manual_seed(f)
    x = torch.randn(n, f, generator=gen, device=cuda, requires_grad=True)
    w = torch.randn(m, f, generator=gen, device=cuda, requires_grad=True)
    dy = torch.randn(n, m, generator=gen, device=cuda)
    y0, y8 = linear_nobias(x, w), linear_nobias(x, w, act_bits=8)
    assert torch.equal(y0, y8)
    (dx0, dw0), (dx8, dw8) = (torch.autograd.grad(y, (x, w), dy) for y in (y0, y8))
    assert torch.equal(dx0, dx8)
    step = torch.exp2(act8_pack(x.detach()).exps.double().repeat_interleave(32, 1)[:, :f] - 127)
    ref = dy.double().t() @ x.detach().double()
    mag = dy.double().abs().t() @ x.detach().double().abs()
    bound = dy.double().abs().t() @ (step / 2) + (n + 8) * 2.0 ** -24 * 1.01 * mag
    assert ((dw8.double() - ref).abs() <= bound).all()


def test_linear_keeps_a_quarter_of_the_memory(cuda):
    """Bytes the layer holds for its backward pass besides the weight: 4 N F, and (1 + 1 / 32) N F in 8 bits."""
    from magic_amd.model.gat import linear_nobias
    x = torch.randn(2000, 256, device=cuda)
    w = torch.randn(64, 256, device=cuda, requires_grad=True)
    held = {}
    for bits in (32, 8):
        y = linear_nobias(x, w, act_bits=bits)              # (kept: the node lives as long as its output)
        saved = y.grad_fn.saved_tensors
        held[bits] = sum(t.numel() * t.element_size() for t in saved if t.data_ptr() != w.data_ptr())
    assert held == {32: 4 * x.numel(), 8: x.numel() + x.numel() // 32}


def test_expanded_and_overlapping_rows(cuda):
    """Operands whose rows share memory, as broadcasts and their gradients do."""
    from magic_amd.model.act8 import act8_pack, act8_weight_grad
    from magic_amd.model.gat import linear_nobias
    row = torch.randn(1, 40, device=cuda)
    a, b = act8_pack(row.expand(50, 40)), act8_pack(row.repeat(50, 1))
    assert torch.equal(a.codes, b.codes) and torch.equal(a.exps, b.exps)
    dy = torch.randn(1, 12, device=cuda)
    assert torch.equal(act8_weight_grad(dy.expand(50, 12), a), act8_weight_grad(dy.repeat(50, 1), a))
    w = torch.randn(12, 40, device=cuda, requires_grad=True)
    x = torch.randn(50, 40, device=cuda, requires_grad=True)
    y = linear_nobias(x, w, act_bits=8)
    got = torch.autograd.grad((y * dy).sum(), (x, w), retain_graph=True)
    via = torch.autograd.grad(y, (x, w), dy.expand(50, 12))
    assert all(torch.equal(p, q) for p, q in zip(got, via))
    window = torch.randn(89, device=cuda).as_strided((50, 40), (1, 1))
    assert torch.equal(act8_pack(window).codes, act8_pack(window.contiguous()).codes)
    assert torch.equal(linear_nobias(row.expand(50, 40), w, act_bits=8), linear_nobias(row.repeat(50, 1), w, act_bits=8))


@pytest.mark.parametrize("m", [1, 40, 64, 96, 130])
@pytest.mark.parametrize("n,f,pad", [(1, 32, 0), (33, 64, 0), (700, 176, 0), (259, 192, 4), (64, 52, 12), (97, 96, 0), (65, 100, 3),
                                     (2000, 256, 0)])
def test_codes_written_beside_the_product(cuda, n, f, pad, m):
    """The product's pass over x writes the codes that a pass of its own writes, whichever kernel takes the shape."""
    from magic_amd import _lib
    gen = torch.Generator(device=cuda).manual_seed(f + m)
    x = (torch.randn(n, f + pad, generator=gen, device=cuda) * torch.exp2(torch.randint(-30, 30, (n, 1), generator=gen, device=cuda).float()))[:, :f]
    x[n // 2, f // 3] = float("inf")
    x[n - 1, :] = 0.0
    w = torch.randn(m, f, generator=gen, device=cuda)
    y, codes, exps = _lib.act8_linear_fwd(x, w)
    want = _lib.act8_pack(x)
    assert torch.equal(codes, want[0]) and torch.equal(exps, want[1])
    assert torch.equal(y.view(torch.int32), _lib.proj_fwd(x, w, m, 0, 0)[0].view(torch.int32))
    assert torch.ops.magic.act8_unpack(codes, exps, f).shape == (n, f)


def test_linear_of_one_row_and_of_none(cuda):
    from magic_amd.model.gat import linear_nobias
    w = torch.randn(6, 40, device=cuda, requires_grad=True)
    col = torch.randn(40, 1, device=cuda)
    x = col.t().requires_grad_(True)                     # one row, row stride 1
    y = linear_nobias(x, w, act_bits=8)
    dx, dw = torch.autograd.grad(y, (x, w), torch.randn(6, 1, device=cuda).t())
    assert torch.equal(y.detach(), linear_nobias(col.t().clone().view(1, 40), w.detach())) and torch.isfinite(dx).all() and torch.isfinite(dw).all()
    with torch.no_grad():
        assert torch.equal(linear_nobias(col.t(), w, act_bits=8), y)
    none = torch.zeros(0, 40, device=cuda, requires_grad=True)
    y = linear_nobias(none, w, act_bits=8)
    dx, dw = torch.autograd.grad(y.sum(), (none, w))
    assert y.shape == (0, 6) and dx.shape == (0, 40) and not dw.any()


def test_every_width_up_to_two_blocks(cuda):
    """Row ends of every kind: the last columns of the last row are the tensor's last."""
    from magic_amd.model.act8 import act8_pack, act8_unpack
    for f in range(1, 70):
        x = torch.randn(5, f, generator=torch.Generator().manual_seed(f))
        a = act8_pack(x.to(cuda))
        codes, exps = definition(x)
        assert np.array_equal(a.codes.cpu().numpy(), codes) and np.array_equal(a.exps.cpu().numpy(), exps), f
        assert np.array_equal(act8_unpack(a).cpu().double().numpy(), codes[:, :f] * 2.0 ** (np.repeat(exps, 32, 1)[:, :f] - 127.0)), f


def test_second_derivative_is_refused(cuda):
    """The backward pass forms plain values: a derivative of them raises instead of coming out as a constant's."""
    from magic_amd.model.gat import linear_nobias
    x = torch.randn(20, 32, device=cuda, requires_grad=True)
    w = torch.randn(4, 32, device=cuda, requires_grad=True)
    dy = torch.randn(20, 4, device=cuda, requires_grad=True)
    dx, dw = torch.autograd.grad(linear_nobias(x, w, act_bits=8), (x, w), dy, create_graph=True)
    for g in (dx, dw):                                    # (beside a term that has a derivative)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (g.sum() + x.sum() + w.sum()).backward(retain_graph=True)
