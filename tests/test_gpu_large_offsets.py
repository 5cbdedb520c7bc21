"""Operands whose offsets pass 2^31 elements: sampled rows against the same rows in small tensors."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n_q", [1, 3, 700])
def test_rows_of_a_wide_store(cuda, n_q, dtype):
    """Keys and values as columns of a store whose rows are 2^22 elements apart: 700 rows reach past 2^31 elements."""
    from magic_amd.model.attention import attention_plan, segment_attention
    gen = torch.Generator(device=cuda).manual_seed(n_q)
    n, h, D, ld = 700, 2, 64, 1 << 22
    store = torch.empty(n * ld, dtype=dtype, device=cuda)
    wide = [store[i * h * D:].as_strided((n, h, D), (ld, D, 1)) for i in range(2)]
    flat = [torch.randn(n, h, D, generator=gen, device=cuda).to(dtype) for _ in range(2)]
    for w, f in zip(wide, flat):
        w.copy_(f)
    q = torch.randn(n_q, h, D, generator=gen, device=cuda).to(dtype)
    d = torch.randn(n_q, h, D, generator=gen, device=cuda).to(dtype)
    mask = torch.rand(n, generator=gen, device=cuda) < 0.8
    plan = attention_plan([n_q], [n], cuda)
    res = []
    for k, v in (flat, wide):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = segment_attention(*leaves, plan, key_mask=mask)
        res.append([out.detach(), *torch.autograd.grad(out, leaves, d)])
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize("dtype,rows,lens,masked", [(torch.bfloat16, 600000, 40, False), (torch.bfloat16, 600000, 600, True),
                                                    (torch.float32, 600000, 600, False)], ids=["bf16", "bf16-gathered", "f32-scaled"])
def test_attention_of_more_than_2_31_elements(cuda, dtype, rows, lens, masked):
    from magic_amd.model.attention import attention_plan, segment_attention
    h, D = 60, 64
    assert rows * h * D > 1 << 31
    gen = torch.Generator(device=cuda).manual_seed(1)
    q, k, v, d = (torch.empty(rows, h, D, dtype=dtype, device=cuda).normal_(generator=gen) for _ in range(4))
    mask = torch.rand(rows, generator=gen, device=cuda) < 0.5 if masked else None
    seg = rows // lens
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = segment_attention(*leaves, attention_plan([lens] * seg, device=cuda), key_mask=mask)
    grads = torch.autograd.grad(out, leaves, d)
    part = list(range(8)) + list(range(seg // 2, seg // 2 + 4)) + list(range(seg - 8, seg))      # (enough for the same tiles)
    at = torch.cat([torch.arange(s * lens, (s + 1) * lens, device=cuda) for s in part])
    small = [t.detach()[at].requires_grad_(True) for t in leaves]
    want = segment_attention(*small, attention_plan([lens] * len(part), device=cuda), key_mask=None if mask is None else mask[at])
    wgrads = torch.autograd.grad(want, small, d[at])
    for a, b in zip((out, *grads), (want, *wgrads)):
        assert torch.equal(a[at], b)


def test_head_norm_of_more_than_2_31_elements(cuda):
    from magic_amd.model.attention import head_norm_rope
    rows, h, D = 600000, 60, 64
    gen = torch.Generator(device=cuda).manual_seed(2)
    q = torch.empty(rows, h, D, dtype=torch.bfloat16, device=cuda).normal_(generator=gen)
    k = torch.empty(rows, 1, D, dtype=torch.bfloat16, device=cuda).normal_(generator=gen)
    w = torch.rand(D, generator=gen, device=cuda) + 0.5
    pos = torch.arange(rows, dtype=torch.int32, device=cuda)
    d = torch.empty(rows, h, D, dtype=torch.bfloat16, device=cuda).normal_(generator=gen)
    at = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device=cuda)
    ql = q.requires_grad_(True)
    y = head_norm_rope(ql, k, w, w, pos)[0]
    g = torch.autograd.grad(y, ql, d)[0]
    qs = q.detach()[at].requires_grad_(True)
    ys = head_norm_rope(qs, k[at], w, w, pos[at])[0]
    assert torch.equal(y[at], ys) and torch.equal(g[at], torch.autograd.grad(ys, qs, d[at])[0])


@pytest.mark.parametrize("f", [1, 4])
def test_codes_of_more_than_2_30_blocks(cuda, f):
    """Block numbers that no longer fit the 32-bit form of the pack kernel; codes past 2^32 bytes."""
    from magic_amd.model.act8 import act8_pack, act8_unpack, act8_weight_grad
    n = (1 << 30) + 77
    x = torch.empty(n, f, device=cuda).normal_(generator=torch.Generator(device=cuda).manual_seed(f))
    a = act8_pack(x)
    at = torch.tensor([0, 1, n // 3, 1 << 28, (1 << 30) - 1, 1 << 30, n - 1], device=cuda)
    b = act8_pack(x[at])
    assert torch.equal(a.codes[at], b.codes) and torch.equal(a.exps[at], b.exps)
    back = act8_unpack(a)
    assert torch.equal(back[at], act8_unpack(b))
    dy = torch.zeros(n, 1, device=cuda)
    dy[at] = 1.0
    del x
    want, mag = act8_unpack(b).double().sum(0), act8_unpack(b).double().abs().sum(0)
    assert ((act8_weight_grad(dy, a)[0].double() - want).abs() <= 8 * 2.0 ** -24 * mag).all()     # (six sums and the zeros)
