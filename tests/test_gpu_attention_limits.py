"""Segment attention at the ends of its ranges.

The cases are built so that their exact answers are simple: one key (or a few with equal logits) is ahead of all others by
more than 100, so that the others' probabilities, below 2^-144, are zeros in float32.  u = 2^-24, half a step of float32."""
import math

import pytest
import torch

from tests.test_gpu_attention import U, check, make, rope_reference, run

pytestmark = pytest.mark.gpu


def _close(got, want, mag, n=8):
    """|got - want| <= (n + 4) u mag plus the rounding of the result: n terms, and four roundings of the chain (or 2^-22 of
    the two planes)."""
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).abs()
    tol = (n + 4) * U * mag + half * want.abs() + 2.0 ** -120
    assert (err <= tol).all(), (float(err.max()), float((err / tol).max()))


# rows, keys, heads, width: two scaled planes, blocks of 32 rows, columns without tiles, three planes, narrow heads
SHAPES = {"planes": ([700, 30], [700, 41], 16, 64), "narrow_planes": ([2100], [2100], 16, 16), "small": ([50], [70], 4, 64),
          "whole_tiles": ([640], [640], 16, 64), "whole_tiles_of_one": ([64], [128], 4, 128), "few": ([1, 3], [700, 1100], 1, 32), "wide": ([300], [300], 8, 128), "ranges": ([1300], [1300], 2, 64)}


def _ahead(cuda, q_lens, kv_lens, h, D, dtype, far, kind):
    """Operands, options and the index of the key that takes everything, for every segment."""
    q, k, v, d, _ = make(cuda, q_lens, kv_lens, h, h, D, dtype, seed=5)
    if kind == "positions":
        # keys 20,000 apart, rows `far` behind the last: slope 1/8 or 1/16 leaves 1,250 or more between two keys
        k_pos = torch.cat([20000 * torch.arange(n, device=cuda) for n in kv_lens])
        q_pos = torch.cat([torch.full((n,), 20000 * (m - 1) + far, device=cuda) for n, m in zip(q_lens, kv_lens)])
        opts = dict(slopes=2.0 ** -(3.0 + torch.arange(h, device=cuda) % 2), q_pos=q_pos.int(), k_pos=k_pos.int())
    else:
        # q.k / sqrt(D) = D a b_j / sqrt(D), b_j = b (1 + j / n): `far` for the first key, far / n more for every further one
        b = torch.cat([1.0 + torch.arange(n, device=cuda) / n for n in kv_lens])
        a = math.sqrt(far / math.sqrt(D))
        q = torch.full_like(q, a)
        k = (a * b)[:, None, None].expand_as(k).to(dtype).contiguous()
        opts = {}
    last = torch.tensor(kv_lens, device=cuda).cumsum(0) - 1
    return q, k, v, d, opts, torch.repeat_interleave(last, torch.tensor(q_lens, device=cuda))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind,far", [("positions", 8000), ("positions", 700000), ("positions", 190000000), ("positions", 2100000000),
                                      ("scores", 1e8), ("scores", 1e11)])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_one_key_takes_everything(cuda, shape, kind, far, dtype):
    """Whatever its logit, p = 1 for one key: the output is its value, all others get no gradient, and no gradient is lost in
    an overflow of a probability.  (How far the gradients of huge scores are off is not bounded here: a score that the
    backward pass recomputes differs from the forward pass's by up to (D + 8) u sum |q||k| scale.)"""
    q_lens, kv_lens, h, D = SHAPES[shape]
    if kind == "scores" and dtype == torch.bfloat16:           # (as many steps of b as bfloat16 tells apart)
        q_lens, kv_lens = q_lens[:1], [min(kv_lens[0], 60)]
    far = min(far, 2 ** 31 - 1 - 20000 * max(kv_lens)) if kind == "positions" else far
    q, k, v, d, opts, win = _ahead(cuda, q_lens, kv_lens, h, D, dtype, far, kind)
    got = run(q, k, v, d, q_lens, kv_lens, **opts)
    want = v[win].double()
    _close(got["out"], want, want.abs())
    lost = torch.ones(k.shape[0], dtype=torch.bool, device=cuda)
    lost[win] = False
    assert not got["dv"][lost].any() and not got["dk"][lost].any()
    for name in got:
        assert torch.isfinite(got[name]).all(), name


def _half_step(dtype):
    """What a bfloat16 call rounds inside its products, relative."""
    return torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("far", [80, 8000, 80000, 700000, 8000000, 2100000000])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_gradients_where_one_key_takes_everything(cuda, shape, far, dtype):
    """p = 1 in the backward pass too, however far the key is: dv is the sum of the rows' gradients, and dq, dk what is left
    of do.v - do.o, zero but for rounding.  q and k are quarters up to 2, so that a score is exact in any order."""
    q_lens, kv_lens, h, D = SHAPES[shape]
    q, k, v, d, opts, win = _ahead(cuda, q_lens, kv_lens, h, D, dtype, min(far, 2 ** 31 - 1 - 20000 * max(kv_lens)), "positions")
    q, k = ((t.float() * 4).round().clamp(-8, 8).div(4).to(dtype) for t in (q, k))
    got = run(q, k, v, d, q_lens, kv_lens, **opts)
    want = v[win].double()
    dv, mag = torch.zeros_like(v, dtype=torch.float64), torch.zeros_like(v, dtype=torch.float64)
    dv.index_add_(0, win, d.double())
    mag.index_add_(0, win, d.double().abs())
    _close(got["dv"], dv, mag, n=max(q_lens))
    # do.v and do.o: D products and sums each; a bfloat16 o and its low part leave half^2 of it, twice with do.v's own part
    half = _half_step(dtype)
    size = (d.double().abs() * want.abs()).sum(-1, keepdim=True)
    bound = (2 * (D + 8) * U + 2 * half * half) * size / math.sqrt(D) * 1.01
    assert (got["dq"].double().abs() <= bound * k[win].double().abs() + 2.0 ** -120).all()
    kb = torch.zeros_like(dv)
    kb.index_add_(0, win, bound * q.double().abs())
    assert (got["dk"].double().abs() <= kb + 2.0 ** -120).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("far", [0, 8000, 700000, 100000000])
@pytest.mark.parametrize("q_lens,kv_lens,h,D", [([40], [90], 2, 32), ([3], [3000], 1, 64), ([700], [700], 16, 64), ([1300], [1300], 2, 64),
                                                ([2], [9000], 4, 128), ([20], [9000], 4, 128)])
def test_keys_of_equal_logits_far_away(cuda, q_lens, kv_lens, h, D, far, dtype):
    """Three keys at one position share everything, one near the first key and two near the last (so that ranges of keys
    hold one and two of them), the others 1e6 positions behind them: p = 1/3 each, in the output and in dv."""
    q, k, v, d, _ = make(cuda, q_lens, kv_lens, h, h, D, dtype, seed=8)
    k[:] = 0                                                  # all scores are zeros: the logits are the positions'
    n, m = q_lens[0], kv_lens[0]
    k_pos = torch.full((m,), -1000000, dtype=torch.int32, device=cuda)
    win = torch.tensor([1, m - 3, m - 2], device=cuda)
    k_pos[win] = 0
    slopes = torch.full((h,), 0.125, device=cuda)
    got = run(q, k, v, d, q_lens, kv_lens, slopes=slopes, k_pos=k_pos, q_pos=torch.full((n,), far, dtype=torch.int32, device=cuda))
    half = _half_step(dtype)                              # of a probability in a product
    want, mag = v[win].double().mean(0), v[win].double().abs().mean(0)
    _close(got["out"], want.expand(n, h, D), (1 + half / U / 8) * mag.expand(n, h, D))
    dv, dmag = d.double().sum(0) / 3, d.double().abs().sum(0) / 3
    _close(got["dv"][win], dv.expand(3, h, D), (1 + half / U / 8) * dmag.expand(3, h, D), n=n + 8)


@pytest.mark.parametrize("cap,scale", [(1e-3, 2e3), (1.0, 1e6), (1e-3, 1e30), (1e30, 1e30)])
@pytest.mark.parametrize("n", [40, 700])
def test_zero_rows_under_steep_caps(cuda, cap, scale, n):
    """A row of zeros scores zero everywhere and gets the mean of the values, whatever scale / cap is."""
    q, k, v, d, _ = make(cuda, [n], [n], 4, 4, 64, torch.bfloat16, seed=3)
    q[:] = 0
    got = run(q, k, v, d, [n], [n], cap=cap, scale=scale)
    # (a probability of the product is 2^0 before the division by the sum: no bfloat16 rounding)
    _close(got["out"], v.double().mean(0).expand(n, 4, 64), v.double().abs().mean(0).expand(n, 4, 64), n=n)
    assert not torch.isnan(got["dk"]).any() and not torch.isnan(got["dv"]).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("lens,blind,hq,hk,D", [([40, 70, 33], 1, 4, 2, 64), ([700, 600, 33], 1, 16, 8, 64), ([2, 1, 3], 0, 2, 2, 32), ([300], 0, 1, 1, 128)])
@pytest.mark.parametrize("opts", ["plain", "all"])
def test_rows_that_see_no_key_may_hold_anything(cuda, lens, blind, hq, hk, D, opts, dtype):
    """NaN and infinities in q and in the incoming gradient of rows whose keys are all masked: zeros, and nothing of it in
    any other result."""
    q, k, v, d, kw = make(cuda, lens, lens, hq, hk, D, dtype, seed=4, slopes=opts == "all", mask=0.7)
    if opts == "all":
        kw["cap"] = 9.0
    at = sum(lens[:blind])
    rows = slice(at, at + lens[blind])
    kw["key_mask"][rows] = False
    clean = run(q, k, v, d, lens, lens, **kw)
    check(clean, q, k, v, d, lens, lens, **kw)
    for poison in (float("nan"), float("inf"), -float("inf")):
        q2, d2 = q.clone(), d.clone()
        q2[rows], d2[rows] = poison, poison
        dirty = run(q2, k, v, d2, lens, lens, **kw)
        assert not dirty["out"][rows].any() and not dirty["dq"][rows].any()
        for name in clean:
            assert torch.equal(clean[name], dirty[name]), (name, poison)


@pytest.mark.parametrize("size", [1e-20, 1e-30, 1e-34])
def test_tiny_values(cuda, size):
    """Values far below one, under the two scaled planes: the outputs and gradients are theirs."""
    lens = [700, 30]
    q, k, v, d, _ = make(cuda, lens, lens, 16, 16, 64, torch.float32, seed=6)
    v = v * size
    check(run(q, k, v, d, lens, lens), q, k, v, d, lens, lens)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape,strides", [((1, 4, 16), (67, 16, 1)), ((1, 4, 16), (2 ** 22 + 72, 16, 1)), ((1, 1, 16), (3, 5, 1)),
                                           ((6, 1, 16), (64, 7, 1)), ((0, 4, 16), (67, 16, 1)), ((1, 2, 8), (2 ** 23, 8, 1))])
def test_single_rows_and_heads_of_any_stride(cuda, shape, strides, dtype):
    """One row cut from a store, one head cut from a row: a stride that is never taken may be any number."""
    from magic_amd.model.attention import head_norm_rope
    n, h, D = shape
    base = torch.randn(8, 4 * D, device=cuda).to(dtype)
    cut = lambda i: base.flatten()[i * 8:].as_strided(shape, strides) if n * h else base[:0].view(0, h, D)  # noqa: E731
    rows = [cut(i) for i in range(4)]
    plain = [t.clone(memory_format=torch.contiguous_format).reshape(-1).clone().view(shape) for t in rows]
    got, want = (run(*ts, [n], [n]) for ts in (rows, plain))
    assert all(torch.equal(got[k], want[k]) for k in want)
    w, pos = torch.rand(D, device=cuda) + 0.5, torch.arange(n, device=cuda, dtype=torch.int32)
    # (strides that are no whole 16 bytes take single columns there: another order of a row's sum of squares)
    for got, x in zip(head_norm_rope(rows[0], rows[1], w, w, pos), plain):
        want, tol = rope_reference(x, w, pos, D, 1e-6, 10000.0, torch.zeros_like(x))[0]
        assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("nq,nk,hq,hk,D", [(3, 5000, 16, 4, 128), (40, 900, 4, 2, 64), (500, 500, 8, 8, 16), (2000, 700, 4, 4, 32)])
def test_bfloat16_outputs_where_low_parts_of_probabilities_are_taken(cuda, nq, nk, hq, hk, D):
    """Blocks of few rows: what is left of a probability's rounding is the square of half a step, so that an output is
    off by its own rounding and the float32 chain: where the sum nearly cancels, by next to nothing.  (Terms as in
    test_gpu_attention.reference, whose bound holds a whole half step of the probabilities.)"""
    q, k, v, d, _ = make(cuda, [nq], [nk], hq, hk, D, torch.bfloat16, seed=D)
    got, r = run(q, k, v, d, [nq], [nk])["out"].double(), 2.0 ** -8
    for h in range(hq):
        Q, K, V = q[:, h].double(), k[:, h * hk // hq].double(), v[:, h * hk // hq].double()
        s, w = Q @ K.T / math.sqrt(D), Q.abs() @ K.abs().T / math.sqrt(D)
        delta = ((D + 8) * U * w).amax(1, keepdim=True) + 4 * U * s.abs().amax(1, keepdim=True)
        p = torch.softmax(s, 1)
        out, ep = p @ V, 2 * delta + (nk + 16) * U
        tol = (ep + r * r + (nk + 16) * U) * (p @ V.abs()) + r * out.abs()
        err = (got[:, h] - out).abs()
        assert (err <= tol).all(), (h, float((err / tol).max()))


@pytest.mark.parametrize("far", [1e6, 1e8])
@pytest.mark.parametrize("shape,dtype", [(s, torch.float32) for s in ("planes", "narrow_planes", "small", "whole_tiles", "whole_tiles_of_one", "wide")]
                         + [(s, torch.bfloat16) for s in SHAPES], ids=str)
def test_both_passes_take_large_scores_for_the_same_numbers(cuda, shape, dtype, far):
    """Where the two passes split their operands alike (bfloat16, and these float32 shapes), a score is the same bits in both,
    and p = 1 in the gradients of a key that is ahead by its scores too."""
    q_lens, kv_lens, h, D = SHAPES[shape]
    if dtype == torch.bfloat16:
        q_lens, kv_lens = q_lens[:1], [min(kv_lens[0], 60)]
    q, k, v, d, opts, win = _ahead(cuda, q_lens, kv_lens, h, D, dtype, far, "scores")
    got = run(q, k, v, d, q_lens, kv_lens, **opts)
    dv, mag = torch.zeros_like(v, dtype=torch.float64), torch.zeros_like(v, dtype=torch.float64)
    dv.index_add_(0, win, d.double())
    mag.index_add_(0, win, d.double().abs())
    _close(got["dv"], dv, mag, n=max(q_lens))
