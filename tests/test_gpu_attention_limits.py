"""Segment attention at the ends of its ranges.

The cases are built so that their exact answers are simple: one key (or a few with equal logits) is ahead of all others by
more than 100, so that the others' probabilities, below 2^-144, are zeros in float32.  u = 2^-24, half a step of float32."""
import math

import pytest
import torch

from tests.test_gpu_attention import U, check, make, run

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
          "few": ([1, 3], [700, 1100], 1, 32), "wide": ([300], [300], 8, 128), "ranges": ([1300], [1300], 2, 64)}


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
