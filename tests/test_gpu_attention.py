"""Segment attention, head norm + rotation: against plain 64-bit implementations, element by element.

The bounds are worst cases of the arithmetic the header promises, formed from the inputs.  u = 2^-24 (half a step of
float32), r = 2^-8 (half a step of bfloat16, relative), 0 for float32 operands.  With w = sum |q||k| scale, a score is
off by at most (D + 8) u w (products and sums in float32), a logit by delta = that + 4 u |l| + 4 u cap (tanh, bias,
subtraction); a probability exp(l - lse) by a factor 1 +- e_p, e_p = 2 delta + (nk + 16) u (both logits, the sum over the
keys), and the p of a product by r more where it is rounded to bfloat16.  The rest follows by the product rule."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0


def reference(q, k, v, q_lens, kv_lens, scale, cap, slopes, q_pos, k_pos, key_mask, d_out):
    """float64 outputs, gradients and the elementwise bounds of the float32 / bfloat16 kernels."""
    r = _half_step(q.dtype)
    dev = q.device
    q, k, v, d_out = (t.detach().double() for t in (q, k, v, d_out))
    hq, hk, D = q.shape[1], k.shape[1], q.shape[2]
    g = hq // hk
    res = {n: torch.zeros_like(t) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    tol = {n: torch.zeros_like(t) for n, t in res.items()}
    res["ds"], tol["ds"] = (torch.zeros(hq, dtype=torch.float64, device=dev) for _ in range(2))
    a = b = 0
    for nq, nk in zip(q_lens, kv_lens):
        rows = torch.arange(a, a + nq, device=dev)
        cols = torch.arange(b, b + nk, device=dev)
        a, b = a + nq, b + nk
        if key_mask is not None:
            cols = cols[key_mask[cols].bool()]
        if rows.numel() == 0 or cols.numel() == 0:
            continue
        n = cols.numel()
        for h in range(hq):
            j = h // g
            Q, K, V, G = q[rows, h], k[cols, j], v[cols, j], d_out[rows, h]
            s = scale * Q @ K.T
            w = abs(scale) * Q.abs() @ K.abs().T
            t = torch.tanh(s / cap) if cap else torch.zeros_like(s)
            c = cap * t if cap else s
            dist = torch.zeros_like(s)
            if slopes is not None:
                dist = (q_pos[rows].double()[:, None] - k_pos[cols].double()[None]).abs()
                l = c - slopes[h].double() * dist
            else:
                l = c
            delta = ((D + 8) * U * w).amax(1, keepdim=True) + 4 * U * l.abs().amax(1, keepdim=True) + 4 * U * cap
            if slopes is not None:
                delta = delta + 4 * U * (slopes[h].abs().double() * dist).amax(1, keepdim=True)
            p = torch.softmax(l, 1)
            ep = 2 * delta + (n + 16) * U
            O = p @ V
            res["out"][rows, h] = O
            tol["out"][rows, h] = (ep + r + (n + 16) * U) * (p @ V.abs()) + r * O.abs()
            # gradients
            res["dv"][cols, j] += p.T @ G
            tol["dv"][cols, j] += ((ep + r) * p).T @ G.abs() + (len(rows) + 16) * U * (p.T @ G.abs())
            dp, ad = G @ V.T, G.abs() @ V.abs().T
            dd, add = (G * O).sum(1, keepdim=True), (G.abs() * O.abs()).sum(1, keepdim=True)
            e_dp = (D + 8) * U * (ad + add) + (G.abs() * (tol["out"][rows, h] + r * O.abs())).sum(1, keepdim=True)
            dl = p * (dp - dd)
            e_dl = ep * dl.abs() + p * e_dp
            f = 1 - t * t if cap else torch.ones_like(t)
            ef = (2 * delta / cap + 8 * U) if cap else 0.0
            ds = scale * dl * f
            e_ds = abs(scale) * (e_dl * f + dl.abs() * ef) + r * ds.abs() + 8 * U * ds.abs()
            res["dq"][rows, h] = ds @ K
            tol["dq"][rows, h] = e_ds @ K.abs() + (n + 16) * U * (ds.abs() @ K.abs())
            res["dk"][cols, j] += ds.T @ Q
            tol["dk"][cols, j] += e_ds.T @ Q.abs() + (g * len(rows) + 16) * U * (ds.abs().T @ Q.abs())
            if slopes is not None:
                res["ds"][h] -= (dl * dist).sum()
                tol["ds"][h] += (e_dl * dist).sum() + (n + len(rows) + 64) * U * (dl.abs() * dist).sum()
    for name in ("dq", "dk", "dv"):
        tol[name] += r * res[name].abs()
    for name in tol:
        tol[name] += 2.0 ** -120
    return res, tol


def make(cuda, q_lens, kv_lens, hq, hk, D, dtype, seed=0, slopes=False, mask=None, std=1.0):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    nq, nk = sum(q_lens), sum(kv_lens)
    q, k, v = (rn(nq, hq, D) * std).to(dtype), (rn(nk, hk, D) * std).to(dtype), rn(nk, hk, D).to(dtype)
    d = (rn(nq, hq, D) * 0.1).to(dtype)
    kw = {}
    if slopes:
        kw = dict(slopes=2.0 ** -(3.0 + 4.0 * torch.rand(hq, generator=gen, device=cuda)),
                  q_pos=torch.randint(0, 500, (nq,), generator=gen, device=cuda, dtype=torch.int32),
                  k_pos=torch.randint(0, 500, (nk,), generator=gen, device=cuda, dtype=torch.int32))
    if mask is not None:
        kw["key_mask"] = torch.rand(nk, generator=gen, device=cuda) < mask
    return q, k, v, d, kw


def run(q, k, v, d, q_lens, kv_lens, cap=0.0, scale=None, **kw):
    from magic_amd.model.attention import attention_plan, segment_attention
    plan = attention_plan(q_lens, kv_lens, q.device)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    if kw.get("slopes") is not None:
        kw = dict(kw, slopes=kw["slopes"].detach().requires_grad_(True))
        leaves.append(kw["slopes"])
    out = segment_attention(*leaves[:3], plan, scale=scale, cap=cap, **kw)
    got = dict(zip(("dq", "dk", "dv", "ds"), torch.autograd.grad(out, leaves, d)))
    got["out"] = out.detach()
    return got


def check(got, q, k, v, d, q_lens, kv_lens, cap=0.0, scale=None, slopes=None, q_pos=None, k_pos=None, key_mask=None):
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    want, tol = reference(q, k, v, q_lens, kv_lens, scale, cap, slopes, q_pos, k_pos, key_mask, d)
    for name, g in got.items():
        err = (g.double() - want[name]).abs()
        bad = ~(err <= tol[name])
        assert not bad.any(), (name, int(bad.sum()), float(err.max()), float((err / tol[name]).nan_to_num(1e9).max()),
                               bad.nonzero()[0].tolist())


LENS = {
    "one": ([1], [1]),
    "tiny": ([3, 0, 1, 2], [1, 4, 0, 5]),
    "tile_edges": ([31, 32, 33, 64], [63, 64, 65, 33]),
    "ragged": ([1, 127, 129, 0, 257, 70], [1, 127, 129, 0, 257, 70]),
    "cross": ([5, 200, 130], [333, 1, 129]),
    "few_rows": ([1, 2, 1], [700, 1500, 3]),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hq,hk,D", [(4, 4, 16), (4, 4, 64), (4, 2, 24), (6, 2, 128), (1, 1, 8), (2, 1, 40)])
@pytest.mark.parametrize("lens", list(LENS))
def test_attention_forward_and_gradients(cuda, lens, hq, hk, D, dtype):
    q_lens, kv_lens = LENS[lens]
    q, k, v, d, kw = make(cuda, q_lens, kv_lens, hq, hk, D, dtype, seed=len(lens) + D)
    check(run(q, k, v, d, q_lens, kv_lens, **kw), q, k, v, d, q_lens, kv_lens, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("cap,slopes,mask", [(20.0, False, None), (0.0, True, None), (3.0, True, 0.4), (0.0, False, 0.1),
                                             (0.0, False, 0.0), (50.0, True, 0.9)])
@pytest.mark.parametrize("lens,D", [("ragged", 64), ("few_rows", 16), ("cross", 128)])
def test_attention_cap_bias_mask(cuda, lens, D, cap, slopes, mask, dtype):
    q_lens, kv_lens = LENS[lens]
    q, k, v, d, kw = make(cuda, q_lens, kv_lens, 4, 2, D, dtype, seed=3, slopes=slopes, mask=mask, std=2.0)
    check(run(q, k, v, d, q_lens, kv_lens, cap=cap, **kw), q, k, v, d, q_lens, kv_lens, cap=cap, **kw)


def test_attention_scale_signs_and_large_scores(cuda):
    q_lens, kv_lens = LENS["ragged"]
    q, k, v, d, kw = make(cuda, q_lens, kv_lens, 4, 4, 32, torch.float32, seed=5, std=4.0)
    for scale in (0.0, -0.3, 2.0):
        check(run(q, k, v, d, q_lens, kv_lens, scale=scale), q, k, v, d, q_lens, kv_lens, scale=scale)


@pytest.mark.parametrize("dtype,hq,hk,D", [(torch.float32, 4, 2, 64), (torch.float32, 16, 8, 64), (torch.float32, 16, 16, 16),
                                           (torch.bfloat16, 16, 4, 128)])
@pytest.mark.parametrize("keep", [0.5, 0.02, 1.0])
def test_masked_keys_of_long_segments(cuda, dtype, hq, hk, D, keep):
    """Long enough for the unmasked keys to be gathered; one segment without any, one whose mask starts off a word."""
    q_lens = kv_lens = [700, 5, 1301, 260, 33]
    q, k, v, d, kw = make(cuda, q_lens, kv_lens, hq, hk, D, dtype, seed=17, slopes=True, mask=keep)
    kw["key_mask"][2006:2266] = False
    kw["key_mask"][705:900] = False
    mask = kw["key_mask"]
    got = run(q, k, v, d, q_lens, kv_lens, **kw)
    check(got, q, k, v, d, q_lens, kv_lens, **kw)
    assert not got["out"][2006:2266].any() and not got["dq"][2006:2266].any()
    k2, v2 = k.clone(), v.clone()
    k2[~mask], v2[~mask] = float("nan"), float("inf")
    dirty = run(q, k2, v2, d, q_lens, kv_lens, **kw)
    byte = run(q, k, v, d, q_lens, kv_lens, **dict(kw, key_mask=mask.to(torch.uint8) * 200))
    for name in got:
        assert torch.equal(got[name], dirty[name]) and torch.equal(got[name], byte[name]), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_rows_without_a_visible_key_and_what_masked_keys_hold(cuda, dtype):
    """Masked keys may hold NaN, infinities and the type's lowest value; rows behind a segment's end may too (they
    belong to the next segment); a row that sees nothing gives zeros."""
    from magic_amd.model.attention import attention_plan, segment_attention
    q_lens = kv_lens = [40, 70, 5, 33]
    q, k, v, d, _ = make(cuda, q_lens, kv_lens, 4, 2, 64, dtype, seed=9)
    mask = torch.rand(148, device=cuda) < 0.6
    mask[110:115] = False                                     # the third segment sees nothing
    clean = run(q, k, v, d, q_lens, kv_lens, key_mask=mask)
    check(clean, q, k, v, d, q_lens, kv_lens, key_mask=mask)
    assert not clean["out"][110:115].any() and not clean["dq"][110:115].any()
    assert not clean["dk"][~mask].any() and not clean["dv"][~mask].any()
    for poison in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
        k2, v2 = k.clone(), v.clone()
        k2[~mask], v2[~mask] = poison, poison
        dirty = run(q, k2, v2, d, q_lens, kv_lens, key_mask=mask)
        for name in clean:
            assert torch.equal(clean[name], dirty[name]), (name, poison)
    # a NaN row stays inside its own segment and head group
    k3 = k.clone()
    k3[45, 0] = float("nan")
    out = segment_attention(q, k3, v, attention_plan(q_lens, None, cuda))
    ref = segment_attention(q, k, v, attention_plan(q_lens, None, cuda))
    hit = torch.zeros(148, 4, dtype=torch.bool, device=cuda)
    hit[40:110, :2] = True
    assert torch.equal(out[~hit], ref[~hit]) and torch.isnan(out[hit]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_attention_strides(cuda, dtype):
    """Views of one projection output, head-major storage, rows off 16-byte addresses, expanded gradients."""
    lens = [50, 91]
    n, h, D = 141, 4, 32
    qkv = torch.randn(n, 3 * h * D, device=cuda).to(dtype)
    q, k, v = (qkv[:, i * h * D:(i + 1) * h * D].view(n, h, D) for i in range(3))
    d = torch.randn(n, h, D, device=cuda).to(dtype)
    want = run(q.contiguous(), k.contiguous(), v.contiguous(), d, lens, lens)
    forms = {"view": (q, k, v),
             "head_major": tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)),
             "unaligned": tuple(torch.empty(n * h * D + 1, device=cuda, dtype=dtype)[1:].view(n, h, D).copy_(t)
                                for t in (q, k, v)),
             "inner_stride": tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))}
    for name, (a, b, c) in forms.items():
        got = run(a, b, c, d.transpose(0, 1).contiguous().transpose(0, 1), lens, lens)
        for key in want:
            assert torch.equal(got[key], want[key]), (name, key)
    one = run(q, k, v, torch.ones((), device=cuda, dtype=dtype).expand(n, h, D), lens, lens)
    check(one, q, k, v, torch.ones(n, h, D, device=cuda, dtype=dtype), lens, lens)


@pytest.mark.parametrize("D,hq,hk", [(64, 16, 16), (40, 12, 6), (128, 16, 8)])
@pytest.mark.parametrize("opts", ["plain", "all"])
def test_attention_large_float32(cuda, D, hq, hk, opts):
    """Enough rows and heads for the launches that split float32 into two fp16 pieces, forward and backward, with
    segments next to each other that they do not serve: one whose rows differ by 2^20 in size, one with zero rows only in
    v, one of zeros, one with an infinity.  The bounds are the ones of the other kernels."""
    q_lens = kv_lens = [1030, 520, 129, 33, 600, 70]
    q, k, v, d, kw = make(cuda, q_lens, kv_lens, hq, hk, D, torch.float32, seed=D + hq, slopes=opts == "all",
                          mask=0.7 if opts == "all" else None)
    cap = 9.0 if opts == "all" else 0.0
    k[1030:1550:7] *= 2.0 ** -10
    v[1030:1550:5] *= 2.0 ** -20
    d[1030:1550:3] *= 2.0 ** 12
    v[1550:1679] = 0.0
    q[1679:1712] = 0.0
    d[1712:2312:2] = 0.0                                       # rows without a gradient
    check(run(q, k, v, d, q_lens, kv_lens, cap=cap, **kw), q, k, v, d, q_lens, kv_lens, cap=cap, **kw)
    v2 = v.clone()
    v2[2320, 0, 3] = float("inf")                              # the last segment
    if opts == "plain":
        a, b = run(q, k, v, d, q_lens, kv_lens), run(q, k, v2, d, q_lens, kv_lens)
        assert torch.equal(a["out"][:2312], b["out"][:2312]) and torch.equal(a["dk"][:2312], b["dk"][:2312])
        assert not torch.isfinite(b["out"][2312:, :hq // hk, 3]).any()
        assert torch.isfinite(b["out"][2312:, hq // hk:]).all()


@pytest.mark.parametrize("dtype,D,hq,hk", [(torch.float32, 64, 4, 2), (torch.float32, 128, 2, 1), (torch.float32, 40, 4, 4),
                                           (torch.bfloat16, 128, 4, 4), (torch.bfloat16, 64, 16, 4)])
@pytest.mark.parametrize("opts", ["plain", "all", "wide_range"])
def test_few_long_segments(cuda, dtype, D, hq, hk, opts):
    """Tiles of 128 rows whose keys are cut into ranges, beside a short and an empty segment; rows of very different
    sizes in one segment (the scaled planes leave it to the other launch) and a segment whose keys are all masked."""
    q_lens, kv_lens = [1700, 3, 0, 90], [1810, 600, 5, 90]
    q, k, v, d, kw = make(cuda, q_lens, kv_lens, hq, hk, D, dtype, seed=D + hq, slopes=opts == "all", mask=None if opts == "plain" else 0.6)
    if opts == "all":
        kw["cap"] = 30.0
    if opts == "wide_range":
        k[:900] *= 2.0 ** -20
        kw["key_mask"][1810:2410] = False
    check(run(q, k, v, d, q_lens, kv_lens, **kw), q, k, v, d, q_lens, kv_lens, **kw)


@pytest.mark.parametrize("D,hq,hk,n", [(16, 4, 2, 2100), (24, 2, 2, 4200), (32, 3, 1, 4300)])
@pytest.mark.parametrize("opts", ["plain", "all"])
def test_long_segments_of_narrow_heads(cuda, D, hq, hk, n, opts):
    """From 2,048 keys on narrow heads take their products from two scaled planes too."""
    lens = [n, 40, 0, 1]
    q, k, v, d, kw = make(cuda, lens, lens, hq, hk, D, torch.float32, seed=D, slopes=opts == "all", mask=0.7 if opts == "all" else None)
    if opts == "all":
        kw["cap"] = 25.0
    check(run(q, k, v, d, lens, lens, **kw), q, k, v, d, lens, lens, **kw)


def test_attention_long_tail_of_small_probabilities(cuda):
    """A distance bias leaves thousands of keys whose terms are each below half a unit of the running sums: together they
    count.  Relative 2-norm error of a float32 result, as small as one formed with whole-row sums."""
    from magic_amd.model.attention import attention_plan, segment_attention
    n, h, D = 6000, 8, 64
    gen = torch.Generator(device=cuda).manual_seed(1)
    q, k, v = (torch.randn(n, h, D, generator=gen, device=cuda) for _ in range(3))
    v += 1.0
    pos = torch.arange(n, device=cuda, dtype=torch.int32)
    slopes = torch.full((h,), 0.003, device=cuda)
    out = segment_attention(q, k, v, attention_plan([n], device=cuda), slopes=slopes, q_pos=pos, k_pos=pos)
    dist = (pos.double()[:, None] - pos.double()[None]).abs()
    for j in (0, 5):
        p = torch.softmax(q[:, j].double() @ k[:, j].double().T / 8 - slopes[j].double() * dist, 1)
        want = p @ v[:, j].double()
        # logits off by (D + 8) u |q||k| / 8 at most, 1/50 of it as a 2-norm of random signs; sums of 6,000 terms
        assert float((out[:, j].double() - want).norm() / want.norm()) < 1e-6


def test_attention_gradient_against_differences(cuda):
    """Central differences of the 64-bit definition along random directions against the kernel's gradients."""
    lens = [37, 66]
    q, k, v, d, kw = make(cuda, lens, lens, 4, 2, 16, torch.float32, seed=21, slopes=True, mask=0.8)
    got = run(q, k, v, d, lens, lens, cap=5.0, **kw)

    def value(q, k, v, slopes):
        kw2 = dict(kw, slopes=slopes)
        want, _ = reference(q, k, v, lens, lens, 0.25, 5.0, d_out=d, **kw2)
        return float((want["out"] * d.double()).sum())

    gen = torch.Generator(device=cuda).manual_seed(4)
    base = [q.double(), k.double(), v.double(), kw["slopes"].double()]
    for i, name in enumerate(("dq", "dk", "dv", "ds")):
        e = torch.randn(base[i].shape, generator=gen, device=cuda, dtype=torch.float64) * (0.01 if name == "ds" else 1.0)
        step = 1e-5
        hi, lo = ([t + s * step * e if j == i else t for j, t in enumerate(base)] for s in (1.0, -1.0))
        diff = (value(*hi) - value(*lo)) / (2 * step)
        mine = float((got[name].double() * e).sum())
        # second-order term of the difference (step^2) and the rounding of the float32 gradient
        size = float((got[name].double() * e).abs().sum())
        assert abs(diff - mine) <= 1e-4 * size + 1e-9, (name, diff, mine)


def test_attention_is_reproducible_and_partial_gradients(cuda):
    from magic_amd.model.attention import attention_plan, segment_attention
    lens = [700, 33, 1200]
    q, k, v, d, kw = make(cuda, lens, lens, 4, 4, 64, torch.float32, seed=2, slopes=True)
    a, b = (run(q, k, v, d, lens, lens, **kw) for _ in range(2))
    for name in a:
        assert torch.equal(a[name], b[name]), name
    plan = attention_plan(lens, device=cuda)
    for want in (("dq",), ("dk",), ("dv",), ("ds",)):
        ts = {"dq": q.clone(), "dk": k.clone(), "dv": v.clone(), "ds": kw["slopes"].clone()}
        for n in want:
            ts[n].requires_grad_(True)
        out = segment_attention(ts["dq"], ts["dk"], ts["dv"], plan, **dict(kw, slopes=ts["ds"]))
        g, = torch.autograd.grad(out, [ts[want[0]]], d)
        assert torch.equal(g, a[want[0]]), want


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.float32, 16), (torch.bfloat16, 128)])
def test_partial_gradients_of_a_long_segment(cuda, dtype, D):
    """Each gradient asked for alone, with its ranges of keys and their joins, within the bounds of the full call.  (Not
    its bits: where dq is not wanted, another kernel forms do . o of a row, D float32 terms in another order.)"""
    from magic_amd.model.attention import attention_plan, segment_attention
    lens = [4300, 30]
    q, k, v, d, kw = make(cuda, lens, lens, 2, 1, D, dtype, seed=D, slopes=True, mask=0.8)
    plan = attention_plan(lens, device=cuda)
    got = {}
    for i, name in enumerate(("dq", "dk", "dv", "ds")):
        ts = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v, kw["slopes"]))]
        out = segment_attention(*ts[:3], plan, cap=20.0, **dict(kw, slopes=ts[3]))
        got[name] = torch.autograd.grad(out, ts[i], d)[0]
    check(got, q, k, v, d, lens, lens, cap=20.0, **kw)


def test_attention_streams_and_captured_graph(cuda):
    """Two calls in flight on two streams, and forward + backward replayed from a captured graph on new inputs."""
    from magic_amd import _lib
    from magic_amd.model.attention import attention_plan
    lens = [300, 41]
    q, k, v, d, kw = make(cuda, lens, lens, 4, 4, 64, torch.float32, seed=12)
    plan = attention_plan(lens, device=cuda)

    def step(q, k, v, d):
        out, lse = _lib.attn_fwd(q, k, v, plan, 0.125)
        return (out,) + _lib.attn_bwd(q, k, v, plan, 0.125, out, lse, d)[:3]

    want = step(q, k, v, d)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(3):
                outs.append(step(q, k, v, d))
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for got in outs:
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    ins = [t.clone() for t in (q, k, v, d)]
    graphs = []
    for _ in range(2):                                       # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(*ins)
        graphs.append((g, res))
    for rep in range(3):
        new = make(cuda, lens, lens, 4, 4, 64, torch.float32, seed=100 + rep)[:4]
        for a, b in zip(ins, new):
            a.copy_(b)
        eager = step(*new)
        for g, res in graphs:
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(res, eager):
                assert torch.equal(x, y)


def test_registered_attention_operators(cuda):
    from magic_amd.model.attention import attention_plan
    lens = [45, 80]
    q, k, v, d, kw = make(cuda, lens, lens, 4, 2, 32, torch.float32, seed=31, slopes=True, mask=0.7)
    plan = attention_plan(lens, device=cuda)
    args = (q, k, v, plan.q_tiles, plan.k_tiles, plan.max_q, plan.max_k, plan.n_seg, 32 ** -0.5, 4.0, kw["slopes"], kw["q_pos"], kw["k_pos"], kw["key_mask"])
    out, lse = torch.ops.magic.attn_fwd(*args)
    grads = torch.ops.magic.attn_bwd(*args, out, lse, d)
    want = run(q, k, v, d, lens, lens, cap=4.0, **kw)
    for x, name in zip((out,) + tuple(grads), ("out", "dq", "dk", "dv", "ds")):
        assert torch.equal(x, want[name]), name


def test_attention_refusals(cuda):
    """What the operators do not serve raises before anything is launched."""
    from magic_amd._lib import MagicHipError
    from magic_amd.model.attention import attention_plan, head_norm_rope, segment_attention
    q, k, v, d, kw = make(cuda, [9], [9], 4, 2, 16, torch.float32, slopes=True)
    plan = attention_plan([9], device=cuda)
    ok = dict(slopes=kw["slopes"], q_pos=kw["q_pos"], k_pos=kw["k_pos"])
    segment_attention(q, k, v, plan, **ok)
    bad = [((q.half(), k.half(), v.half()), {}), ((q, k.bfloat16(), v), {}), ((q[:, :3], k, v), {}), ((q[..., :12], k[..., :12], v[..., :12]), {}),
           ((q, k[:8], v[:8]), {}), ((q[:8], k, v), {}), ((q, k, v[:, :1]), {}), ((q[0], k, v), {}),
           ((q, k, v), dict(cap=-1.0)), ((q, k, v), dict(cap=1e-9)), ((q, k, v), dict(cap=float("nan"))),
           ((q, k, v), dict(scale=float("inf"))), ((q, k, v), dict(slopes=ok["slopes"])),
           ((q, k, v), dict(ok, slopes=ok["slopes"][:2])), ((q, k, v), dict(ok, q_pos=ok["q_pos"].long())),
           ((q, k, v), dict(ok, k_pos=ok["k_pos"].cpu())), ((q, k, v), dict(key_mask=torch.ones(8, dtype=torch.bool, device=cuda))),
           ((q, k, v), dict(key_mask=torch.ones(9, device=cuda)))]
    for args, opt in bad:
        with pytest.raises(MagicHipError):
            segment_attention(*args, plan, **opt)
    with pytest.raises(MagicHipError):
        segment_attention(q, k, v, attention_plan([9], device="cpu"))
    wide = torch.zeros(3, 1, 136, device=cuda)
    with pytest.raises(MagicHipError):
        segment_attention(wide, wide, wide, attention_plan([3], device=cuda))
    w, pos = torch.ones(16, device=cuda), torch.arange(9, device=cuda, dtype=torch.int32)
    for args, opt in [((q, k, w, w, pos), dict(rotary_dim=15)), ((q, k, w, w, pos), dict(rotary_dim=18)), ((q, k, w[:8], w, pos), {}),
                      ((q, k, w, w, pos.long()), {}), ((q, k[:8], w, w, pos), {}), ((q, k, w.bfloat16(), w, pos), {}),
                      ((q, k, w, w, pos), dict(eps=-1.0)), ((q, k, w, w, pos), dict(base=0.0)), ((q.half(), k.half(), w, w, pos), {})]:
        with pytest.raises(MagicHipError):
            head_norm_rope(*args, **opt)


def test_plan_is_not_built_during_a_capture(cuda):
    from magic_amd._lib import MagicHipError
    from magic_amd.model.attention import attention_plan
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(8, device=cuda)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = x + 1
        with pytest.raises(MagicHipError):
            attention_plan([4], device=cuda)
    graph.replay()
    torch.cuda.synchronize()
    assert (y == 1).all()


@pytest.mark.parametrize("cap", [1e-3, 1e6, 1e30])
def test_caps_far_from_the_scores(cuda, cap):
    """One far below the scores makes them its sign.  One far above leaves them as they are (tanh takes less than 1e-10
    of a score off, a two-hundredth of a half step): the reference has none then."""
    q, k, v, d, _ = make(cuda, [40], [40], 2, 2, 16, torch.float32)
    got = run(q, k, v, d, [40], [40], cap=cap)
    check(got, q, k, v, d, [40], [40], cap=cap if cap < 1 else 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("cap", [1e9, 4e9, 1e20])
def test_capped_scores_of_many_millions(cuda, cap, dtype):
    """Scores of 4e8 and 2e8, capped at some times as much: one key takes the whole probability (2^-1e8 of it is left for
    the other, which gets exact zeros).  The output is its value: p v / p, with a rounding for p v, one for the quotient
    and one for the result's type.  (Nothing is promised of the winning key's gradients: a logit of 4e8 is off by 4 u 4e8 =
    95, and e^95 = 2^137 is no float32 number.)"""
    from magic_amd.model.attention import attention_plan, segment_attention
    q = torch.full((3, 1, 16), 1e4, device=cuda).to(dtype).requires_grad_(True)
    k = torch.tensor([0.5e4, 1e4], device=cuda).view(2, 1, 1).expand(2, 1, 16).to(dtype).contiguous().requires_grad_(True)
    v = torch.randn(2, 1, 16, device=cuda).to(dtype).requires_grad_(True)
    out = segment_attention(q, k, v, attention_plan([3], [2], cuda), cap=cap)
    want = v.detach()[1:].expand(3, 1, 16).double()
    assert ((out.double() - want).abs() <= (2.01 * U + torch.finfo(dtype).eps / 2) * want.abs()).all()
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert not dk[0].any() and not dv[0].any()


def test_registered_operators_check_their_tables(cuda):
    from magic_amd._lib import MagicHipError
    from magic_amd.model.attention import attention_plan
    q, k, v, _, _ = make(cuda, [9], [9], 2, 2, 16, torch.float32)
    p = attention_plan([9], device=cuda)
    call = lambda qt, kt, mq, mk, ns: torch.ops.magic.attn_fwd(q, k, v, qt, kt, mq, mk, ns, 0.25, 0.0, None, None, None, None)  # noqa: E731
    call(p.q_tiles, p.k_tiles, 9, 9, 1)
    for bad in ((p.q_tiles.long(), p.k_tiles, 9, 9, 1), (p.q_tiles, p.k_tiles[:, :7], 9, 9, 1), (p.q_tiles.cpu(), p.k_tiles, 9, 9, 1),
                (p.q_tiles[:0], p.k_tiles, 9, 9, 1), (p.q_tiles, p.k_tiles, 10, 9, 1), (p.q_tiles, p.k_tiles, 9, 9, -1)):
        with pytest.raises(MagicHipError):
            call(*bad)


def test_attention_one_tensor_thrice_broadcast_operands_and_gradients(cuda):
    """q, k and v the same leaf; slopes, positions and masks as views; the expanded gradient of a sum; no segment."""
    from magic_amd.model.attention import attention_plan, segment_attention
    lens = [5, 40, 1]
    x = torch.randn(46, 2, 16, device=cuda)
    plan = attention_plan(lens, device=cuda)
    slopes, pos = torch.full((1,), 0.25, device=cuda), torch.arange(92, device=cuda, dtype=torch.int32)
    mask = torch.rand(46, 2, device=cuda) < 0.7
    views = dict(slopes=slopes.expand(2), q_pos=pos[::2], k_pos=pos[::2], key_mask=mask[:, 0])
    plain = {n: t.contiguous() for n, t in views.items()}
    leaf = x.clone().requires_grad_(True)
    segment_attention(leaf, leaf, leaf, plan, **views).sum().backward()
    parts = [x.clone().requires_grad_(True) for _ in range(3)]
    out = segment_attention(*parts, plan, **plain)
    want = torch.autograd.grad(out, parts, torch.ones_like(out))
    assert torch.allclose(leaf.grad, want[0] + want[1] + want[2], rtol=1e-6, atol=1e-6)       # (sums of three, any order)
    none = segment_attention(x[:0], x[:0], x[:0], attention_plan([], device=cuda))
    assert none.shape == (0, 2, 16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_calls_on_two_streams_at_once(cuda, dtype):
    """Calls of two streams share no workspace: each gives the result it gives alone."""
    sets = [([900, 700], 64), ([1, 640, 3], 64)]
    jobs = [make(cuda, lens, lens, 4, 2, D, dtype, seed=i, slopes=True, mask=0.5) + (lens,) for i, (lens, D) in enumerate(sets)]
    alone = [run(q, k, v, d, lens, lens, cap=20.0, **kw) for q, k, v, d, kw, lens in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(4):
        got = []
        for s, (q, k, v, d, kw, lens) in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(run(q, k, v, d, lens, lens, cap=20.0, **kw))
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert all(torch.equal(a[n], b[n]) for n in b)


def test_attention_serves_without_rows_or_keys(cuda):
    from magic_amd.model.attention import attention_plan, segment_attention
    q, k, v, d, _ = make(cuda, [5], [7], 4, 2, 16, torch.float32)
    out = segment_attention(q[:0], k, v, attention_plan([0], [7], cuda))
    assert out.shape == (0, 4, 16)
    got = run(q[:0], k, v, d[:0], [0], [7])
    assert not got["dk"].any() and not got["dv"].any() and got["dk"].shape == k.shape
    got = run(q, k[:0], v[:0], d, [5], [0])
    assert not got["out"].any() and not got["dq"].any()


# ------------------------------------------------------------------------------------------- head norm + rotation
def rope_reference(x, w, pos, rot, eps, base, dy):
    r = _half_step(x.dtype)
    x, w, dy = x.detach().double(), w.detach().double(), dy.double()
    d, half = x.shape[-1], rot // 2
    inv = base ** (-torch.arange(half, dtype=torch.float64, device=x.device) * 2 / max(rot, 1))
    ang = (pos.double()[:, None] * inv)[:, None]
    c, s = torch.cos(ang), torch.sin(ang)

    def turn(y, s):
        return torch.cat([y[..., :half] * c - y[..., half:rot] * s, y[..., half:rot] * c + y[..., :half] * s,
                          y[..., rot:]], -1)

    q = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    u = x * q * w
    mag = torch.cat([u[..., :half].abs() + u[..., half:rot].abs()] * 2 + [u[..., rot:].abs()], -1)
    y = turn(u, s)
    # rsqrt of a float32 sum of D squares: (D / 2 + 4) u; sine and cosine of an angle reduced in double: 8 u absolute
    ty = (d / 2 + 24) * U * mag + r * y.abs()
    gu = turn(dy, -s)
    gmag = torch.cat([dy[..., :half].abs() + dy[..., half:rot].abs()] * 2 + [dy[..., rot:].abs()], -1)
    dw = (gu * x * q).sum((0, 1))
    n = x.shape[0] * x.shape[1]
    tw = ((d / 2 + 32) * U + min(n, 4096) * U) * (gmag * x.abs() * q).sum((0, 1))
    g = gu * w
    dx = q * (g - x * q * q * (g * x).mean(-1, keepdim=True))
    am = q * (gmag * w.abs() + x.abs() * q * q * (gmag * w.abs() * x.abs()).mean(-1, keepdim=True))
    tx = (2.5 * d + 48) * U * am + r * dx.abs()
    return (y, ty + 1e-30), (dx, tx + 1e-30), (dw, tw + 1e-30)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,hq,hk,D,rot", [(1, 4, 4, 64, 64), (77, 4, 2, 16, 16), (1000, 8, 2, 128, 64), (33, 3, 1, 24, 12),
                                           (50, 2, 2, 63, 62), (129, 1, 1, 128, 2), (64, 4, 4, 64, 0), (9, 2, 1, 1, 0),
                                           (5000, 4, 4, 64, 64)])
def test_head_norm_rope(cuda, n, hq, hk, D, rot, dtype):
    from magic_amd.model.attention import head_norm_rope
    gen = torch.Generator(device=cuda).manual_seed(n + D)
    rn = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    qkv = rn(n, (hq + 2 * hk) * D).to(dtype)
    q, k = qkv[:, :hq * D].view(n, hq, D), qkv[:, hq * D:(hq + hk) * D].view(n, hk, D)
    wq, wk = 1 + 0.2 * rn(D), 1 + 0.2 * rn(D)
    pos = torch.randint(-5, 700000, (n,), generator=gen, device=cuda, dtype=torch.int32)
    dq, dk = rn(n, hq, D).to(dtype), rn(n, hk, D).to(dtype)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    yq, yk = head_norm_rope(*leaves, pos, rotary_dim=rot)
    gq, gk, gwq, gwk = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    for x, w, dy, y, g, gw in ((q, wq, dq, yq, gq, gwq), (k, wk, dk, yk, gk, gwk)):
        for got, (want, tol) in zip((y, g, gw), rope_reference(x, w, pos, rot, 1e-6, 10000.0, dy)):
            err = (got.double() - want).abs()
            assert (err <= tol).all(), (float(err.max()), float((err / tol).max()))
    again = torch.autograd.grad(head_norm_rope(*leaves, pos, rotary_dim=rot), leaves, (dq, dk))
    for a, b in zip(again, (gq, gk, gwq, gwk)):
        assert torch.equal(a, b)


def test_head_norm_rope_strides_and_operators(cuda):
    from magic_amd.model.attention import head_norm_rope
    n, h, D = 91, 4, 32
    x = torch.randn(n, h, D, device=cuda)
    w = torch.rand(D, device=cuda) + 0.5
    pos = torch.arange(n, device=cuda, dtype=torch.int32)
    want = head_norm_rope(x, x, w, w, pos)
    odd = torch.empty(n * h * D + 1, device=cuda)[1:].view(n, h, D).copy_(x)
    for form in (x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(1, 2).contiguous().transpose(1, 2), odd):
        for a, b in zip(head_norm_rope(form, x, w, w, pos), want):
            assert (a - b).abs().max() <= 2e-6 * b.abs().max()           # (another order of the same sum)
    assert torch.equal(torch.ops.magic.head_norm_rope_fwd(x, x, w, w, pos, D, 1e-6, 10000.0)[0], want[0])
    empty = head_norm_rope(x[:0], x[:0], w, w, pos[:0])
    assert empty[0].shape == (0, h, D)
    lw = w.clone().requires_grad_(True)
    y = head_norm_rope(x[:0], x[:0], lw, w, pos[:0])[0]
    assert not torch.autograd.grad(y.sum(), lw)[0].any()


@pytest.mark.parametrize("q_lens,kv_lens,D,hq,hk", [([2, 531], [2, 4], 128, 4, 2), ([700], [3], 16, 4, 4), ([300, 40], [7, 2000], 64, 4, 1),
                                                    ([3, 2], [900, 5], 64, 1, 1)])
def test_bfloat16_gradients_over_few_keys(cuda, q_lens, kv_lens, D, hq, hk):
    """do . o takes the output before its rounding: with few keys what that rounding takes reaches every score gradient of
    a row with one sign.  In the 2-norm the gradients are off by their own rounding and that of the score gradients or
    probabilities in the products, each at most r = 2^-8 relative of a term, r / sqrt(3) as root mean square of a rounding
    uniform in (-r, r): sqrt(2) r / sqrt(3) together where the terms are independent, at most 2 r / sqrt(3) allowed here.
    (Without the low part dq and dk are off by 3.7e-3 and 2.4 times the plain form.)"""
    q, k, v, d, kw = make(cuda, q_lens, kv_lens, hq, hk, D, torch.bfloat16, seed=D, slopes=True)
    got = run(q, k, v, d, q_lens, kv_lens, **kw)
    want, _ = reference(q, k, v, q_lens, kv_lens, D ** -0.5, 0.0, kw["slopes"], kw["q_pos"], kw["k_pos"], None, d)
    check(got, q, k, v, d, q_lens, kv_lens, **kw)
    for name in ("dq", "dk", "dv"):
        err = float((got[name].double() - want[name]).norm() / want[name].norm())
        assert err <= 2 * 2.0 ** -8 / math.sqrt(3), (name, err)
