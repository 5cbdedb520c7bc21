"""Host side of the global-attention block: plans, argument checks (no GPU)."""
import numpy as np
import pytest
import torch


def test_plan_tiles_cover_every_row_once():
    from magic_amd import _lib
    from magic_amd.model.attention import attention_plan
    rng = np.random.default_rng(0)
    for _ in range(20):
        s = int(rng.integers(1, 12))
        ql, kl = (rng.integers(0, 400, s) * (rng.random(s) < 0.8)).tolist(), rng.integers(0, 400, s).tolist()
        plan = attention_plan(ql, kl, device="cpu")
        for tiles, rows, others in ((plan.q_tiles, ql, kl), (plan.k_tiles, kl, ql)):
            seen = np.zeros(sum(rows), int)
            r0, o0 = np.cumsum([0] + rows), np.cumsum([0] + others)
            for a, n, b, m, g, s0, sn, _ in tiles.tolist():
                assert 1 <= n <= _lib.ATTN_TILE
                seg = int(np.searchsorted(r0, a, side="right")) - 1
                while rows[seg] == 0:
                    seg += 1
                assert r0[seg] <= a and a + n <= r0[seg] + rows[seg]
                assert (b, m, g, s0, sn) == (o0[seg], others[seg], seg, r0[seg], rows[seg])
                assert (a - s0) % _lib.ATTN_TILE == 0
                seen[a:a + n] += 1
            assert (seen == 1).all()
    assert attention_plan([], device="cpu").q_tiles.shape == (0, 8)


def test_plan_refusals():
    from magic_amd._lib import MagicHipError
    from magic_amd.model.attention import attention_plan
    for args in (([1, 2], [1]), ([-1], [1]), ([1 << 31], [1])):
        with pytest.raises(MagicHipError):
            attention_plan(*args, device="cpu")


def test_operators_refuse_cpu_tensors():
    from magic_amd._lib import MagicHipError
    from magic_amd.model.act8 import act8_pack
    from magic_amd.model.attention import attention_plan, head_norm_rope, segment_attention
    from magic_amd.model.gat import linear_nobias
    x = torch.randn(4, 2, 16)
    with pytest.raises(MagicHipError, match="GPU"):
        segment_attention(x, x, x, attention_plan([4], device="cpu"))
    with pytest.raises(MagicHipError, match="GPU"):
        head_norm_rope(x, x, torch.ones(16), torch.ones(16), torch.arange(4, dtype=torch.int32))
    with pytest.raises(MagicHipError):
        act8_pack(torch.randn(4, 16))
    with pytest.raises(MagicHipError, match="act_bits"):
        linear_nobias(torch.randn(4, 16), torch.randn(8, 16), act_bits=4)


@pytest.mark.parametrize("n_rows", [0, 5])
def test_c_entry_points_check_their_arguments(n_rows):
    """Status codes of calls that must return before anything is launched."""
    import ctypes as C

    from magic_amd import _lib
    lib = _lib.load()
    a = _lib.MagicAttn()
    assert lib.magic_attn_fwd(None, None, 0, 0, None, None, 0, None) == -1
    a.dtype, a.q_heads, a.kv_heads, a.head_dim = 7, 4, 2, 64
    assert lib.magic_attn_fwd(C.byref(a), None, 0, 0, None, None, 0, None) == -2          # type
    a.dtype, a.kv_heads = 0, 3
    assert lib.magic_attn_fwd(C.byref(a), None, 0, 0, None, None, 0, None) == -1          # 4 heads over 3
    for d in (12, 136):
        a.kv_heads, a.head_dim = 2, d
        assert lib.magic_attn_fwd(C.byref(a), None, 0, 0, None, None, 0, None) == -2
    a.head_dim, a.n_q = 64, n_rows
    assert lib.magic_attn_fwd(C.byref(a), None, 0, 0, None, None, 0, None) == (0 if n_rows == 0 else -1)
    args = [n_rows, 4, 2, 64, 64, 0, None, 0, 0, None, 0, 0, None, None, None, 1e-6, 1e4, None, None, None]
    assert lib.magic_head_norm_rope_fwd(*args) == (0 if n_rows == 0 else -1)
    for i, bad, want in ((1, 0, -1), (3, 129, -2), (4, 65, -1), (4, 63, -1), (5, 2, -2), (15, -1.0, -1)):
        wrong = list(args)
        wrong[i] = bad
        assert lib.magic_head_norm_rope_fwd(*wrong) == want, (i, bad)
    assert lib.magic_act8_code_stride(5) == 16 and lib.magic_act8_code_stride(0) == 0
    assert lib.magic_act8_pack(n_rows, 8, None, 8, None, None, None) == (0 if n_rows == 0 else -1)
    assert lib.magic_act8_pack(n_rows, 0, None, 8, None, None, None) == -1
    assert lib.magic_act8_weight_grad(5, 4, 8, None, 4, None, None, None, None, 0, None) == -1


def test_cap_polynomial_is_as_close_to_tanh_as_its_comment_says():
    """tanh(t) / t from the kernels' float32 coefficients, exactly evaluated: 4.2e-8 off at most on its range, 1 at zero."""
    import re
    from pathlib import Path
    text = (Path(__file__).parent.parent / "magic_amd" / "csrc" / "attn_common.h").read_text()
    k = [float(np.float32(re.search(rf"\bK{i} = ([-0-9.e]+)f", text).group(1))) for i in range(4)]
    top = float(np.float32(re.search(r"TANH_SMALL = ([0-9.]+)f", text).group(1)))
    t = np.linspace(0, top, 20001)[1:]
    z = t * t
    poly = k[0] + z * (k[1] + z * (k[2] + z * k[3]))
    assert np.abs(poly * t / np.tanh(t) - 1).max() <= 4.2e-8 and k[0] == 1.0


def test_scales_far_below_the_cap_are_refused():
    """scale / cap would be no normal float32 number: capped scores lose bits."""
    import ctypes as C

    from magic_amd import _lib
    from magic_amd.model.attention import attention_plan, segment_attention
    a = _lib.MagicAttn()
    a.dtype, a.q_heads, a.kv_heads, a.head_dim = 0, 4, 2, 64
    for cap, scale, want in ((1e30, 1e-7, 0), (1e30, 1e-9, -1), (1e30, 0.0, 0), (0.0, 1e-38, 0), (50.0, 1e-36, 0), (50.0, 1e-37, -1)):      # (1e-36 / 50 = 2e-38, 2^-126 = 1.2e-38)
        a.cap, a.scale = cap, scale
        assert _lib.load().magic_attn_fwd(C.byref(a), None, 0, 0, None, None, 0, None) == want, (cap, scale)
    x = torch.randn(4, 2, 16)
    with pytest.raises(_lib.MagicHipError, match="of the cap"):
        segment_attention(x, x, x, attention_plan([4], device="cpu"), cap=1e30, scale=1e-9)
