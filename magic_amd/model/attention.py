"""Attention of a node over all nodes of its own component graph.

``GATConv`` (``gat.py``) reaches as far as its layers hop along edges; the operators here let every node of a batch of
component graphs see all nodes of its own graph:

* ``head_norm_rope``: RMS norm of every head of the queries and keys, with the rotation by a node's position (its
  order of appearance), in one pass;
* ``segment_attention``: softmax attention inside segments (the component graphs), with scores capped by a tanh, a
  bias that falls with the distance of two positions, a mask over keys and grouped heads, and its gradients;
* ``GlobalAttention``: the block ``x + W_o attention(norm_rope(W_q x), norm_rope(W_k x), W_v x)`` that
  ``GMAEModel(global_attention=True)`` puts behind its encoder.

No counterpart in the reference, whose only attention is the one along edges (``model/gat.py:302-312``).
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import numpy as np
import torch
import torch.nn as nn

from .. import _lib
from ..graph import Graph
from .gat import linear_nobias


class AttentionPlan:
    """Segments of ``segment_attention`` and the tables of tiles its kernels walk (on the device)."""

    def __init__(self, q_lens, kv_lens, q_tiles, k_tiles):
        self.q_lens, self.kv_lens = q_lens, kv_lens
        self.n_q, self.n_k = sum(q_lens), sum(kv_lens)
        self.max_q, self.max_k = max(q_lens, default=0), max(kv_lens, default=0)
        self.n_seg = len(q_lens)
        self.q_tiles, self.k_tiles = q_tiles, k_tiles
        self._stream = _stream_of(q_tiles.device)

    @property
    def device(self):
        return self.q_tiles.device

    def hold(self, *more):
        """Keeps the memory of the tables (and of ``more`` that came with them) from being handed out again while work of
        the current stream, if it is not the one they were made on, still reads them."""
        if _stream_of(self.device) != self._stream:
            for t in (self.q_tiles, self.k_tiles) + more:
                t.record_stream(torch.cuda.current_stream(self.device))


def _stream_of(device):
    return _lib.stream_on(device) if device.type == "cuda" else None


def _tiles(rows, others):
    """int32 [tiles, 8]: {first row, rows, first row of the other side, its rows, segment, the segment's own first row
    and rows, 0} of every tile of up to ``_lib.ATTN_TILE`` rows, longest segments' tiles first (they take longest; results do not depend on the order)."""
    rows, others = np.asarray(rows, np.int64), np.asarray(others, np.int64)
    n = -(-rows // _lib.ATTN_TILE)
    seg = np.repeat(np.arange(rows.size), n)
    at = (np.arange(seg.size) - np.repeat(np.cumsum(n) - n, n)) * _lib.ATTN_TILE
    r0, o0 = np.cumsum(rows) - rows, np.cumsum(others) - others
    t = np.stack([r0[seg] + at, np.minimum(rows[seg] - at, _lib.ATTN_TILE), o0[seg], others[seg], seg, r0[seg], rows[seg], 0 * seg], 1)
    return t[np.argsort(-others[seg], kind="stable")].astype(np.int32)


def attention_plan(q_lens: Sequence[int], kv_lens: Optional[Sequence[int]] = None, device="cuda") -> AttentionPlan:
    """Plan for segments of ``q_lens[i]`` query rows over ``kv_lens[i]`` key rows (host integers, in row order; keys =
    queries when ``kv_lens`` is None).  Lengths may be zero.  A plan serves any heads, types and options, and can be
    kept as long as the lengths stay the same (all layers of a step, all calls against one stored graph), on any stream of
    its device.  Its tables are on the device when this returns: build it before recording a graph."""
    q_lens = [int(x) for x in q_lens]
    kv_lens = q_lens if kv_lens is None else [int(x) for x in kv_lens]
    if len(q_lens) != len(kv_lens):
        raise _lib.MagicHipError(f"{len(q_lens)} query segments but {len(kv_lens)} key segments")
    if any(x < 0 for x in q_lens + kv_lens):
        raise _lib.MagicHipError("segment lengths must not be negative")
    if max(sum(q_lens), sum(kv_lens)) > 0x7fff0000:
        raise _lib.MagicHipError("segment attention serves up to 2,147,418,112 rows")
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    sides = ((q_lens, kv_lens), (kv_lens, q_lens))[:1 if kv_lens == q_lens else 2]      # (both sides' tables are one then)
    tabs = [torch.from_numpy(_tiles(a, b)) for a, b in sides]
    if device.type == "cuda":
        if torch.cuda.is_current_stream_capturing():
            raise _lib.MagicHipError("build the plan before the capture: its tables would not outlive it")
        # (blocking copies: the kernels take the tables' entries as offsets, on whatever stream a call comes)
        tabs = [t.to(device) for t in tabs]
    return AttentionPlan(q_lens, kv_lens, tabs[0], tabs[-1])


class _SegmentAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, plan, scale, cap, q_pos, k_pos, key_mask):
        _lib.attn_check(q, k, v, plan.n_q, plan.n_k, plan.device, cap, slopes, q_pos, k_pos, key_mask)
        plan.hold()
        operands = _lib.attn_operands(q, k, v, slopes, q_pos, k_pos, key_mask)
        # A score gradient is p (do.v - do.o): with few keys the rounding of a bfloat16 o is twice what else is off
        out_lo = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q.dtype == torch.bfloat16 and any(ctx.needs_input_grad) else None
        out, lse = _lib.attn_fwd_checked(operands, plan, scale, cap, out_lo)
        ctx.save_for_backward(*operands, out, lse, out_lo)
        ctx.plan, ctx.scale, ctx.cap = plan, scale, cap
        return out

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, d_out):
        *operands, out, lse, out_lo = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv, ds = _lib.attn_bwd_checked(operands, ctx.plan, ctx.scale, ctx.cap, out, lse, d_out, need[0],
                                               need[1] or need[2], need[3], out_lo)
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, ds) + (None,) * 6


def segment_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: AttentionPlan, *,
                      scale: Optional[float] = None, cap: float = 0.0, slopes: Optional[torch.Tensor] = None,
                      q_pos: Optional[torch.Tensor] = None, k_pos: Optional[torch.Tensor] = None,
                      key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of the rows of every segment over the keys of the same segment.

    q [n_q, q_heads, head_dim]; k, v [n_k, kv_heads, head_dim], query head h reads key head h // (q_heads //
    kv_heads).  float32 or bfloat16, any row and head strides, head_dim a multiple of 8 up to 128.
    ``s = scale q.k`` (scale: 1 / sqrt(head_dim)); ``cap`` (1e-3 to 1e30, 0: none): ``cap tanh(s / cap)``;
    ``slopes`` [q_heads] float32: minus ``slopes[h] |q_pos[i] - k_pos[j]|`` (int32 positions); ``key_mask`` [n_k] bool: False = the key takes no part,
    whatever its rows hold.  A row that sees no key gets zeros, and zero gradients.
    Differentiable in q, k, v and slopes; the sums have a fixed order."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if not abs(scale) <= 1e30:
        raise _lib.MagicHipError(f"scale must be at most 1e30 in size (got {scale})")
    if cap and scale and abs(scale) < cap * 2.0 ** -126:
        raise _lib.MagicHipError(f"scale must be at least 2^-126 of the cap (got {scale}, {cap})")
    return _SegmentAttentionFn.apply(q, k, v, slopes, plan, float(scale), float(cap), q_pos, k_pos, key_mask)


class _HeadNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, pos, rotary_dim, eps, base):
        ctx.save_for_backward(q, k, wq, wk, pos)
        ctx.opts = (rotary_dim, eps, base)
        return _lib.head_norm_rope_fwd(q, k, wq, wk, pos, rotary_dim, eps, base)

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dyq, dyk):
        q, k, wq, wk, pos = ctx.saved_tensors
        return _lib.head_norm_rope_bwd_checked(q, k, wq, wk, pos, *ctx.opts, dyq, dyk) + (None,) * 4


def head_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, pos: torch.Tensor, *,
                   rotary_dim: Optional[int] = None, eps: float = 1e-6, base: float = 10000.0):
    """``(q', k')``: every head of q [n, q_heads, head_dim] and k [n, kv_heads, head_dim] divided by its root mean
    square (``rsqrt(mean(x^2) + eps)``), times ``q_weight`` / ``k_weight`` [head_dim] float32, and its column pairs
    (i, i + R/2), i < R/2, turned by ``pos * base^(-2i/R)``; R = ``rotary_dim`` (head_dim unless given; 0: norm only).
    float32 or bfloat16, any strides, head_dim up to 128, ``pos`` [n] int32.  Differentiable in q, k and the weights."""
    rotary_dim = q.shape[-1] if rotary_dim is None else int(rotary_dim)
    return _HeadNormRopeFn.apply(q, k, q_weight, k_weight, pos, rotary_dim, float(eps), float(base))


class GlobalAttention(nn.Module):
    """Every node attends the nodes of its own component graph: ``x + W_o attention(q, k, W_v x)`` with ``q, k`` = heads
    of ``W_q x, W_k x`` after RMS norm and rotation by the node's position, scores capped at ``cap`` (0: not), and a
    learned bias per head that falls with the distance of two positions.  ``W_o`` starts as zeros: the block is the
    identity until it has learned something.

    ``act_bits=8`` keeps the input of its first linear layer for the backward pass as 8-bit codes (``act8.py``).  That saves
    memory where nothing else keeps ``x``; an activation or a graph layer that made it does.  (The input of the last linear
    layer is the attention's result, which its own backward pass reads in float32.)"""

    def __init__(self, dim: int, n_heads: int, cap: float = 50.0, act_bits: int = 32):
        super().__init__()
        if dim % n_heads or (dim // n_heads) % 8 or dim // n_heads > _lib.ATTN_MAX_DIM:
            raise _lib.MagicHipError(f"head width {dim} / {n_heads} must be a multiple of 8 up to {_lib.ATTN_MAX_DIM}")
        if act_bits not in (8, 32):
            raise _lib.MagicHipError(f"act_bits must be 32 or 8 (got {act_bits})")
        self.n_heads, self.head_dim, self.cap, self.act_bits = n_heads, dim // n_heads, float(cap), act_bits
        self.qkv = nn.Linear(dim, 3 * dim, bias=False)
        self.out = nn.Linear(dim, dim, bias=False)
        self.q_weight = nn.Parameter(torch.ones(self.head_dim))
        self.k_weight = nn.Parameter(torch.ones(self.head_dim))
        # 1/8 of a unit of score per position down to 2^-11, from head to head
        self.slopes = nn.Parameter(2.0 ** -torch.linspace(3.0, 11.0, n_heads))
        nn.init.xavier_uniform_(self.qkv.weight)
        nn.init.zeros_(self.out.weight)

    def forward(self, graph: Graph, x: torch.Tensor, key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``key_mask`` [N] bool: nodes that may be attended (all when None)."""
        n, dim = x.shape
        plan, pos = graph.component_attention()
        parts = linear_nobias(x, self.qkv.weight, self.act_bits).split(dim, dim=1)
        q, k, v = (t.view(n, self.n_heads, self.head_dim) for t in parts)
        q, k = head_norm_rope(q, k, self.q_weight, self.k_weight, pos)
        o = segment_attention(q, k, v, plan, cap=self.cap, slopes=self.slopes, q_pos=pos, k_pos=pos, key_mask=key_mask)
        return x + linear_nobias(o.view(n, dim), self.out.weight)
