"""Workloads of the global-attention block of the masked graph auto-encoder.

Three operators that a training step or a serving call runs one after the other:

* ``attention``: every row attends the keys of its own component graph (``segment_attention``): scores capped
  by a tanh, a bias that falls with the distance of two positions, a mask over keys, grouped heads;
* ``norm_rope``: RMS norm of every head of the queries and keys, with the position rotation (``head_norm_rope``);
* ``act8``: the inputs of linear layers kept for the backward pass as 8-bit codes with a power-of-two scale for 32
  columns (``act8_pack`` / ``act8_unpack``, ``linear_nobias(..., act_bits=8)``).

``own`` selects the framework's kernels; otherwise ``run`` computes the plain form in float32.
"""
import math
import random

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new node per stored graph scored against the nodes of a StreamSpot-shaped batch of twelve graphs
        dict(name="attn_serve_streamspot", op="attention", train=False, dtype="f32", hq=4, hk=4, d=64,
             q_lens="1*12", kv_lens="8206,7310,8971,8000,7777,9013,8555,6901,8192,7643,8420,8012", cap=0.0, bias=True,
             mask=False),
        # few new nodes against one long entity-level history, shared key heads, bfloat16 store
        dict(name="attn_serve_long_bf16", op="attention", train=False, dtype="bf16", hq=16, hk=4, d=128,
             q_lens="3", kv_lens="262147", cap=30.0, bias=False, mask=False),
        # a step on one small graph at the entity-level model's width (hidden 64, 4 heads)
        dict(name="attn_train_small", op="attention", train=True, dtype="f32", hq=4, hk=4, d=16, q_lens="301",
             kv_lens="301", cap=20.0, bias=True, mask=True),
        # embedding of many small ragged graphs, one of them empty, one of a single node
        dict(name="attn_embed_ragged", op="attention", train=False, dtype="f32", hq=4, hk=4, d=16,
             q_lens="1,0," + ",".join(str(17 + (i * 389) % 1500) for i in range(62)),
             kv_lens="1,0," + ",".join(str(17 + (i * 389) % 1500) for i in range(62)), cap=0.0, bias=False, mask=True),
        # a training step on the batch of twelve StreamSpot-shaped graphs (hidden 256, 4 heads)
        dict(name="attn_train_streamspot", op="attention", train=True, dtype="f32", hq=4, hk=4, d=64,
             q_lens="8206,7310,8971,8000,7777,9013,8555,6901,8192,7643,8420,8012",
             kv_lens="8206,7310,8971,8000,7777,9013,8555,6901,8192,7643,8420,8012", cap=0.0, bias=True, mask=False),
        # the same in bfloat16 with grouped heads of width 128 and graphs of very different sizes
        dict(name="attn_train_grouped_bf16", op="attention", train=True, dtype="bf16", hq=8, hk=2, d=128,
             q_lens="15001,257,4099,1,8888,63,2050", kv_lens="15001,257,4099,1,8888,63,2050", cap=50.0, bias=False,
             mask=True),
        # the new nodes of a serving call before their attention
        dict(name="norm_rope_serve", op="norm_rope", train=False, dtype="f32", hq=4, hk=4, d=64, n=12, rot=64),
        # the rows of the StreamSpot-shaped batch, training
        dict(name="norm_rope_train_streamspot", op="norm_rope", train=True, dtype="f32", hq=4, hk=4, d=64, n=97000,
             rot=64),
        # grouped heads of width 128, bfloat16, half of each head rotated
        dict(name="norm_rope_train_grouped_bf16", op="norm_rope", train=True, dtype="bf16", hq=16, hk=4, d=128,
             n=131071, rot=64),
        # a small linear layer of odd sizes
        dict(name="act8_linear_small", op="act8", kind="linear", n=1201, f=69, m=37),
        # the encoder-to-decoder projection of the THEIA-shaped model (three hidden states of 64 side by side)
        dict(name="act8_linear_theia", op="act8", kind="linear", n=700000, f=192, m=64),
        # codes and back, the concatenated hidden states of the StreamSpot-shaped batch
        dict(name="act8_pack_streamspot", op="act8", kind="pack", n=97000, f=1024, m=0),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    kind = rng.choice(["serve", "train", "train", "embed", "norm_rope", "norm_rope", "linear", "linear", "pack"])
    if kind in ("serve", "train", "embed"):
        dtype = rng.choice(["f32", "bf16"])
        d = rng.choice([16, 24, 32, 64, 64, 128])
        hk = rng.choice([1, 2, 4])
        hq = hk * rng.choice([1, 1, 2, 4])
        budget = 2.0e11 if kind != "serve" else 2.0e10       # multiply-adds of one product
        segs = _logint(rng, 1, 40)
        q_lens, kv_lens = [], []
        for _ in range(segs):
            if kind == "serve":
                q, k = rng.randint(1, 8), _logint(rng, 1, 60000)
            else:
                q = _logint(rng, 1, 9000)
                k = q if rng.random() < 0.8 else _logint(rng, 1, 9000)
            cost = float(q) * k * hq * d
            if cost > budget:
                continue
            budget -= cost
            q_lens.append(q)
            kv_lens.append(k)
        if not q_lens:
            q_lens, kv_lens = [5], [77]
        return dict(op="attention", train=kind == "train", dtype=dtype, hq=hq, hk=hk, d=d,
                    q_lens=",".join(map(str, q_lens)), kv_lens=",".join(map(str, kv_lens)),
                    cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.5, mask=rng.random() < 0.4)
    if kind == "norm_rope":
        d = rng.choice([16, 24, 32, 64, 128])
        hk = rng.choice([1, 2, 4])
        return dict(op="norm_rope", train=rng.random() < 0.7, dtype=rng.choice(["f32", "bf16"]),
                    hq=hk * rng.choice([1, 2, 4]), hk=hk, d=d, n=_logint(rng, 1, 100000),
                    rot=rng.choice([d, d, d // 2, 8]))
    if kind == "linear":
        return dict(op="act8", kind="linear", n=_logint(rng, 1, 200000), f=_logint(rng, 4, 1024), m=_logint(rng, 4, 320))
    return dict(op="act8", kind="pack", n=_logint(rng, 1, 100000), f=_logint(rng, 4, 1024), m=0)


def _lens(text):
    out = []
    for part in text.split(","):
        if "*" in part:
            a, b = part.split("*")
            out += [int(a)] * int(b)
        else:
            out.append(int(part))
    return out


# ------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * std

    st = {"case": case}
    if case["op"] == "attention":
        dt = _DT[case["dtype"]]
        ql, kl = _lens(case["q_lens"]), _lens(case["kv_lens"])
        nq, nk, hq, hk, d = sum(ql), sum(kl), case["hq"], case["hk"], case["d"]
        st["q_lens"], st["kv_lens"] = ql, kl
        st["q"] = randn(nq, hq, d, std=1.3).to(dt)
        st["k"] = randn(nk, hk, d, std=1.3).to(dt)
        st["v"] = randn(nk, hk, d, std=0.7).to(dt)
        st["slopes"] = st["q_pos"] = st["k_pos"] = st["key_mask"] = None
        if case["bias"]:
            st["slopes"] = torch.tensor([2.0 ** -(6.0 + 5.0 * h / hq) for h in range(hq)], device="cuda") \
                * (1.0 + 0.1 * torch.rand(hq, generator=gen, device="cuda"))
            st["k_pos"] = _positions(kl, gen)
            st["q_pos"] = st["k_pos"] if ql == kl else _positions(ql, gen, start=kl)
        if case["mask"]:
            st["key_mask"] = torch.rand(nk, generator=gen, device="cuda") < 0.5      # the masked half of the nodes
        if case["train"]:
            st["d_out"] = randn(nq, hq, d, std=0.01).to(dt)
        if own:
            from magic_amd.model.attention import attention_plan
            st["plan"] = attention_plan(ql, kl, device="cuda")
            if case["train"]:
                for key in ("q", "k", "v", "slopes"):
                    if st[key] is not None:
                        st[key].requires_grad_(True)
    elif case["op"] == "norm_rope":
        dt = _DT[case["dtype"]]
        n, hq, hk, d = case["n"], case["hq"], case["hk"], case["d"]
        # queries, keys and values of a row lie side by side, as one projection writes them
        qkv = randn(n, (hq + 2 * hk) * d, std=0.8).to(dt)
        st["qkv"] = qkv
        st["q"] = qkv[:, :hq * d].view(n, hq, d)
        st["k"] = qkv[:, hq * d:(hq + hk) * d].view(n, hk, d)
        st["wq"] = 1.0 + randn(d, std=0.1)
        st["wk"] = 1.0 + randn(d, std=0.1)
        st["pos"] = torch.randint(0, 700000, (n,), generator=gen, device="cuda", dtype=torch.int32)
        if case["train"]:
            st["d_q"] = randn(n, hq, d, std=0.01).to(dt)
            st["d_k"] = randn(n, hk, d, std=0.01).to(dt)
        if own and case["train"]:
            for key in ("q", "k", "wq", "wk"):
                st[key] = st[key].detach().requires_grad_(True)
    else:
        n, f, m = case["n"], case["f"], case["m"]
        x = randn(n, f)
        # activations after a PReLU: the negative side is small
        st["x"] = torch.where(x > 0, x, 0.25 * x) * torch.exp(randn(n, 1, std=0.5))
        if case["kind"] == "linear":
            st["w"] = randn(m, f, std=1.0 / math.sqrt(f))
            st["d_y"] = randn(n, m, std=0.01)
            if own:
                st["x"].requires_grad_(True)
                st["w"].requires_grad_(True)
    return st


def _positions(lens, gen, start=None):
    """Order of appearance with gaps: ascending whole numbers within a graph."""
    n = sum(lens)
    step = torch.randint(0, 3, (max(n, 1),), generator=gen, device="cuda", dtype=torch.int64)
    tot = torch.cumsum(step, 0)
    out, at = [], 0
    for i, ln in enumerate(lens):
        if ln:
            base = 0 if start is None else start[i]
            out.append(tot[at:at + ln] - tot[at] + base)
        at += ln
    return (torch.cat(out) if out else tot[:0]).to(torch.int32)


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_attention(st):
    case = st["case"]
    hq, hk, d, cap = case["hq"], case["hk"], case["d"], case["cap"]
    g, scale, train = hq // hk, 1.0 / math.sqrt(d), case["train"]
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    out = torch.zeros_like(q)
    if train:
        do = st["d_out"].float()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dslope = torch.zeros(hq, device=q.device) if case["bias"] else None
    q0 = k0 = 0
    for nq, nk in zip(st["q_lens"], st["kv_lens"]):
        qs, ks = slice(q0, q0 + nq), slice(k0, k0 + nk)
        q0, k0 = q0 + nq, k0 + nk
        if nq == 0 or nk == 0:
            continue
        qh = q[qs].view(nq, hk, g, d).permute(1, 2, 0, 3).reshape(hk, g * nq, d)       # [hk, g*nq, d]
        kh = k[ks].transpose(0, 1).contiguous()                                       # [hk, nk, d]
        vh = v[ks].transpose(0, 1).contiguous()
        c = (torch.matmul(qh, kh.transpose(1, 2).contiguous()) * scale).view(hk, g, nq, nk)
        if cap > 0:
            c = cap * torch.tanh(c / cap)
        logit = c
        if case["bias"]:
            dist = (st["q_pos"][qs].long()[:, None] - st["k_pos"][ks].long()[None, :]).abs().float()
            logit = c - st["slopes"].view(hk, g, 1, 1) * dist
        if case["mask"]:
            logit = logit.masked_fill(~st["key_mask"][ks], float("-inf"))
        top = logit.amax(-1, keepdim=True)
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        p = torch.exp(logit - top)
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, torch.zeros_like(p)).view(hk, g * nq, nk)
        oh = torch.matmul(p, vh)
        out[qs] = oh.view(hk, g, nq, d).permute(2, 0, 1, 3).reshape(nq, hq, d)
        if not train:
            continue
        doh = do[qs].view(nq, hk, g, d).permute(1, 2, 0, 3).reshape(hk, g * nq, d)
        dv[ks] = torch.matmul(p.transpose(1, 2).contiguous(), doh).transpose(0, 1)
        dp = torch.matmul(doh, vh.transpose(1, 2).contiguous())
        dl = p * (dp - (doh * oh).sum(-1, keepdim=True))
        if case["bias"]:
            dslope -= (dl.view(hk, g, nq, nk) * dist).sum((2, 3), dtype=torch.float64).view(hq).float()
        if cap > 0:
            dl = dl * (1.0 - (c / cap) ** 2).view(hk, g * nq, nk)
        ds = dl * scale
        dq[qs] = torch.matmul(ds, kh).view(hk, g, nq, d).permute(2, 0, 1, 3).reshape(nq, hq, d)
        dk[ks] = torch.matmul(ds.transpose(1, 2).contiguous(), qh).transpose(0, 1)
    dt = st["q"].dtype
    if not train:
        return {"out": out.to(dt)}
    res = {"out": out.to(dt), "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt)}
    if case["bias"]:
        res["dslopes"] = dslope
    return res


def _plain_norm_rope(st):
    case = st["case"]
    d, rot, eps = case["d"], case["rot"], 1e-6
    half = rot // 2
    inv = torch.pow(10000.0, -torch.arange(half, dtype=torch.float64, device="cuda") * 2.0 / rot)
    ang = st["pos"].double()[:, None] * inv                              # far positions: angles in 64 bits
    cos, sin = torch.cos(ang).float()[:, None, :], torch.sin(ang).float()[:, None, :]

    def turn(y, sn):
        a, b = y[..., :half], y[..., half:rot]
        return torch.cat([a * cos - b * sn, b * cos + a * sn, y[..., rot:]], -1)

    def one(x, w, dy):
        dt = x.dtype
        x = x.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        y = turn(x * r * w, sin).to(dt)
        if dy is None:
            return y, None, None
        gy = turn(dy.float(), -sin)
        dw = (gy * x * r).sum((0, 1), dtype=torch.float64).float()
        gw = gy * w
        dx = r * (gw - x * (r * r) * (gw * x).mean(-1, keepdim=True))
        return y, dx.to(dt), dw

    train = case["train"]
    yq, dxq, dwq = one(st["q"], st["wq"], st["d_q"] if train else None)
    yk, dxk, dwk = one(st["k"], st["wk"], st["d_k"] if train else None)
    if not train:
        return {"q": yq, "k": yk}
    return {"q": yq, "k": yk, "dq": dxq, "dk": dxk, "dwq": dwq, "dwk": dwk}


def _plain_round8(x):
    n, f = x.shape
    blocks = (f + 31) // 32
    xp = torch.zeros(n, blocks * 32, device=x.device, dtype=x.dtype)
    xp[:, :f] = x
    xb = xp.view(n, blocks, 32)
    amax = xb.abs().amax(-1, keepdim=True)
    _, ex = torch.frexp(amax)                                # amax = m 2^ex, m in [0.5, 1)
    e = (ex - 7).clamp(min=-126)
    e = torch.where(torch.ldexp(amax, -e) >= 127.5, e + 1, e)
    val = torch.ldexp(torch.round(torch.ldexp(xb, -e)), e)
    return val.reshape(n, blocks * 32)[:, :f].contiguous()


def _plain_act8(st):
    xh = _plain_round8(st["x"])
    if st["case"]["kind"] == "pack":
        return {"values": xh}
    return {"y": torch.matmul(st["x"], st["w"].t()), "dx": torch.matmul(st["d_y"], st["w"]),
            "dw": torch.matmul(st["d_y"].t(), xh)}


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        return {"attention": _plain_attention, "norm_rope": _plain_norm_rope, "act8": _plain_act8}[case["op"]](state)
    if case["op"] == "attention":
        from magic_amd.model.attention import segment_attention
        leaves = [state[key] for key in ("q", "k", "v")]
        with torch.set_grad_enabled(case["train"]):
            out = segment_attention(*leaves, state["plan"], cap=case["cap"], slopes=state["slopes"],
                                    q_pos=state["q_pos"], k_pos=state["k_pos"], key_mask=state["key_mask"])
        if not case["train"]:
            return {"out": out}
        names = ["dq", "dk", "dv"]
        if case["bias"]:
            leaves.append(state["slopes"])
            names.append("dslopes")
        return dict(out=out.detach(), **dict(zip(names, torch.autograd.grad(out, leaves, state["d_out"]))))
    if case["op"] == "norm_rope":
        from magic_amd.model.attention import head_norm_rope
        args = (state["q"], state["k"], state["wq"], state["wk"])
        with torch.set_grad_enabled(case["train"]):
            q, k = head_norm_rope(*args, state["pos"], rotary_dim=case["rot"])
        if not case["train"]:
            return {"q": q, "k": k}
        grads = torch.autograd.grad((q, k), args, (state["d_q"], state["d_k"]))
        return dict(q=q.detach(), k=k.detach(), **dict(zip(("dq", "dk", "dwq", "dwk"), grads)))
    if case["kind"] == "pack":
        from magic_amd.model.act8 import act8_pack, act8_unpack
        return {"values": act8_unpack(act8_pack(state["x"]))}
    from magic_amd.model.gat import linear_nobias
    y = linear_nobias(state["x"], state["w"], act_bits=8)
    dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["d_y"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def work(case):
    if case["op"] == "attention":
        size = 4 if case["dtype"] == "f32" else 2
        ql, kl = _lens(case["q_lens"]), _lens(case["kv_lens"])
        pairs = float(sum(a * b for a, b in zip(ql, kl)))
        rows_q, rows_k = sum(ql) * case["hq"] * case["d"], sum(kl) * case["hk"] * case["d"]
        extra = (4 * (sum(ql) + sum(kl)) if case["bias"] else 0) + (sum(kl) if case["mask"] else 0)
        one = pairs * case["hq"] * case["d"]
        if not case["train"]:
            return {"bytes": size * (2 * rows_q + 2 * rows_k) + extra, "flops": 4 * one}
        return {"bytes": size * (4 * rows_q + 4 * rows_k) + extra, "flops": 14 * one}
    if case["op"] == "norm_rope":
        size = 4 if case["dtype"] == "f32" else 2
        elems = case["n"] * (case["hq"] + case["hk"]) * case["d"]
        if not case["train"]:
            return {"bytes": 2 * size * elems + 4 * case["n"], "flops": 8 * elems}
        return {"bytes": 4 * size * elems + 4 * case["n"], "flops": 24 * elems}
    n, f, m = case["n"], case["f"], case["m"]
    if case["kind"] == "pack":
        return {"bytes": 8 * n * f, "flops": 4 * n * f}
    return {"bytes": 4 * (2 * n * f + 2 * n * m + 2 * m * f), "flops": 6 * n * f * m}


# ------------------------------------------------------------------------------------------------- definition, 64 bits
def _exact_attention(case, st):
    hq, hk, d = case["hq"], case["hk"], case["d"]
    train = case["train"]
    q, k, v = (st[key].double() for key in ("q", "k", "v"))
    res = {"out": torch.zeros_like(q)}
    if train:
        res.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
        if case["bias"]:
            res["dslopes"] = torch.zeros(hq, dtype=torch.float64, device=q.device)
    q0 = k0 = 0
    for nq, nk in zip(st["q_lens"], st["kv_lens"]):
        rows, cols = slice(q0, q0 + nq), torch.arange(k0, k0 + nk, device=q.device)
        q0, k0 = q0 + nq, k0 + nk
        if case["mask"]:
            cols = cols[st["key_mask"][cols]]                # a masked key takes no part at all
        if nq == 0 or cols.numel() == 0:
            continue
        for h in range(hq):
            j = h // (hq // hk)
            a = q[rows, h].clone().requires_grad_(train)
            b, c = k[cols, j].clone().requires_grad_(train), v[cols, j].clone().requires_grad_(train)
            s = a.mm(b.t()) / math.sqrt(d)
            if case["cap"]:
                s = torch.tanh(s / case["cap"]) * case["cap"]
            wrt = [a, b, c]
            if case["bias"]:
                far = (st["q_pos"][rows].double()[:, None] - st["k_pos"][cols].double()[None]).abs()
                slope = st["slopes"][h].detach().double().requires_grad_(train)
                wrt.append(slope)
                s = s - slope * far
            o = torch.exp(s - torch.logsumexp(s, 1, keepdim=True)).mm(c)
            res["out"][rows, h] = o.detach()
            if train:
                grads = torch.autograd.grad(o, wrt, st["d_out"][rows, h].double())
                res["dq"][rows, h] = grads[0]
                res["dk"][:, j].index_add_(0, cols, grads[1])
                res["dv"][:, j].index_add_(0, cols, grads[2])
                if case["bias"]:
                    res["dslopes"][h] += grads[3]
    return res


def _exact_norm_rope(case, st):
    rot, train = case["rot"], case["train"]
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    phase = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), st["pos"].double()[:, None] * freq)

    def one(x, w):
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        z = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * phase[:, None]
        return torch.cat([z.real, z.imag, y[..., rot:]], -1)

    args = [st[key].detach().double().requires_grad_(train) for key in ("q", "k", "wq", "wk")]
    yq, yk = one(args[0], args[2]), one(args[1], args[3])
    res = {"q": yq.detach(), "k": yk.detach()}
    if train:
        grads = torch.autograd.grad((yq, yk), args, (st["d_q"].double(), st["d_k"].double()))
        res.update(zip(("dq", "dk", "dwq", "dwk"), grads))
    return res


def _exact_act8(case, st):
    x = st["x"].detach().double()
    n, f = x.shape
    val = torch.empty_like(x)
    for c in range(0, f, 32):
        part = x[:, c:c + 32]
        top = part.abs().amax(1, keepdim=True)
        # the smallest power of two that holds the block in whole steps up to 127
        step = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -120))) - 6.0)
        step = torch.where(torch.round(top / step) > 127, 2.0 * step, step)
        val[:, c:c + 32] = torch.round(part / step) * step
    if case["kind"] == "pack":
        return {"values": val}
    w, dy = st["w"].detach().double(), st["d_y"].double()
    return {"y": x.mm(w.t()), "dx": dy.mm(w), "dw": dy.t().mm(val)}


def exact(case, seed):
    st = prepare(case, seed)
    with torch.enable_grad():
        return {"attention": _exact_attention, "norm_rope": _exact_norm_rope, "act8": _exact_act8}[case["op"]](case, st)
