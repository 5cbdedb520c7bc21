"""The global-attention block and the 8-bit checkpoints as the model uses them: the block against a float64 restatement,
the model's loss and gradients, one training loop."""
import copy
import math

import pytest
import torch

from tests.util import small_graph, to_graph

pytestmark = pytest.mark.gpu


def restated(block, x, lens, key_mask=None):
    """float64 statement of GlobalAttention on component graphs of ``lens`` nodes."""
    b = copy.deepcopy(block).double()
    h, d = b.n_heads, b.head_dim
    dim = h * d
    y = x @ b.qkv.weight.t()
    q, k, v = (t.reshape(-1, h, d) for t in y.split(dim, 1))
    out, at = [], 0
    inv = 10000.0 ** (-torch.arange(d // 2, dtype=torch.float64, device=x.device) * 2 / d)
    for n in lens:
        pos = torch.arange(n, device=x.device, dtype=torch.float64)
        c, s = torch.cos(pos[:, None] * inv)[:, None], torch.sin(pos[:, None] * inv)[:, None]

        def prep(t, w):
            t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
            a, e = t[..., :d // 2], t[..., d // 2:]
            return torch.cat([a * c - e * s, e * c + a * s], -1)

        rows = slice(at, at + n)
        at += n
        sc = torch.einsum("ihd,jhd->hij", prep(q[rows], b.q_weight), prep(k[rows], b.k_weight)) / math.sqrt(d)
        sc = b.cap * torch.tanh(sc / b.cap) - b.slopes[:, None, None] * (pos[:, None] - pos[None]).abs()
        if key_mask is not None:
            sc = sc.masked_fill(~key_mask[rows], -float("inf"))
        out.append(torch.einsum("hij,jhd->ihd", torch.softmax(sc, -1), v[rows]).reshape(n, dim))
    return x + torch.cat(out) @ b.out.weight.t(), b


@pytest.mark.parametrize("dim,heads", [(64, 4), (256, 4)])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_block_matches_float64(cuda, dim, heads, masked, bits):
    import magic_amd as G
    from magic_amd.model.attention import GlobalAttention
    torch.manual_seed(3)
    lens = [130, 700, 1, 57]
    graphs = [G.graph((torch.zeros(1, dtype=torch.long), torch.zeros(1, dtype=torch.long)), num_nodes=n) for n in lens]
    g = G.batch([x.to(cuda) for x in graphs])
    assert g.batch_num_nodes() == lens
    block = GlobalAttention(dim, heads, act_bits=bits).to(cuda)
    x = torch.randn(sum(lens), dim, device=cuda)
    assert torch.equal(block(g, x), x)                        # W_o = 0: the identity
    with torch.no_grad():
        block.out.weight.normal_(std=dim ** -0.5)
        block.q_weight.uniform_(0.5, 1.5)
    mask = None
    if masked:
        mask = torch.rand(sum(lens), device=cuda) < 0.5
        mask[830] = True                                       # (the graph of one node keeps its key)
    x.requires_grad_(True)
    y = block(g, x, key_mask=mask)
    d = torch.randn_like(y)
    params = dict(block.named_parameters())
    grads = torch.autograd.grad(y, [x] + list(params.values()), d)
    x64 = x.detach().double().requires_grad_(True)
    want, twin = restated(block, x64, lens, mask)
    wg = torch.autograd.grad(want, [x64] + [dict(twin.named_parameters())[k] for k in params], d.double())
    # float32 chains of about dim + n terms: relative 2-norm errors of some 1e-6.  The weight gradients of the 8-bit layers
    # see inputs off by up to half a step, 2^-7 of the largest of 32 values, which is up to four times their root mean
    # square: dY^T E against dY^T X is then at most about 2^-7 * 4 = 2^-5.
    def rel(a, b):
        return float((a.detach().double() - b.detach()).norm() / b.detach().norm())
    assert rel(y, want) < 1e-5
    for name, a, b in zip(["x"] + list(params), grads, wg):
        assert rel(a, b) < (2.0 ** -5 if bits == 8 and name in ("qkv.weight", "out.weight") else 2e-5), name


@pytest.mark.parametrize("bits", [32, 8])
def test_model_with_global_attention(cuda, bits):
    """Loss and every parameter's gradient against the same model with the block restated in float64 torch, and the
    embedding; without the options the model is the reference's."""
    from magic_amd.model.autoencoder import GMAEModel
    n_dim, e_dim, n, e = 5, 7, 300, 1500
    src, dst, nt, et = small_graph(n, e, n_dim, e_dim, seed=5, hub_deg=90)
    args = (n_dim, e_dim, 64, 3, 4, "prelu", 0.1, 0.2, True, "BatchNorm", 0.5, "sce", 3)
    torch.manual_seed(0)
    plain = GMAEModel(*args)
    torch.manual_seed(0)
    model = GMAEModel(*args, global_attention=True, act_bits=bits)
    for k, v in plain.state_dict().items():
        assert torch.equal(v, model.state_dict()[k])
    extra = set(model.state_dict()) - set(plain.state_dict())
    assert extra == {f"global_attn.{k}" for k in ("qkv.weight", "out.weight", "q_weight", "k_weight", "slopes")}
    model, plain = model.to(cuda).eval(), plain.to(cuda).eval()
    gen = torch.Generator().manual_seed(1)
    kw = dict(perm=torch.randperm(n, generator=gen).to(cuda), pos_idx=torch.randperm(src.size, generator=gen)[:n],
              neg_pairs=tuple(torch.randint(0, n, (2, n), generator=gen)))
    make = lambda: to_graph(src, dst, n, nt, et, n_dim, e_dim, cuda)  # noqa: E731
    with torch.no_grad():
        assert torch.equal(model.embed(make()), plain.embed(make()))      # the block starts as the identity
    # and so does training, up to the order of the layer-by-layer path's sums
    l0, l1 = plain.compute_loss(make(), **kw), model.compute_loss(make(), **kw)
    assert abs(l0.item() - l1.item()) < 1e-5 * abs(l0.item())
    with torch.no_grad():
        model.global_attn.out.weight.normal_(std=0.1)
    loss, parts = model.compute_loss(make(), return_parts=True, **kw)
    loss.backward()
    for name, p in model.named_parameters():
        if "fc_node_embedding" in name:
            continue
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    # gradient of the block's parameters against central differences of the loss (float32 loss: step 1e-2, 2 % of it)
    for name in ("out.weight", "qkv.weight"):
        p = dict(model.global_attn.named_parameters())[name]
        dirn = p.grad / p.grad.norm()
        vals = []
        for s in (1e-2, -1e-2):
            with torch.no_grad():
                p.add_(dirn, alpha=s)
                vals.append(float(model.compute_loss(make(), **kw)))
                p.add_(dirn, alpha=-s)
        slope = (vals[0] - vals[1]) / 2e-2
        assert abs(slope - float(p.grad.norm())) < 0.05 * float(p.grad.norm()) + 1e-4, name


def test_training_loop_and_refusals(cuda):
    """The batch-level loop with both options runs and moves the block's parameters; what is not served is refused."""
    from magic_amd import _lib
    import magic_amd as G
    from magic_amd.model.attention import GlobalAttention
    from magic_amd.model.autoencoder import build_model
    from magic_amd.utils.config import build_args
    args = build_args(["--global_attention", "--act_bits", "8"])
    args.n_dim, args.e_dim, args.num_hidden, args.num_layers = 5, 7, 64, 3
    torch.manual_seed(0)
    model = build_model(args).to(cuda).train()
    graphs = []
    for seed in range(3):
        src, dst, nt, et = small_graph(120 + 30 * seed, 700, 5, 7, seed=seed)
        graphs.append(to_graph(src, dst, 120 + 30 * seed, nt, et, 5, 7, cuda))
    opt = torch.optim.Adam(model.parameters(), lr=1e-3)
    before = {k: v.clone() for k, v in model.global_attn.state_dict().items()}
    for _ in range(3):
        g = G.batch(graphs)
        g.ndata["attr"] = torch.nn.functional.one_hot(g.ndata["type"].view(-1).long(), 5).float()
        loss = model(g)
        opt.zero_grad()
        loss.backward()
        opt.step()
        assert torch.isfinite(loss)
    for k, v in model.global_attn.state_dict().items():
        assert not torch.equal(v, before[k]), k
    for bad in (lambda: GlobalAttention(60, 5), lambda: GlobalAttention(64, 4, act_bits=4)):
        with pytest.raises(_lib.MagicHipError):
            bad()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_step_of_the_block(cuda, bits):
    """Forward and backward through autograd in a captured graph (scaled planes, gathered keys, rotation, 8-bit linear
    layers), replayed on new inputs with eager steps between the replays."""
    import magic_amd as G
    from magic_amd.model.attention import GlobalAttention
    torch.manual_seed(4)
    lens = [650, 1, 90]
    g = G.batch([G.graph((torch.zeros(1, dtype=torch.long), torch.zeros(1, dtype=torch.long)), num_nodes=n).to(cuda) for n in lens])
    block = GlobalAttention(256, 4, act_bits=bits).to(cuda)
    with torch.no_grad():
        block.out.weight.normal_(std=1 / 16)
    params = list(block.parameters())
    draw = lambda: (torch.randn(sum(lens), 256, device=cuda), torch.randn(sum(lens), 256, device=cuda), torch.rand(sum(lens), device=cuda) < 0.6)  # noqa: E731

    def step(x, d, mask):
        y = block(g, x, key_mask=mask)
        return [y.detach(), *torch.autograd.grad(y, [x] + params, d)]

    ins = [t.clone() for t in draw()]
    ins[0].requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*ins)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(*ins)
    for _ in range(4):
        new = draw()
        with torch.no_grad():
            for a, b in zip(ins, new):
                a.copy_(b)
        graph.replay()
        got = [t.clone() for t in res]
        eager = step(new[0].requires_grad_(True), *new[1:])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def _two_component_graphs(cuda, lens):
    import magic_amd as G
    edge = torch.zeros(1, dtype=torch.long)
    return G.batch([G.graph((edge, edge), num_nodes=n).to(cuda) for n in lens])


def test_component_plan_made_on_one_stream_and_read_on_another(cuda):
    """The tables are whole for a second stream although the first, which made them, is busy."""
    from magic_amd.model.attention import attention_plan
    lens = [130, 70, 1]
    g, want = _two_component_graphs(cuda, lens), attention_plan(lens, device="cpu")
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        torch.cuda._sleep(5_000_000)
        plan, pos = g.component_attention()
    with torch.cuda.stream(b):
        got = plan.q_tiles.clone(), plan.k_tiles.clone(), pos.clone()
    torch.cuda.synchronize()
    assert torch.equal(got[0].cpu(), want.q_tiles) and torch.equal(got[1].cpu(), want.k_tiles)
    assert torch.equal(got[2].cpu(), torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]))


def test_component_plan_dropped_while_another_stream_reads_it(cuda):
    """The plan's stream gets its memory back only behind the work of the other one.  (What that stream writes next is
    another valid plan of the same size: whichever of the two a call reads, it stays inside its operands.)"""
    from magic_amd.model.attention import attention_plan, segment_attention
    lens, other = [130, 70, 1], [1, 70, 130]
    x = torch.randn(201, 4, 32, device=cuda)
    want = segment_attention(x, x, x, attention_plan(lens, device=cuda))
    fill = attention_plan(other, device=cuda).q_tiles
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    g = _two_component_graphs(cuda, lens)
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        plan, _ = g.component_attention()
    with torch.cuda.stream(b):
        torch.cuda._sleep(5_000_000)
        got = segment_attention(x, x, x, plan)
    del plan, g
    with torch.cuda.stream(a):
        again = [fill.clone() for _ in range(64)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(again) == 64


def _held(fn, owned):
    """Bytes of the distinct memory that the backward pass of ``fn()`` holds beside ``owned`` tensors."""
    seen = {}

    def pack(t):
        s = t.untyped_storage()
        seen[s.data_ptr()] = s.nbytes()
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = fn()
    own = {t.untyped_storage().data_ptr() for t in owned}
    return sum(n for p, n in seen.items() if p not in own), y


def test_what_8_bit_checkpoints_save_in_the_block_and_the_model(cuda):
    """The inputs that only the 8-bit layers keep shrink from 4 to 1 + 1 / 32 bytes an element, and nothing is added
    anywhere else."""
    from magic_amd.model.attention import GlobalAttention
    from magic_amd.model.autoencoder import GMAEModel
    lens = [130, 200]
    g, n = _two_component_graphs(cuda, lens), 330
    x0 = torch.randn(n, 64, device=cuda, requires_grad=True)
    held = {}
    for bits in (32, 8):
        block = GlobalAttention(64, 4, act_bits=bits).to(cuda)
        held[bits], _ = _held(lambda: block(g, x0 * 2.0), [x0, *block.parameters()])     # (x0 * 2 keeps nothing of its result)
    assert held[32] - held[8] == n * 64 * 3 - n * 64 // 32
    n_dim, e_dim, n, e, layers = 5, 7, 300, 1500, 3
    src, dst, nt, et = small_graph(n, e, n_dim, e_dim, seed=5, hub_deg=90)
    gen = torch.Generator().manual_seed(1)
    kw = dict(perm=torch.randperm(n, generator=gen).to(cuda), pos_idx=torch.randperm(src.size, generator=gen)[:n],
              neg_pairs=tuple(torch.randint(0, n, (2, n), generator=gen)))
    for bits in (32, 8):
        torch.manual_seed(0)
        model = GMAEModel(n_dim, e_dim, 64, layers, 4, "prelu", 0.1, 0.2, True, "BatchNorm", 0.5, "sce", 3,
                          global_attention=True, act_bits=bits).to(cuda).eval()
        graph = to_graph(src, dst, n, nt, et, n_dim, e_dim, cuda)
        held[bits], loss = _held(lambda: model.compute_loss(graph, **kw), model.parameters())
    elements = n * 64 * layers + 2 * n * 2 * 64 * layers                  # hidden states side by side; rows of 2 n node pairs
    assert held[32] - held[8] == elements * 3 - elements // 32
