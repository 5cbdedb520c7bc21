"""Library calls inside a recorded HIP graph: no memory-set nodes (such nodes have left old contents standing in replays
after the first), and the eager result in every replay, with other work on the same memory in between."""
import collections
import ctypes

import pytest
import torch

from tests.util import small_graph, to_graph

pytestmark = pytest.mark.gpu
MEMSET = 2          # hipGraphNodeTypeMemset


def node_types(graph):
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    hip, g, n = ctypes.CDLL(path), ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(g, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert hip.hipGraphGetNodes(g, nodes, ctypes.byref(n)) == 0
    kinds = collections.Counter()
    for node in nodes:
        t = ctypes.c_int(-1)
        assert hip.hipGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(t)) == 0
        kinds[t.value] += 1
    return kinds


def _calls(cuda):
    from magic_amd import _lib
    from magic_amd.model.loss_func import sce_loss_masked
    x = torch.randn(3000, 12, device=cuda, requires_grad=True)
    t, idx = torch.rand(3000, 12, device=cuda), torch.randperm(3000, device=cuda)[:1500]
    none = torch.empty(0, 12, device=cuda)
    return {"sce": lambda: torch.autograd.grad(sce_loss_masked(x, t, idx, 3), x)[0],
            "weight_gradient_of_no_rows": lambda: _lib.proj_bwd_weight(torch.empty(0, 7, device=cuda), none),
            "readout_of_no_rows": lambda: _lib.readout(none, None, 0, False),
            "mean_of_no_rows": lambda: _lib.readout(none, None, 0, True).nan_to_num(5.0)}


@pytest.mark.parametrize("name", ["sce", "weight_gradient_of_no_rows", "readout_of_no_rows", "mean_of_no_rows"])
def test_recorded_calls_clear_their_results_in_every_replay(cuda, name):
    call = _calls(cuda)[name]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        got = call()
    assert node_types(graph)[MEMSET] == 0
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        got.fill_(float("inf"))
        assert torch.equal(call(), want)


def test_recorded_training_step_holds_no_memset(cuda, monkeypatch):
    from magic_amd.model.autoencoder import GMAEModel
    from magic_amd.model.step import CapturedTrainStep, make_adam
    whole = torch.cuda.CUDAGraph
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda **kw: whole(keep_graph=True))
    model = GMAEModel(5, 7, 64, 3, 4, "prelu", 0.1, 0.2, True, "BatchNorm", 0.5, "sce", 3).to(cuda)
    src, dst, nt, et = small_graph(9000, 40000, 5, 7, seed=91, hub_deg=300, hub_out=150)
    step = CapturedTrainStep(model, make_adam(model, 1e-3, 5e-4), to_graph(src, dst, 9000, nt, et, 5, 7, cuda), 5, capture=True)
    for _ in range(4):
        loss = step()
    torch.cuda.synchronize()
    assert torch.isfinite(loss) and node_types(step._graphs[0])[MEMSET] == 0


@pytest.mark.parametrize("ld,off", [(5, 0), (8, 0), (5, 1)])
def test_fills_of_every_alignment(cuda, ld, off):
    """The cleared rows of the SCE gradient are the operand's, to the last word."""
    from magic_amd import _lib
    lib, n, d = _lib.load(), 1001, 5
    x = torch.randn(n * ld + off + 8, device=cuda)[off:]
    mask = torch.arange(0, n, 3, device=cuda)
    t, loss = torch.rand(d, device=cuda), torch.zeros(1, device=cuda)
    d_x = torch.full((n * ld + 8,), 3.0, device=cuda)
    buf = torch.full((n * ld + 9,), 3.0, device=cuda)[off:off + n * ld + 8]
    for out in (d_x, buf):
        ws = torch.empty(lib.magic_sce_workspace_bytes(mask.numel(), d), dtype=torch.uint8, device=cuda)
        assert lib.magic_sce_fwd_bwd(n, d, mask.numel(), mask.data_ptr(), x.data_ptr(), ld, t.data_ptr(), 0, 3.0, 1.0, loss.data_ptr(),
                                     out.data_ptr(), None, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(d_x, buf) and (d_x[n * ld:] == 3.0).all()
    rows = d_x[:n * ld].view(n, ld)
    keep = torch.ones(n, dtype=torch.bool, device=cuda)
    keep[mask] = False
    assert not rows[keep].any() and not rows[:, d:].any() and rows[mask].any()


def _linear(n, f, m, bits, seed, cuda):
    from magic_amd.model.gat import linear_nobias
    gen = torch.Generator(device=cuda).manual_seed(seed)
    x, w, dy = (torch.randn(*s, generator=gen, device=cuda) for s in ((n, f), (m, f), (n, m)))
    x.requires_grad_(True), w.requires_grad_(True)

    def call():
        y = linear_nobias(x, w, act_bits=bits)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dy)]

    return call


@pytest.mark.parametrize("bits", [32, 8])
def test_linear_layers_on_two_streams_share_no_scratch(cuda, bits):
    calls = [_linear(60000, 256, 256, bits, 1, cuda), _linear(50000, 320, 130, bits, 2, cuda)]
    alone = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        got = []
        for s, call in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append([call() for _ in range(4)])
        torch.cuda.synchronize()
        for many, want in zip(got, alone):
            assert all(torch.equal(a, b) for res in many for a, b in zip(res, want))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_keeps_its_scratch_from_later_calls(cuda, bits):
    """A larger call after the recording, and tensors that take what it gave back: neither reaches the replays, nor they them."""
    call = _linear(3000, 256, 256, bits, 3, cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    for _ in range(3):
        _linear(90000, 512, 300, bits, 4, cuda)()
        other = [torch.full((1 << k,), float(k), device=cuda) for k in range(12, 25)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all((t == float(k)).all() for k, t in zip(range(12, 25), other))
