"""The layer with a relative position bias and an RMS norm ahead of it: the operators as they are used together.

Against the layer written out in float64.  Every step is a sum of at most 512 fp32 products and so off by at most 512 u (u = 2^-24)
of its magnitudes; eight steps follow each other in a forward and a backward (norm, projection, logits, weights, output, and back), and
the cancellation in the norms, the softmax and dP - D is taken as a factor of 4: 8 * 512 * 4 u = 1e-3 of the largest value."""
import math

import pytest
import torch

import spion_amd
from spion_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
B, H, L, d, BS = 2, 2, 256, 32, 32
TOL = 8 * 512 * 4 * 2.0 ** -24


@pytest.fixture(params=["node", "python"], autouse=True)
def both_nodes(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setitem(_lib._cache, "node", None)


def _config(task):
    return dict(transformer_dim=64, head_dim=d, num_head=H, max_seq_len=L, block_size=BS, batch_size=B, attention_dropout=0.0, task=task,
                num_layers=1, threshold=0.9, relative_buckets=16, relative_max_distance=64, rms_norm=True)


def _layer(task, inference=False):
    g = torch.Generator().manual_seed(3)
    layer = spion_amd.Attention(_config(task), inference=inference).to(DEV)
    with torch.no_grad():
        for n, p in layer.named_parameters():
            p.copy_(torch.randn(p.shape, generator=g) * (0.5 if "attn" in n else 0.1) + (1.0 if n.startswith("norm") else 0.0))
    return layer


def _written_out(layer, X, mask, mat):
    P = {n: p.detach().double().requires_grad_() for n, p in layer.named_parameters()}
    X = X.detach().double().requires_grad_()
    x = X / torch.sqrt((X * X).mean(-1, keepdim=True) + layer.norm.eps) * P["norm.weight"]
    q, k, v = ((x @ P[f"W_{n}.weight"].t() + P[f"W_{n}.bias"]).view(B, L, H, d).transpose(1, 2) for n in "qkv")
    rel = (torch.arange(L, device=DEV)[None] - torch.arange(L, device=DEV)[:, None]).clamp(-64, 64) + 64
    t = q @ k.transpose(-1, -2).contiguous() / math.sqrt(d) + P["attn.weight"].t()[:, layer.attn.buckets.long()[rel]]
    if mat is not None:
        at = torch.arange(L, device=DEV) // BS
        inside = mat[at][:, at] != 0
        t = torch.where(inside, t, 0.0)
    if mask is not None:
        left_out = (mask == 0)[:, None, None, :]
        t = t.masked_fill(left_out if mat is None else left_out & inside, -math.inf)
    p = torch.softmax(t, -1)
    w = p if mat is None else p * inside
    out = (w @ v).transpose(1, 2).reshape(B, L, H * d) @ P["ff.weight"].t() + P["ff.bias"]
    return out, p, X, P


def _near(name, got, want):
    top = float(want.abs().max())
    assert float((got.detach().double() - want).abs().max()) <= TOL * max(top, 1e-6), name


@pytest.mark.parametrize("task", ["lra-image", "lra-text"])
def test_both_phases_of_the_layer(task):
    layer = _layer(task)
    names = set(layer.state_dict())
    g = torch.Generator().manual_seed(1)
    X, dout = (torch.randn(B, L, 64, generator=g).to(DEV) for _ in range(2))
    mask = torch.ones(B, L, device=DEV)
    if task == "lra-text":
        mask[0, 200:] = 0
        mask[1, 77:] = 0
    layer.attn.emit_score_map = True
    mat = None
    for phase in ("dense", "sparse"):
        if phase == "sparse":
            mat = spion_amd.generate_pattern_conv_ff([layer.attn.score_map], _config(task))[0][0]
            layer.reconstruct_for_blocksparse(_config(task))
            assert set(layer.state_dict()) == names  # one table, under one name
        x = X.clone().requires_grad_()
        out, attn = layer(x, mask, mat)
        ps = dict(layer.named_parameters())
        got = dict(zip(["x", *ps], torch.autograd.grad(out, [x, *ps.values()], dout)))
        ref, p, x64, p64 = _written_out(layer, X, mask if task == "lra-text" else None, mat)
        want = dict(zip(["x", *p64], torch.autograd.grad(ref, [x64, *p64.values()], dout.double())))
        _near(phase, out, ref)
        for n in got:
            if n != "W_k.bias":  # softmax does not see it but for the keys off a pattern: a sum that cancels
                _near(f"{phase} {n}", got[n], want[n])
        if mat is None:
            _near("map", layer.attn.score_map, p.mean((0, 1)))
    served = _layer(task, inference=True)
    served.load_state_dict(layer.state_dict())
    assert spion_amd.attach_mask_sidecars([served], mat[None, None], _config(task)) == [None]
    with torch.no_grad():
        assert torch.equal(served(X, mask, mat)[0], layer(X, mask, mat)[0])


def test_a_step_of_the_layer_in_a_graph():
    """Forward and backward of norm, projections, core and output projection, recorded and replayed on new inputs, with eager steps and
    synchronizations between the replays."""
    layer = _layer("lra-text")
    mat = (torch.rand(L // BS, L // BS, generator=torch.Generator().manual_seed(0)) < 0.5).float().to(DEV)
    X, dout = (torch.randn(B, L, 64, device=DEV) for _ in range(2))
    X.requires_grad_()
    mask = torch.ones(B, L, device=DEV)
    leaves = [X, *layer.parameters()]

    def step():
        dense, sparse = layer(X, mask)[0], layer(X, mask, mat)[0]
        return [dense.detach(), sparse.detach(), *torch.autograd.grad(dense + sparse, leaves, dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for turn in range(4):
        with torch.no_grad():
            X.copy_(torch.randn(X.shape, generator=torch.Generator().manual_seed(turn)))
            mask.copy_((torch.arange(L)[None] < torch.tensor([[40 + 50 * turn], [256 - turn]])).float())
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(outs, eager):
            _near("replay", a, b.double())


def test_two_streams_at_once():
    """Calls on two streams, without a wait between them, have workspaces of their own: the bits of the calls one after the other."""
    g = torch.Generator().manual_seed(1)
    sets = []
    for n in (1000, 700):
        heads = [torch.randn(3, n, 4, 64, generator=g).to(DEV).transpose(1, 2) for _ in range(4)]
        sets.append([*heads, torch.randn(16, 4, generator=g).to(DEV)])
    buckets = spion_amd.relative_position_buckets(16, 64, DEV)

    def step(q, k, v, do, w):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, w)]
        out = spion_amd.relative_bias_attention(*leaves, buckets)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


@pytest.mark.parametrize("mat", [False, True])
def test_half_rows_under_autocast(mat):
    """Autocast leaves rows in fp16, which a layer without the norm takes as well: they are normalised in fp32."""
    layer = _layer("lra-listops")
    mask, pattern = torch.ones(B, L, device=DEV), torch.ones(L // BS, L // BS, device=DEV) if mat else None
    X = torch.randn(B, L, 64, generator=torch.Generator().manual_seed(5)).half().to(DEV)
    got = []
    for x in (X.detach().requires_grad_(), X.float().requires_grad_()):
        with torch.autocast("cuda", torch.float16):
            y, _ = layer(x, mask, pattern)
        got.append((y, *torch.autograd.grad(y.float().sum(), (x, layer.norm.weight))))
    (a, da, wa), (b, db, wb) = got
    assert torch.equal(a, b) and torch.equal(da, db.half()) and torch.equal(wa, wb)
