"""Attention with a learned relative position bias against its 64-bit statement (bias_oracle.py says what the bounds count)."""
import ctypes
import math

import pytest
import torch

import spion_amd
from spion_amd import _lib, workloads
from spion_amd import relative_bias as rb
from tests.bias_oracle import bias_reference, check

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(params=["node", "python"], autouse=True)
def both_nodes(request, monkeypatch):
    """Every test runs through the compiled node and through the Python function."""
    if request.param == "python":
        monkeypatch.setitem(_lib._cache, "node", None)


def _inputs(dtype, B, H, Lq, Lk, d, buckets=16, distance=40, seed=0, views=True):
    g = torch.Generator().manual_seed(seed)

    def heads(L):
        x = torch.randn(B, L, H, d, generator=g).to(dtype).to(DEV)
        return x.transpose(1, 2) if views else x.transpose(1, 2).contiguous()

    q, k, v, do = heads(Lq), heads(Lk), heads(Lk), heads(Lq)
    w = (0.8 * torch.randn(buckets, H, generator=g)).to(dtype).to(DEV)
    return q, k, v, w, spion_amd.relative_position_buckets(buckets, distance, DEV), do


def _lengths_mask(B, L, seed, kind):
    g = torch.Generator().manual_seed(seed)
    m = (torch.arange(L)[None] < torch.randint(1, L + 1, (B, 1), generator=g))
    if kind == "holes":
        m = m & (torch.rand(B, L, generator=g) < 0.6)
        m[0] = False  # a sample without any key
    return m.to(DEV)


def _run(q, k, v, w, buckets, do, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v, w)]
    out = spion_amd.relative_bias_attention(*leaves, buckets, **kw)
    return dict(zip(("out", "dq", "dk", "dv", "dw"), [out, *torch.autograd.grad(out, leaves, do)]))


def _compare(got, ref):
    for n, t in got.items():
        check(n, t, ref[n])


# lengths of one, tile edges (32), more queries than keys, few queries, pieces of a long row, chunks of 16384 on either side
SIZES = [(1, 1, 1, 1), (1, 2, 32, 32), (2, 1, 31, 33), (1, 3, 64, 65), (2, 2, 129, 127), (1, 2, 100, 7), (3, 1, 1, 300), (2, 2, 5, 4111)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(size, d, dtype):
    B, H, Lq, Lk = size
    q, k, v, w, buckets, do = _inputs(dtype, B, H, Lq, Lk, d, seed=Lk)
    off = Lk - Lq
    ref = bias_reference(q, k, v, w, buckets, offset=off, do=do)
    _compare(_run(q, k, v, w, buckets, do, offset=off), ref)
    with torch.no_grad():  # the form without a backward rounds the weights once
        check("out", spion_amd.relative_bias_attention(q, k, v, w, buckets, offset=off), ref["out"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Lq,Lk", [(40, 17000), (17000, 40)])
def test_long_sides(Lq, Lk, dtype):
    q, k, v, w, buckets, do = _inputs(dtype, 1, 2, Lq, Lk, 32, buckets=32, distance=1024)
    mask = _lengths_mask(1, Lk, 3, "lengths")
    _compare(_run(q, k, v, w, buckets, do, key_mask=mask, offset=100), bias_reference(q, k, v, w, buckets, mask, offset=100, do=do))


# calls that fill the machine take strips of 128 rows: ragged strips and stages, wavefronts without rows, few or many other rows,
# ranges of differences that tiles lie within, across and outside of
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,Lq,Lk,d,distance,offset", [(32, 16, 60, 60, 32, 40, 0), (64, 4, 200, 130, 64, 9, -50), (32, 4, 500, 700, 32, 100, 200),
                                                         (128, 4, 33, 1, 64, 40, 0), (16, 8, 512, 520, 64, 200, 0), (43, 12, 128, 96, 32, 4, 5),
                                                         (128, 4, 300, 310, 64, 30, 0), (64, 8, 520, 260, 32, 64, -100)])
@pytest.mark.parametrize("kind", [None, "lengths", "holes"])
def test_calls_that_fill_the_machine(B, H, Lq, Lk, d, distance, offset, kind, dtype):
    q, k, v, w, buckets, do = _inputs(dtype, B, H, Lq, Lk, d, 12, distance)
    mask = None if kind is None else _lengths_mask(B, Lk, 7, kind)
    if mask is not None:  # whatever lies in keys that are left out
        hidden = ~mask[:, None, :, None].expand_as(k)
        k = torch.where(hidden, torch.tensor(math.nan, dtype=dtype, device=DEV), k)
        v = torch.where(hidden, torch.tensor(math.inf, dtype=dtype, device=DEV), v)
    ref = bias_reference(q, k, v, w, buckets, mask, offset=offset, do=do)
    _compare(_run(q, k, v, w, buckets, do, key_mask=mask, offset=offset), ref)
    with torch.no_grad():
        out, mean = spion_amd.relative_bias_attention(q, k, v, w, buckets, key_mask=mask, offset=offset, score_map=True)
    check("out", out, ref["out"])
    p, bound = ref["p"]
    check("mean", mean, (p.mean((0, 1)), (bound + p * (B * H + 2) * 2.0 ** -24).mean((0, 1))))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("buckets,distance", [(4, 2), (8, 33), (32, 128), (64, 1024), (1024, 1000)])
@pytest.mark.parametrize("offset", [-700, 0, 23])
def test_buckets_and_offsets(buckets, distance, offset, dtype):
    q, k, v, w, bk, do = _inputs(dtype, 1, 2, 200, 333, 32, buckets, distance)
    _compare(_run(q, k, v, w, bk, do, offset=offset), bias_reference(q, k, v, w, bk, offset=offset, do=do))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["lengths", "holes"])
@pytest.mark.parametrize("mask_type", [torch.bool, torch.float32, torch.int64])
def test_key_masks(kind, mask_type, dtype):
    """Keys that are left out may hold anything; their gradients are zeros, and so is the output of a sample without keys."""
    q, k, v, w, buckets, do = _inputs(dtype, 3, 2, 150, 230, 64)
    mask = _lengths_mask(3, 230, 5, kind)
    hidden = ~mask[:, None, :, None].expand_as(k)
    k = torch.where(hidden, torch.tensor(math.nan, dtype=dtype, device=DEV), k)
    v = torch.where(hidden, torch.tensor(math.inf, dtype=dtype, device=DEV), v)
    got = _run(q, k, v, w, buckets, do, key_mask=mask.to(mask_type))
    _compare(got, bias_reference(q, k, v, w, buckets, mask, do=do))
    assert not bool(got["dk"][hidden].any()) and not bool(got["dv"][hidden].any())
    if kind == "holes":
        assert not bool(got["out"][0].any()) and not bool(got["dq"][0].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L,block", [(256, 32), (300, 64), (1000, 96), (33, 32)])
@pytest.mark.parametrize("masked", [False, True])
def test_block_patterns(L, block, masked, dtype):
    """Rows with no block at all, full rows and columns; keys off the pattern count with a logit of 0."""
    q, k, v, w, buckets, do = _inputs(dtype, 2, 2, L, L, 32, seed=L)
    nb = -(-L // block)
    mat = torch.from_numpy(workloads.band_random_block_mask(nb, 0, extra_frac=0.3, seed=L)).to(DEV)
    mat[-1] = 0.0
    mat[0] = 1.0
    mat[:, nb // 2] = 1.0 if nb > 2 else 0.0
    mask = _lengths_mask(2, L, 9, "holes") if masked else None
    got = _run(q, k, v, w, buckets, do, key_mask=mask, mat=mat, block_size=block)
    _compare(got, bias_reference(q, k, v, w, buckets, mask, mat, block, do=do))


# strips of 128 rows over patterns of 64 x 64 blocks and more, in pieces (B = 32: 384 strips) and whole
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,block,d", [(32, 700, 64, 32), (32, 700, 64, 64), (44, 650, 192, 32), (64, 300, 64, 64), (256, 300, 64, 64), (256, 290, 128, 32)])
@pytest.mark.parametrize("masked", [False, True])
def test_block_patterns_that_fill_the_machine(B, L, block, d, masked, dtype):
    q, k, v, w, buckets, do = _inputs(dtype, B, 2, L, L, d, seed=L)
    nb = -(-L // block)
    mat = torch.from_numpy(workloads.band_random_block_mask(nb, 0, extra_frac=0.3, seed=L)).to(DEV)
    mat[-1] = 0.0
    mat[0] = 1.0
    mat[:, nb // 2] = 1.0
    mask = _lengths_mask(B, L, 9, "holes") if masked else None
    if masked:
        k = torch.where(mask[:, None, :, None], k, torch.tensor(math.nan, dtype=dtype, device=DEV))
    got = _run(q, k, v, w, buckets, do, key_mask=mask, mat=mat, block_size=block)
    _compare(got, bias_reference(q, k, v, w, buckets, mask, mat, block, do=do))


# fewer strips than work-groups wanted: the other side in pieces
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,Lq,Lk,d", [(4, 4, 1000, 1100, 64), (2, 3, 1500, 3000, 32), (8, 8, 90, 2000, 64), (8, 8, 2000, 70, 32), (1, 2, 3000, 3100, 64)])
@pytest.mark.parametrize("kind", [None, "holes"])
def test_calls_in_pieces(B, H, Lq, Lk, d, kind, dtype):
    q, k, v, w, buckets, do = _inputs(dtype, B, H, Lq, Lk, d, 12, 100)
    mask = None if kind is None else _lengths_mask(B, Lk, 7, kind)
    _compare(_run(q, k, v, w, buckets, do, key_mask=mask, offset=7), bias_reference(q, k, v, w, buckets, mask, offset=7, do=do))


def test_an_empty_pattern():
    q, k, v, w, buckets, do = _inputs(torch.float32, 1, 1, 64, 64, 32)
    got = _run(q, k, v, w, buckets, do, mat=torch.zeros(2, 2, device=DEV), block_size=32)
    assert not any(bool(t.any()) for t in got.values())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_buckets_of_minus_infinity_are_a_window(dtype):
    """A table entry of -infinity takes its pairs out; rows that lose everything (the queries beyond the keys) give zeros."""
    q, k, v, w, buckets, do = _inputs(dtype, 1, 2, 200, 120, 32, buckets=8, distance=20)
    w[3] = w[7] = -math.inf
    ref = bias_reference(q, k, v, w, buckets, do=do)
    got = _run(q, k, v, w, buckets, do)
    _compare(got, ref)
    assert not bool(got["dw"][3].any()) and not bool(got["out"][:, :, 180:].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_logits(dtype):
    """Logits of some hundreds: the running maximum is raised in the middle of a row."""
    q, k, v, w, buckets, do = _inputs(dtype, 1, 1, 96, 400, 32)
    q = (q * torch.linspace(0.1, 30, 96, device=DEV)[:, None]).to(dtype)
    k = (k * torch.linspace(0.1, 3, 400, device=DEV)[:, None]).to(dtype)
    _compare(_run(q, k, v, w, buckets, do), bias_reference(q, k, v, w, buckets, do=do))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("how", ["contiguous", "fused", "unaligned", "shared", "transposed", "ones"])
def test_layouts(how, dtype):
    B, H, L, d = (1, 1, 1, 32) if how == "ones" else (2, 3, 70, 32)
    q, k, v, w, buckets, do = _inputs(dtype, B, H, L, L, d, views=how != "contiguous")
    if how == "fused":
        x = torch.stack([t.transpose(1, 2) for t in (q, k, v)], 2).contiguous()
        q, k, v = (x[:, :, i].transpose(1, 2) for i in range(3))
    elif how == "unaligned":
        q, k, v, do = (torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape) for t in (q, k, v, do))
    elif how == "shared":  # one K / V head for all query heads, one sample's for all samples
        k, v = k[:, :1].expand(B, H, L, d), v[:1].expand(B, H, L, d)
        do = do[:, :, :1].expand(B, H, L, d)
        w = w[:, :1].expand(-1, H)
    elif how == "transposed":
        q, k, v = (t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in (q, k, v))
    elif how == "ones":
        q = torch.as_strided(q.reshape(-1), (1, 1, 1, d), (3, 1, 5, 1))
    _compare(_run(q, k, v, w, buckets, do), bias_reference(q, k, v, w, buckets, do=do))


def test_gradients_of_shared_leaves():
    """One K / V head expanded to all heads, and K = V: autograd adds up what the heads and operands give."""
    q, k, v, w, buckets, do = _inputs(torch.float32, 2, 3, 70, 70, 32)
    kv = k[:, :1].contiguous().requires_grad_()
    out = spion_amd.relative_bias_attention(q, kv.expand(2, 3, 70, 32), kv.expand(2, 3, 70, 32), w, buckets)
    g, = torch.autograd.grad(out, kv, do)
    e = kv.detach().expand(2, 3, 70, 32)
    ref = bias_reference(q, e, e, w, buckets, do=do)
    check("dkv", g, tuple(sum(ref[n][i].sum(1, keepdim=True) for n in ("dk", "dv")) * (1 + i * 1e-6) for i in (0, 1)))


def test_gradient_against_differences():
    """The directional derivative of <out, do> along each operand, by central differences: curvature leaves h^2 / 6 of the third
    derivative (directions scaled so that logits move by some 1e-2: 1e-5 of the value), fp32 outputs leave
    2^-23 sqrt(n) |do| |out| / h."""
    q, k, v, w, buckets, do = _inputs(torch.float32, 2, 2, 70, 90, 32)
    got = _run(q, k, v, w, buckets, do)
    ops = [q, k, v, w]
    h = 1e-2
    with torch.no_grad():
        for i, n in enumerate(("dq", "dk", "dv", "dw")):
            g = torch.Generator().manual_seed(i)
            u = torch.randn(ops[i].shape, generator=g).to(DEV)
            f = []
            for sign in (1, -1):
                moved = list(ops)
                moved[i] = ops[i] + sign * h * u
                f.append(float((spion_amd.relative_bias_attention(*moved, buckets).double() * do).sum()))
            slope = (f[0] - f[1]) / (2 * h)
            want = float((got[n].double() * u).sum())
            size = float((got[n].double().abs() * u.abs()).sum())
            noise = 2.0 ** -23 * math.sqrt(do.numel()) * float(do.abs().max()) * float(got["out"].abs().max()) / h
            assert abs(slope - want) <= 1e-3 * size + 4 * noise, (n, slope, want, size, noise)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B", [3, 128])
def test_the_same_call_gives_the_same_bits(B, dtype):
    q, k, v, w, buckets, do = _inputs(dtype, B, 2, 300, 300, 64)
    mask = _lengths_mask(B, 300, 5, "holes")
    a, b = (_run(q, k, v, w, buckets, do, key_mask=mask) for _ in range(2))
    for n in a:
        assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,L,d,masked", [(3, 2, 100, 32, True), (2, 5, 65, 64, False), (1, 1, 1, 32, False), (5, 3, 257, 64, True)])
def test_mean_map(B, H, L, d, masked, dtype):
    q, k, v, w, buckets, _ = _inputs(dtype, B, H, L, L + 3, d)
    mask = _lengths_mask(B, L + 3, 11, "holes") if masked else None
    out, mean = spion_amd.relative_bias_attention(q, k, v, w, buckets, key_mask=mask, offset=3, score_map=True)
    ref = bias_reference(q, k, v, w, buckets, mask, offset=3)
    check("out", out, ref["out"])
    p, bound = ref["p"]
    n = B * H
    check("mean", mean, (p.mean((0, 1)), (bound + p * (n + 2) * 2.0 ** -24).mean((0, 1))))


def test_streams_and_replays():
    """A step recorded on a side stream, replayed on new inputs, masks and patterns with eager work in between: every replay has the
    bits of the eager step.  Two recorded steps with workspaces of their own do not disturb each other."""
    cases = []
    for L, block in ((200, 0), (192, 32)):
        q, k, v, w, buckets, do = _inputs(torch.bfloat16, 2, 2, L, L, 32)
        mask = _lengths_mask(2, L, 5, "holes")
        mat = torch.ones(L // block, L // block, device=DEV) if block else None
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, w)]
        kw = dict(key_mask=mask, mat=mat, block_size=block or None)

        def step(leaves=leaves, buckets=buckets, do=do, kw=kw):
            out = spion_amd.relative_bias_attention(*leaves, buckets, **kw)
            return [out.detach(), *torch.autograd.grad(out, leaves, do)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        cases.append((leaves, mask, mat, step, graph, outs))
    for turn in range(4):
        for leaves, mask, mat, *_ in cases:
            with torch.no_grad():
                for i, t in enumerate(leaves):
                    t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(10 * turn + i)))
                mask.copy_(_lengths_mask(*mask.shape, turn, "holes"))
                if mat is not None:
                    mat.copy_(torch.rand(mat.shape, generator=torch.Generator().manual_seed(turn)) < 0.5)
        for case in cases:
            case[4].replay()
        torch.cuda.synchronize()
        for _, _, _, step, _, outs in cases:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                eager = step()
            torch.cuda.current_stream().wait_stream(side)
            for a, b in zip(outs, eager):
                assert torch.equal(a, b), turn


@pytest.mark.parametrize("L", [0, 40])
def test_nothing_to_attend_to(L):
    q, k, v, w, buckets, do = _inputs(torch.float32, 2, 2, 40 - L, L, 32)
    got = _run(q, k, v, w, buckets, do)
    assert all(got[n].shape == t.shape and not bool(got[n].any()) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v), ("dw", w)))


def test_a_second_derivative_is_refused():
    q, k, v, w, buckets, do = _inputs(torch.float32, 1, 1, 40, 40, 32)
    q = q.detach().requires_grad_()
    out = spion_amd.relative_bias_attention(q, k, v, w, buckets)
    g, = torch.autograd.grad(out.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_a_mask_changed_before_the_backward_is_refused():
    q, k, v, w, buckets, do = _inputs(torch.float32, 1, 1, 40, 40, 32)
    mask = torch.ones(1, 40, device=DEV)
    q = q.detach().requires_grad_()
    out = spion_amd.relative_bias_attention(q, k, v, w, buckets, key_mask=mask)
    mask.zero_()
    with pytest.raises(RuntimeError):
        out.backward(do)


def test_module_from_the_dense_phase_to_the_sparse_one():
    """The dense phase leaves the score map, discovery makes the block mask of it, the sparse phase runs on the mask with the same
    table: forward and gradients of both against the 64-bit statement."""
    B, H, L, d, bs = 2, 2, 256, 32, 32
    cfg = dict(head_dim=d, num_head=H, max_seq_len=L, batch_size=B, block_size=bs, relative_buckets=16, relative_max_distance=64,
               threshold=0.9, num_layers=1)
    mod = spion_amd.RelativeBiasAttention(cfg, key_mask=True).to(DEV)
    with torch.no_grad():
        mod.weight.copy_(torch.randn(mod.weight.shape, generator=torch.Generator().manual_seed(1)))
    q, k, v, _, _, do = _inputs(torch.float32, B, H, L, L, d)
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    mask = _lengths_mask(B, L, 2, "lengths").float()
    mod.emit_score_map = True
    for mat in (None, "discover"):
        if mat is not None:
            mat = spion_amd.generate_pattern_conv_ff([mod.score_map], cfg)[0][0]
            assert mat.shape == (L // bs, L // bs) and 0 < float(mat.mean()) < 1
        out, attn = mod(q, k, v, mask, mat)
        assert attn == 0
        got = [out, *torch.autograd.grad(out, (q, k, v, mod.weight), do)]
        ref = bias_reference(q, k, v, mod.weight, mod.buckets, mask, mat, bs, do=do)
        for n, t in zip(("out", "dq", "dk", "dv", "dw"), got):
            check(n, t, ref[n])
        if mat is None:
            p, bound = ref["p"]
            check("map", mod.score_map, (p.mean((0, 1)), (bound + p * 8 * 2.0 ** -24).mean((0, 1))))


def test_module_with_bf16_heads_trains_an_fp32_table():
    cfg = dict(head_dim=32, num_head=2, max_seq_len=96, batch_size=2, block_size=32)
    mod = spion_amd.RelativeBiasAttention(cfg).to(DEV)
    q, k, v, _, _, do = _inputs(torch.bfloat16, 2, 2, 96, 96, 32)
    out, _ = mod(q, k, v, None)
    out.backward(do)
    ref = bias_reference(q, k, v, mod.weight.to(torch.bfloat16), mod.buckets, do=do)
    assert mod.weight.grad.dtype == torch.float32
    check("dw", mod.weight.grad, ref["dw"])


def test_c_entry_points_keep_to_their_buffers():
    """Through the C entry points, with rows behind the last query and key marked: they stay as they were."""
    B, H, L, d = 1, 2, 45, 32
    q, k, v, w, buckets, do = _inputs(torch.float32, B, H, L, L, d, views=False)
    ref = bias_reference(q, k, v, w, buckets, do=do)
    lib = rb._lib_typed()
    outs = {n: torch.full((B, H, L + 9, d), 7.0, device=DEV) for n in ("Out", "dQ", "dK", "dV")}
    lse, dw = torch.full((B * H * L + 8,), 7.0, device=DEV), torch.full((w.numel() + 8,), 7.0, device=DEV)
    call = rb._call_of(q, k, w, buckets, None, None, 0, 0)
    call.Q, call.K, call.V, call.dO = (rb._heads(t) for t in (q, k, v, do))
    for n, t in outs.items():
        setattr(call, n, rb._heads(t))
    call.Lse, call.dweight = lse.data_ptr(), dw.data_ptr()
    n = lib.spion_bias_workspace(ctypes.addressof(call), 1)
    ws = torch.full((n + 8,), 7.0, device=DEV)
    call.workspace, call.workspace_floats = ws.data_ptr(), n
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.spion_bias_attention_forward(ctypes.addressof(call), stream) == 0
    assert lib.spion_bias_attention_backward(ctypes.addressof(call), stream) == 0
    for name, t in outs.items():
        assert bool((t[:, :, L:] == 7.0).all()), name
        check(name, t[:, :, :L], ref[{"Out": "out", "dQ": "dq", "dK": "dk", "dV": "dv"}[name]])
    assert bool((lse[B * H * L:] == 7.0).all()) and bool((dw[w.numel():] == 7.0).all()) and bool((ws[n:] == 7.0).all())
    check("dw", dw[: w.numel()].view(w.shape), ref["dw"])
    call.workspace_floats = n - 1
    assert lib.spion_bias_attention_backward(ctypes.addressof(call), stream) != 0
    with pytest.raises(_lib.SpionLibraryError, match="workspace"):
        _lib.check_error()


# the widest range of differences: the bias, the tiles of heads of 64 and the histograms together take nearly all of a CU's LDS
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,block", [(1, 1100, 0), (1, 1100, 32), (33, 1100, 64), (44, 700, 0)])
def test_the_widest_range(B, L, block, dtype):
    q, k, v, w, buckets, do = _inputs(dtype, B, 2, L, L, 64, 64, 1024)
    mat = None
    if block:
        nb = -(-L // block)
        mat = torch.from_numpy(workloads.band_random_block_mask(nb, 1, extra_frac=0.2, seed=L)).to(DEV)
    kw = dict(mat=mat, block_size=block) if block else {}
    _compare(_run(q, k, v, w, buckets, do, **kw), bias_reference(q, k, v, w, buckets, mat=mat, block=block, do=do))


# sides of more than two tiles that leave fewer than a work-group for each CU, of either type: strips of 32 and of 128 next to each other
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,Lq,Lk,d", [(8, 8, 320, 320, 64), (8, 8, 320, 320, 32), (4, 4, 1500, 1030, 32), (6, 8, 1030, 1000, 64), (1, 4, 2100, 4200, 64)])
def test_between_strips_of_32_and_of_128(B, H, Lq, Lk, d, dtype):
    q, k, v, w, buckets, do = _inputs(dtype, B, H, Lq, Lk, d)
    mask = _lengths_mask(B, Lk, 4, "lengths")
    _compare(_run(q, k, v, w, buckets, do, key_mask=mask, offset=-3), bias_reference(q, k, v, w, buckets, mask, offset=-3, do=do))


# the column pass in strips of 64 rows, two wavefronts to the same rows: strips, halves and stages that end anywhere, keys left out
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,Lq,Lk,offset", [(64, 4, 100, 127, 0), (64, 4, 31, 97, 5), (32, 4, 300, 161, -70), (40, 8, 64, 66, 0)])
@pytest.mark.parametrize("kind", [None, "holes"])
def test_columns_in_strips_of_64(B, H, Lq, Lk, offset, kind, dtype):
    q, k, v, w, buckets, do = _inputs(dtype, B, H, Lq, Lk, 32, 16, 90)
    mask = None if kind is None else _lengths_mask(B, Lk, 8, kind)
    _compare(_run(q, k, v, w, buckets, do, key_mask=mask, offset=offset), bias_reference(q, k, v, w, buckets, mask, offset=offset, do=do))


# maps that no division into ranges makes: buckets that come back, neighbours that all differ, one bucket for everything
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L", [(2, 150), (128, 150)])
@pytest.mark.parametrize("how", ["random", "cyclic", "pairs", "one"])
def test_any_map_of_buckets(how, B, L, dtype):
    q, k, v, w, _, do = _inputs(dtype, B, 4, L, L, 32, 12)
    n = torch.arange(2 * 75 + 1)
    buckets = {"random": torch.randint(0, 12, n.shape, generator=torch.Generator().manual_seed(0)), "cyclic": n % 12,
               "pairs": (n // 2) % 5, "one": torch.full_like(n, 7)}[how].to(torch.int32).to(DEV)
    got = _run(q, k, v, w, buckets, do)
    _compare(got, bias_reference(q, k, v, w, buckets, do=do))
    again = _run(q, k, v, w, buckets, do)
    assert all(torch.equal(got[x], again[x]) for x in got)


def test_far_buckets_of_a_pattern_have_no_bias():
    """fp32, rows whose probabilities lie on the pattern by half: the table's gradient adds up P (dP - D) over 3 x 1500 rows a head, where
    an error of one sign in dP grows with their number n and roundings with its root.  A row's dP and D are off by a few
    2^-24 of |dO| |v| ~ d, of which its sum keeps at most a quarter (S (1 - S)): 4 * 2^-24 * 32 / 4 * sqrt(n) / 4 for rounding
    (n = 4500: 3.2e-5 where every row has the same buckets), against 2.8e-8 / 4 * n = 3.1e-5 an error of 2^-25 in every dP leaves.
    Their mean over 24 tables tells them apart: rounding leaves 3.2e-5 / sqrt(24) = 6.5e-6, so 1e-5 is between them."""
    total = 0.0
    for seed in range(6):
        q, k, v, w, buckets, do = _inputs(torch.float32, 3, 4, 1500, 1500, 32, 8, 16, seed=seed)
        mat = (torch.rand(47, 47, generator=torch.Generator().manual_seed(seed)) < 0.5).float().to(DEV)
        got = _run(q, k, v, w, buckets, do, mat=mat, block_size=32)["dw"].double()
        ref = bias_reference(q, k, v, w, buckets, mat=mat, block=32, do=do)["dw"][0]
        total += float((got - ref)[3].sum())  # everything far behind
    assert abs(total / 24) <= 1e-5, total / 24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("grad", [False, True])
def test_a_traced_call_computes(grad, dtype):
    """A traced call gives on other inputs what the function gives, with gradients and with the mean map."""
    first, other = (_inputs(dtype, 2, 2, 70, 70, 32, seed=s) for s in (1, 2))
    buckets, mask = first[4], _lengths_mask(2, 70, 3, "lengths")
    call = lambda *x: spion_amd.relative_bias_attention(*x, buckets, key_mask=mask, score_map=not grad)  # noqa: E731
    leaves = [t.detach().requires_grad_(grad) for t in other[:4]]
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(call, tuple(t.detach().requires_grad_(grad) for t in first[:4]), check_trace=False)
        got, want = traced(*leaves), call(*leaves)
    if grad:
        got, want = ([y, *torch.autograd.grad(y, leaves, other[5])] for y in (got, want))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_calls_go_by_their_own_status():
    """A call that the library refuses raises; what another call has left in the process-wide error slot neither fails a call nor is
    taken by it."""
    lib = _lib.core()
    q, k, v, w, buckets, do = _inputs(torch.float32, 1, 2, 40, 40, 32)
    lib.spion_set_stream(None, None)  # a failure: no handle
    try:
        got = _run(q, k, v, w, buckets, do)
        with pytest.raises(_lib.SpionLibraryError, match="32767 buckets"):
            _run(q, k, v, torch.zeros(32768, 2, device=DEV), buckets, do)
        assert lib.spion_last_error().startswith(b"spion_set_stream")
    finally:
        lib.spion_clear_error()
    _compare(got, bias_reference(q, k, v, w, buckets, do=do))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("how", ["interleaved", "shared"])
def test_more_heads_than_rows_of_them_may_lie_apart(how, dtype):
    """Heads next to each other in rows of more than 2^24 bytes: the operands are read from copies, and outputs and gradients lie
    as the copies do.  One head shared by all is read in place, and its output would have such rows."""
    H = (1 << 24) // (32 * (4 if dtype == torch.float32 else 2)) + 1
    q, k, v, w, buckets, do = _inputs(dtype, 1, H, 2, 2, 32)
    if how == "shared":
        q, k, v = (t[:, :1].expand(1, H, 2, 32) for t in (q, k, v))
    _compare(_run(q, k, v, w, buckets, do), bias_reference(q, k, v, w, buckets, do=do))


# fewer strips of 128 rows than work-groups wanted, over a pattern: pieces of its stages in both passes
@pytest.mark.parametrize("H,L,block,d", [(9, 2000, 128, 32), (12, 1000, 64, 64), (12, 1000, 128, 64)])
@pytest.mark.parametrize("masked", [False, True])
def test_block_patterns_in_pieces(H, L, block, d, masked):
    q, k, v, w, buckets, do = _inputs(torch.float32, 1, H, L, L, d, seed=L)
    nb = -(-L // block)
    mat = torch.from_numpy(workloads.band_random_block_mask(nb, 0, extra_frac=0.3, seed=L)).to(DEV)
    mat[-1] = 0.0
    mat[0] = 1.0
    mask = _lengths_mask(1, L, 9, "lengths") if masked else None
    call = rb._call_of(q, k, w, buckets, mask, mat, block, 0)
    lib = rb._lib_typed()
    assert lib.spion_bias_workspace(ctypes.addressof(call), 0) >= 2 * H * -(-L // 32) * 32 * d  # sums of two pieces at least
    assert lib.spion_bias_workspace(ctypes.addressof(call), 1) >= 2 * H * -(-L // 32) * 64 * d
    got = _run(q, k, v, w, buckets, do, key_mask=mask, mat=mat, block_size=block)
    _compare(got, bias_reference(q, k, v, w, buckets, mask, mat, block, do=do))


# every walk: strips of 32, whole and in pieces, of 128, of 64 over a pattern; the NaN in a key that takes part, in one head of one sample
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,Lq,Lk,d,block", [(2, 2, 70, 90, 32, 0), (1, 2, 3, 3000, 64, 0), (64, 4, 200, 200, 64, 0), (2, 2, 160, 160, 32, 32),
                                               (40, 2, 300, 300, 64, 64)])
def test_a_nan_is_not_hidden(B, H, Lq, Lk, d, block, dtype):
    """A NaN among a row's logits makes all of its probabilities NaN: the output, the map and dV show it, for the rows (with a pattern:
    of the blocks) that see the key, and nowhere else."""
    q, k, v, w, buckets, do = _inputs(dtype, B, H, Lq, Lk, d)
    mask = torch.ones(B, Lk, dtype=torch.bool, device=DEV)
    mask[:, -5:] = False
    k[1 if B > 1 else 0, 1, 17, 3] = math.nan
    mat = None
    rows, keys = torch.ones(Lq, dtype=torch.bool, device=DEV), mask[0]
    if block:
        nb = -(-Lk // block)
        mat = torch.eye(nb, device=DEV)
        mat[2, 0] = mat[2, 1] = 1.0
        at = torch.arange(Lk, device=DEV) // block
        rows = mat[at, 0] != 0
        keys = keys & (at <= 2)  # blocks that rows of the first block or of the third see
    kw = dict(key_mask=mask, mat=mat, block_size=block) if block else dict(key_mask=mask)
    got = _run(q, k, v, w, buckets, do, **kw)
    for n, t, seen in (("out", got["out"], rows), ("dq", got["dq"], rows), ("dv", got["dv"], keys)):
        bad = torch.isnan(t)
        hit = bad[1 if B > 1 else 0, 1]
        assert bool(hit[seen].all()) and not bool(hit[~seen].any()), n
        assert int(bad.sum()) == int(hit.sum()), n
    if not block:
        with torch.no_grad():
            mean = spion_amd.relative_bias_attention(q, k, v, w, buckets, score_map=True, **kw)[1]
        assert bool(torch.isnan(mean[:, mask[0]]).all()) and not bool(mean[:, ~mask[0]].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_buckets_of_the_lowest_value_are_left_out_too(dtype):
    """The type's lowest value times log2(e) is -infinity: the same bits as with -infinity, rows that lose everything among them."""
    q, k, v, w, buckets, do = _inputs(dtype, 1, 2, 200, 120, 32, buckets=8, distance=20)
    got = []
    for x in (-math.inf, torch.finfo(dtype).min):
        w[3] = w[7] = x
        got.append(_run(q, k, v, w, buckets, do))
    assert all(torch.equal(got[0][n], got[1][n]) for n in got[0])


def test_refused_calls_in_another_thread(monkeypatch):
    """One thread's calls are all refused by the library while another's steps run: each raises for its own, and no step is disturbed."""
    import threading

    monkeypatch.setenv("SPION_QUIET", "1")
    q, k, v, w, buckets, do = _inputs(torch.float32, 1, 2, 40, 40, 32)
    many = torch.zeros(32768, 2, device=DEV)
    first = _run(q, k, v, w, buckets, do)
    torch.cuda.synchronize()
    refused, began, stop = [0, 0], threading.Event(), threading.Event()

    def refuse():
        while not stop.is_set():
            try:
                spion_amd.relative_bias_attention(q, k, v, many, buckets)
            except _lib.SpionLibraryError as e:
                refused["32767 buckets" not in str(e)] += 1
            began.set()

    other = threading.Thread(target=refuse)
    other.start()
    try:
        assert began.wait(60)
        steps = [_run(q, k, v, w, buckets, do) for _ in range(200)]
    finally:
        stop.set()
        other.join()
    assert refused[0] > 0 and refused[1] == 0
    assert _lib.core().spion_error_pending() == 0
    for got in steps:
        assert all(torch.equal(got[n], first[n]) for n in first)
