"""Relative position buckets and what the bias operators refuse, without a GPU."""
import ctypes
import math

import pytest
import torch

import spion_amd
from spion_amd import _lib
from spion_amd import relative_bias as rb


@pytest.fixture(params=["node", "python"], autouse=True)
def both_nodes(request, monkeypatch):
    """Every test runs through the compiled node and through the Python function."""
    if request.param == "python":
        monkeypatch.setitem(_lib._cache, "node", None)


@pytest.mark.parametrize("buckets,distance", [(4, 2), (8, 27), (32, 128), (64, 1000), (256, 100)])
def test_buckets_by_their_definition(buckets, distance):
    got = spion_amd.relative_position_buckets(buckets, distance)
    assert got.dtype == torch.int32 and got.shape == (2 * distance + 1,)
    half, exact = buckets // 2, buckets // 4
    for diff in range(-distance, distance + 1):
        n = abs(diff)
        k = n
        if n >= exact:
            x = math.log(n / exact) / math.log(distance / exact) * (half - exact)
            if abs(x - round(x)) < 1e-9:
                x = round(x)  # a border: the logarithm may be off either way
            k = min(half - 1, exact + int(x))
        assert int(got[diff + distance]) == (half if diff > 0 else 0) + k, diff


@pytest.mark.parametrize("buckets,distance", [(0, 10), (6, 10), (32, 8), (32, 1025), (-4, 10)])
def test_buckets_refuse(buckets, distance):
    with pytest.raises(ValueError):
        spion_amd.relative_position_buckets(buckets, distance)


def _ok():
    x = torch.zeros(2, 3, 40, 32)
    return dict(query=x, key=x, value=x, weight=torch.zeros(8, 3), buckets=spion_amd.relative_position_buckets(8, 20))


@pytest.mark.parametrize("change,error", [
    (dict(query=torch.zeros(3, 40, 32)), ValueError),
    (dict(key=torch.zeros(2, 2, 40, 32)), ValueError),
    (dict(value=torch.zeros(2, 3, 41, 32)), ValueError),
    (dict(query=torch.zeros(2, 3, 40, 32).half()), TypeError),
    (dict(key=torch.zeros(2, 3, 40, 32).bfloat16()), (TypeError, RuntimeError)),
    (dict(weight=torch.zeros(8, 2)), ValueError),
    (dict(weight=torch.zeros(0, 3)), ValueError),
    (dict(buckets=torch.zeros(10, dtype=torch.int32)), ValueError),
    (dict(buckets=torch.zeros(2051, dtype=torch.int32)), ValueError),
    (dict(buckets=torch.zeros(41, dtype=torch.int64)), TypeError),
    (dict(key_mask=torch.ones(2, 41)), ValueError),
    (dict(offset=1 << 30), ValueError),
    (dict(mat=torch.ones(2, 2)), ValueError),
    (dict(mat=torch.ones(2, 2), block_size=16), ValueError),
    (dict(mat=torch.ones(3, 3), block_size=32), ValueError),
    (dict(mat=torch.ones(2, 2), block_size=32, offset=1), ValueError),
    (dict(mat=torch.ones(2, 2), block_size=32, score_map=True), ValueError),
    (dict(), RuntimeError),  # everything in order, but not on a GPU
])
def test_operator_refuses(change, error):
    with pytest.raises(error):
        spion_amd.relative_bias_attention(**{**_ok(), **change})


def test_head_dimensions_other_than_32_and_64_are_refused():
    x = torch.zeros(1, 1, 8, 48)
    with pytest.raises(ValueError, match="head dimension"):
        spion_amd.relative_bias_attention(x, x, x, torch.zeros(8, 1), spion_amd.relative_position_buckets(8, 20))


def test_module_refuses_heads_of_another_shape():
    mod = spion_amd.RelativeBiasAttention(dict(head_dim=32, num_head=2))
    assert mod.weight.shape == (32, 2) and list(mod.state_dict()) == ["weight"]
    with pytest.raises(ValueError, match="2 heads of 32"):
        mod(*[torch.zeros(1, 3, 8, 32)] * 3, None)


def test_c_entry_points_refuse_before_any_gpu_work():
    lib = rb._lib_typed()
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16  # never read: every call below is refused

    def call(**kw):
        c = rb._Call(weight=at, dweight=at, buckets=at, Lse=at, workspace=at, workspace_floats=1 << 40, batch=1, heads=1, q_len=64,
                     k_len=64, head_dim=32, num_buckets=8, max_distance=20)
        for n in ("Q", "K", "V", "Out", "dO", "dQ", "dK", "dV"):
            setattr(c, n, rb._Heads(at, 2048, 2048, 32))
        for n, x in kw.items():
            setattr(c, n, x)
        return c

    bad = [dict(batch=0), dict(q_len=0), dict(k_len=-1), dict(head_dim=48), dict(num_buckets=0), dict(num_buckets=32768), dict(max_distance=0),
           dict(max_distance=1025), dict(offset=1 << 30), dict(q_len=(1 << 29) + 1), dict(batch=1 << 20, heads=1 << 10),
           dict(mat=at, block_size=16), dict(mat=at, block_size=32, offset=1), dict(mat=at, block_size=32, k_len=65),
           dict(key_mask=at, mask_bytes=2), dict(weight=None), dict(Lse=None), dict(buckets=None),
           dict(Q=rb._Heads(None, 0, 0, 32)), dict(K=rb._Heads(at + 4, 0, 0, 32)), dict(V=rb._Heads(at, 2, 0, 32)),
           dict(Out=rb._Heads(at, 0, -32, 32)),
           dict(Q=rb._Heads(at, 0, 0, 1 << 23)), dict(V=rb._Heads(at, 0, 0, 1 << 20), k_len=4096)]
    for kw in bad + [dict(Out=rb._Heads(at, 0, 0, 0)), dict(Mean=at, mat=at, block_size=32)]:
        assert lib.spion_bias_attention_forward(ctypes.addressof(call(**kw)), None) != 0, kw
        with pytest.raises(_lib.SpionLibraryError, match="spion_bias_attention_forward"):
            _lib.check_error()
    for kw in bad + [dict(dQ=rb._Heads(at, 0, 0, 28)), dict(dO=rb._Heads(None, 0, 0, 32)), dict(workspace=None), dict(dweight=None),
                     dict(workspace_floats=63), dict(workspace=at + 4)]:
        assert lib.spion_bias_attention_backward(ctypes.addressof(call(**kw)), None) != 0, kw
        with pytest.raises(_lib.SpionLibraryError, match="spion_bias_attention_backward"):
            _lib.check_error()
    assert lib.spion_bias_attention_forward(None, None) != 0 and lib.spion_bias_workspace(None, 1) == -1
    assert lib.spion_bias_workspace(ctypes.addressof(call(head_dim=16)), 0) == -1
    _lib.core().spion_clear_error()
    assert lib.spion_bias_workspace(ctypes.addressof(call()), 1) == 64 + 2 * 8


def _huge(*shape):
    return torch.zeros(()).expand(*shape)  # no memory behind it


@pytest.mark.parametrize("change", [
    dict(mat=torch.ones(1, 1), block_size=(1 << 32) + 32),  # 32 in 32 bits, and the pattern would be read past its end
    dict(key=_huge(2, 3, (1 << 32) + 40, 32), value=_huge(2, 3, (1 << 32) + 40, 32)),
    dict(query=_huge(2, 3, (1 << 32) + 40, 32)),
    dict(weight=_huge((1 << 32) + 8, 3)),
])
def test_sizes_past_32_bits_are_refused(change):
    with pytest.raises(ValueError):
        spion_amd.relative_bias_attention(**{**_ok(), **change})


def _c_call(**sizes):
    c = rb._Call(batch=1, heads=1, q_len=40, k_len=40, head_dim=32, num_buckets=8, max_distance=20)
    for n, x in sizes.items():
        setattr(c, n, x)
    return rb._lib_typed().spion_bias_workspace(ctypes.addressof(c), 1)


@pytest.mark.parametrize("sizes", [dict(mat=16, block_size=(1 << 31) - 32), dict(batch=1 << 20, q_len=1000, k_len=1000),
                                   dict(num_buckets=32767, heads=1 << 10)])
def test_c_entry_points_refuse_what_no_launch_holds(sizes):
    assert _c_call() > 0
    assert _c_call(**sizes) == -1
    with pytest.raises(_lib.SpionLibraryError, match="spion_bias_workspace"):
        _lib.check_error()


def test_strides_past_64_bits_of_bytes_are_refused():
    """A row stride whose bytes come out as 0 in 64 bits."""
    lib = rb._lib_typed()
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16  # never read
    c = rb._Call(weight=at, buckets=at, Lse=at, batch=1, heads=1, q_len=1, k_len=1, head_dim=32, num_buckets=8, max_distance=20)
    for n in ("K", "V", "Out"):
        setattr(c, n, rb._Heads(at, 32, 32, 32))
    c.Q = rb._Heads(at, 32, 32, 1 << 62)
    assert lib.spion_bias_attention_forward(ctypes.addressof(c), None) != 0
    with pytest.raises(_lib.SpionLibraryError, match="Q: rows up to"):
        _lib.check_error()


def _aligned(*shape):
    x = torch.zeros(math.prod(shape) + 4)
    return x[(-x.data_ptr() % 16) // 4:][: math.prod(shape)].view(shape)


def test_heads_are_copied_only_where_they_have_to_be(monkeypatch):
    views = _aligned(2, 40, 3, 32).transpose(1, 2), _aligned(2, 3, 40, 32), _aligned(2, 40, 3, 3, 32)[:, :, 1].transpose(1, 2)
    off = _aligned(2 * 3 * 40 * 32 + 1)[1:].view(2, 3, 40, 32)  # contiguous, 4 bytes off
    turned = _aligned(2, 3, 32, 40).transpose(2, 3)
    copies = []
    contiguous, clone = torch.Tensor.contiguous, torch.Tensor.clone
    monkeypatch.setattr(torch.Tensor, "contiguous", lambda t, *a, **k: (copies.append("contiguous"), contiguous(t, *a, **k))[1])
    monkeypatch.setattr(torch.Tensor, "clone", lambda t, *a, **k: (copies.append("clone"), clone(t, *a, **k))[1])
    for t in views:
        assert rb._readable(t) is t
    assert copies == []
    for t, how in ((off, ["contiguous", "clone"]), (turned, ["contiguous"])):
        copies.clear()
        got = rb._readable(t)
        assert copies == how and rb._fits(got) and torch.equal(got, t)


@pytest.mark.parametrize("dtype,H,L,d,interleaved", [
    (torch.float32, 64, (1 << 17) - 1, 64, True), (torch.float32, 64, 1 << 17, 64, False),  # 2^29 elements to a head's rows
    (torch.float32, 1 << 17, 2, 32, True), (torch.float32, (1 << 17) + 1, 2, 32, False),  # 2^24 bytes from row to row
    (torch.bfloat16, 1 << 18, 2, 32, True), (torch.bfloat16, (1 << 18) + 1, 2, 32, False)])
def test_outputs_lie_as_the_kernels_take_them(dtype, H, L, d, interleaved):
    """Outputs follow the operands' memory order, but not where the library would refuse it: the operands are copied then."""
    shared = torch.empty(1, 1, L, d, dtype=dtype, device="meta").expand(1, H, L, d)  # fits, its heads' stride is 0
    for t in (torch.empty(1, L, H, d, dtype=dtype, device="meta").transpose(1, 2), shared):
        out = rb._empty_like_heads(t)
        assert out.shape == t.shape and out.stride()[1:] == ((d, H * d, 1) if interleaved else (L * d, d, 1))
        call = rb._Call(weight=16, buckets=16, Lse=16, batch=1, heads=H, q_len=L, k_len=L, head_dim=d, bf16=int(dtype == torch.bfloat16),
                        num_buckets=8, max_distance=20, Mean=16, mat=16, block_size=1 << 29)
        for n in ("Q", "K", "V"):
            setattr(call, n, rb._Heads(16, 0, 0, d))
        call.Out = rb._Heads(16, *out.stride()[:3])
        # refused for the map with a pattern, which is looked at after the heads: these are in order
        assert rb._lib_typed().spion_bias_attention_forward(ctypes.addressof(call), None) != 0
        with pytest.raises(_lib.SpionLibraryError, match="mean map"):
            _lib.check_error()


def _floats(nb, Lq, Lk, d, backward, **more):
    c = rb._Call(batch=nb, heads=1, q_len=Lq, k_len=Lk, head_dim=d, num_buckets=32, max_distance=128, **more)
    return rb._lib_typed().spion_bias_workspace(ctypes.addressof(c), backward)


@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize("nb,L", [(257, 2048), (130, 4096), (1030, 4096), (131000, 4096)])
def test_calls_that_fill_the_machine_many_times_over_are_not_cut(nb, L, d):
    """(A machine of 256 CUs.)  Only D and the table's gradient by strips of 128 rows are left in the workspace; the pieces of 257 heads
    of 2048 took 1.1 GB forward and 2.2 GB backward, and of 131000 heads of 4096 more work-groups than a launch holds."""
    assert _floats(nb, L, L, d, 0) == 0
    assert _floats(nb, L, L, d, 1) == nb * L + nb * (L // 128) * 32


@pytest.mark.parametrize("d", [32, 64])
def test_pieces_leave_a_bounded_workspace(d):
    """Eight work-groups of 128 rows for each of 256 CUs at most, whatever the sizes; strips of 32 rows in the forward come in pieces of
    fewer."""
    groups, slot = 8 * 256, 4 * (32 * d + 96)
    for nb in (1, 3, 12, 40, 100, 128, 200, 257, 300, 512, 700, 1000):
        for Lq in (65, 200, 700, 1030, 2048, 5000):
            for Lk in (90, Lq, 3000, 40000):
                for more in ({},) if Lq != Lk else ({}, dict(mat=16, block_size=64), dict(mat=16, block_size=32)):
                    assert _floats(nb, Lq, Lk, d, 0, **more) <= groups * slot, (nb, Lq, Lk)
                    base = nb * Lq + 3 + 32 * max(groups, nb * -(-Lk // 32)) + 3
                    assert _floats(nb, Lq, Lk, d, 1, **more) <= base + groups * max(slot, 4 * 64 * d), (nb, Lq, Lk)
