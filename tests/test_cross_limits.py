"""The sizes that a call of the attention to an encoder's states may have, without a GPU."""
import ctypes

import pytest
import torch

from spion_amd import _lib
from spion_amd import attention_cross as ac


def _workspace(backward, **sizes):
    c = ac._Call(**{**dict(heads=2, key_heads=2, head_dim=64, bf16=1), **sizes})
    return ac._lib_typed().spion_cross_workspace(ctypes.addressof(c), backward)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("sizes", [
    dict(batch=16384, heads=8, key_heads=8, q_len=1, k_len=4096),  # one token of many samples over states that they share
    dict(batch=1 << 17, q_len=33, k_len=2049), dict(batch=1 << 17, q_len=2049, k_len=33), dict(batch=1 << 17, q_len=8064, k_len=8064)])
def test_calls_of_more_strips_of_32_than_a_launch_holds(sizes, d):
    for bf16 in (0, 1):
        for backward in (0, 1):
            assert _workspace(backward, bf16=bf16, head_dim=d, **sizes) >= 0, _lib.core().spion_take_call_error()


@pytest.mark.parametrize("sizes", [dict(q_len=1, k_len=8065), dict(q_len=8065, k_len=1), dict(heads=4, q_len=4033, k_len=1)])
def test_calls_of_as_many_strips_of_128_are_refused(sizes):
    """2^17 samples of two heads of keys, 64 strips each: 2^24."""
    for backward in (0, 1):
        assert _workspace(backward, batch=1 << 17, **sizes) == -1
        with pytest.raises(_lib.SpionLibraryError, match="strips"):
            _lib.check_error()


@pytest.mark.parametrize("dtype,H,d", [(torch.bfloat16, 8, 128), (torch.float32, 4, 128), (torch.bfloat16, 2, 32), (torch.float32, 1, 64)])
def test_long_heads_are_read_in_place(dtype, H, d):
    """Heads within 2^31 bytes, in either order: what the library takes is not copied ahead of it."""
    most = (1 << 31) // (H * d * dtype.itemsize)
    for L, fits in ((most // 2, True), (most - 1, True), (most + 1, False)):
        assert ac._fits(torch.empty(1, L, H, d, dtype=dtype, device="meta").transpose(1, 2), 1) == fits, L
    most = (1 << 31) // (d * dtype.itemsize)
    for L, together, fits in ((most // 2, 1, True), (most - 1, 1, True), (most + 1, 1, False), (most // 2 + 1, 2, False)):
        assert ac._fits(torch.empty(1, 2 * H, L, d, dtype=dtype, device="meta"), together) == fits, L
