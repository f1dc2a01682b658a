"""The sizes that a call of the attention to an encoder's states may have, without a GPU."""
import ctypes

import pytest

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
