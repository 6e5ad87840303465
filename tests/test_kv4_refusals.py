"""What the entry points of the paged 4-bit KV cache refuse before a launch: without
a GPU."""

import os

import pytest

from moe_fused_inference_b200 import _lib, build, kv4


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    return _lib.load()


def test_no_workspace_for_a_cache_on_the_host(lib):
    with pytest.raises(RuntimeError, match="must be cuda"):
        kv4.attention_workspace(1, 4, kv4.KV4Cache(1, 16, 4, 64, device="cpu"))


@pytest.mark.parametrize("D", [64, 128])
def test_tokens_past_31_bits(lib, D):
    """Tokens so close to 2^31 that the last block's would pass it (a broadcast row
    needs no memory for them): refused before the pointers are used."""
    for T in (2 ** 31 - 1, 2 ** 31 - 8):
        args = (2, 4096, 4096, T, 1, D, 64, 8, None)
        assert lib.mfi_kv4_write(4096, 0, D, 4096, 0, D, *args) == 1
        assert b"too many rows" in lib.mfi_last_error()
        assert lib.mfi_kv4_read(4096, 4096, 4096, 4096, 2, *args[3:]) == 1
        assert b"too many rows" in lib.mfi_last_error()
