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
