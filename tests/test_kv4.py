"""The paged 4-bit KV cache without a GPU: the restatement in oracle/kv4.py
against the MXFP4 quantiser's, its layout, and what the entry points refuse."""

import numpy as np
import pytest
import torch

from moe_fused_inference_b200 import _lib, build, kv4
from oracle import kv4 as ok
from oracle import mxfp4 as mx

import os


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    return _lib.load()


def test_codes_are_those_of_the_weight_quantiser():
    """Nibbles and codes equal the MXFP4 quantiser's on ordinary blocks; only a
    block of zeros (code 28 instead of 127) differs."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((64, 128)) * np.exp(rng.uniform(-20, 20, (64, 1)))).astype(np.float32)
    x[5, 32:64] = 0
    nib, codes = ok.encode(x)
    packed, want = mx.quantize_rows(x)
    assert np.array_equal((nib[:, 0::2] | (nib[:, 1::2] << 4)), packed)
    keep = np.ones_like(codes, bool)
    keep[5, 1] = False
    assert np.array_equal(codes[keep], want[keep])
    assert codes[5, 1] == 28 and want[5, 1] == 127


@pytest.mark.parametrize("D", [64, 128])
def test_write_then_read_gives_the_encoded_values(D):
    rng = np.random.default_rng(D)
    pool = rng.integers(0, 256, (3, 2, 3, 17 * D), dtype=np.uint8)
    before = pool.copy()
    k, v = rng.standard_normal((2, 5, 2, D)).astype(np.float32)
    slots = np.array([0, 47, -1, 100, 143])
    ok.write(pool, k, v, slots)
    gk, gv = ok.read(pool, slots)
    live = slots >= 0
    assert np.array_equal(gk[live], ok.decode(*ok.encode(k[live])))
    assert np.array_equal(gv[live], ok.decode(*ok.encode(v[live])))
    assert not gk[2].any() and not gv[2].any()
    others = np.setdiff1d(np.arange(144), slots)
    for a, b in zip(ok.read(pool, others), ok.read(before, others)):
        assert np.array_equal(a, b, equal_nan=True)


@pytest.mark.parametrize("D", [64, 128])
def test_every_byte_of_a_tile_has_one_place(D):
    """The interleaved rows are permutations: each byte holds two elements."""
    for piece in (8, 4):
        at = ok._at(D, piece)
        assert np.array_equal(np.sort(at), np.repeat(np.arange(D // 2), 2))


def test_sizes(lib):
    assert lib.mfi_kv4_pool_bytes(10, 64, 4, 128) == 10 * 4 * 4 * 2176
    assert lib.mfi_kv4_pool_bytes(10, 16, 1, 64) == 10 * 1088
    for bad in ((0, 64, 4, 128), (10, 63, 4, 128), (10, 64, 0, 128), (10, 64, 4, 96)):
        assert lib.mfi_kv4_pool_bytes(*bad) == 0
    assert lib.mfi_kv4_attn_workspace_bytes(1, 32, 4, 128, 1) > 0
    for bad in ((0, 32, 4, 128, 1), (1, 30, 4, 128, 1), (1, 32, 4, 80, 1), (1, 32, 4, 128, 0)):
        assert lib.mfi_kv4_attn_workspace_bytes(*bad) == 0


def test_c_entries_refuse(lib):
    """Statuses and messages of the C entries; nothing is launched."""
    P = 4096  # stands for a device pointer: every check comes before its use

    def write(k=P, v=P, dtype=2, pool=P, slots=P, T=1, H=4, D=128, page=64, pages=8):
        return lib.mfi_kv4_write(k, 512, 128, v, 512, 128, dtype, pool, slots, T, H, D, page, pages,
                                 None)

    def read(k=P, v=P, dtype=2, pool=P, slots=P, T=1, H=4, D=128, page=64, pages=8):
        return lib.mfi_kv4_read(pool, slots, k, v, dtype, T, H, D, page, pages, None)

    for f in (write, read):
        for kw, msg in ((dict(T=-1), b"negative"), (dict(dtype=7), b"dtype"), (dict(D=96), b"head_dim"),
                        (dict(H=0), b"Hkv"), (dict(page=24), b"multiple of 16"),
                        (dict(pages=0), b"no pages"), (dict(pool=None), b"null"),
                        (dict(pool=P + 8), b"aligned"), (dict(k=None), b"null"),
                        (dict(v=None), b"null"), (dict(slots=None), b"null")):
            assert f(**kw) == 1 and msg in lib.mfi_last_error(), (f.__name__, kw)
        assert f(T=0) == 0
    assert read(k=P + 4) == 1 and b"aligned" in lib.mfi_last_error()

    def attn(q=P, dtype=2, pool=P, table=P, lens=P, cu=None, out=P, T=2, max_q=1, n=2, Hq=32, H=4,
             D=128, page=64, pages=8, width=4, ws=P, nws=1 << 40):
        return lib.mfi_kv4_attn(q, dtype, 4096, 128, pool, table, width, lens, cu, out, T, max_q, n,
                                Hq, H, D, page, pages, width, 0.1, ws, nws, None)

    for kw, msg in ((dict(dtype=0), b"MFI_F16"), (dict(D=256), b"head_dim"), (dict(page=8), b"multiple"),
                    (dict(Hq=30), b"multiple of Hkv"), (dict(Hq=0), b"multiple of Hkv"),
                    (dict(T=-1), b"negative"), (dict(n=-1), b"negative"), (dict(width=-1), b"negative"),
                    (dict(T=3), b"cu_q"), (dict(q=None), b"null"), (dict(table=None), b"null"),
                    (dict(lens=None), b"null"), (dict(out=None), b"null"), (dict(ws=None), b"null"),
                    (dict(pool=None), b"null")):
        assert attn(**kw) == 1 and msg in lib.mfi_last_error(), kw
    assert attn(nws=16) == 3 and b"workspace" in lib.mfi_last_error()
    assert attn(T=0, n=0) == 0
    assert attn(T=0, max_q=0) == 0
    assert lib.mfi_kv4_attn_init_workspace(None, 256, None) == 1


def test_python_refusals(lib):
    with pytest.raises(RuntimeError, match="head_dim"):
        kv4.KV4Cache(4, 64, 4, 96, device="cpu")
    with pytest.raises(RuntimeError, match="multiple of 16"):
        kv4.KV4Cache(4, 40, 4, 128, device="cpu")
    with pytest.raises(RuntimeError, match="positive"):
        kv4.KV4Cache(0, 64, 4, 128, device="cpu")
    with pytest.raises(RuntimeError, match="contiguous uint8"):
        kv4.KV4Cache.wrap(torch.zeros((4, 4, 4, 17 * 128), dtype=torch.int8))
    with pytest.raises(RuntimeError, match="head_dim"):
        kv4.KV4Cache.wrap(torch.zeros((4, 4, 4, 2048), dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="no pages"):
        kv4.KV4Cache.wrap(torch.zeros((0, 4, 4, 17 * 128), dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="aligned"):
        flat = torch.zeros(17 * 128 + 64, dtype=torch.uint8)
        off = (8 - flat.data_ptr()) % 16
        kv4.KV4Cache.wrap(flat[off:off + 17 * 128].view(1, 1, 1, 17 * 128))
    cache = kv4.KV4Cache(4, 64, 4, 128, device="cpu")
    assert (cache.page, cache.kv_heads, cache.head_dim, cache.capacity) == (64, 4, 128, 256)
    k = torch.zeros((2, 4, 128))
    slots = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="must be cuda"):
        kv4.kv4_write(cache, k, k, slots)
    with pytest.raises(RuntimeError, match="must be cuda"):
        kv4.kv4_read(cache, slots)
    with pytest.raises(RuntimeError, match="must be cuda"):
        kv4.kv4_attention(k, cache, torch.zeros((2, 1), dtype=torch.int32),
                          torch.zeros(2, dtype=torch.int32))
