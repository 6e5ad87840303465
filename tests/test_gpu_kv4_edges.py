"""Attention over the paged 4-bit KV cache where numbers run out of range: small,
large and NaN keys, values and queries, against oracle/kv4.py in 64 bits."""

import numpy as np
import pytest
import torch

from moe_fused_inference_b200 import _lib, kv4
from oracle import kv4 as ok
from tests.test_gpu_kv4 import _call, _compare, _errors, _make, _np

pytestmark = pytest.mark.gpu


def _cache(k, v, page=32):
    """A cache that holds the tokens k, v (L, Hkv, D) on its pages in order, and
    the page table of that one sequence."""
    L, H, D = k.shape
    cache = kv4.KV4Cache(max(1, -(-L // page)), page, H, D)
    kv4.kv4_write(cache, k, v, torch.arange(L, device="cuda"))
    return cache, np.arange(cache.num_pages, dtype=np.int32)[None]


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


# ---- small queries over small keys ----------------------------------------------
@pytest.mark.parametrize("rows", [1, 140])
@pytest.mark.parametrize("key_std", [0.0, 2.0 ** -60, 2.0 ** -30, 1.0])
@pytest.mark.parametrize("q_std,scale", [(0.0, None), (2.0 ** -120, None), (2.0 ** -30, None),
                                         (2.0 ** -24, None), (1.0, 0.0), (1.0, 2.0 ** -100)])
def test_scores_too_small_to_tell_apart(rows, key_std, q_std, scale):
    """The mean of the tokens that a row sees, not NaN: queries, keys or scales
    whose product with the other two leaves fp32."""
    L, H, G, D = 200, 2, 4, 128
    k, v = _randn(1, 2, L, H, D)
    cache, table = _cache(k * key_std, v)
    q = (_randn(2, rows, H * G, D) * q_std).bfloat16()
    _compare(_call(q, cache, table, [L], [rows], scale=scale), q, cache, table, [L], [rows], scale)
    assert _errors() == 0


@pytest.mark.parametrize("rows", [1, 140])
@pytest.mark.parametrize("length", [0, 1, 200])
def test_zero_rows_over_a_fresh_cache(rows, length):
    """A padded or warm-up call: a pool that nobody wrote to, rows of zeros, and
    rows that see no token give zeros."""
    cache = kv4.KV4Cache(8, 32, 2, 64)
    table = np.arange(8, dtype=np.int32)[None]
    for q in (torch.zeros((rows, 8, 64), device="cuda").bfloat16(), _randn(3, rows, 8, 64).half()):
        got = _call(q, cache, table, [length], [rows])
        assert torch.equal(got, torch.zeros_like(q))
    assert _errors() == 0


# ---- a value that is NaN under a weight that rounds to zero ------------------------
@pytest.mark.parametrize("rows", [1, 3, 8, 20, 140])
@pytest.mark.parametrize("at", [0, 100, 250, 292, 297])
@pytest.mark.parametrize("D", [64, 128])
def test_nan_value_of_a_token_that_hardly_counts(rows, at, D):
    """0 x NaN: the rows that see the token have NaN in its block of 32, wherever
    the token lies and however small its weight, the others do not."""
    L, H, G = 300, 2, 4
    k, v = _randn(4, 2, L, H, D)
    k[at] = -8.0                       # a score some 4 x 8 sqrt(D) below the others
    v[at, 1, 40] = float("nan")
    cache, table = _cache(k, v)
    q = (4.0 + 0.1 * _randn(5, rows, H * G, D)).bfloat16()
    got = _call(q, cache, table, [L], [rows])
    first = max(0, at - (L - rows))    # first row that sees the token
    want = torch.zeros_like(got, dtype=torch.bool)
    want[first:, G:, 32:64] = True
    assert torch.equal(got.isnan(), want)
    assert _errors() == 0


# ---- values of very different strength -----------------------------------------------
def _compare_blocks(got, q, cache, table, L):
    """The bound of oracle/kv4.py for each block of 32 channels by itself, with the
    largest value that the row sees in that block instead of the whole head; and
    2^-31 of it for each token, whose weight and scale may fall below fp16."""
    pool, (R, Hq, D) = cache.data.cpu().numpy(), q.shape
    want, bound = ok.attention(_np(q), pool, table, [L], [R])
    pos = np.arange(L)
    _, v = ok.read(pool, table[0][pos // cache.page].astype(np.int64) * cache.page + pos % cache.page)
    err = np.abs(_np(got) - want)
    for r in range(R):
        for h in range(Hq):
            seen = np.abs(v[:L - R + r + 1, h * pool.shape[1] // Hq])
            top = seen.reshape(len(seen), D // 32, 32).max((0, 2))
            tol = np.repeat((bound[r, h, 0] / seen.max() + L * 2.0 ** -31) * top, 32)
            assert (err[r, h] <= tol + 2.0 ** -8 * np.abs(want[r, h])).all(), (r, h)


@pytest.mark.parametrize("rows", [1, 3, 8, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_weak_channels_beside_strong_ones(rows, D):
    """Blocks of channels 2^-70 to 2^40 of each other keep their own accuracy."""
    L, H, G = 333, 2, 4
    k, v = _randn(6, 2, L, H, D)
    strength = torch.tensor([2.0 ** 20, 2.0 ** -20, 2.0 ** 30, 2.0 ** -40][:D // 32], device="cuda")
    cache, table = _cache(k, v * strength.repeat_interleave(32))
    q = (2.0 * _randn(7, rows, H * G, D)).bfloat16()
    _compare_blocks(_call(q, cache, table, [L], [rows]), q, cache, table, L)
    assert _errors() == 0


@pytest.mark.parametrize("L,rows", [(3000, 1), (3000, 40), (300, 140)])
def test_values_that_grow_along_the_sequence(L, rows):
    """The references of the values move with the tokens: 2^-90 to 2^60, one block
    falling while the others rise, in parts that are joined as well."""
    H, G, D = 1, 4, 128
    k, v = _randn(8, 2, L, H, D)
    power = torch.linspace(-90.0, 60.0, L, device="cuda")[:, None] * torch.tensor([1.0, -1.0, 0.5, 0.0], device="cuda")
    cache, table = _cache(k, v * torch.exp2(power.floor()).repeat_interleave(32, 1)[:, None])
    q = _randn(9, rows, H * G, D).bfloat16()
    _compare_blocks(_call(q, cache, table, [L], [rows]), q, cache, table, L)
    assert _errors() == 0


@pytest.mark.parametrize("rows", [1, 3, 140])
@pytest.mark.parametrize("key,query,scale", [(110, -110, None), (-90, 92, None), (112, -95, 2.0 ** -20),
                                             (110, 0, 2.0 ** -113), (-80, -30, 2.0 ** 108)])
def test_scores_of_ordinary_size_from_extreme_factors(rows, key, query, scale):
    """Keys, queries and scales far from 1 whose product is not."""
    L, H, G, D = 300, 2, 4, 128
    k, v = _randn(10, 2, L, H, D)
    cache, table = _cache(k * 2.0 ** key, v)
    q = (_randn(11, rows, H * G, D) * 2.0 ** query).bfloat16()
    _compare(_call(q, cache, table, [L], [rows], scale=scale), q, cache, table, [L], [rows], scale)
    assert _errors() == 0


# ---- a workspace that an aborted call has left -------------------------------------
def test_counters_that_an_aborted_call_left_do_not_reach_the_next():
    """A CTA of the kernel for many rows that gives up a wait does not arrive at its
    parts' counters.  The next call on the workspace starts them anew: with ones in
    the words after the few-row kernel's 3 x 444, rows joined from parts are those of
    a fresh workspace."""
    L, rows, H, G, D = 3050, 100, 1, 8, 128
    k, v = _randn(12, 2, L, H, D)
    cache, table = _cache(k, v)
    q = _randn(13, rows, H * G, D).bfloat16()
    want = _call(q, cache, table, [L], [rows])
    ws = kv4.attention_workspace(1, H * G, cache, max_q=rows)
    words = ws[:16384].view(torch.int32)
    for _ in range(2):
        words[3 * 444:] = 1
        assert torch.equal(_call(q, cache, table, [L], [rows], workspace=ws), want)
        assert not words[:3 * 444].any()
    assert _errors() == 0


# ---- another device is current -------------------------------------------------------
def test_calls_run_on_their_tensors_device(monkeypatch):
    """With another device current every entry point makes its tensors' device
    current for its launches.  (One device is enough: the query says 1 until the
    entry point changes it.)"""
    L, H, G, D = 70, 2, 4, 64
    k, v = _randn(14, 2, L, H, D)
    cache, table = _cache(k, v)
    q = _randn(15, 3, H * G, D).bfloat16()
    table = torch.from_numpy(table).cuda()
    lens = torch.tensor([L], dtype=torch.int32, device="cuda")
    slots = torch.arange(L, device="cuda")
    want = kv4.kv4_attention(q, cache, table, lens), *kv4.kv4_read(cache, slots)
    current, entered = [1], []

    class device:
        def __init__(self, to):
            self.to = torch.device(to)

        def __enter__(self):
            self.was, current[0] = current[0], self.to.index
            entered.append(self.to)

        def __exit__(self, *exc):
            current[0] = self.was

    monkeypatch.setattr(kv4, "_device", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    other = kv4.KV4Cache.wrap(torch.zeros_like(cache.data))
    kv4.kv4_write(other, k, v, slots)
    ws = kv4.attention_workspace(1, H * G, other, max_q=3)
    got = kv4.kv4_attention(q, other, table, lens, workspace=ws), *kv4.kv4_read(other, slots)
    assert entered == [cache.device] * 4 and current == [1]
    assert torch.equal(other.data, cache.data)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- wide page tables -------------------------------------------------------------------
@pytest.mark.parametrize("n,heads,rows,width", [(500, 8, 1, 1 << 19), (500, 16, 4, 282144),
                                                (4096, 32, 4, 24000)])
def test_many_short_sequences_under_a_wide_table(n, heads, rows, width):
    """The count of work that a call may have goes by its rows and the table's room,
    not by more sets of vectors than there are: rows is the largest count of a
    sequence, the others have one."""
    H, D = 8, 64
    k, v = _randn(16, 2, 16, H, D)
    cache, table = _cache(k, v, page=16)
    each = [rows] + [1] * (n - 1)
    q = _randn(17, sum(each), heads, D).bfloat16()
    wide = torch.from_numpy(table).cuda().expand(n, width)
    lens = torch.full((n,), 16, dtype=torch.int32, device="cuda")
    cu = torch.tensor(np.concatenate([[0], np.cumsum(each)]), dtype=torch.int32, device="cuda")
    got = kv4.kv4_attention(q, cache, wide, lens, cu_q=cu, max_q=rows)
    assert _errors() == 0
    some = list(range(rows)) + [len(q) // 2, len(q) - 1]
    lens_of = [16 - rows + 1 + r for r in range(rows)] + [16, 16]
    _compare(got[some], q[some], cache, np.repeat(table, len(some), 0), lens_of, [1] * len(some))


def test_more_work_than_31_bits_is_refused():
    cache = kv4.KV4Cache(1, 16, 8, 64)
    q = torch.zeros((600, 8, 64), device="cuda").bfloat16()
    wide = torch.zeros((1, 1), dtype=torch.int32, device="cuda").expand(600, 1 << 19)
    lens = torch.ones(600, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="2\\^31 tiles"):
        kv4.kv4_attention(q, cache, wide, lens)


# ---- both sizes of CTA of the kernel for few rows --------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [32, 33])  # 64 and 66 pairs of a sequence and KV head
@pytest.mark.parametrize("most,G", [(1, 8), (3, 5)])
def test_either_side_of_64_pieces(n, most, G, D):
    rows = [1 + i % most for i in range(n)]
    lens = [(97 * i) % 613 for i in range(n)]
    q, cache, table = _make(40 + n, rows, lens, 2, G, D, 48, torch.bfloat16)
    _compare(_call(q, cache, table, lens, rows), q, cache, table, lens, rows)
    assert _errors() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,Hkv", [([3, 1], 2), ([6, 6], 2), ([6, 7], 2), ([8], 3), ([8, 2], 3)])
def test_either_side_of_24_sets_of_vectors(rows, Hkv, D):
    lens = [700, 41][:len(rows)]
    q, cache, table = _make(50, rows, lens, Hkv, 8, D, 32, torch.float16)
    _compare(_call(q, cache, table, lens, rows), q, cache, table, lens, rows)
    assert _errors() == 0


# ---- huge scores -----------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 3, 8, 40, 140])
@pytest.mark.parametrize("power", [6, 9, 12, 16, 30, 50])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_huge_scores_leave_one_weight(rows, power, sign):
    """Scores of 2^(2 power) and more, all positive or all negative: the tokens of the
    largest one alone (the others are an eighth of it away at least)."""
    L, H, G, D = 300, 2, 4, 64
    g = np.random.default_rng(power)
    e = g.permutation(L) % 24
    score = np.exp2(e // 3 + power) * np.array([1.0, 1.25, 1.5])[e % 3]    # exact in 4 bits, two blocks
    k = torch.zeros((L, H, D), device="cuda")
    k[:, :, 0] = sign * torch.from_numpy(np.exp2(e // 3 + power)).float().cuda()[:, None]
    k[:, :, 32] = sign * torch.from_numpy(score - np.exp2(e // 3 + power)).float().cuda()[:, None]
    v = _randn(20, L, H, D)
    cache, table = _cache(k, v)
    q = torch.zeros((rows, H * G, D), device="cuda")
    q[:, :, 0] = q[:, :, 32] = 2.0 ** power
    got = _np(_call(q.bfloat16(), cache, table, [L], [rows], scale=1.0))
    _, held = kv4.kv4_read(cache, torch.arange(L, device="cuda"), dtype=torch.float32)
    held = _np(held)
    for r in range(rows):
        s = sign * score[:L - rows + r + 1]
        want = held[:len(s)][s == s.max()].mean(0)          # (H, D): equal scores share
        tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -11 * np.abs(held).max()
        assert (np.abs(got[r].reshape(H, G, D) - want[:, None]) <= tol[:, None]).all()
    assert _errors() == 0


# ---- strong tokens that a row does not see --------------------------------------------------
@pytest.mark.parametrize("rows", [2, 5, 8, 33, 140])
@pytest.mark.parametrize("back", [1, 2, 30])
@pytest.mark.parametrize("what", ["values", "keys", "both"])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_do_not_depend_on_tokens_after_theirs(rows, back, what, D):
    """A token 2^100 stronger than the others takes nothing from the rows before it;
    the rows that see it stay within the bound of what they see."""
    L, H, G = 300, 2, 4
    k, v = _randn(18, 2, L, H, D)
    at = L - min(back, rows - 1)
    if what != "keys":
        v[at] *= 2.0 ** 100
        v[at + 1:at + 2, 0] *= 2.0 ** 50
    if what != "values":
        k[at] *= 2.0 ** 60
    cache, table = _cache(k, v)
    q = _randn(19, rows, H * G, D).bfloat16()
    got = _call(q, cache, table, [L], [rows])
    _compare_blocks(got, q, cache, table, L)
    assert got.isfinite().all() and _errors() == 0


@pytest.mark.parametrize("L,rows", [(1, 1), (7, 3), (40, 40), (3000, 1), (3000, 30)])
def test_values_near_the_end_of_fp32(L, rows):
    """Values of up to 2^126: the weights' factor has no room beside them."""
    H, G, D = 1, 8, 128
    k, v = _randn(21, 2, L, H, D)
    cache, table = _cache(0.1 * k, v.clamp(-2, 2) * 2.0 ** 125)
    q = _randn(22, rows, H * G, D).bfloat16() * (1.0 if L < 3000 else 40.0)   # few tokens count
    got = _call(q, cache, table, [L], [rows])
    assert got.isfinite().all()
    _compare_blocks(got, q, cache, table, L)
    assert _errors() == 0


@pytest.mark.parametrize("rows", [1, 3, 8, 140])
@pytest.mark.parametrize("L", [17, 300, 2000])
@pytest.mark.parametrize("power", [20, 26, 70])
@pytest.mark.parametrize("first", [True, False])
def test_hugely_negative_scores_beside_ordinary_ones(rows, L, power, first):
    """Half of the tokens of a weight of zero, in tiles and parts of their own: the other
    half's alone count."""
    H, G, D = 2, 4, 64
    k, v = _randn(23, 2, L, H, D)
    q = _randn(24, rows, H * G, D).bfloat16()
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    k[: L // 2 if first else None, :, :32] = 0.0
    (k[: L // 2] if first else k[1 - L % 2::2])[..., 0] = -2.0 ** power
    cache, table = _cache(k, v, page=16)
    got = _call(q, cache, table, [L], [rows])
    want, _ = ok.attention(_np(q), cache.data.cpu().numpy(), table, [L], [rows])
    # the scores that count are ordinary: the bound without the others' size
    held, vals = (_np(x) for x in kv4.kv4_read(cache, torch.arange(L, device="cuda"), dtype=torch.float32))
    live = held[:, 0, 0] == 0
    if rows > L:
        return
    for r in range(rows):
        see = np.arange(L) <= L - rows + r
        if not (live & see).any():
            continue
        ds = 2 * D * 2.0 ** -24 * np.abs(held[live]).max() * np.abs(_np(q)[r]).max() * D ** 0.5
        tol = (2.0 ** -12 + 2 * ds + 2.0 ** -18 + L * 2.0 ** -31) * np.abs(vals).max() + 2.0 ** -8 * np.abs(want[r])
        assert (np.abs(_np(got[r]) - want[r]) <= tol).all()
    assert got.isfinite().all() and _errors() == 0
