"""The paged 4-bit KV cache on the GPU against oracle/kv4.py.

Write and read-back are compared for equality (bytes and values).  Attention is
compared value by value with the restatement in 64 bits: within the bound that
its docstring derives plus half a unit in the last place of the output's type.
"""

import numpy as np
import pytest
import torch

from moe_fused_inference_b200 import _lib, kv4
from oracle import kv4 as ok

pytestmark = pytest.mark.gpu

ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # twice half a unit: see _compare


def _errors():
    torch.cuda.synchronize()
    return _lib.device_error(clear=True)


def _np(t):
    return t.double().cpu().numpy()


# ---- write and read -----------------------------------------------------------
def _round_trip(k, v, slots, pages, page):
    """Write into a pool of random bytes, compare every byte, read back."""
    H, D = k.shape[1:]
    rng = np.random.default_rng(pages)
    pool = rng.integers(0, 256, (pages, H, page // 16, 17 * D), dtype=np.uint8)
    cache = kv4.KV4Cache.wrap(torch.from_numpy(pool).cuda())
    st = torch.tensor(slots, dtype=torch.int64, device="cuda")
    kv4.kv4_write(cache, k, v, st)
    ok.write(pool, _np(k), _np(v), slots)
    assert np.array_equal(cache.data.cpu().numpy(), pool)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for got, want in zip(kv4.kv4_read(cache, st, dtype=dtype), ok.read(pool, slots)):
            want = torch.from_numpy(want).float().to(dtype)
            assert got.dtype == dtype and got.shape == want.shape
            assert torch.equal(torch.nan_to_num(got.cpu(), nan=7.0), torch.nan_to_num(want, nan=7.0))
            assert torch.equal(got.cpu().isnan(), want.isnan())
    assert _errors() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H,D,page", [(1, 4, 128, 64), (1, 1, 64, 16), (3, 2, 64, 48),
                                        (37, 4, 128, 16), (130, 3, 128, 80), (257, 1, 64, 256),
                                        (65, 8, 64, 32)])
def test_write_and_read_equal_the_restatement(T, H, D, page, dtype):
    g = torch.Generator(device="cuda").manual_seed(T * 7 + H)
    x = torch.randn((2, T, H, D), generator=g, device="cuda")
    x *= torch.exp(4 * torch.randn((2, T, H, 1), generator=g, device="cuda"))
    k, v = x.clamp(-6e4, 6e4).to(dtype)
    pages = T // page + 3
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].tolist()
    if T > 3:
        slots[1] = -1
        slots[T // 2] = -7
    _round_trip(k, v, slots, pages, page)


def test_write_every_bf16_pattern():
    """All 65,536 bit patterns, infinities and NaN (their blocks read as NaN)."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    perm = torch.randperm(65536, generator=torch.Generator().manual_seed(1))
    k = bits.view(512, 1, 128).cuda()
    v = bits[perm].view(512, 1, 128).cuda()
    _round_trip(k, v, list(range(16, 528)), 9, 64)


def test_write_special_blocks():
    x = torch.zeros((6, 1, 64))
    x[0, 0, :32] = 1e-38             # below the floor of the exponent
    x[0, 0, 40] = -2.0 ** -149
    x[1, 0, 3], x[1, 0, 35] = float("inf"), float("nan")
    x[2, 0] = 3.4e38
    x[3, 0, 5] = 6.0
    x[3, 0, 37] = 6.0000005
    x[4, 0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])  # ties
    x[4, 0, 32:40] = -x[4, 0, :8]
    x[5] = -1e-30
    _round_trip(x.cuda(), x.flip(2).contiguous().cuda(), [5, 4, 3, 2, 1, 0], 1, 16)


def test_write_strided_inputs():
    """Slices of a fused projection, heads before tokens, a broadcast row, rows
    that start off a 16-byte boundary, elements that are not contiguous."""
    g = torch.Generator(device="cuda").manual_seed(3)
    T, H, D = 21, 2, 128
    fused = torch.randn((T, 7 * H, D), generator=g, device="cuda").bfloat16()
    slots = list(range(T))
    _round_trip(fused[:, 5 * H:6 * H], fused[:, 6 * H:], slots, 2, 32)
    heads_first = torch.randn((2, H, T, D), generator=g, device="cuda").half()
    _round_trip(heads_first[0].transpose(0, 1), heads_first[1].transpose(0, 1), slots, 2, 32)
    one = torch.randn((1, H, D), generator=g, device="cuda")
    _round_trip(one.expand(T, H, D), fused[:, :H].float(), slots, 2, 32)
    odd = torch.randn(T * (H * D + 3) + 1, generator=g, device="cuda").bfloat16()
    odd = odd[1:].view(T, H * D + 3)[:, 1:1 + H * D].unflatten(1, (H, D))
    _round_trip(odd, odd.flip(0), slots, 2, 32)
    _round_trip(fused[:, :H].transpose(1, 2).contiguous().transpose(1, 2), odd, slots, 2, 32)


def test_slots_past_the_pool_are_reported():
    cache = kv4.KV4Cache(2, 16, 1, 64)
    x = torch.ones((3, 1, 64), device="cuda")
    slots = torch.tensor([31, 32, 1 << 40], device="cuda")
    kv4.kv4_write(cache, x, x, slots)
    assert _errors() == 12
    k, v = kv4.kv4_read(cache, slots, dtype=torch.float32)
    assert _errors() == 12
    assert k[0].eq(1).all() and v[0].eq(1).all() and not k[1:].any() and not v[1:].any()


def test_no_tokens():
    cache = kv4.KV4Cache(2, 16, 1, 64)
    none = torch.empty((0, 1, 64), device="cuda")
    slots = torch.empty(0, dtype=torch.int64, device="cuda")
    kv4.kv4_write(cache, none, none, slots)
    k, v = kv4.kv4_read(cache, slots)
    assert k.shape == v.shape == (0, 1, 64)
    q = torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    lens = torch.empty(0, dtype=torch.int32, device="cuda")
    assert kv4.kv4_attention(q, cache, lens.view(0, 1), lens).shape == (0, 2, 64)
    assert _errors() == 0


# ---- attention -------------------------------------------------------------------
def _make(seed, rows, lens, Hkv, G, D, page, dtype, q_std=2.0, spread=0.0):
    """A pool with the tokens on shuffled pages; every byte that no sequence
    sees is poisoned (codes 255: NaN if it took part)."""
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) + 1
    pages = sum(need) + 3
    pool = np.full((pages, Hkv, page // 16, 17 * D), 255, np.uint8)
    ids = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lens), width), ids[-1], np.int32)
    at = 0
    cache = kv4.KV4Cache.wrap(torch.from_numpy(pool).cuda())
    for i, (n, L) in enumerate(zip(need, lens)):
        table[i, :n] = ids[at:at + n]
        at += n
        if L == 0:
            continue
        x = rng.standard_normal((2, L, Hkv, D)) * np.exp(spread * rng.standard_normal((2, L, Hkv, 1)))
        k, v = torch.from_numpy(x.astype(np.float32)).cuda()
        pos = np.arange(L)
        slots = torch.from_numpy(table[i][pos // page].astype(np.int64) * page + pos % page).cuda()
        kv4.kv4_write(cache, k, v, slots)
    q = torch.from_numpy(rng.standard_normal((sum(rows), Hkv * G, D)).astype(np.float32) * q_std)
    return q.to(dtype).cuda(), cache, table


def _call(q, cache, table, lens, rows, **kw):
    cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    return kv4.kv4_attention(q, cache, torch.from_numpy(table).cuda(),
                             torch.tensor(lens, dtype=torch.int32, device="cuda"),
                             cu_q=torch.from_numpy(cu).cuda(), max_q=max(rows + [1]), **kw)


def _compare(got, q, cache, table, lens, rows, scale=None):
    """|got - want| <= bound + ulp |want|: the output is rounded to nearest, off
    by half a unit, at most 2^-9 (bf16) or 2^-12 (fp16, plus half of its smallest
    number) of a value that is itself off by up to the bound."""
    want, bound = ok.attention(_np(q), cache.data.cpu().numpy(), table, lens, rows, scale)
    err = np.abs(_np(got) - want)
    tol = bound + ULP[q.dtype] * np.abs(want) + 2.0 ** -25
    assert got.shape == q.shape and got.dtype == q.dtype
    assert np.isfinite(_np(got)).all()
    assert (err <= tol).all(), (np.argwhere(err > tol)[:5], (err / tol).max())


CASES = [
    # rows, lens, Hkv, G, D, page
    ([1], [1], 1, 1, 64, 16),
    ([1], [1], 4, 8, 128, 64),
    ([1], [17], 2, 8, 128, 16),
    ([1], [64], 1, 8, 128, 64),
    ([1], [1152], 4, 8, 128, 64),
    ([1, 1, 1, 1], [63, 65, 128, 129], 2, 4, 64, 48),
    ([1, 1, 1], [5, 0, 700], 2, 5, 128, 32),              # an empty sequence
    ([5], [1021], 4, 8, 128, 16),                         # speculative verification
    ([3, 1, 8, 2], [200, 1, 8, 333], 1, 3, 64, 80),
    ([8, 4], [5, 2], 2, 2, 128, 16),                      # fewer tokens than rows
    ([1], [300], 1, 16, 128, 64),
    ([2], [300], 1, 20, 64, 64),                          # more heads than a tile
    ([1, 0, 2], [40, 70, 33], 8, 1, 128, 16),             # no grouping, a sequence without rows
    ([1], [20011], 1, 8, 128, 256),
    ([1] * 70, [1 + 13 * i % 97 for i in range(70)], 1, 8, 64, 16),
    ([9, 17], [100, 17], 2, 8, 128, 64),
    ([64, 37, 50], [64, 500, 29], 2, 8, 128, 64),         # prompt chunks
    ([130], [130], 1, 1, 128, 16),
    ([257], [700], 1, 2, 64, 48),
    ([129, 3, 300], [400, 3, 300], 1, 5, 128, 32),
    ([200], [1500], 2, 3, 64, 1024),
    ([100], [3050], 1, 8, 128, 64),                       # few items: their tokens in parts
    ([70, 1, 90, 2], [5000, 900, 90, 1], 1, 4, 64, 16),   # parts, whole items and few rows together
    ([40, 40], [8000, 4100], 2, 2, 128, 48),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_matches_the_restatement(case, dtype):
    rows, lens, Hkv, G, D, page = CASES[case]
    q, cache, table = _make(case, rows, lens, Hkv, G, D, page, dtype)
    got = _call(q, cache, table, lens, rows)
    assert _errors() == 0
    _compare(got, q, cache, table, lens, rows)
    # the same bits again, with a workspace that earlier calls have used
    ws = kv4.attention_workspace(len(lens), Hkv * G, cache, max(rows))
    for _ in range(2):
        assert torch.equal(_call(q, cache, table, lens, rows, workspace=ws), got)


@pytest.mark.parametrize("rows,lens,q_std,spread", [
    ([1], [500], 0.0, 1.0),        # all weights equal
    ([2], [400], 40.0, 0.0),       # one weight carries almost all
    ([1], [600], 1.0, 3.0),        # tokens of very different strength
    ([150], [300], 12.0, 2.0),
    ([150], [400], 0.0, 3.0),
])
def test_attention_of_strong_and_weak_tokens(rows, lens, q_std, spread):
    q, cache, table = _make(11, rows, lens, 2, 4, 128, 32, torch.bfloat16, q_std, spread)
    _compare(_call(q, cache, table, lens, rows), q, cache, table, lens, rows)


@pytest.mark.parametrize("rows", [1, 140])
def test_attention_strides_and_scale(rows):
    """q as the slice of a fused projection, and with heads before rows; a scale
    of its own; rows without cu_q."""
    lens, Hkv, G, D = [211, 150], 2, 4, 64
    q, cache, table = _make(5, [rows, rows], lens, Hkv, G, D, 16, torch.bfloat16)
    T, Hq = q.shape[:2]
    fused = torch.randn((T, Hq + 2 * Hkv, D), device="cuda").bfloat16()
    fused[:, :Hq] = q
    odd = torch.zeros(T * (Hq * D + 5) + 3, dtype=torch.bfloat16, device="cuda")
    odd = odd[3:].view(T, Hq * D + 5)[:, :Hq * D].unflatten(1, (Hq, D))
    odd.copy_(q)
    base = _call(q, cache, table, lens, [rows, rows], scale=0.3)
    _compare(base, q, cache, table, lens, [rows, rows], scale=0.3)
    forms = [fused[:, :Hq], q.transpose(0, 1).contiguous().transpose(0, 1), odd,
             q.transpose(1, 2).contiguous().transpose(1, 2)]
    for x in forms:
        assert torch.equal(_call(x, cache, table, lens, [rows, rows], scale=0.3), base)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 9.0)
    same = kv4.kv4_attention(q, cache, torch.from_numpy(table).cuda(), lens_t, scale=0.3, out=out)
    assert same is out and torch.equal(out, base)


@pytest.mark.parametrize("rows", [1, 140])
def test_attention_nan_only_where_it_is_seen(rows):
    """A key or value that is NaN makes NaN of the rows that see it on its head,
    and of no others."""
    lens, Hkv, G, D, page = [220], 2, 2, 128, 32
    q, cache, table = _make(9, [rows], lens, Hkv, G, D, page, torch.bfloat16)
    clean = _call(q, cache, table, lens, [rows])
    at = 200
    slot = int(table[0, at // page]) * page + at % page
    k, v = kv4.kv4_read(cache, torch.tensor([slot], device="cuda"), dtype=torch.float32)
    for which in range(2):
        bad = (k.clone(), v.clone())
        bad[which][0, 1, 40] = float("nan")
        kv4.kv4_write(cache, *bad, torch.tensor([slot], device="cuda"))
        got = _call(q, cache, table, lens, [rows])
        first = max(0, at - (lens[0] - rows))    # first row that sees the token
        hit = got[first:, G:]
        if which == 1:                           # block 1 of the values
            assert hit[..., 32:64].isnan().all() and hit[..., :32].isfinite().all()
        else:
            assert hit.isnan().all()
        assert torch.equal(got[:, :G], clean[:, :G])
        assert torch.equal(got[:first], clean[:first])
        kv4.kv4_write(cache, k, v, torch.tensor([slot], device="cuda"))
    q2 = q.clone()
    q2[0, 3, 7] = float("inf")
    got = _call(q2, cache, table, lens, [rows])
    assert got[0, 3].isnan().all()
    got[0, 3] = clean[0, 3]
    assert torch.equal(got, clean)


def test_attention_out_of_range_arguments_are_reported():
    rows, lens = [2, 3], [100, 90]
    q, cache, table = _make(2, rows, lens, 1, 4, 64, 16, torch.bfloat16)
    good = _call(q, cache, table, lens, rows)
    assert _errors() == 0
    for bad_id in (-1, cache.num_pages, 2 ** 31 - 1):
        t = table.copy()
        t[1, 2] = bad_id
        got = _call(q, cache, t, lens, rows)
        assert _errors() == 11
        assert torch.equal(got[:2], good[:2])
    room = table.shape[1] * 16
    full = _call(q, cache, table, [100, room], rows)
    assert _errors() == 0
    got = _call(q, cache, table, [100, room + 1], rows)
    assert _errors() == 11
    assert torch.equal(got.isnan(), full.isnan()) and torch.equal(got.nan_to_num(), full.nan_to_num())
    got = _call(q, cache, table, [100, -5], rows)
    assert _errors() == 11
    assert torch.equal(got[:2], good[:2]) and not got[2:].any()
    tt, lt = torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    for cu in ([0, 2, 6], [0, 2, 1], [-1, 2, 5], [0, 5, 5]):
        out = torch.zeros_like(q)
        kv4.kv4_attention(q, cache, tt, lt, cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"),
                          max_q=3, out=out)
        assert _errors() == 11
        assert out.isfinite().all()


def test_attention_in_a_graph_with_moving_lengths():
    """A captured step: write one token a sequence, attend, advance."""
    B, Hkv, G, D, page, steps = 3, 2, 8, 128, 16, 40
    g = torch.Generator(device="cuda").manual_seed(8)
    cache = kv4.KV4Cache(B * 5, page, Hkv, D)
    table = torch.randperm(B * 5, generator=g, device="cuda").to(torch.int32).view(B, 5)
    ks, vs = torch.randn((2, steps, B, Hkv, D), generator=g, device="cuda").bfloat16()
    qs = torch.randn((steps, B, Hkv * G, D), generator=g, device="cuda").bfloat16()
    k, v, q = torch.zeros_like(ks[0]), torch.zeros_like(vs[0]), torch.zeros_like(qs[0])
    lens = torch.tensor([0, 7, 20], dtype=torch.int32, device="cuda")
    start = lens.clone()
    out = torch.zeros_like(q)
    ws = kv4.attention_workspace(B, Hkv * G, cache)

    def step():
        pos = lens.long()
        page_id = table.gather(1, (pos // page)[:, None])[:, 0].long()
        kv4.kv4_write(cache, k, v, page_id * page + pos % page)
        lens.add_(1)
        kv4.kv4_attention(q, cache, table, lens, out=out, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    lens.copy_(start)
    cache.data.zero_()
    for t in range(steps):
        k.copy_(ks[t]); v.copy_(vs[t]); q.copy_(qs[t])
        graph.replay()
        if t in (0, 8, 9, steps - 1):
            torch.cuda.synchronize()
            _compare(out, q, cache, table.cpu().numpy(), lens.tolist(), [1] * B)
    assert _errors() == 0


def test_attention_of_many_rows_under_a_wide_table():
    """Rows of a prompt times the tiles that its page table has room for pass 2^31
    (8 heads x 38400 x 8192 sets of 8): no limit of the kernel for many rows."""
    q, cache, table = _make(9, [20], [20], 8, 8, 64, 1024, torch.bfloat16)
    rows = 8192
    wide = np.full((1, 600), table[0, 0], np.int32)
    many = torch.zeros((rows, 64, 64), dtype=q.dtype, device="cuda")
    many[-20:] = q
    got = _call(many, cache, wide, [20], [rows])
    assert _errors() == 0
    assert not got[:-20].any()  # rows that see no token
    _compare(got[-20:], q, cache, table, [20], [20])


def test_one_workspace_serves_calls_of_all_shapes_in_turn():
    """Every call leaves the workspace as it found it, and repeats bit for bit."""
    cases = [([1], [20011], 1, 8), ([100], [3050], 1, 8), ([1] * 40, [1 + 61 * i for i in range(40)], 1, 8),
             ([257], [700], 1, 8), ([5], [4099], 1, 8), ([0, 0], [9, 9], 1, 8)]
    made = [_make(20 + i, rows, lens, H, G, 128, 64, torch.bfloat16) + (lens, rows)
            for i, (rows, lens, H, G) in enumerate(cases)]
    want = [_call(*m) for m in made]
    ws = kv4.attention_workspace(40, 8, made[0][1], max_q=257)
    for i in [0, 1, 2, 3, 4, 5, 1, 0, 2, 4, 3, 3, 0, 1] * 3:
        assert torch.equal(_call(*made[i], workspace=ws), want[i])
    assert _errors() == 0


@pytest.mark.parametrize("rows", [1, 140])
def test_attention_of_a_table_without_pages(rows):
    """No sequence can have a token: zeros."""
    cache = kv4.KV4Cache(2, 16, 2, 64)
    q = torch.randn((2 * rows, 2, 64), device="cuda").half()
    none = torch.empty((2, 0), dtype=torch.int32, device="cuda")
    got = kv4.kv4_attention(q, cache, none, torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert not got.any() and _errors() == 0


@pytest.mark.parametrize("rows,lens,Hkv,G", [
    ([1] * 12, [1, 5000, 0, 17, 3, 2100, 16, 0, 1, 1030, 33, 2], 4, 4),     # whole and split pieces, empty ones
    ([1] * 9, [1, 1, 1, 1, 1, 1, 1, 1, 9000], 8, 2),
    ([3, 1, 4, 2, 1], [3, 1100, 2500, 0, 1], 8, 5),
    ([1] * 300, [i % 5 * 7 for i in range(300)], 2, 2),                     # more pieces than CTAs
])
def test_attention_of_very_unequal_lengths(rows, lens, Hkv, G):
    q, cache, table = _make(31, rows, lens, Hkv, G, 64, 16, torch.bfloat16)
    got = _call(q, cache, table, lens, rows)
    assert _errors() == 0
    _compare(got, q, cache, table, lens, rows)


def test_attention_on_another_stream():
    rows, lens = [1, 1], [900, 33]
    q, cache, table = _make(4, rows, lens, 2, 8, 128, 64, torch.bfloat16)
    want = _call(q, cache, table, lens, rows)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q2 = q + 0
        got = _call(q2, cache, table, lens, rows)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_offsets_past_32_bits():
    """A pool of more than 4 GB: the last pages are written, read and attended."""
    page, Hkv, D = 256, 8, 128
    pages = (1 << 32) // (Hkv * 16 * 17 * D) + 40
    cache = kv4.KV4Cache.wrap(torch.empty((pages, Hkv, page // 16, 17 * D), dtype=torch.uint8,
                                          device="cuda"))
    assert cache.data.numel() > (1 << 32)
    g = torch.Generator(device="cuda").manual_seed(6)
    for L, rows in ((300, 1), (300, 140)):
        k, v = torch.randn((2, L, Hkv, D), generator=g, device="cuda").bfloat16()
        table = np.array([[pages - 1, pages - 3]], np.int32)
        pos = np.arange(L)
        slots = torch.from_numpy(table[0][pos // page].astype(np.int64) * page + pos % page).cuda()
        kv4.kv4_write(cache, k, v, slots)
        gk, gv = kv4.kv4_read(cache, slots, dtype=torch.float32)
        assert np.array_equal(_np(gk), ok.decode(*ok.encode(_np(k))))
        assert np.array_equal(_np(gv), ok.decode(*ok.encode(_np(v))))
        q = torch.randn((rows, Hkv, D), generator=g, device="cuda").bfloat16()
        got = _call(q, cache, table, [L], [rows])
        # the restatement reads a small pool of the same two pages
        small = kv4.KV4Cache.wrap(cache.data[[pages - 1, pages - 3]].contiguous())
        _compare(got, q, small, np.array([[0, 1]], np.int32), [L], [rows])
    assert _errors() == 0
