"""Positions past a runner's caches are refused on the host, before any launch: the
indexing of a page table or cache past its end would be a fault of the device."""

from types import SimpleNamespace

import pytest
import torch

from moe_fused_inference_b200.model import GraphDecoder, QwenConfig, Runner

CFG = QwenConfig(hidden=64, layers=1, heads=2, kv_heads=1, head_dim=64, vocab=97, experts=8, top_k=2, inter=32)


def _runner(kv, max_len=40, **kw):
    return Runner(SimpleNamespace(cfg=CFG, final_norm=torch.ones(64)), None, 2, max_len, kv=kv, **kw)


@pytest.mark.parametrize("kv", ["fp8", "mxfp4"])
@pytest.mark.parametrize("base,rows", [(40, 1), (39, 2), (0, 41), (-1, 1), (200, 1)])
def test_forward_refuses_positions_past_the_caches(kv, base, rows):
    with pytest.raises(RuntimeError, match="outside the caches' 40"):
        _runner(kv).forward(torch.zeros((2, rows), dtype=torch.long), base)


@pytest.mark.parametrize("kv", ["fp8", "mxfp4"])
def test_graph_decoder_counts_its_steps(kv):
    """Steps since start() are bounded by max_steps and by the caches, over
    several calls of decode()."""
    replays = []
    gd = GraphDecoder(_runner(kv), 8)
    gd.graph = SimpleNamespace(replay=lambda: replays.append(1))
    prompt = torch.zeros((2, 36), dtype=torch.long)
    gd.start(prompt, prefill=False)
    gd.decode(3)
    gd.decode(2)                      # positions 35 .. 39
    with pytest.raises(RuntimeError, match="outside the caches' 40"):
        gd.decode(1)
    gd.start(prompt[:, :10], prefill=False)
    gd.decode(5)
    gd.decode(3)
    with pytest.raises(RuntimeError, match="at most 8 steps"):
        gd.decode(1)
    assert len(replays) == 13
    with pytest.raises(RuntimeError, match="leave the caches' 40"):
        gd.start(torch.zeros((2, 41), dtype=torch.long), prefill=False)


def test_runner_refuses_pages_of_no_size():
    for page in (0, -16):
        with pytest.raises(RuntimeError, match="must be positive"):
            _runner("mxfp4", page=page)
    with pytest.raises(RuntimeError, match="must be positive"):
        _runner("mxfp4", max_len=0)


@pytest.mark.gpu
@pytest.mark.parametrize("base", [39, 40, 47, 48, 5000])
def test_rows_past_the_caches_under_a_device_position_are_reported(base):
    """A captured step's position is read on the device: a row past max_len writes
    nothing and is reported; the caches and the device go on."""
    from moe_fused_inference_b200 import _lib
    from moe_fused_inference_b200.model import LibBackend, SyntheticQwen
    cfg = QwenConfig(hidden=512, layers=1, heads=8, kv_heads=2, head_dim=64, vocab=4099, experts=16,
                     top_k=4, inter=256)
    model = SyntheticQwen.build(cfg, seed=1)
    r = Runner(model, LibBackend(model), 2, 40, kv="mxfp4", page=16)
    prompt = torch.randint(0, cfg.vocab, (2, 40), generator=torch.Generator().manual_seed(2)).cuda()
    r.prefill(prompt)
    before = r.kv4[0].data.clone()
    step = torch.full((1,), base, dtype=torch.int32, device="cuda")
    logits, _ = r.forward(prompt[:, -1:], step, last_only=True)
    assert logits.shape == (2, cfg.vocab)
    assert (_lib.device_error(clear=True) == 12) == (base >= 40)
    assert torch.equal(r.kv4[0].data, before) == (base >= 40)
    want, _ = r.forward(prompt[:, -1:], 39, last_only=True)
    assert want.isfinite().all() and _lib.device_error(clear=True) == 0
    if base == 39:
        assert torch.equal(want, logits)
