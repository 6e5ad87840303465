"""The model runner over paged 4-bit KV caches (Runner(kv="mxfp4")): every layer's
attention, on the rows that the runner gives it, against the same in torch from
the cache's values; eager decoding against its captured graph."""

import math

import pytest
import torch

from moe_fused_inference_b200 import _lib, kv4
from moe_fused_inference_b200.model import (GraphDecoder, LibBackend, QwenConfig, Runner,
                                            SyntheticQwen, synthetic_prompts)

pytestmark = pytest.mark.gpu

CFG = QwenConfig(hidden=512, layers=3, heads=8, kv_heads=2, head_dim=64, vocab=4099, experts=16,
                 top_k=4, inter=256)


@pytest.fixture(scope="module")
def model():
    return SyntheticQwen.build(CFG, seed=3)


class CheckedAttention(LibBackend):
    """The library, each attention call compared with torch in 32 bits: off by
    half a unit of bf16, and by the bound of oracle/kv4.py's attention (weights
    of 11 bits, scores in 32 bits: the latter here under 2^-12 as well)."""

    calls = 0

    def attention_kv4(self, q, cache, table, lens, M, workspace):
        got = super().attention_kv4(q, cache, table, lens, M, workspace)
        G = q.shape[1] // cache.kv_heads
        for b, L in enumerate(lens.tolist()):
            pos = torch.arange(L, device=q.device)
            k, v = kv4.kv4_read(cache, table[b].long()[pos // cache.page] * cache.page + pos % cache.page,
                                dtype=torch.float32)
            rows = q[b * M:(b + 1) * M].double()
            s = torch.einsum("mhd,lhd->hml", rows, k.double().repeat_interleave(G, 1)) / math.sqrt(q.shape[2])
            s.masked_fill_(pos > (L - M + torch.arange(M, device=q.device))[:, None], -math.inf)
            want = torch.einsum("hml,lhd->mhd", s.softmax(-1), v.double().repeat_interleave(G, 1))
            err = (got[b * M:(b + 1) * M].double() - want).abs()
            assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * v.abs().max()).all()
        self.calls += 1
        return got


@pytest.mark.parametrize("batch,chunk", [(1, 64), (3, 64), (2, 17), (2, 4)])
def test_every_layers_attention_in_a_prompt_and_a_decode_step(model, batch, chunk):
    """Chunks of a prompt (few and many rows), then decode steps."""
    prompt = synthetic_prompts(batch, 150, CFG.vocab, seed=batch)
    be = CheckedAttention(model)
    r = Runner(model, be, batch, 160, kv="mxfp4", page=32)
    tokens, margins = r.greedy(prompt, 5, chunk=chunk)
    assert be.calls == CFG.layers * (-(-149 // chunk) + 5)
    assert tokens.shape == (batch, 5) and margins.isfinite().all()
    assert _lib.device_error(clear=True) == 0


def test_graph_decode_matches_eager_greedy(model):
    prompt = synthetic_prompts(4, 70, CFG.vocab, seed=9)
    greedy, _ = Runner(model, LibBackend(model), 4, 128, kv="mxfp4").greedy(prompt, 40)
    gd = GraphDecoder(Runner(model, LibBackend(model), 4, 128, kv="mxfp4"), 40)
    gd.start(prompt)
    assert torch.equal(gd.decode(40), greedy)
    assert _lib.device_error(clear=True) == 0


def test_runner_refuses_other_caches(model):
    with pytest.raises(RuntimeError, match="kv must be"):
        Runner(model, None, 1, 16, kv="int4")
