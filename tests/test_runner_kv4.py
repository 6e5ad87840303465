"""Runner(kv="mxfp4") without a GPU, on the comparison backend with the 4-bit cache of
oracle/kv4.py: the places of the rows in the pool, the lengths and the page table.  The
same rows over a second, contiguous record of what the cache holds give the same
attention; chunks and page sizes do not change the tokens."""

import numpy as np
import pytest
import torch

from moe_fused_inference_b200.layer import MoELayerWeights
from moe_fused_inference_b200.model import LayerWeights, QwenConfig, Runner, SyntheticQwen, synthetic_prompts
from oracle import kv4 as ok
from oracle import mxfp4 as mx
from tests.torch_backend import TorchBackend

CFG = QwenConfig(hidden=64, layers=2, heads=4, kv_heads=2, head_dim=64, vocab=97, experts=8, top_k=2,
                 inter=32)


@pytest.fixture(scope="module")
def model():
    rng = np.random.default_rng(4)

    def packed(n, k):
        p, c = mx.quantize_rows(mx.bf16_round(rng.standard_normal((n, k)).astype(np.float32) * 0.2))
        return torch.from_numpy(p), torch.from_numpy(c)

    def norm(n):
        return torch.from_numpy(1.0 + 0.02 * rng.standard_normal(n).astype(np.float32)).bfloat16()

    H, D = CFG.hidden, CFG.head_dim
    m = SyntheticQwen(CFG, packed(CFG.vocab, H), packed(CFG.vocab, H), norm(H))
    for _ in range(CFG.layers):
        W = mx.make_layer(rng, n_experts=CFG.experts, hidden=H, inter=CFG.inter, std=0.2)
        moe = MoELayerWeights(*(torch.from_numpy(x) for x in (W.wg, W.sg, W.wu, W.su, W.wd, W.sd, W.wr, W.sr)))
        m.layers.append(LayerWeights(packed(CFG.heads * D, H), packed(CFG.kv_heads * D, H),
                                     packed(CFG.kv_heads * D, H), packed(H, CFG.heads * D), norm(D), norm(D),
                                     norm(H), norm(H), moe))
    return m


class Kv4OnHost(TorchBackend):
    """The comparison backend over the restated cache.  ``seen`` records each
    layer's rows in the order of their sequence, as the cache holds them."""

    def __init__(self, model):
        super().__init__(model)
        self.seen = {}

    def workspace_kv4(self, cache, B, M):
        return None

    def write_kv4(self, cache, k, v, slots):
        k, v = k.float().numpy(), v.float().numpy()
        ok.write(cache.data.numpy(), k, v, slots.numpy())
        self.rows = [ok.decode(*ok.encode(x)) for x in (k, v)]

    def attention_kv4(self, q, cache, table, lens, M, workspace):
        B, lens = len(lens), lens.tolist()
        out, _ = ok.attention(q.float().numpy(), cache.data.numpy(), table.numpy(), lens, [M] * B)
        for x, held in zip(self.rows, self.seen.setdefault(id(cache), ([[] for _ in range(B)], [[] for _ in range(B)]))):
            for b in range(B):
                held[b] += list(x[b * M:(b + 1) * M])
        G = q.shape[1] // cache.kv_heads
        for b in range(B):
            k, v = (np.repeat(np.stack(x[b]), G, 1) for x in self.seen[id(cache)])
            assert len(k) == lens[b]
            for r in range(M):
                n = lens[b] - M + r + 1
                s = np.einsum("hd,lhd->hl", q[b * M + r].double().numpy(), k[:n]) / 8.0
                p = np.exp(s - s.max(-1, keepdims=True))
                want = np.einsum("hl,lhd->hd", p / p.sum(-1, keepdims=True), v[:n])
                assert np.allclose(out[b * M + r], want, rtol=0, atol=1e-12)
        return torch.from_numpy(out).float()


@pytest.mark.parametrize("page,chunk", [(16, 64), (16, 7), (32, 16), (48, 5)])
def test_rows_find_their_places(model, page, chunk):
    prompt = synthetic_prompts(2, 40, CFG.vocab, seed=3, motif=8, device="cpu")
    toks, margins = Runner(model, Kv4OnHost(model), 2, 50, kv="mxfp4", page=page).greedy(prompt, 6, chunk=chunk)
    assert toks.shape == (2, 6) and bool((margins >= 0).all())
    base, _ = Runner(model, Kv4OnHost(model), 2, 50, kv="mxfp4", page=64).greedy(prompt, 6)
    assert torch.equal(toks, base)


def test_pages_of_a_sequence_are_its_own(model):
    r = Runner(model, Kv4OnHost(model), 3, 50, kv="mxfp4", page=16)
    assert sorted(r.table.flatten().tolist()) == list(range(r.kv4[0].num_pages))
    assert r.table.shape == (3, 4) and len(r.kv4) == CFG.layers
