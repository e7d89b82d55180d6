"""The serving operators together on the GPU: a decoder with 4-bit pooled caches, an adapter per request and
log probabilities through the engine backend, against the same decoder with the three operators
replaced by the oracle's (everything else the same kernels).  Tolerance: the operators' own are far
below the decoder tests' ``LOGITS_TOL``, which covers what a different rounding of one layer (a
code of the cache one step further, say) does to the next.  The second run takes the experts that the
first one chose, after checking that they are its own choice except where its logits nearly tie: another
expert changes a token's output outright."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ccut_b200.backend import GenericBackend
from tests.gpu_helpers import gpu_layer
from tests.model_helpers import make_tiny, quantized_layers
from tests.serving_helpers import banks, use_standins
from tests.test_z_gpu_engine import LOGITS_TOL, _decoder, _rel_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from ccut_b200 import build
    build.build()


class _Replayed:
    """A ``MoeLayer`` that keeps the routing of its calls, and in a second run replays it in order."""

    def __init__(self, layer):
        self.layer, self.routes, self.replay = layer, [], False

    def forward(self, x, out_dtype=torch.bfloat16):
        if not self.replay:
            out, r = self.layer.forward(x, out_dtype, return_routing=True)
            self.routes.append(r)
            return out
        r = self.routes.pop(0)
        own = self.layer.route(x, want_logits=True)
        k = self.layer.top_k
        best = own.logits.sort(dim=1, descending=True).values
        other = (own.ids.sort(dim=1).values != r.ids.sort(dim=1).values).any(1)
        tie = best[:, k - 1] - best[:, k] <= 2 * LOGITS_TOL * own.logits.abs().amax(1)
        assert bool((~other | tie).all())
        perm = self.layer.permute(r)
        return self.layer.combine(self.layer.expert_ffn(x, perm), perm, x.shape[0], out_dtype=out_dtype)


@pytest.mark.parametrize("kv_heads, head_dim, pool", [(2, 64, True), (1, 128, False)])
def test_backend_serves_int4_caches_adapters_and_logprobs(monkeypatch, kv_heads, head_dim, pool):
    """Prompts of different lengths (one long enough for the long-block attention), then greedy steps with
    adapters 0, 1 and none; logits, tokens' log probabilities and a scored prompt."""
    t = make_tiny(51, kv_heads=kv_heads, head_dim=head_dim)
    qlayers = quantized_layers(t, "awq_int4_g128", seed=51)
    ffns = [_Replayed(gpu_layer(ol.lw)) for ol in qlayers]
    dec = _decoder(t, ffns)
    dec.set_adapters(banks(t, 2, 24, 3, "cuda"))
    rng = np.random.default_rng(1)
    prompts = [[int(x) for x in rng.integers(0, t.vocab, n)] for n in (150, 37, 5)]
    adapters = (1, None, 0)

    def run(steps):
        be = GenericBackend(dec, max_seqs=3, max_len=256, pool=pool, kv_dtype="int4", prefill_chunk=96)
        out = []
        seqs = [list(p) for p in prompts]
        for feed in steps:
            lg = torch.stack(be.logits_batch(seqs, adapters)).cpu().numpy()
            out.append(lg)
            for s, x in zip(seqs, feed):
                s.append(int(x))
        info = [i for _, i in be.generate_batch([(s, {"temperature": 0.0, "adapter": a}) for s, a in zip(seqs, adapters)], 5)]
        return out, info, be.score(prompts[1], 3, adapter=1)

    feeds = rng.integers(0, t.vocab, (4, 3))
    got, info, score = run(feeds)
    use_standins(monkeypatch)
    for f in ffns:
        f.replay = True
    want, info2, score2 = run(feeds)
    assert all(not f.routes for f in ffns)
    for g, w in zip(got, want):
        assert _rel_rows(g, w) <= LOGITS_TOL
    scale = max(float(np.abs(w).max()) for w in want)  # a logit off by LOGITS_TOL * scale moves lp by twice that
    for a, b in zip(info + score, info2 + score2):
        assert abs(a["entropy"] - b["entropy"]) <= 8 * LOGITS_TOL * scale
        assert len(a["top"]) == len(b["top"]) and a["top"] == sorted(a["top"], key=lambda e: -e[1])
    for a, b in zip(score, score2):
        assert abs(a["logprob"] - b["logprob"]) <= 2 * LOGITS_TOL * scale


def test_decoder_loaded_with_int4_caches(tmp_path):
    """``[quant] kv_cache_dtype = "int4"`` of the engine's config reaches the caches of a loaded decoder."""
    from ccut_b200.blocks.attn_kv4 import Kv4Cache, Kv4Pool
    from ccut_b200.checkpoint import load_decoder
    from tests.ckpt_helpers import write_decoder_checkpoint

    t = make_tiny(52, kv_heads=2)
    write_decoder_checkpoint(tmp_path / "m", t, "awq_int4_g128", quantized_layers(t, "awq_int4_g128", seed=52))
    dec = load_decoder(tmp_path / "m", app_config={"quant": {"kv_cache_dtype": "int4"}})
    assert isinstance(dec.new_cache(8), Kv4Cache) and isinstance(dec.new_pool(2, 8), Kv4Pool)
    be = GenericBackend(dec, max_seqs=2, max_len=64, pool=True)
    toks = be.generate_batch([([1, 2, 3], {"temperature": 0.0}), ([4, 5], {"temperature": 0.0})])
    assert all(0 <= x < t.vocab for x in toks) and be._pool.k.dtype == torch.uint8
