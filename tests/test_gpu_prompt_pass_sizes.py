"""Prompts in several passes are what they are in one: the decoder's scores, its cache and the steps behind it.

Tolerance: one fp32 twin's of test_gpu_prompt_pass, twice (either side is as far from the twin as that).  The products' sums
may go by another order for another number of rows; everything else of a sequence is the same."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")

from test_gpu_prompt_pass import CONFIGS, _prompts, _slack, _want  # noqa: E402
from test_gpu_spec_decode_configs import _pair, _rel  # noqa: E402


def test_prompts_in_several_passes(cuda_dev):
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    mdl, twin = _pair(CONFIGS["qwen3"](), cuda_dev)
    lens = [130, 1, 0, 217, 64, 33, 0]
    prompts = _prompts(3, lens)
    slack = 2 * _slack(_want(twin, prompts[3], cuda_dev), mdl)
    steps = torch.tensor(_prompts(4, [9] * len(lens)), device=cuda_dev)
    dec = TreeSpeculativeDecoder(mdl, batch=len(lens), max_len=300, page=16, packed=True)
    scores = dec.score(prompts, top=3)
    dec.prefill_packed(prompts)
    logits, keys, ctx = dec.forward(steps), dec.cache.k.clone(), dec.ctx.clone()
    for most in (1, 100, 218, 300):
        dec.pass_tokens = most
        for s, w in zip(dec.score(prompts, top=3, rows=50), scores):
            assert s.top_tokens.shape == w.top_tokens.shape
            for x, y in ((s.logprobs, w.logprobs), (s.top_logprobs, w.top_logprobs)):
                assert x.shape == y.shape and (not x.numel() or float((x - y).abs().max()) <= slack)
        dec.cache.k.zero_()
        dec.prefill_packed(prompts)
        assert torch.equal(dec.ctx, ctx) and dec.ctx.tolist() == lens
        assert _rel(dec.forward(steps), logits) <= 2 * 2e-2
        assert torch.equal((dec.cache.k != 0).any(-1), (keys != 0).any(-1))
