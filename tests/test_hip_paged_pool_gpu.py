"""generate() on a paged cache whose pool is too small ends within the next eight steps, on both of its loops."""
import pytest
import torch

from test_hip_paged_generate_gpu import setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(), dict(output_scores=True, return_dict_in_generate=True)])
def test_a_pool_that_is_too_small_is_reported_within_eight_steps(golden, monkeypatch, kw):
    from vilmedic_amd import generation
    g, cfg, dec, call = setup(golden)
    call["max_length"] = 40
    call["eos_token_id"] = cfg["vocab_size"] - 1              # (hardly ever chosen: the rows do not end early)
    steps, step = [], generation.DecodeState.step
    monkeypatch.setattr(generation.DecodeState, "step", lambda self, tokens, t: (steps.append(t), step(self, tokens, t))[1])
    for pages in (g["B"] - 1, 2 * g["B"] - 1):                # the first token, and the seventeenth, finds no page
        steps.clear()
        with pytest.raises(RuntimeError, match="kv_pages"):
            dec.generate(kv_cache="paged", kv_pages=pages, **call, **kw)
        assert len(steps) <= (8 if pages < g["B"] else 24), steps
    steps.clear()
    out = dec.generate(kv_cache="paged", kv_pages=3 * g["B"], **call, **kw)
    assert len(steps) > 24 and (out if torch.is_tensor(out) else out.sequences).shape[0] == g["B"]
