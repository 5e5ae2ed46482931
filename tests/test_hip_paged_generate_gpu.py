"""generate() on the paged cache and with the log probabilities of the emitted tokens, against the contiguous cache and the golden sequences."""
import pytest
import torch

from test_hip_models_gpu import _g7_setup

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda:0")


def setup(golden):
    g, cfg, dec, st, enc, start, common = _g7_setup(golden)
    kw = dict(input_ids=start, encoder_hidden_states=enc.to(dev()), encoder_attention_mask=g["enc_mask"].to(dev()), **common)
    return g, cfg, dec, kw


def peak_pages(seq, eos, page):
    """most pages that are in use at once: a row at position t holds t + 1 tokens, and gives its pages back in the plan after its eos, whose pages can be
    taken from the plan after that on"""
    rows, n = seq.shape
    last = [(seq[b, 1:] == eos).nonzero()[0].item() + 1 if bool((seq[b, 1:] == eos).any()) else n for b in range(rows)]     # tokens fed: positions 0 .. last - 1
    return max(sum(-(-min(t + 1, m) // page) for m in last if t <= m) for t in range(n - 1))


@pytest.mark.parametrize("page", [16, 32])
def test_greedy_on_pages_emits_the_golden_sequences(golden, page):
    g, cfg, dec, kw = setup(golden)
    ref = g["beams1_lp1.0"]["sequences"]
    for _ in range(2):                                   # the second call runs on the kept state and its captured steps
        assert torch.equal(dec.generate(kv_cache="paged", kv_page_size=page, **kw).cpu(), ref)
    assert torch.equal(dec.generate(**kw).cpu(), ref)


def test_eager_steps_on_pages(golden, monkeypatch):
    from vilmedic_amd import generation
    monkeypatch.setattr(generation, "DECODE_GRAPH", False)
    g, cfg, dec, kw = setup(golden)
    assert torch.equal(dec.generate(kv_cache="paged", **kw).cpu(), g["beams1_lp1.0"]["sequences"])


def test_a_pool_of_just_the_pages_in_use_is_enough_and_a_smaller_one_is_refused(golden):
    g, cfg, dec, kw = setup(golden)
    ref = g["beams1_lp1.0"]["sequences"]
    need = peak_pages(ref, 2, 16)
    assert torch.equal(dec.generate(kv_cache="paged", kv_pages=need, **kw).cpu(), ref)
    with pytest.raises(RuntimeError, match="kv_pages"):
        dec.generate(kv_cache="paged", kv_pages=ref.shape[0] - 1, **kw)


def test_bf16_steps_on_pages_stay_near_the_contiguous_ones(golden):
    """the same model step by step on the same tokens: the two caches hold the same bf16 keys and values, their attention kernels round differently"""
    from vilmedic_amd.generation import DecodeState
    g, cfg, dec, kw = setup(golden)
    enc, mask, ref = kw["encoder_hidden_states"], kw["encoder_attention_mask"], g["beams1_lp1.0"]["sequences"].to(dev())
    for dtype, tol in (("fp32", 2e-5), ("bf16", 0.05)):
        a = DecodeState(dec.decoder, enc, mask, 1, ref.shape[1], dtype)
        b = DecodeState(dec.decoder, enc, mask, 1, ref.shape[1], dtype, paged=(16, None))
        for t in range(ref.shape[1] - 1):
            x, y = a.step(ref[:, t], t), b.step(ref[:, t], t)
            assert float((x - y).norm() / x.norm()) <= tol, (dtype, t)
            assert b.paged.lengths.tolist() == [t + 1] * ref.shape[0]


def test_rows_that_finish_give_their_pages_back(golden):
    from vilmedic_amd import generation
    g, cfg, dec, kw = setup(golden)
    generation._STATE_CACHE.pop(dec.decoder, None)
    dec.generate(kv_cache="paged", **kw)
    (st,) = generation._STATE_CACHE[dec.decoder].values()
    lens = st.paged.lengths.tolist()
    seq = g["beams1_lp1.0"]["sequences"]
    done = [bool((seq[b, 1:-1] == 2).any()) for b in range(seq.shape[0])]
    assert all(n == 0 for n, d in zip(lens, done) if d)
    assert st.paged.free_ring[1].item() == st.paged.free_pages.shape[0] - sum(-(-n // 16) for n in lens)


@pytest.mark.parametrize("scores", [False, True])
def test_logprobs_of_the_emitted_tokens(golden, scores):
    """against log_softmax (fp64) of the scores of the step-by-step loop; the fused selection loop must give the same fields"""
    g, cfg, dec, kw = setup(golden)
    ref = dec.generate(output_scores=True, return_dict_in_generate=True, **kw)
    kept = [s.clone() for s in ref.scores]
    out = dec.generate(output_logprobs=3, output_scores=scores, return_dict_in_generate=True, **kw)
    seq = out.sequences
    assert torch.equal(seq.cpu(), g["beams1_lp1.0"]["sequences"])
    B, n = seq.shape[0], seq.shape[1] - 1
    lp = torch.log_softmax(torch.stack(kept, 1).double(), -1)
    assert out.logprobs.logp.shape == (B, n) and out.logprobs.top_ids.shape == (B, n, 3)
    for b in range(B):
        ended = False
        for t in range(n):
            f = [x[b, t] for x in out.logprobs]
            if ended:
                assert f[0] == 0 and f[1] == 0 and not f[2].any() and not f[3].any()
                continue
            tok = int(seq[b, t + 1])
            assert abs(float(f[0]) - float(lp[b, t, tok])) <= 1e-4 and int(f[3][0]) == tok         # greedy: the token is its own best alternative
            assert abs(float(f[1]) + float((lp[b, t].exp() * lp[b, t]).sum())) <= 1e-4
            assert torch.allclose(f[2].double(), lp[b, t, f[3]], atol=1e-4)
            ended = tok == 2


def test_sampled_tokens_have_their_logprobs_too(golden):
    g, cfg, dec, kw = setup(golden)
    out = dec.generate(do_sample=True, top_k=20, bad_words_ids=[[1], [0]], output_logprobs=0, kv_cache="paged", return_dict_in_generate=True,
                       generator=torch.Generator().manual_seed(3), **kw)
    assert out.logprobs.logp.shape == (g["B"], out.sequences.shape[1] - 1) and bool((out.logprobs.logp <= 0).all()) and bool(torch.isfinite(out.logprobs.entropy).all())
    assert out.logprobs.top_ids.shape[-1] == 0 and bool((out.logprobs.logp[:, 0] < 0).all())


def test_the_step_by_step_loop_on_pages(golden):
    g, cfg, dec, kw = setup(golden)
    ref = g["beams1_lp1.0"]["sequences"]
    out = dec.generate(kv_cache="paged", output_scores=True, output_logprobs=1, return_dict_in_generate=True, **kw)
    assert torch.equal(out.sequences.cpu(), ref) and len(out.scores) == ref.shape[1] - 1 and out.logprobs.logp.shape[1] == ref.shape[1] - 1
    need = peak_pages(ref, 2, 16)
    assert torch.equal(dec.generate(kv_cache="paged", kv_pages=need, output_scores=True, return_dict_in_generate=True, **kw).sequences.cpu(), ref)


def test_logprobs_of_an_ensemble_are_those_of_the_summed_logits(golden):
    g, cfg, dec, kw = setup(golden)
    eo = dict(encoder_hidden_states=kw.pop("encoder_hidden_states"), encoder_attention_mask=kw.pop("encoder_attention_mask"))
    call = dict(hf_models=[dec.decoder, dec.decoder], encoders_outputs=[eo, eo], return_dict_in_generate=True, **kw)
    ref = dec.generate(output_scores=True, **call)
    kept = torch.log_softmax(torch.stack([s.clone() for s in ref.scores], 1).double(), -1)
    out = dec.generate(output_logprobs=0, **call)
    assert torch.equal(out.sequences, ref.sequences)
    want = kept.gather(2, out.sequences[:, 1:, None])[..., 0]
    is_eos = (out.sequences[:, 1:] == 2).long()
    live = (torch.cumsum(is_eos, 1) - is_eos) == 0
    assert float((out.logprobs.logp.double() - want)[live].abs().max()) <= 1e-4 and not bool(out.logprobs.logp[~live].any())
