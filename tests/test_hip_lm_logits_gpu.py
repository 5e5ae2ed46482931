"""A decoder's logits carry a gradient (called without labels): decoder -> logits -> token_logprobs -> loss -> gradients of every parameter, and the head alone against
64 bits, for vocabularies that are no multiple of 8."""
import pytest
import torch

import golden_recipes as R
from test_hip_models_gpu import build_decoder, cosine, rel_l2

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


@pytest.mark.parametrize("B,L,V", [(3, 20, 97), (4, 16, 1000), (2, 32, 1003), (1, 1, 9)])
def test_head_against_64_bits(B, L, V):
    """logits off by (D + 2) u sum |h||E|, so a probability by twice that and token_logprobs' own (V / 64 + 64 + 8 |log p|) u; the gradient of the logits is rounded to
    bf16 once (2^-8), the products run in fp32, dh is rounded to bf16"""
    from vilmedic_amd import ops
    D, Vp, M = 128, (V + 7) // 8 * 8, B * L
    g = torch.Generator().manual_seed(V)
    h = torch.randn(B, L, D, generator=g).to(BF)
    emb = torch.zeros(Vp, D, dtype=BF)
    emb[:V] = (0.15 * torch.randn(V, D, generator=g)).to(BF)
    bias = torch.randn(V, generator=g)
    t = torch.randint(0, V, (B, L), generator=g)
    t[0, 0] = -1
    gl, gh = torch.randn(B, L, generator=g), 0.3 * torch.randn(B, L, generator=g)
    hd = h.to(dev()).requires_grad_(True)
    g_emb, g_bias = torch.zeros(V, D, device=dev()), torch.zeros(V, device=dev())
    old = torch.full((M * Vp * 4,), float("nan"), device=dev())            # what the next buffers held before
    del old
    logits = ops.lm_logits(hd, emb.to(dev()), bias.to(dev()), V, g_emb=g_emb, g_bias=g_bias)
    assert logits.shape == (B, L, V) and logits.dtype == F32 and logits.requires_grad
    out = ops.token_logprobs(logits, t.to(dev()))
    ((out.logp * gl.to(dev())).sum() + (out.entropy * gh.to(dev())).sum()).backward()
    torch.cuda.synchronize()
    h2, E, b = h.double().view(M, D), emb[:V].double(), bias.double()
    x = h2 @ E.t() + b
    lp = torch.log_softmax(x, 1)
    p = lp.exp()
    H = -(p * lp).sum(1, keepdim=True)
    w, wh, tt = torch.where(t >= 0, gl, torch.zeros_like(gl)).double().view(M, 1), gh.double().view(M, 1), t.view(M, 1)
    dl = -p * (w + wh * (lp + H))
    dl.scatter_add_(1, tt.clamp(min=0), w)
    e_x = ((D + 2) * U * (h2.abs() @ E.abs().t() + b.abs())).amax(1, keepdim=True)
    rel = 2 * e_x + (V / 64 + 64 + 8 * lp.abs()) * U
    e_dl = p * ((w.abs() + wh.abs() * (lp.abs() + H)) * rel + wh.abs() * 2 * (rel + (V / 64 + 64) * U * (1 + H))) + 2.0 ** -8 * dl.abs()
    checks = [("dh", hd.grad.view(M, D), dl @ E, e_dl @ E.abs() + (Vp + 4) * U * (dl.abs() @ E.abs()), 2.0 ** -8),
              ("dE", g_emb, dl.t() @ h2, e_dl.t() @ h2.abs() + (M + 4) * U * (dl.abs().t() @ h2.abs()), U),
              ("db", g_bias, dl.sum(0), e_dl.sum(0) + (M + 4) * U * dl.abs().sum(0), U)]
    for name, got, want, tol, half in checks:
        err = (got.double().cpu() - want).abs()
        tol = 1.01 * tol + half * (want.abs() + tol) + 1e-30
        assert bool((err <= tol).all()), (name, (err / tol).max())


@pytest.mark.parametrize("mt", [None, "bert"])
def test_policy_gradient_with_an_entropy_bonus_through_a_decoder(golden, tmp_path, mt):
    from oracle import torch_ref as O
    from vilmedic_amd import ops
    from vilmedic_amd.blocks.huggingface.decoder.decoder_model import DecoderModel
    if mt is None:
        cfg, specials = dict(R.DEC_TINY), {}
        dec, st = build_decoder(cfg, 31)
    else:
        d = golden("g23_proto_towers")[mt + "_dec"]
        cfg, specials = dict(d["cfg"], model_type=mt), d["specials"]
        st = R.rand_state(R.causal_lm_shapes(d["cfg"], mt), 77)
        dec = DecoderModel(dict(proto=R.write_proto_dir(str(tmp_path / "ckpt"), mt, d["cfg"], st))).to(dev())
    B, L, S = 4, 24, 10
    ids, am = R.make_reports(B, L, cfg["vocab_size"], seed=78, **specials)
    gen = torch.Generator().manual_seed(79)
    enc = torch.randn(B, S, cfg["hidden_size"], generator=gen)
    mask = torch.ones(B, S, dtype=torch.bool)
    mask[2, 6:] = False
    enc[~mask] = 0.0
    w = torch.randn(B, L - 1, generator=gen) * am[:, 1:].float()
    stg = {k: v.clone().requires_grad_(True) for k, v in st.items()}
    encg = enc.clone().requires_grad_(True)
    ref = torch.log_softmax(O.decoder_forward(ids, am, encg, mask, stg, cfg)[1][:, :-1], -1)
    ref_loss = -(w * ref.gather(2, ids[:, 1:, None])[..., 0]).sum() / B + 0.1 * (ref.exp() * ref).sum(-1).sum() / B
    ref_loss.backward()
    enc_d = enc.to(dev()).to(BF).requires_grad_(True)
    dec.train()
    call = dict(input_ids=ids.to(dev()), attention_mask=am.to(dev()), encoder_hidden_states=enc_d, encoder_attention_mask=mask.to(dev()))
    logits = dec.decoder(**call)["logits"]
    out = ops.token_logprobs(logits[:, :-1], ids[:, 1:].to(dev()))
    loss = -(w.to(dev()) * out.logp).sum() / B - 0.1 * out.entropy.sum() / B
    assert abs(loss.item() - ref_loss.item()) <= 1e-2 * max(1.0, abs(ref_loss.item())), (loss.item(), ref_loss.item())
    loss.backward()
    torch.cuda.synchronize()
    named = dict(dec.decoder.named_parameters())
    seen = 0
    for n in stg:
        if stg[n].grad is None or n not in named or float(stg[n].grad.norm()) < 1e-6:
            continue
        got = named[n].grad.float().cpu()
        # (a key bias shifts all scores of a row alike: its gradient is rounding noise on both sides)
        if n.endswith("key.bias"):
            continue
        assert cosine(got, stg[n].grad) >= 0.999 and rel_l2(got, stg[n].grad) <= 3e-2, (n, cosine(got, stg[n].grad), rel_l2(got, stg[n].grad))
        seen += 1
    assert seen > 20
    assert cosine(enc_d.grad.float().cpu(), encg.grad) >= 0.999
    with torch.no_grad():
        again = dec.decoder(**call)["logits"]
    assert not again.requires_grad and torch.equal(again, logits.detach())


def test_logits_may_be_changed_in_place_and_the_ones_beside_a_loss_carry_no_gradient():
    from vilmedic_amd import ops
    dec, _ = build_decoder(R.DEC_TINY, 31)
    ids, am = R.make_reports(2, 9, 97, seed=1)
    enc = torch.randn(2, 5, 128, generator=torch.Generator().manual_seed(2)).to(dev()).to(BF)
    dec.eval()
    call = dict(input_ids=ids.to(dev()), attention_mask=am.to(dev()), encoder_hidden_states=enc, encoder_attention_mask=torch.ones(2, 5, dtype=torch.bool, device=dev()))
    logits = dec.decoder(**call)["logits"]
    keep = logits.detach().clone()
    logits[..., 0] = -float("inf")
    out = ops.token_logprobs(logits[:, :-1], ids[:, 1:].to(dev()).clamp(min=1))
    out.logp.sum().backward()
    torch.cuda.synchronize()
    grad = dict(dec.decoder.named_parameters())["lm_head.bias"].grad
    assert bool(torch.isfinite(grad).all()) and grad[0].item() == 0.0 and grad[1:].abs().sum().item() > 0
    assert torch.equal(logits.detach()[..., 1:], keep[..., 1:])
    assert not dec.decoder(**call, labels=call["input_ids"])["logits"].requires_grad
