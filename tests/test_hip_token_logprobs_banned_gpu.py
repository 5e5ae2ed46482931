"""Gradients of token_logprobs through log probabilities of columns at -inf: a banned target, alternatives where fewer columns are left."""
import pytest
import torch

from test_hip_token_logprobs_gpu import close, dev, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,top", [(12, 0), (12, 12), (700, 3), (4003, 32), (40001, 5)])
def test_gradient_of_banned_targets_and_alternatives_as_log_softmax_has_it(dtype, V, top):
    from vilmedic_amd import ops
    R = 6
    x, _, (gl, gh) = make(R, V, dtype, seed=V + top)
    t = torch.tensor([4, 0, V - 1, 4, 2, 5])
    x[0, 4] = -float("inf")                                   # one banned target
    x[1, :V // 2] = -float("inf")
    x[2, V - 1] = x[2, 0] = -float("inf")
    x[3, 1:] = -float("inf")                                  # one column left, the target and the other alternatives banned
    gt = torch.randn(R, top, generator=torch.Generator().manual_seed(1))
    xd = x.to(dev()).requires_grad_(True)
    out = ops.token_logprobs(xd, t.to(dev()), top)
    (logp, e_l), _, _, ids, (dx, e_dx) = reference(x, t, top, (gl, gh, gt))
    close(out.logp.detach(), logp, e_l, "logp")
    assert torch.isinf(out.logp[:4]).all() and torch.equal(out.top_ids.cpu(), ids)
    outs, gs = [out.logp, out.entropy], [gl.to(dev()), gh.to(dev())]
    if top:
        outs, gs = outs + [out.top_logp], gs + [gt.to(dev())]
    grad = torch.autograd.grad(outs, xd, gs)[0]
    close(grad, dx, e_dx, "gradient", dtype)
    assert bool(torch.isfinite(grad).all())
    # columns at -inf that are neither target nor alternative: exactly nothing
    own = torch.zeros(R, V, dtype=torch.bool)
    own.scatter_(1, t[:, None], True)
    own.scatter_(1, ids, True)
    assert not bool(grad.cpu()[torch.isinf(x) & ~own].any())
