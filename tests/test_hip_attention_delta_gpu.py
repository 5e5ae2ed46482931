"""Gradients of attention where the keys, and the values, are nearly alike, as in the last layers of a deep encoder: dS_j = P_j (dP_j - delta) is then a
small difference of large numbers, and an error of delta = sum_j P_j dP_j moves dQ along the mean key.  Against 64 bits, with bounds that count the
roundings of the kernels: dS to bf16 once, the results to bf16 once, everything else in fp32."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
U = 2.0 ** -24          # half a step of fp32


def dev():
    return torch.device("cuda:0")


def reference(q, k, v, do, mask, causal):
    """one head, float64: -> (dq, bound, dk, bound), the bounds without the results' own rounding"""
    L, dh = q.shape
    n = k.shape[0]
    scale = dh ** -0.5
    dead = torch.zeros(L, n, dtype=torch.bool)
    if mask is not None:
        dead |= ~mask[None, :].bool()
    if causal:
        dead |= torch.arange(n)[None, :] > torch.arange(L)[:, None]
    s, size = q @ k.t() * scale, q.abs() @ k.abs().t() * scale
    p = torch.softmax(s.masked_fill(dead, float("-inf")), 1)
    dp = do @ v.t()
    delta = (p * dp).sum(1, keepdim=True)
    ds = p * (dp - delta)
    # P: the scores' sums (dh products), scaled and exponentiated, twice (row maximum and own score), relative
    rel = 2 * ((dh + 2) * U * size.amax(1, keepdim=True) + 4 * U * s.abs().amax(1, keepdim=True) + 4 * U)
    e_dp = (dh + 2) * U * (do.abs() @ v.abs().t())
    # delta: dP's errors, P's errors on dP - delta (their common part cancels but for the fp32 sum of P), its own sum
    e_delta = (p * e_dp).sum(1, keepdim=True) + rel * (p * (dp - delta).abs()).sum(1, keepdim=True) + 2 * (n + 16) * U * ((p * dp.abs()).sum(1, keepdim=True) + delta.abs())
    e = (2.0 ** -8 + rel + (max(L, n) + 4) * U) * ds.abs() + p * (e_dp + e_delta)
    return ds @ k * scale, e @ k.abs() * scale, ds.t() @ q * scale, e.t() @ q.abs() * scale


@pytest.mark.parametrize("dh,L,n,causal,masked", [
    (96, 49, 49, False, False), (96, 197, 50, False, True), (32, 64, 64, False, False), (32, 1, 33, False, False), (128, 60, 60, True, True), (96, 300, 17, False, False)])
def test_attention_gradients_of_keys_that_are_nearly_alike(dh, L, n, causal, masked):
    from vilmedic_amd import ops
    B, H = 2, 3
    g = torch.Generator().manual_seed(dh + n)

    def rows(count, mean, spread):
        return (mean * torch.randn(B, 1, H * dh, generator=g) + spread * torch.randn(B, count, H * dh, generator=g)).to(BF)
    q, k, v, do = rows(L, 0.0, 1.0), rows(n, 1.0, 0.1), rows(n, 4.0, 0.05), rows(L, 0.0, 1.0)
    mask = None
    if masked:
        mask = torch.ones(B, n, dtype=torch.uint8)
        mask[1, n - n // 3:] = 0
    x = [t.to(dev()).requires_grad_(True) for t in (q, k, v)]
    ops.AttentionFn.apply(*x, mask.to(dev()) if masked else None, H, causal, 0.0).backward(do.to(dev()))
    torch.cuda.synchronize()
    for b in range(B):
        for h in range(H):
            c = slice(h * dh, (h + 1) * dh)
            dq, tq, dk, tk = reference(*(t[b, :, c].double() for t in (q, k, v, do)), mask[b] if masked else None, causal)
            for name, got, want, tol in (("dq", x[0].grad, dq, tq), ("dk", x[1].grad, dk, tk)):
                err = (got[b, :, c].double().cpu() - want).abs()
                tol = tol * 1.01 + torch.finfo(BF).eps / 2 * (want.abs() + tol) + 1e-30
                assert bool((err <= tol).all()), (name, b, h, (err / tol).max())
