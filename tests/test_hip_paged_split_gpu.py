"""The two bf16 parts of a probability in the bf16 attention: together they hold it to 2^-16.  Three keys a row, of probabilities 1, p and 1 before the division: values
-b, 1 and -c with b + c next to p cancel in the sum, so the result is what the parts leave out (and fp32 roundings)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def bf16(x):
    return torch.from_numpy(x).to(BF).double().numpy()


def test_parts_of_a_probability_leave_out_at_most_2_16():
    from vilmedic_amd import ops
    N = 8192
    x = np.random.default_rng(0).uniform(-np.log(2.0), 0.0, N)
    hi = bf16(x)
    lo = bf16((x - hi) * 256)
    score = hi + lo / 256                                     # 16 bits: exact in fp32
    p = np.exp(score)
    b = bf16(p)
    c = bf16(p - b)
    k, v = torch.zeros(N, 1, 16, 8), torch.zeros(N, 1, 16, 8)
    k[:, 0, 1, 0], k[:, 0, 1, 1] = torch.from_numpy(hi).float(), torch.from_numpy(lo).float()
    v[:, 0, 0], v[:, 0, 1], v[:, 0, 2] = -torch.from_numpy(b).float()[:, None], 1.0, -torch.from_numpy(c).float()[:, None]
    q = torch.tensor([1, 1 / 256, 0, 0, 0, 0, 0, 0]).expand(N, 1, 8).contiguous()
    dev = torch.device("cuda:0")
    table, lengths = torch.arange(N, dtype=torch.int32, device=dev)[:, None].contiguous(), torch.full((N,), 3, dtype=torch.int32, device=dev)
    got = ops.paged_attention(q.to(BF).to(dev), k.to(BF).to(dev), v.to(BF).to(dev), table, lengths, 1.0).double().cpu().numpy()[:, 0]
    want = ((p - b - c) / (2 + p))[:, None]
    # fp32: the score's change of base and the exponential move p by at most 4 steps, the sum of three products of at most 1 by at most 4 half steps
    tol = ((2.0 ** -16 + 4 * 2.0 ** -23) * p + 4 * 2.0 ** -24 * 3)[:, None] / (2 + p)[:, None] + 2.0 ** -8 * np.abs(want) + 2.0 ** -24 * np.abs(want) * 8
    # (the result's own rounding to bf16, of the result with that error in it)
    tol = tol * (1 + 2.0 ** -8)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


def test_infinite_values_of_tiny_weights_stay_infinite():
    """a weight of 2^-60 .. 2^-100 times infinity is infinity, in every column, whatever the weight's bits"""
    from vilmedic_amd import ops
    N = 512
    score = torch.linspace(-100 * 0.6931, -60 * 0.6931, N).to(BF)
    k, v = torch.zeros(N, 1, 16, 16, dtype=BF), torch.randn(N, 1, 16, 16, generator=torch.Generator().manual_seed(1)).to(BF)
    k[:, 0, 1, 0] = score
    v[:, 0, 1] = float("inf")
    v[::2, 0, 1] = float("-inf")
    q = torch.zeros(N, 1, 16, dtype=BF)
    q[:, :, 0] = 1
    dev = torch.device("cuda:0")
    got = ops.paged_attention(q.to(dev), k.to(dev), v.to(dev), torch.arange(N, dtype=torch.int32, device=dev)[:, None].contiguous(),
                              torch.full((N,), 2, dtype=torch.int32, device=dev), 1.0).cpu()
    assert bool((got[::2] == float("-inf")).all()) and bool((got[1::2] == float("inf")).all())
