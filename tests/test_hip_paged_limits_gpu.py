"""The paged-cache operators and token_logprobs at the ends of the sizes that they accept: sums that pass 31 bits, launches of more than 2^32 threads."""
import pytest
import torch

pytestmark = pytest.mark.gpu

I32, BF, F32 = torch.int32, torch.bfloat16, torch.float32


def dev():
    return torch.device("cuda:0")


def ints(*v):
    return torch.tensor(v, dtype=I32, device=dev())


def test_plan_on_a_ring_of_more_than_2_30_pages():
    """head + P passes 2^31: pages are taken around the ring's end and go back behind its tail"""
    from vilmedic_amd import ops
    P, head = 1_500_000_000, 1_000_000_000
    free = torch.arange(P, dtype=I32, device=dev())
    for at in (head, head - P, P - 1):                        # (a negative head is the same place)
        lengths, table, ring = ints(0, 0, 0), torch.full((3, 2), -1, dtype=I32, device=dev()), ints(at, 1000)
        slots, positions, cu, granted = ops.paged_plan(lengths, ints(20, 0, 5), table, free, ring, 16, 25)
        pages = [(at % P + k) % P for k in range(3)]
        assert table.tolist() == [pages[:2], [-1, -1], [pages[2], -1]] and granted.tolist() == [20, 0, 5] and cu.tolist() == [0, 20, 20, 25]
        assert slots.tolist() == [pages[j // 16] * 16 + j % 16 for j in range(20)] + [pages[2] * 16 + j for j in range(5)]
        assert ring.tolist() == [(at % P + 3) % P, 997]
        ops.paged_plan(lengths, ints(-1, -1, -1), table, free, ring, 16, 0)
        back = torch.tensor([(at + 1000 + k) % P for k in range(3)], device=dev())
        assert free[back].tolist() == pages and ring.tolist() == [(at % P + 3) % P, 1000] and not lengths.any()
        free[back] = back.to(I32)


@pytest.mark.parametrize("rows", [2, 1500])
def test_plan_with_pages_of_more_than_2_30_tokens(rows):
    """length + page_size passes 2^31 where the page size is no power of two; one launch (2 rows) and two (1500)"""
    from vilmedic_amd import ops
    s, length = 1_200_000_000, 1_100_000_000
    lengths, table = torch.full((rows,), length, dtype=I32, device=dev()), torch.arange(5, 5 + rows, dtype=I32, device=dev())[:, None].contiguous()
    new = torch.zeros(rows, dtype=I32, device=dev())
    new[0], new[-1] = 2, 1
    free, ring = torch.arange(rows + 10, dtype=I32, device=dev()), ints(1, 3)
    slots, positions, cu, granted = ops.paged_plan(lengths, new, table, free, ring, s, 3)
    assert positions.tolist() == [length, length + 1, length] and granted.tolist() == new.tolist()
    assert slots.tolist() == [5 * s + length, 5 * s + length + 1, (4 + rows) * s + length]
    assert ring.tolist() == [1, 3] and table.flatten().tolist() == list(range(5, 5 + rows)) and lengths.tolist() == (length + new).tolist()


def test_write_of_more_than_2_24_tokens():
    from vilmedic_amd import ops
    T = (1 << 24) + 5
    k = torch.randint(-100, 100, (T, 1, 8), dtype=torch.int16, device=dev()).view(BF)
    v = torch.randint(-100, 100, (T, 1, 8), dtype=torch.int16, device=dev()).view(BF)
    P = -(-T // 16)
    pages = torch.zeros(2, P, 1, 16, 8, dtype=BF, device=dev())
    slots = torch.arange(P * 16 - 1, P * 16 - 1 - T, -1, device=dev())
    ops.paged_kv_write(k, v, pages[0], pages[1], slots)
    bits = pages.view(torch.int16).view(2, P * 16, 8).flip(1)
    assert torch.equal(bits[0, :T], k.view(torch.int16)[:, 0]) and torch.equal(bits[1, :T], v.view(torch.int16)[:, 0]) and not bits[:, T:].any()


def test_attention_of_more_than_2_26_rows():
    from vilmedic_amd import ops
    period, N = 4096, (1 << 26) + 4096
    g = torch.Generator().manual_seed(3)
    q = torch.randn(period, 1, 8, generator=g).to(BF).to(dev()).repeat(N // period, 1, 1)
    k, v = (torch.randn(5, 1, 16, 8, generator=g).to(BF).to(dev()) for _ in range(2))
    table = torch.randint(0, 5, (period, 1), generator=g).to(I32).to(dev()).repeat(N // period, 1)
    lengths = torch.randint(0, 17, (period,), generator=g).to(I32).to(dev()).repeat(N // period)
    got = ops.paged_attention(q, k, v, table, lengths)
    few = ops.paged_attention(q[:period], k, v, table[:period], lengths[:period])         # (a wave per row here too)
    assert few.abs().sum() > 0
    assert bool((got.view(N // period, period, 8).view(torch.int16) == few.view(1, period, 8).view(torch.int16)).all())


def test_logprobs_of_more_than_2_26_rows():
    from vilmedic_amd import ops
    period, R, V = 4096, (1 << 26) + 4096, 16
    g = torch.Generator().manual_seed(4)
    x0 = torch.randn(period, V, generator=g).to(BF).to(dev())
    t0 = torch.randint(-1, V, (period,), generator=g).to(dev())
    g0 = torch.randn(period, generator=g).to(dev())

    def both(n):
        x = x0.repeat(n, 1).requires_grad_(True)
        out = ops.token_logprobs(x, t0.repeat(n), 1)
        dx, = torch.autograd.grad([out.logp, out.entropy], [x], [g0.repeat(n), torch.ones(n * period, device=dev())])
        return [out.logp.detach(), out.entropy.detach(), out.top_logp.detach(), out.top_ids, dx]
    for many, few in zip(both(R // period), both(1)):
        assert few.abs().sum() > 0
        assert bool((many.view(R // period, -1) == few.view(1, -1)).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dh,length", [(64, 1), (64, 40), (40, 33), (64, 9000), (192, 70)])
def test_attention_of_rows_whose_scores_are_all_minus_infinity(dtype, dh, length):
    """no key with a score above -inf: zeros, also where the values are infinite (and in one launch as well as in split rows)"""
    from vilmedic_amd import ops
    M = -(-length // 16)
    k, v = torch.zeros(M + 1, 2, 16, dh, dtype=dtype, device=dev()), torch.ones(M + 1, 2, 16, dh, dtype=dtype, device=dev())
    k[..., dh - 1] = -float("inf")
    v[:, 1] = float("inf")
    q = torch.ones(2, 4, dh, dtype=dtype, device=dev())
    table = torch.arange(1, M + 1, dtype=I32, device=dev()).expand(2, M).contiguous()
    lengths = ints(length, length)
    assert not ops.paged_attention(q, k, v, table, lengths).any()
    k[1, :, 0] = 0                                            # one key of weight 1 in page 1, which both rows start with
    out = ops.paged_attention(q, k, v, table, lengths)
    assert bool((out[:, :2] == 1).all())
