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
