"""Sizes that the paged-cache operators and token_logprobs refuse, and calls that would drop a derivative (no GPU needed)."""
import pytest
import torch

from vilmedic_amd import ops
from vilmedic_amd._lib import lib

I32 = torch.int32


def test_plan_refuses_more_than_2_30_rows():
    N = (1 << 30) + 1
    row = torch.empty(N, dtype=I32, device="meta")
    with pytest.raises(ValueError, match="2\\^30 rows"):
        ops.paged_plan(row, row, torch.empty(N, 1, dtype=I32, device="meta"), torch.empty(8, dtype=I32, device="meta"), torch.empty(2, dtype=I32, device="meta"), 16, 4)
    fake = 1 << 20                  # a non-null address that is never followed: the refusal is about the numbers
    assert lib().vm_paged_plan(fake, fake, fake, 1, N, 1, fake, fake, 8, 16, fake, fake, 4, fake, fake, fake, 1 << 40, None) == -1


def test_write_refuses_tokens_of_2_29_columns():
    k = torch.empty(1, 1 << 21, 256, dtype=torch.bfloat16, device="meta")
    pages = torch.empty(1, 1 << 21, 16, 256, dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="2\\^29 columns"):
        ops.paged_kv_write(k, k, pages, pages, torch.zeros(1, dtype=torch.int64, device="meta"))
    fake = 1 << 20
    assert lib().vm_paged_kv_write(fake, 0, 0, fake, 0, 0, fake, fake, fake, 1, 1 << 21, 256, 1, 16, 1, None) == -1
