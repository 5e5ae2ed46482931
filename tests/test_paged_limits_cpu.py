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


@pytest.mark.parametrize("which", ["k", "v", "k_pages", "v_pages", "q", "logits", "no rows"])
def test_forward_mode_derivatives_are_refused_and_not_dropped(which):
    from torch.autograd import forward_ad
    from vilmedic_amd._lib import VmHipError
    t = dict(k=torch.zeros(5, 2, 16), v=torch.zeros(5, 2, 16), k_pages=torch.zeros(3, 2, 16, 16), v_pages=torch.zeros(3, 2, 16, 16), q=torch.zeros(5, 4, 16),
             logits=torch.zeros(5, 10))
    table, lengths, slots, targets = torch.zeros(5, 1, dtype=I32), torch.zeros(5, dtype=I32), torch.zeros(5, dtype=torch.int64), torch.zeros(5, dtype=torch.int64)
    if which == "no rows":
        t["logits"], targets = t["logits"][:0], targets[:0]
    calls = {"paged_kv_write": lambda: ops.paged_kv_write(t["k"], t["v"], t["k_pages"], t["v_pages"], slots),
             "paged_attention": lambda: ops.paged_attention(t["q"], t["k_pages"], t["v_pages"], table, lengths),
             "token_logprobs": lambda: ops.token_logprobs(t["logits"], targets)}
    meant = {"k": ["paged_kv_write"], "v": ["paged_kv_write"], "q": ["paged_attention"], "logits": ["token_logprobs"], "no rows": ["token_logprobs"]}
    meant = meant.get(which, ["paged_kv_write", "paged_attention"])
    key = "logits" if which == "no rows" else which
    with forward_ad.dual_level():
        plain = t[key]
        for name in calls if which != "no rows" else []:
            with pytest.raises(VmHipError):                   # no tangent: the call goes on (to the refusal of CPU tensors)
                calls[name]()
        for grad in (False, True):
            t[key] = forward_ad.make_dual(plain, torch.ones_like(plain))
            for name in meant:
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match=name + ".*forward-mode"):
                    calls[name]()


@pytest.mark.parametrize("kw", [dict(kv_page_size=0), dict(kv_page_size=24), dict(kv_page_size=8), dict(kv_page_size=-16), dict(kv_pages=0), dict(kv_pages=-3)])
def test_generate_refuses_page_sizes_and_pools(kw):
    from vilmedic_amd.generation import generate

    class Cfg:
        eos_token_id, pad_token_id, bos_token_id = 2, 1, 0

    class Dec:
        config = Cfg()
    with pytest.raises(ValueError, match="kv_page_size must be"):
        generate(Dec(), input_ids=torch.zeros(2, 1, dtype=torch.long), encoder_hidden_states=torch.zeros(2, 3, 8), kv_cache="paged", **kw)
