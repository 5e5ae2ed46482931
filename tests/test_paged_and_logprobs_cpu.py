"""Refusals of the paged-cache operators and of token_logprobs (no GPU needed: every check of shapes, types, strides and devices comes before the first
device pointer), and the exported workspace sizes."""
import pytest
import torch

from vilmedic_amd import ops
from vilmedic_amd._lib import VmHipError, lib

I32, BF = torch.int32, torch.bfloat16


def plan_args(**kw):
    a = dict(lengths=torch.zeros(3, dtype=I32), new_tokens=torch.ones(3, dtype=I32), block_table=torch.full((3, 4), -1, dtype=I32),
             free_pages=torch.arange(8, dtype=I32), free_ring=torch.tensor([0, 8], dtype=I32), page_size=16, max_tokens=8)
    a.update(kw)
    return a


@pytest.mark.parametrize("bad", [
    dict(lengths=torch.zeros(3, dtype=torch.int64)), dict(lengths=torch.zeros(4, dtype=I32)), dict(new_tokens=torch.ones(2, dtype=I32)),
    dict(new_tokens=torch.ones(6, dtype=I32)[::2]), dict(block_table=torch.zeros(12, dtype=I32)), dict(block_table=torch.zeros(4, 3, dtype=I32).t()),
    dict(block_table=torch.zeros(1, 4, dtype=I32).expand(3, 4)), dict(free_pages=torch.zeros(0, dtype=I32)), dict(free_ring=torch.zeros(3, dtype=I32)),
    dict(page_size=0), dict(max_tokens=-1), dict(max_tokens=(1 << 30) + 1), dict(page_size=1 << 30),
    dict(lengths=torch.zeros(0, dtype=I32), new_tokens=torch.zeros(0, dtype=I32), block_table=torch.zeros(0, 4, dtype=I32)),
])
def test_plan_refuses(bad):
    with pytest.raises(ValueError, match="paged_plan"):
        ops.paged_plan(**plan_args(**bad))


def test_plan_has_no_cpu_fallback():
    with pytest.raises(VmHipError):
        ops.paged_plan(**plan_args())


def kv(T=5, H=2, dh=16, P=3, s=16, dtype=BF):
    return dict(k=torch.zeros(T, H, dh, dtype=dtype), v=torch.zeros(T, H, dh, dtype=dtype), k_pages=torch.zeros(P, H, s, dh, dtype=dtype),
                v_pages=torch.zeros(P, H, s, dh, dtype=dtype), slots=torch.zeros(T, dtype=torch.int64))


@pytest.mark.parametrize("bad", [
    dict(k=torch.zeros(5, 2, 8, dtype=BF)), dict(v=torch.zeros(5, 2, 16)), dict(slots=torch.zeros(5, dtype=I32)), dict(slots=torch.zeros(4, dtype=torch.int64)),
    dict(slots=torch.zeros(10, dtype=torch.int64)[::2]), dict(k_pages=torch.zeros(3, 2, 16, 16)), dict(k_pages=torch.zeros(3, 2, 32, 16, dtype=BF)[:, :, ::2]),
    dict(k=torch.zeros(5, 2, 32, dtype=BF)[..., ::2]), dict(k=torch.zeros(5, 2, 16, dtype=torch.float16), v=torch.zeros(5, 2, 16, dtype=torch.float16)),
    dict(k=torch.zeros(5, 2, 16, dtype=BF, requires_grad=True)), dict(k=torch.zeros(5, 3, 16, dtype=BF), v=torch.zeros(5, 3, 16, dtype=BF)),
    dict(slots=torch.zeros(5, dtype=torch.int64, device="meta")),
])
def test_write_refuses(bad):
    with pytest.raises(ValueError, match="paged_kv_write"):
        ops.paged_kv_write(**{**kv(), **bad})


@pytest.mark.parametrize("shape", [dict(dh=12), dict(dh=264), dict(s=8), dict(s=24), dict(s=48)])
def test_write_and_attention_refuse_the_page_shape(shape):
    a = kv(**shape)
    with pytest.raises(ValueError, match="paged_kv_write"):
        ops.paged_kv_write(**a)
    with pytest.raises(ValueError, match="paged_attention"):
        ops.paged_attention(a["k"], a["k_pages"], a["v_pages"], torch.zeros(5, 1, dtype=I32), torch.zeros(5, dtype=I32))


def test_pages_must_be_aligned():
    a = kv()
    a["k_pages"] = torch.zeros(3 * 2 * 16 * 16 + 8, dtype=BF)[1:1 + 3 * 2 * 16 * 16].view(3, 2, 16, 16)
    with pytest.raises(ValueError, match="multiple of 16 bytes"):
        ops.paged_kv_write(**a)


def attn(N=3, Hq=4, H=2, dh=16, P=3, s=16, M=2, dtype=BF):
    return dict(q=torch.zeros(N, Hq, dh, dtype=dtype), k_pages=torch.zeros(P, H, s, dh, dtype=dtype), v_pages=torch.zeros(P, H, s, dh, dtype=dtype),
                block_table=torch.zeros(N, M, dtype=I32), lengths=torch.zeros(N, dtype=I32))


@pytest.mark.parametrize("bad", [
    dict(q=torch.zeros(3, 4, 24, dtype=BF)), dict(q=torch.zeros(3, 3, 16, dtype=BF)), dict(q=torch.zeros(3, 0, 16, dtype=BF)), dict(q=torch.zeros(3, 4, 16)),
    dict(q=torch.zeros(3, 16, 4, dtype=BF).transpose(1, 2)), dict(q=torch.zeros(3, 4, 16, dtype=BF, requires_grad=True)), dict(q=torch.zeros(3, 64, dtype=BF)),
    dict(block_table=torch.zeros(3, 2, dtype=torch.int64)), dict(block_table=torch.zeros(2, 2, dtype=I32)), dict(block_table=torch.zeros(3, 0, dtype=I32)),
    dict(block_table=torch.zeros(2, 3, dtype=I32).t()), dict(block_table=torch.zeros(1, 2, dtype=I32).expand(3, 2)), dict(lengths=torch.zeros(3, dtype=torch.int64)),
    dict(lengths=torch.zeros(3, 1, dtype=I32)), dict(lengths=torch.zeros(6, dtype=I32)[::2]), dict(lengths=torch.zeros(3, dtype=I32, device="meta")),
])
def test_attention_refuses(bad):
    with pytest.raises(ValueError, match="paged_attention"):
        ops.paged_attention(**{**attn(), **bad})


def test_attention_and_write_have_no_cpu_fallback_and_take_no_rows():
    with pytest.raises(VmHipError):
        ops.paged_attention(**attn())
    with pytest.raises(VmHipError):
        ops.paged_kv_write(**kv())
    ops.paged_kv_write(**kv(T=0))                        # no tokens: nothing to do, nothing launched


@pytest.mark.parametrize("logits,targets,top", [
    (torch.zeros(3, 10, dtype=torch.float16), torch.zeros(3, dtype=torch.int64), 0), (torch.zeros(3, 10, dtype=torch.float64), torch.zeros(3, dtype=torch.int64), 0),
    (torch.zeros(3, 10), torch.zeros(3, dtype=I32), 0), (torch.zeros(3, 10), torch.zeros(4, dtype=torch.int64), 0),
    (torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64), 11), (torch.zeros(3, 100), torch.zeros(3, dtype=torch.int64), 33),
    (torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64), -1), (torch.zeros(3, 0), torch.zeros(3, dtype=torch.int64), 0),
    (torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64, device="meta"), 0),
])
def test_logprobs_refuse(logits, targets, top):
    with pytest.raises(ValueError, match="token_logprobs"):
        ops.token_logprobs(logits, targets, top)


def test_logprobs_without_rows_or_device():
    x = torch.zeros(0, 10, requires_grad=True)
    out = ops.token_logprobs(x, torch.zeros(0, dtype=torch.int64), 3)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0, 3), (0, 3)]
    assert torch.autograd.grad(out.logp.sum() + out.entropy.sum(), x)[0].shape == (0, 10)
    with pytest.raises(VmHipError):
        ops.token_logprobs(torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64))


def test_c_entries_refuse_without_touching_the_device():
    L = lib()
    assert L.vm_paged_plan(None, None, None, 4, 1, 4, None, None, 8, 16, None, None, 0, None, None, None, 0, None) == -1
    assert L.vm_paged_kv_write(None, 0, 0, None, 0, 0, None, None, None, 1, 1, 8, 1, 16, 1, None) == -1
    assert L.vm_paged_attention(None, 0, 0, None, None, None, 1, None, None, 1, 1, 1, 8, 1, 16, 1, 1.0, 1, None, 0, None) == -1
    assert L.vm_token_logprobs_fwd(None, 0, 0, 1, None, 1, 8, 0, None, None, None, None, None, 1, None) == -1
    fake = 1 << 20                                       # a non-null address that is never followed: the refusal is about the numbers
    assert L.vm_token_logprobs_fwd(fake, 8, 8, 1, fake, 1, 8, 9, fake, fake, fake, fake, fake, 1, None) == -1
    assert L.vm_paged_attention(fake, 8, 8, fake, fake, fake, 1, fake, fake, 1, 1, 1, 12, 1, 16, 1, 1.0, 1, None, 0, None) == -1
    assert L.vm_paged_attention(fake, 8, 8, fake, fake, fake, 1, fake, fake, 1, 1, 1, 16, 1, 24, 1, 1.0, 1, None, 0, None) == -1
    assert L.vm_paged_plan(fake, fake, fake, 4, 2000, 4, fake, fake, 8, 16, fake, fake, 8, fake, fake, fake, 8, None) == -1      # workspace too small
    assert L.vm_paged_plan_ws(0, 4, 5) == 0 and L.vm_paged_plan_ws(64, 16, 64) == 0 and L.vm_paged_plan_ws(2000, 4, 5) >= 2000 * 16


def test_paged_cache_holds_its_tensors_and_refuses():
    from vilmedic_amd.paged import PagedKVCache
    c = PagedKVCache(2, 3, 4, 16, 33, dtype=torch.float32, device="cpu")
    assert c.pages.shape == (2, 2, 9, 4, 16, 16) and c.block_table.shape == (3, 3) and c.free_ring.tolist() == [0, 9]
    c.free_ring[0], c.free_ring[1], c.lengths[1] = 5, 2, 7
    c.free_pages.fill_(3)
    c.reset()
    assert c.free_ring.tolist() == [0, 9] and c.free_pages.tolist() == list(range(9)) and not c.lengths.any() and bool((c.block_table == -1).all())
    for bad in (dict(page_size=24), dict(page_size=8), dict(pages=0), dict(max_tokens=0), dict(rows=0), dict(layers=0)):
        with pytest.raises(ValueError, match="PagedKVCache"):
            PagedKVCache(**{**dict(layers=1, rows=2, heads=1, head_dim=16, max_tokens=20, device="cpu"), **bad})


def test_generate_refuses_paged_caches_where_they_do_not_serve():
    from vilmedic_amd.generation import generate

    class Cfg:
        eos_token_id, pad_token_id, bos_token_id = 2, 1, 0

    class Dec:
        config = Cfg()
    ids, enc = torch.zeros(2, 1, dtype=torch.long), torch.zeros(2, 3, 8)
    for kw, err in ((dict(kv_cache="pages"), ValueError), (dict(output_logprobs=3), ValueError), (dict(kv_cache="paged", num_beams=4), NotImplementedError),
                    (dict(output_logprobs=3, num_beams=4, return_dict_in_generate=True), NotImplementedError)):
        with pytest.raises(err):
            generate(Dec(), input_ids=ids, encoder_hidden_states=enc, **kw)
    with pytest.raises(NotImplementedError):
        generate(Dec(), input_ids=ids, hf_models=[Dec(), Dec()], encoders_outputs=[dict(encoder_hidden_states=enc)] * 2, kv_cache="paged")
