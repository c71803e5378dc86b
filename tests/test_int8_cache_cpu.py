"""Refusals of the operators of a cache held in 8 bits: what they check before anything is launched needs no device."""
import pytest
import torch

from llm_b200 import ops
from llm_b200.errors import KernelError


def pages(n=3, kv=2, dim=16, block=16):
    return ops.Int8Pages(torch.zeros(n, kv, 64, dim, dtype=torch.int8), torch.ones(n, kv, 64 // block))


@pytest.mark.parametrize("values, scales", [
    (torch.zeros(3, 2, 64, 16), torch.ones(3, 2, 4)),                                       # not 8 bits
    (torch.zeros(3, 2, 32, 16, dtype=torch.int8), torch.ones(3, 2, 4)),                     # no pages of 64
    (torch.zeros(3, 2, 16, 64, dtype=torch.int8).transpose(2, 3), torch.ones(3, 2, 4)),     # not contiguous
    (torch.zeros(3, 2, 64, 16, dtype=torch.int8), torch.ones(3, 2, 3)),                     # no block of 64 / 3
    (torch.zeros(3, 2, 64, 16, dtype=torch.int8), torch.ones(3, 2, 128)),
    (torch.zeros(3, 2, 64, 16, dtype=torch.int8), torch.ones(3, 1, 4)),
    (torch.zeros(3, 2, 64, 16, dtype=torch.int8), torch.ones(3, 2, 4, dtype=torch.float64)),
    (torch.zeros(3 * 2 * 64 * 16 + 1, dtype=torch.int8)[1:].view(3, 2, 64, 16), torch.ones(3, 2, 4)),      # off 16 bytes
])
def test_pages_that_are_none(values, scales):
    with pytest.raises(KernelError, match="Int8Pages"):
        ops.Int8Pages(values, scales)


def test_what_pages_stand_for():
    p = pages(block=32)
    p.values.copy_(torch.arange(-64, 64).repeat(48).view(p.values.shape))
    p.scales.copy_(torch.exp2(torch.arange(12).float() - 20).view(3, 2, 2))
    want = p.values.double() * p.scales.double().repeat_interleave(32, 2)[..., None]
    assert torch.equal(p.held().double(), want) and torch.equal(p.held(torch.float32).double(), want) and p.block == 32


def step(n=4, heads=4, kv=2, dim=16):
    i32 = dict(dtype=torch.int32)
    return dict(qkv=torch.zeros(n, (heads + 2 * kv) * dim), rope_table=torch.zeros(64, dim), tok_pos=torch.zeros(n, **i32), tok_seq=torch.zeros(n, **i32),
                cu_seqlens=torch.tensor([0, n], **i32), block_table=torch.zeros(1, 2, **i32), ring_pages=2, keys=pages(), values=pages(), n_heads=heads,
                n_kv_heads=kv, head_dim=dim)


@pytest.mark.parametrize("wrong", [
    dict(qkv=torch.zeros(4, 100)), dict(qkv=torch.zeros(4, 128, dtype=torch.float16)), dict(qkv=torch.zeros(128, 4).T), dict(rope_table=torch.zeros(64, 18)),
    dict(rope_table=torch.zeros(64, 7)), dict(rope_table=torch.zeros(64, 16, dtype=torch.float64)), dict(tok_pos=torch.zeros(3, dtype=torch.int32)),
    dict(tok_seq=torch.zeros(4, dtype=torch.int64)), dict(block_table=torch.zeros(2, 2, dtype=torch.int32)), dict(ring_pages=3), dict(ring_pages=0),
    dict(keys=torch.zeros(3, 2, 64, 16)), dict(values=pages(block=64)), dict(values=pages(n=4)), dict(keys=pages(dim=32)), {}])
def test_appends_that_are_refused(wrong):
    with pytest.raises(KernelError):                            # ({}: a call on the CPU)
        ops.rope_cache_write_int8(**{**step(), **wrong})


def attended(n=4, heads=4, kv=2, dim=16):
    i32 = dict(dtype=torch.int32)
    return dict(qkv=torch.zeros(n, heads * dim), keys=pages(), values=pages(), block_table=torch.zeros(1, 2, **i32), ring_pages=2,
                seq_lens=torch.tensor([n], **i32), cu_seqlens=torch.tensor([0, n], **i32), n_heads=heads, n_kv_heads=kv, head_dim=dim, scale=0.25,
                max_new=n, max_len=n)


@pytest.mark.parametrize("wrong", [
    dict(qkv=torch.zeros(4, 60)), dict(qkv=torch.zeros(64, 4).T), dict(qkv=torch.zeros(4, 64, dtype=torch.float16)), dict(n_heads=3), dict(n_kv_heads=1),
    dict(seq_lens=torch.zeros(1)), dict(cu_seqlens=torch.zeros(1, dtype=torch.int32)), dict(seq_order=torch.zeros(2, dtype=torch.int32)), dict(max_new=0),
    dict(max_len=0), dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(ring_pages=3), dict(block_table=torch.zeros(1, 2)),
    dict(values=pages(block=1)), dict(keys=pages(kv=1)), {}])
def test_attentions_that_are_refused(wrong):
    with pytest.raises(KernelError):
        ops.attention_int8(**{**attended(), **wrong})


def test_what_an_integer_does_not_hold_is_refused():
    far = torch.empty_strided((4, 64), (1 << 31, 1), device="meta")
    with pytest.raises(KernelError, match="apart"):
        ops.attention_int8(**{**attended(), "qkv": far})
    table = torch.empty_strided((1, 2), (1 << 31, 1), dtype=torch.int32, device="meta")
    with pytest.raises(KernelError, match="apart"):
        ops.attention_int8(**{**attended(), "block_table": table})
    with pytest.raises(KernelError, match="apart"):
        ops.rope_cache_write_int8(**{**step(), "block_table": table})
    with pytest.raises(KernelError, match="table of angles"):                              # (no rows: not the same as no table)
        ops.rope_cache_write_int8(**{**step(), "rope_table": torch.zeros(0, 16)})
