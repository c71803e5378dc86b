"""Plain statements of the operators of a cache held in 8 bits, for CPU tests of the engine's host logic (with plain_ops.install)."""
import math

import torch

PAGE = 64
exact = None        # where it is a dict: address of a cache's whole numbers -> its rows in 32 bits, which are read in their place


def held_of(cache):
    return cache.held(torch.float32) if exact is None else exact[cache.values.data_ptr()]


def scale_of(largest):
    """The smallest power of two with which `largest` is at most 127 steps."""
    mantissa, exponent = torch.frexp(largest)
    return torch.ldexp(torch.ones_like(largest), (exponent - 7 + (mantissa > 127 / 128)).clamp(min=-126))


def append(cache, rows, page, row):
    """rows [n, Hkv, D] of one block of the cache, from position `row` of the page on."""
    block = cache.block
    if exact is not None:
        whole = exact.setdefault(cache.values.data_ptr(), torch.zeros(cache.values.shape))
        whole[page, :, row:row + len(rows)] = rows.transpose(0, 1)
    at = row // block
    kept = cache.scales[page, :, at].clone() if row % block else torch.zeros(cache.scales.shape[1])
    wanted = scale_of(rows.abs().amax((0, 2)))
    scale = torch.maximum(kept, wanted) if row % block else wanted
    first = at * block
    older = cache.values[page, :, first:row].float() * (kept / scale)[:, None, None]
    cache.values[page, :, first:row] = torch.round(older).to(torch.int8)
    cache.scales[page, :, at] = scale
    cache.values[page, :, row:row + len(rows)] = torch.round(rows / scale[None, :, None]).to(torch.int8).transpose(0, 1)


def rope_cache_write_int8(qkv, rope_table, tok_pos, tok_seq, cu_seqlens, block_table, ring_pages, keys, values, n_heads, n_kv_heads, head_dim,
                          interleaved=False, write_cache=True, out=None):
    x = qkv.float().view(-1, n_heads + 2 * n_kv_heads, head_dim).clone()
    if rope_table is not None:
        n = rope_table.shape[1]
        angles = rope_table[tok_pos.long()][:, None]
        at0 = torch.arange(0, n, 2) if interleaved else torch.arange(n // 2)
        at1 = at0 + (1 if interleaved else n // 2)
        turned = x[:, :n_heads + n_kv_heads]
        low, high = turned[..., at0].clone(), turned[..., at1].clone()
        c, s = angles[..., :n // 2], angles[..., n // 2:]
        turned[..., at0], turned[..., at1] = low * c - high * s, high * c + low * s
    for b in range(len(cu_seqlens) - 1 if write_cache else 0):
        t, end = int(cu_seqlens[b]), int(cu_seqlens[b + 1])
        while t < end:
            p = int(tok_pos[t])
            assert int(tok_seq[t]) == b
            count = min(keys.block - p % keys.block, end - t)
            page = int(block_table[b, p // PAGE % ring_pages])
            append(keys, x[t:t + count, n_heads:n_heads + n_kv_heads], page, p % PAGE)
            append(values, x[t:t + count, n_heads + n_kv_heads:], page, p % PAGE)
            t += count
    queries = x[:, :n_heads].flatten(1).to(qkv.dtype)
    return queries if out is None else out.copy_(queries)


def attention_int8(qkv, keys, values, block_table, ring_pages, seq_lens, cu_seqlens, n_heads, n_kv_heads, head_dim, scale, window=0, *, max_new,
                   max_len, out=None, seq_order=None):
    result = torch.zeros(qkv.shape[0], n_heads, head_dim)
    held = [held_of(cache) for cache in (keys, values)]
    for b in range(len(seq_lens)):
        t0, t1, length = int(cu_seqlens[b]), int(cu_seqlens[b + 1]), int(seq_lens[b])
        assert t1 - t0 <= max_new and length <= max_len
        row = torch.arange(length)
        page = block_table[b].long()[row // PAGE % ring_pages]
        position = torch.arange(length - (t1 - t0), length)
        hidden = row[None] > position[:, None]
        if window:
            hidden |= row[None] <= position[:, None] - window
        for a in range(n_heads):
            k, v = (cache[page, a * n_kv_heads // n_heads, row % PAGE] for cache in held)
            q = qkv[t0:t1, a * head_dim:(a + 1) * head_dim].float()
            result[t0:t1, a] = torch.softmax((q @ k.T * scale).masked_fill(hidden, -math.inf), -1) @ v
    result = result.flatten(1).to(qkv.dtype)
    return result if out is None else out.copy_(result)


def copy_page_scales(scales, source, target):
    flat = scales.view(-1, *scales.shape[-3:])
    flat[:, list(target)] = flat[:, list(source)]


def install(monkeypatch):
    import llm_b200.ops as ops
    for fn in (rope_cache_write_int8, attention_int8, copy_page_scales):
        monkeypatch.setattr(ops, fn.__name__, fn)
