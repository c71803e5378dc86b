"""The operators of a cache held in 8 bits: what they are timed on, and what they compute in plain form.

Two operators, which belong together. `ops.rope_cache_write_int8` appends a step's keys and values to the pages of the cache: keys
are rotated by their position on the way, keys and values become 8-bit whole numbers with a scale for each block of positions and head,
and the rotated queries are its result. `ops.attention_int8` is causal grouped-query attention over such a cache, for steps of single tokens and
for prompts.

A cache is pages of 64 positions: whole numbers q [pages, kv heads, 64, dim] in 8 bits and scales s [pages, kv heads, 64 / block] in 32 bits, with
q * s the value that is held. Scales are powers of two: the smallest with which the largest value of the block is at most 127 steps. A block
that is continued keeps its scale where that is enough; where it grows, the rows that the block held are divided by the growth and rounded again
(to even), which for a power of two is exact to half a step.

An append case says the heads (`heads` over `kv_heads` of `dim`), the block, how many sequences there are, how many positions each holds
(`held_*`, spread over the sequences) and how many it brings (`new_*`). An attention case says the same; the new tokens' keys are in the cache
already. `window` > 0: a query sees its own position and the window - 1 before it.
"""
from __future__ import annotations

import math

import torch

DEVICE = "cuda:0"
PAGE = 64                       # positions of a page of the cache
own = False                     # False: the plain form; True: the framework's operators


# ----------------------------------------------------------------------------- the cases

def _case(name, kind, heads, dim, seqs, held, new=(1, 1), dtype="bfloat16", block=16, window=0):
    return {"name": name, "kind": kind, "dtype": dtype, "heads": heads[0], "kv_heads": heads[1], "dim": dim, "block": block, "window": window,
            "seqs": seqs, "held_low": held[0], "held_high": held[1], "new_low": new[0], "new_high": new[1]}


def listed():
    return [
        # the smallest append: three sequences of a small 32-bit model, a token each
        _case("append_tiny_fp32", "append", (4, 2), 16, 3, (5, 150), dtype="float32"),
        # a decode step of 64 sequences, most of them in the middle of a block
        _case("append_64", "append", (32, 8), 128, 64, (1, 8000)),
        # the prompts of the benchmark's batch of 16, all in one step
        _case("append_prompts_16", "append", (32, 8), 128, 16, (0, 0), (64, 2048)),
        # the smallest attention: the same small model
        _case("decode_tiny_fp32", "attention", (4, 2), 16, 3, (5, 150), dtype="float32"),
        # one user, a long context: the latency of a layer's attention in a decode step
        _case("decode_1_of_8k", "attention", (32, 8), 128, 1, (8191, 8191)),
        # the benchmark's decode step
        _case("decode_8_of_8k", "attention", (32, 8), 128, 8, (8191, 8191)),
        # the same with all the sequences that it serves at most: the largest decode step
        _case("decode_64_of_8k", "attention", (32, 8), 128, 64, (8191, 8191)),
        # the small model's decode step of requests that came at different times
        _case("decode_64_up_to_8k", "attention", (32, 8), 64, 64, (1, 8191)),
        # the 32-bit path of the small model's decode step
        _case("decode_8_of_4k_fp32", "attention", (32, 8), 64, 8, (3900, 4095), dtype="float32"),
        # a prompt of 2,048 tokens from its start
        _case("prompt_2048", "attention", (32, 8), 128, 1, (0, 0), (2048, 2048)),
        # eight short questions, unequal, each behind a document of its own
        _case("questions_8_behind_8k", "attention", (32, 8), 128, 8, (8100, 8300), (17, 93)),
        # the next turn of four long conversations: the largest prompt step
        _case("turns_4_behind_16k", "attention", (32, 8), 128, 4, (16000, 16500), (120, 510)),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.randrange(10)
    block = rng.choice((16, 16, 16, 1, 4, 64))
    heads, dim = rng.choice((((32, 8), 128), ((32, 8), 128), ((32, 32), 128), ((32, 8), 64), ((32, 4), 64)))
    narrow = heads[1] * dim <= 1024
    if kind == 0:                                        # appends of small 32-bit models
        held, new = rng.randint(0, 200), rng.randint(1, 40)
        case = _case("", "append", (4, 2), 16, rng.randint(1, 8), (rng.randint(0, held), held), (rng.randint(1, new), new), "float32", block)
    elif kind == 1:                                      # appends of decode steps
        held = _log(rng, 1, 8000)
        case = _case("", "append", heads, dim, _log(rng, 1, 64 if narrow else 16), (rng.randint(0, held), held), block=block)
    elif kind == 2:                                      # appends of prompts, some of them continued
        new = _log(rng, 2, 1500 if narrow else 400)
        held = rng.choice((0, rng.randint(1, 300)))
        case = _case("", "append", heads, dim, _log(rng, 1, 12), (rng.randint(0, held), held), (rng.randint(1, new), new), block=block)
    elif kind == 3:                                      # 32-bit decode steps and short prompts
        held, new = _log(rng, 1, 4000), rng.choice((1, 1, rng.randint(2, 40)))
        case = _case("", "attention", *rng.choice((((4, 2), 16), ((32, 8), 64))), _log(rng, 1, 8), (rng.randint(0, held), held), (1, new), "float32", block)
    elif kind in (4, 5, 6):                              # decode steps
        held = _log(rng, 16, 8000 if narrow else 2000)
        case = _case("", "attention", heads, dim, _log(rng, 1, 64), (rng.randint(0, held), held), block=block)
    elif kind == 7:                                      # decode steps of layers with a window
        held = _log(rng, 100, 8000 if narrow else 2000)
        case = _case("", "attention", heads, dim, _log(rng, 1, 32), (rng.randint(0, held), held), block=block, window=_log(rng, 30, 2000))
    elif kind == 8:                                      # prompts from their start
        new = _log(rng, 5, 1500)
        case = _case("", "attention", heads, dim, _log(rng, 1, 6), (0, 0), (rng.randint(1, new), new), block=block, window=rng.choice((0, 0, 333)))
    else:                                                # prompts behind what a cache holds
        new, held = _log(rng, 2, 400), _log(rng, 16, 8000 if narrow else 3000)
        case = _case("", "attention", heads, dim, _log(rng, 1, 6), (rng.randint(0, held), held), (rng.randint(1, new), new), block=block)
    case.pop("name")
    return case


# ----------------------------------------------------------------------------- inputs

def _spread(count, low, high):
    """`count` whole numbers from low to high, evenly spread, long and short ones mixed."""
    at = [low + (high - low) * i // max(count - 1, 1) for i in range(count)]
    stride = next(s for s in (7, 5, 3, 1) if math.gcd(s, count) == 1)
    return [at[i * stride % count] for i in range(count)]


def _batch(case):
    """(positions held before the step, new tokens) of each sequence."""
    return _spread(case["seqs"], case["held_low"], case["held_high"]), _spread(case["seqs"], case["new_low"], case["new_high"])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 31)
    dtype, heads, kv_heads, dim, block = getattr(torch, case["dtype"]), case["heads"], case["kv_heads"], case["dim"], case["block"]
    held, new = _batch(case)
    lengths = [a + b for a, b in zip(held, new)]
    # an append's pool has the pages that it writes to, and a few that it leaves alone; pages in front of those are not looked at
    append = case["kind"] == "append"
    first = [a // PAGE if append else 0 for a in held]
    need = [-(-length // PAGE) - f for length, f in zip(lengths, first)]
    width = max(-(-length // PAGE) for length in lengths) + 1
    n_pages = sum(need) + 3
    free = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()      # a used pool: its pages are scattered
    tables, at = [], 0
    for f, n in zip(first, need):
        tables.append([0] * f + free[at:at + n] + [0] * (width - f - n))
        at += n
    cu = [sum(new[:i]) for i in range(len(new) + 1)]

    def pages():
        """Pages in use: normal values, in blocks whose largest differ."""
        values = torch.empty((n_pages, kv_heads, PAGE, dim), dtype=torch.float16, device=DEVICE)
        whole = torch.empty(values.shape, dtype=torch.int8, device=DEVICE)
        for i in range(0, n_pages, 1024):                # (a part at a time: the cache of the largest case has 10^9 values)
            whole[i:i + 1024] = values[i:i + 1024].normal_(std=30.0, generator=gen).round_().clamp_(-127, 127)
        exponents = torch.randint(-6, -3, (n_pages, kv_heads, PAGE // block), device=DEVICE, generator=gen)
        return whole, torch.exp2(exponents.float())

    (keys, key_scales), (values, value_scales) = pages(), pages()
    state = {"kind": case["kind"], "keys": keys, "key_scales": key_scales, "values": values, "value_scales": value_scales, "table": _ints(tables),
             "seq_lens": _ints(lengths), "cu_seqlens": _ints(cu), "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block,
             "window": case["window"], "scale": dim ** -0.5, "max_new": max(new), "max_len": max(lengths), "ring": width}
    if append:
        # a layer's projection: queries, keys and values side by side; some heads are louder than others, as they are in trained models
        qkv = torch.empty((cu[-1], heads + 2 * kv_heads, dim), dtype=dtype, device=DEVICE).normal_(generator=gen)
        state["qkv"] = qkv.mul_(torch.exp(0.5 * torch.randn((1, heads + 2 * kv_heads, 1), device=DEVICE, generator=gen)).to(dtype)).flatten(1)
        state["tok_seq"] = _ints([i for i, n in enumerate(new) for _ in range(n)])
        state["tok_pos"] = _ints([a + j for a, n in zip(held, new) for j in range(n)])
        angles = torch.arange(width * PAGE, dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        state["angles"] = torch.cat([angles.cos(), angles.sin()], 1).float().to(DEVICE)
        state["held_values"] = [torch.empty(keys.shape, dtype=torch.bfloat16, device=DEVICE) for _ in range(2)]
    else:
        state["q"] = torch.empty((cu[-1], heads * dim), dtype=dtype, device=DEVICE).normal_(generator=gen)
    return state


# ----------------------------------------------------------------------------- one pass

def run(state):
    if state["kind"] == "append":
        queries = _append_own(state) if own else _append_plain(state)
        return queries, _held(state, 0, "keys", "key_scales"), _held(state, 1, "values", "value_scales")
    return _attention_own(state) if own else _attention_plain(state)


def _held(state, i, values, scales):
    """The values that a cache stands for (8 bits times a power of two: exact in bfloat16)."""
    to, whole, s = state["held_values"][i], state[values], state[scales]
    torch.mul(whole.view(*s.shape, -1), s[..., None], out=to.view(*s.shape, -1))
    return to


def _pages_own(state):
    from llm_b200 import ops
    return ops.Int8Pages(state["keys"], state["key_scales"]), ops.Int8Pages(state["values"], state["value_scales"])


def _append_own(state):
    from llm_b200 import ops
    keys, values = _pages_own(state)
    return ops.rope_cache_write_int8(state["qkv"], state["angles"], state["tok_pos"], state["tok_seq"], state["cu_seqlens"], state["table"],
                                     state["ring"], keys, values, state["heads"], state["kv_heads"], state["dim"])


def _append_plain(state):
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    x = state["qkv"].view(-1, heads + 2 * kv_heads, dim).float()
    position, half = state["tok_pos"].long(), dim // 2
    cos, sin = state["angles"][position, None, :half], state["angles"][position, None, half:]
    turned = x[:, :heads + kv_heads]
    low, high = turned[..., :half], turned[..., half:]
    turned = torch.cat([low * cos - high * sin, high * cos + low * sin], -1)
    page = state["table"][state["tok_seq"].long(), position // PAGE].long()
    _store_plain(state, state["keys"], state["key_scales"], turned[:, heads:], page, position)
    _store_plain(state, state["values"], state["value_scales"], x[:, heads + kv_heads:], page, position)
    return turned[:, :heads].flatten(1).to(state["qkv"].dtype)


def _store_plain(state, whole, scales, x, page, position):
    """Rows x [tokens, kv heads, dim] into their pages: the new scale of every block that gets rows, what it held before in steps of
    that scale, then the rows."""
    block, per = state["block"], PAGE // state["block"]
    n_pages, kv_heads = whole.shape[:2]
    row = position % PAGE
    at = page * per + row // block                                                     # the block of each token
    largest = torch.full((n_pages * per, kv_heads), -1.0, device=x.device)
    largest.scatter_reduce_(0, at[:, None].expand(-1, kv_heads), x.abs().amax(-1), "amax")
    first = torch.full((n_pages * per,), block, device=x.device).scatter_reduce_(0, at, row % block, "amin")      # a block's first new row
    mantissa, exponent = torch.frexp(largest)
    wanted = torch.ldexp(torch.ones_like(largest), (exponent - 7 + (mantissa > 127 / 128)).clamp(min=-126))
    before = scales.transpose(1, 2).reshape(n_pages * per, kv_heads)
    kept = (first > 0) & (first < block)                                               # blocks that are continued
    scale = torch.where((first < block)[:, None], torch.where(kept[:, None], torch.maximum(before, wanted), wanted), before)
    steps = whole.view(n_pages, kv_heads, per, block, whole.shape[-1])
    shrink = (before / scale).view(n_pages, per, kv_heads).transpose(1, 2)
    older = torch.arange(block, device=x.device)[None, :] < torch.where(kept, first, 0)[:, None]
    again = torch.round(steps.float() * shrink[..., None, None])
    steps.copy_(torch.where(older.view(n_pages, 1, per, block, 1), again, steps.float()))
    scales.copy_(scale.view(n_pages, per, kv_heads).transpose(1, 2))
    whole[page, :, row] = torch.round(x / scale[at][..., None]).to(torch.int8)


def _attention_own(state):
    from llm_b200 import ops
    keys, values = _pages_own(state)
    return ops.attention_int8(state["q"], keys, values, state["table"], state["ring"], state["seq_lens"], state["cu_seqlens"], state["heads"],
                              state["kv_heads"], state["dim"], state["scale"], state["window"], max_new=state["max_new"], max_len=state["max_len"])


def _attention_plain(state):
    """All sequences at once, as long as the longest: their pages gathered and widened to 32 bits, scores, softmax, values; rounded once
    at the end."""
    heads, kv_heads, dim, share = state["heads"], state["kv_heads"], state["dim"], state["heads"] // state["kv_heads"]
    lengths, cu, device = state["seq_lens"].long(), state["cu_seqlens"].long(), state["q"].device
    n_seqs, pages, most = len(lengths), -(-state["max_len"] // PAGE), state["max_new"]
    table = state["table"][:, :pages].long()

    def gathered(whole, scales):
        x = whole[table].view(n_seqs, pages, *scales.shape[1:], -1).float() * scales[table][..., None]
        return x.view(n_seqs, pages, kv_heads, PAGE, dim).transpose(1, 2).reshape(n_seqs, kv_heads, pages * PAGE, dim)

    new = cu[1:] - cu[:-1]
    ordinal = torch.arange(most, device=device)
    token = (cu[:-1, None] + torch.minimum(ordinal, new[:, None] - 1)).flatten()          # rows behind a sequence's last repeat it
    q = (state["q"][token].float() * state["scale"]).view(n_seqs, most, kv_heads, share, dim).permute(0, 2, 1, 3, 4)
    scores = torch.matmul(q.reshape(n_seqs, kv_heads, most * share, dim), gathered(state["keys"], state["key_scales"]).transpose(2, 3))
    key, position = torch.arange(pages * PAGE, device=device), lengths[:, None] - new[:, None] + ordinal
    hidden = key > position[..., None]
    if state["window"]:
        hidden |= key <= position[..., None] - state["window"]
    scores.view(n_seqs, kv_heads, most, share, -1).masked_fill_(hidden[:, None, :, None], -math.inf)
    weights = torch.exp_(scores.sub_(scores.amax(-1, keepdim=True).clamp_(min=-1e30)))
    out = torch.matmul(weights, gathered(state["values"], state["value_scales"])) / weights.sum(-1, keepdim=True)
    out = out.view(n_seqs, kv_heads, most, share, dim).permute(0, 2, 1, 3, 4).reshape(n_seqs, most, heads * dim)
    return out[ordinal < new[:, None]].to(state["q"].dtype)


# ----------------------------------------------------------------------------- from the definition, in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    return _append_exact(case, state) if case["kind"] == "append" else _attention_exact(case, state)


def _append_exact(case, state):
    """Sequence by sequence and block by block."""
    heads, kv_heads, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    held, new = _batch(case)
    x = state["qkv"].view(-1, heads + 2 * kv_heads, dim).double()
    table, position = state["table"].tolist(), torch.cat([torch.arange(a, a + n, device=DEVICE) for a, n in zip(held, new)])
    angle = state["angles"][position].double()
    pairs = torch.complex(x[:, :heads + kv_heads, :dim // 2], x[:, :heads + kv_heads, dim // 2:])
    pairs = pairs * torch.complex(angle[:, :dim // 2], angle[:, dim // 2:])[:, None]
    turned = torch.cat([pairs.real, pairs.imag], -1)
    outputs = [turned[:, :heads].reshape(-1, heads * dim)]
    for rows, whole, scales in ((turned[:, heads:], state["keys"], state["key_scales"]), (x[:, heads + kv_heads:], state["values"], state["value_scales"])):
        q, s = whole.double(), scales.double()
        token = 0
        for seq, (begin, count) in enumerate(zip(held, new)):
            done = 0
            while done < count:
                p = begin + done
                n = min(block - p % block, count - done)
                page, b, r = table[seq][p // PAGE], p % PAGE // block, p % PAGE
                got = rows[token + done:token + done + n].transpose(0, 1)                     # [kv heads, n, dim]
                size = torch.exp2(torch.ceil(torch.log2(got.abs().amax((1, 2)) / 127)).clamp(min=-126))
                size = torch.where(size * 127 < got.abs().amax((1, 2)), size * 2, torch.where(size * 63.5 >= got.abs().amax((1, 2)), size / 2, size))
                if p % block:
                    size = torch.maximum(size, s[page, :, b])
                    older = q[page, :, b * block:r]
                    older.copy_(torch.round(older * (s[page, :, b] / size)[:, None, None]))
                s[page, :, b] = size
                q[page, :, r:r + n] = torch.round(got / size[:, None, None])
                done += n
            token += count
        outputs.append((q.view(*s.shape, -1) * s[..., None]).view(q.shape))
    return tuple(outputs)


def _attention_exact(case, state):
    heads, dim, share, window = case["heads"], case["dim"], case["heads"] // case["kv_heads"], case["window"]
    held, new = _batch(case)
    tables, out = state["table"].tolist(), torch.zeros((sum(new), heads, dim), dtype=torch.float64, device=DEVICE)
    token = 0
    for seq, (before, count) in enumerate(zip(held, new)):
        length = before + count
        used = torch.tensor(tables[seq][:-(-length // PAGE)], device=DEVICE)
        seen = torch.ones((count, length), dtype=torch.bool, device=DEVICE).tril(before)
        if window:
            seen &= torch.ones_like(seen).triu(before - window + 1)
        for a in range(heads):
            k, v = ((state[n][used, a // share].double() * state[s][used, a // share].double().repeat_interleave(case["block"], 1)[..., None])
                    .reshape(-1, dim)[:length] for n, s in (("keys", "key_scales"), ("values", "value_scales")))
            scores = (state["q"][token:token + count, a * dim:(a + 1) * dim].double() @ k.T * state["scale"]).masked_fill(~seen, -math.inf)
            out[token:token + count, a] = torch.softmax(scores, -1) @ v
        token += count
    return out.reshape(-1, heads * dim)


# ----------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    size, heads, kv_heads, dim = 2 if case["dtype"] == "bfloat16" else 4, case["heads"], case["kv_heads"], case["dim"]
    held, new = _batch(case)
    position = 2 * kv_heads * (dim + 4 / case["block"])                         # a position's key and value in all heads
    if case["kind"] == "append":
        # the projection, the rotated queries, the angles, the new rows in 8 bits
        return {"bytes": sum(new) * (size * dim * (2 * heads + 2 * kv_heads) + 4 * dim + position), "flops": 0}
    read, seen = 0, 0
    for before, count in zip(held, new):
        window = case["window"] or before + count
        read += before + count - max(0, before - window + 1)
        seen += sum(min(before + i + 1, window) for i in range(count))
    return {"bytes": read * position + 2 * sum(new) * heads * dim * size, "flops": 4 * heads * dim * seen}
