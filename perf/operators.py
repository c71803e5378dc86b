"""The operators for sequences that share their first pages: what they are timed on, and what they compute in plain form.

Two operators. `ops.prefix_attention` is the attention of a batch in which groups of sequences have the same first pages of the
cache (several samples of one prompt, several questions behind one document), whose keys and values it reads once for a group.
`ops.copy_pages` is what forking a sequence and compacting a cache do to the pools of pages: whole pages, or the first rows of pages,
copied to other pages in every layer at once.

An attention case says the heads (`heads` over `kv_heads` of `dim`), how many groups there are, how many sequences a group has
(`members_low` to `members_high`, spread over the groups), how many pages of 64 positions its sequences share (`shared_*`, spread over the
groups), how many positions each sequence holds alone (`own_*`) and how many new tokens each brings (`new_*`, spread over the
sequences). The new tokens' keys are in the cache already. A copy case says the pool (`layers` of keys and values, `pages` of them),
how many pages are copied from (`sources`), to how many pages each (`each`), and how many of a page's 64 rows (`rows_*`).
"""
from __future__ import annotations

import math

import torch

DEVICE = "cuda:0"
PAGE = 64                       # positions of a page of the cache
own = False                     # False: the plain form; True: the framework's operators


# ----------------------------------------------------------------------------- the cases

def _attention(name, heads, dim, groups, members, shared, own_held, new=(1, 1), dtype="bfloat16"):
    return {"name": name, "kind": "attention", "dtype": dtype, "heads": heads[0], "kv_heads": heads[1], "dim": dim, "groups": groups,
            "members_low": members[0], "members_high": members[1], "shared_low": shared[0], "shared_high": shared[1],
            "own_low": own_held[0], "own_high": own_held[1], "new_low": new[0], "new_high": new[1]}


def _copy(name, layers, kv_heads, dim, pages, sources, each, rows, dtype="bfloat16"):
    return {"name": name, "kind": "copy", "dtype": dtype, "layers": layers, "kv_heads": kv_heads, "dim": dim, "pages": pages,
            "sources": sources, "each": each, "rows_low": rows[0], "rows_high": rows[1]}


def listed():
    return [
        # the smallest call: three samples of a short prompt on a small 32-bit model
        _attention("tiny_samples_fp32", (4, 2), 16, 1, (3, 3), (1, 1), (5, 17), dtype="float32"),
        # one user asks for four samples: the latency of a layer's attention in a decode step
        _attention("samples_4_of_1k", (32, 8), 128, 1, (4, 4), (16, 16), (37, 101)),
        # one key head per query head, eight samples of a prompt half as long as the model's context
        _attention("samples_8_mha_of_2k", (32, 32), 128, 1, (8, 8), (32, 32), (3, 250)),
        # four prompts of unequal length with eight samples each, a small head size
        _attention("four_prompts_of_8", (32, 8), 64, 4, (5, 11), (9, 130), (1, 700)),
        # sixteen samples of the benchmark's long prompt
        _attention("samples_16_of_8k", (32, 8), 128, 1, (16, 16), (128, 128), (1, 256)),
        # the largest decode step: 64 requests behind one document
        _attention("requests_64_of_32k", (32, 8), 128, 1, (64, 64), (512, 512), (64, 1024)),
        # the 32-bit path of the small model's decode step
        _attention("samples_8_of_4k_fp32", (32, 8), 64, 1, (8, 8), (64, 64), (10, 300), dtype="float32"),
        # eight short questions, unequal, behind one document: a prompt step
        _attention("questions_8_behind_8k", (32, 8), 128, 1, (8, 8), (128, 128), (0, 0), (17, 93)),
        # the largest prompt step: long questions, some of them follow-ups
        _attention("questions_16_behind_16k", (32, 8), 128, 1, (16, 16), (256, 256), (0, 130), (120, 510)),
        # the smallest copy: a second sample of a prompt whose last page holds five tokens
        _copy("fork_1", 16, 8, 64, 64, 1, 1, (5, 5)),
        # sixteen samples of a prompt: the partly filled page to sixteen new ones, in all layers
        _copy("fork_16", 32, 8, 128, 96, 1, 16, (37, 37)),
        # the cache is compacted: whole pages move to the front of the pools
        _copy("compact_100", 32, 8, 128, 256, 100, 1, (64, 64)),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.randrange(10)
    if kind == 0:                                        # small 32-bit models
        low = rng.randint(0, 40)
        case = _attention("", (4, 2), 16, rng.randint(1, 3), (1, rng.randint(2, 6)), (1, rng.randint(1, 20)), (low, low + rng.randint(0, 90)),
                          (1, rng.randint(1, 5)), "float32")
    elif kind == 1:                                      # 32-bit decode steps of the small model
        low = rng.randint(0, 100)
        case = _attention("", (32, 8), 64, 1, (2, _log(rng, 2, 16)), (1, _log(rng, 2, 100)), (low, low + rng.randint(0, 300)), dtype="float32")
    elif kind in (2, 3, 4):                              # decode steps: samples of one or of several prompts
        heads, dim = rng.choice((((32, 8), 128), ((32, 8), 128), ((32, 32), 128), ((32, 8), 64)))
        groups = rng.choice((1, 1, 2, 5))
        members = _log(rng, 2, 64 // groups)
        pages = _log(rng, 2, 400 // (groups if heads[1] == 8 else 4 * groups))
        low = rng.randint(0, 200)
        case = _attention("", heads, dim, groups, (max(1, members - rng.randint(0, 3)), members), (max(1, pages - rng.randint(0, pages)), pages),
                          (low, low + _log(rng, 1, 800)))
    elif kind in (5, 6):                                 # prompt steps behind a document
        new = _log(rng, 2, 400)
        low = rng.randint(0, 70)
        case = _attention("", (32, 8), rng.choice((64, 128)), rng.choice((1, 1, 2)), (2, _log(rng, 2, 8)), (1, _log(rng, 2, 200)),
                          (low, low + rng.randint(0, 70)), (max(1, new - rng.randint(0, new)), new))
    elif kind in (7, 8):                                 # forks
        dim, layers = rng.choice(((64, 16), (128, 32)))
        rows = rng.randint(1, 64)
        case = _copy("", layers, 8, dim, rng.randint(70, 120), rng.randint(1, 4), _log(rng, 1, 16), (max(1, rows - rng.randint(0, 20)), rows),
                     rng.choice(("bfloat16", "bfloat16", "float32")))
    else:                                                # compaction
        dim, layers = rng.choice(((64, 16), (128, 32)))
        case = _copy("", layers, 8, dim, 250, _log(rng, 2, 100), 1, (64, 64))
    case.pop("name")
    return case


# ----------------------------------------------------------------------------- inputs

def _spread(count, low, high):
    """`count` whole numbers from low to high, evenly spread, long and short ones mixed."""
    at = [low + (high - low) * i // max(count - 1, 1) for i in range(count)]
    stride = next(s for s in (7, 5, 3, 1) if math.gcd(s, count) == 1)
    return [at[i * stride % count] for i in range(count)]


def _batch(case):
    """(members of each group, shared pages of each group, own positions before the step and new tokens of each sequence)."""
    members = _spread(case["groups"], case["members_low"], case["members_high"])
    shared = _spread(case["groups"], case["shared_low"], case["shared_high"])
    n = sum(members)
    return members, shared, _spread(n, case["own_low"], case["own_high"]), _spread(n, case["new_low"], case["new_high"])


def _copied(case):
    """(source pages, target pages, rows) of a copy, one entry a target; the pages are scattered over the pool."""
    n = case["sources"]
    order = [(i * 37 + 11) % case["pages"] for i in range(case["pages"])] if case["pages"] % 37 else list(range(case["pages"]))
    rows = _spread(n, case["rows_low"], case["rows_high"])
    source = [order[i] for i in range(n) for _ in range(case["each"])]
    return source, order[n:n + n * case["each"]], [rows[i] for i in range(n) for _ in range(case["each"])]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 23)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape):
        return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(generator=gen)

    if case["kind"] == "copy":
        source, target, rows = _copied(case)
        pool = normal(case["layers"], 2, case["pages"], case["kv_heads"], PAGE, case["dim"])
        return {"kind": "copy", "pool": pool, "source": source, "target": target, "rows": rows}

    members, shared, held, new = _batch(case)
    lengths, tables, own_pages = [], [], []
    at = 0
    for m, p in zip(members, shared):
        for _ in range(m):
            i = len(lengths)
            lengths.append(p * PAGE + held[i] + new[i])
            own_pages.append(-(-lengths[i] // PAGE) - p)
    n_pages = sum(shared) + sum(own_pages)
    free = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()      # a used pool: its pages are scattered
    width = max(-(-n // PAGE) for n in lengths) + 1
    i = 0
    for m, p in zip(members, shared):
        front, at = free[at:at + p], at + p
        for _ in range(m):
            tables.append(front + free[at:at + own_pages[i]])
            at += own_pages[i]
            tables[i] += [0] * (width - len(tables[i]))
            i += 1
    first = [sum(members[:g]) for g in range(len(members) + 1)]
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    qkv = normal(cu[-1], (heads + 2 * kv_heads) * dim)              # a layer's projection: the queries are its first columns
    return {
        "kind": "attention", "q": qkv, "keys": normal(n_pages, kv_heads, PAGE, dim), "values": normal(n_pages, kv_heads, PAGE, dim),
        "table": _ints(tables), "seq_lens": _ints(lengths), "cu_seqlens": _ints(cu), "group_first": _ints(first), "group_pages": _ints(shared),
        "heads": heads, "kv_heads": kv_heads, "dim": dim, "scale": dim ** -0.5,
        "host": {"tables": tables, "lengths": lengths, "cu": cu, "first": first, "shared": shared},
        "max_new": max(new), "max_group": max(cu[first[g + 1]] - cu[first[g]] for g in range(len(members))), "max_shared": max(shared),
        "max_own": max(a + b for a, b in zip(held, new)),
    }


# ----------------------------------------------------------------------------- one pass

def run(state):
    if state["kind"] == "copy":
        return _copy_own(state) if own else _copy_plain(state)
    return _attention_own(state) if own else _attention_plain(state)


def _copy_own(state):
    from llm_b200 import ops
    ops.copy_pages(state["pool"], state["source"], state["target"], state["rows"])
    return state["pool"]


def _copy_plain(state):
    """One indexed copy for each number of rows."""
    pool = state["pool"]
    for rows in sorted(set(state["rows"])):
        pairs = [(s, t) for s, t, r in zip(state["source"], state["target"], state["rows"]) if r == rows]
        source = torch.tensor([s for s, _ in pairs], device=pool.device)
        target = torch.tensor([t for _, t in pairs], device=pool.device)
        pool[:, :, target, :, :rows] = pool[:, :, source, :, :rows]
    return pool


def _attention_own(state):
    from llm_b200 import ops
    return ops.prefix_attention(state["q"], state["keys"], state["values"], state["table"], state["seq_lens"], state["cu_seqlens"],
                                state["group_first"], state["group_pages"], state["heads"], state["kv_heads"], state["dim"], state["scale"],
                                max_new=state["max_new"], max_group=state["max_group"], max_shared=state["max_shared"], max_own=state["max_own"])


def _attention_plain(state):
    """Group by group: the shared keys and values are gathered and multiplied once for all of the group's rows, each sequence's own
    ones behind them; both parts of a row are joined over their maxima and sums. In 32 bits, rounded once at the end."""
    heads, kv_heads, dim, host = state["heads"], state["kv_heads"], state["dim"], state["host"]
    q = state["q"][:, :heads * dim]
    share = heads // kv_heads
    out = torch.empty((q.shape[0], heads * dim), dtype=q.dtype, device=q.device)

    def gathered(cache, table_row, first, last):
        """Pages first .. last - 1 of a sequence, [kv heads, positions, dim] in 32 bits."""
        pages = state["table"][table_row, first:last].long()
        return cache[pages].transpose(0, 1).reshape(kv_heads, (last - first) * PAGE, dim).float()

    def part(rows, keys, values, hidden=None):
        """(maximum, sum, weighted values) of rows [kv heads, n, dim] over keys; `hidden` [n, positions]: what a row does not see."""
        scores = torch.matmul(rows, keys.transpose(1, 2))
        if hidden is not None:
            scores.masked_fill_(hidden, -math.inf)
        top = scores.amax(-1, keepdim=True)
        weights = torch.exp_(scores.sub_(top))
        return top, weights.sum(-1, keepdim=True), torch.matmul(weights, values)

    for g, pages in enumerate(host["shared"]):
        a, b = host["first"][g], host["first"][g + 1]
        t0, t1 = host["cu"][a], host["cu"][b]
        # rows of a key head: token after token, the query heads that share it
        rows = (q[t0:t1].float() * state["scale"]).view(t1 - t0, kv_heads, share, dim).transpose(0, 1).reshape(kv_heads, -1, dim)
        m, l, o = part(rows, gathered(state["keys"], a, 0, pages), gathered(state["values"], a, 0, pages))
        for s in range(a, b):
            n, length = host["cu"][s + 1] - host["cu"][s], host["lengths"][s]
            of = slice((host["cu"][s] - t0) * share, (host["cu"][s + 1] - t0) * share)
            last = -(-length // PAGE)
            keys = gathered(state["keys"], s, pages, last)[:, :length - pages * PAGE]
            values = gathered(state["values"], s, pages, last)[:, :length - pages * PAGE]
            hidden = None
            if n > 1:
                position = torch.arange(length - n, length, device=q.device).repeat_interleave(share)
                hidden = torch.arange(pages * PAGE, length, device=q.device)[None, :] > position[:, None]
            m1, l1, o1 = part(rows[:, of], keys, values, hidden)
            top = torch.maximum(m[:, of], m1)
            w0, w1 = torch.exp(m[:, of] - top), torch.exp(m1 - top)
            mixed = (o[:, of] * w0 + o1 * w1) / (l[:, of] * w0 + l1 * w1)
            out[host["cu"][s]:host["cu"][s + 1]] = mixed.view(kv_heads, n, share, dim).transpose(0, 1).reshape(n, heads * dim).to(q.dtype)
    return out


# ----------------------------------------------------------------------------- from the definition, in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "copy":
        pool = state["pool"].double()
        for s, t, r in zip(state["source"], state["target"], state["rows"]):
            for row in range(r):
                pool[:, :, t, :, row, :] = pool[:, :, s, :, row, :]
        return pool
    heads, dim, share = state["heads"], state["dim"], state["heads"] // state["kv_heads"]
    out = torch.zeros((state["host"]["cu"][-1], heads, dim), dtype=torch.float64, device=DEVICE)
    for s, length in enumerate(state["host"]["lengths"]):
        # position j of the sequence is row j % 64 of its page j // 64; nothing is known of what it shares
        used = _ints(state["host"]["tables"][s][:-(-length // PAGE)]).long()
        t0, t1 = state["host"]["cu"][s], state["host"]["cu"][s + 1]
        for a in range(heads):
            k = state["keys"][used, a // share].double().reshape(-1, dim)[:length]
            v = state["values"][used, a // share].double().reshape(-1, dim)[:length]
            scores = state["q"][t0:t1, a * dim:(a + 1) * dim].double() @ k.T * state["scale"]
            scores = scores.masked_fill(torch.ones_like(scores, dtype=torch.bool).triu(length - (t1 - t0) + 1), -math.inf)
            out[t0:t1, a] = torch.softmax(scores, -1) @ v
    return out.reshape(-1, heads * dim)


# ----------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "copy":
        row = case["layers"] * 2 * case["kv_heads"] * case["dim"] * size
        rows = sum(_spread(case["sources"], case["rows_low"], case["rows_high"]))
        return {"bytes": row * rows * (1 + case["each"]), "flops": 0}
    members, shared, held, new = _batch(case)
    position = 2 * case["kv_heads"] * case["dim"] * size                       # a position's key and value in all heads
    rows = 2 * sum(new) * case["heads"] * case["dim"] * size                   # queries and results
    flops, i = 0, 0
    for m, p in zip(members, shared):
        for _ in range(m):
            seen = new[i] * (p * PAGE + held[i]) + new[i] * (new[i] + 1) // 2
            flops += 4 * case["heads"] * case["dim"] * seen
            i += 1
    return {"bytes": position * (sum(shared) * PAGE + sum(held) + sum(new)) + rows, "flops": flops}
