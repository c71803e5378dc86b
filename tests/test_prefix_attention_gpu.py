"""Attention of sequences that share pages, against the definition in 64 bits.

Every batch is made so that a wrong page, key or row shows: shuffled pages, unequal groups and sequences, and NaN in every
place of the cache that no sequence holds (what lies behind a sequence's last position in its last page included).

The bound on an element of the result is derived from the arithmetic, per row, with u = 2^-24: a score of D products in
32 bits is off by at most (D + 8) u sum |q k| scale, so a weight by twice that at most, relatively; sums over n keys, the parts' maxima
and the division add (n + 16) u; tensor cores may drop bits below the largest term, so all of this counts four times. A
bfloat16 run rounds weights to 8 bits and the result once, each by half a unit in the last place: up to 2^-8 of a value just above a
power of two.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
PAGE = 64
F32, BF16 = torch.float32, torch.bfloat16


def ops():
    import llm_b200.ops as o
    return o


def make(groups, heads, kv_heads, dim, dtype, seed=0, spread=1.0, n_pages=None, extra_width=1, padded=0, poison=float("nan")):
    """groups: [(shared pages, [(own positions held, new tokens), ...]), ...]."""
    gen = torch.Generator().manual_seed(seed)
    lengths, new, first, shared, own_pages = [], [], [0], [], []
    for pages, members in groups:
        for held, n in members:
            lengths.append(pages * PAGE + held + n)
            new.append(n)
            own_pages.append(-(-(held + n) // PAGE))
        first.append(len(lengths))
        shared.append(pages)
    need = sum(shared) + sum(own_pages)
    assert n_pages is None or n_pages >= need + 3
    n_pages = n_pages or need + 3
    free = (torch.randperm(n_pages - 3, generator=gen) + 3).tolist()
    width = max(-(-n // PAGE) for n in lengths) + extra_width
    table = torch.zeros((len(lengths), width), dtype=torch.int32)
    keys = torch.empty((n_pages, kv_heads, PAGE, dim), dtype=dtype, device=DEV)
    values = torch.empty_like(keys)
    if n_pages <= need + 3:
        keys.fill_(poison)
        values.fill_(poison)
    at, filled = 0, {}
    for g, pages in enumerate(shared):
        front, at = free[at:at + pages], at + pages
        for s in range(first[g], first[g + 1]):
            row = front + free[at:at + own_pages[s]]
            at += own_pages[s]
            table[s, :len(row)] = torch.tensor(row, dtype=torch.int32)
            for i, page in enumerate(row):
                filled[page] = max(filled.get(page, 0), min(PAGE, lengths[s] - i * PAGE))
    for page, rows in filled.items():
        if n_pages > need + 3:                               # (a pool too large to be poisoned as a whole)
            keys[page] = poison
            values[page] = poison
        for cache in (keys, values):
            cache[page, :, :rows] = (torch.randn(kv_heads, rows, dim, generator=gen) * spread).to(dtype).to(DEV)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    wide = (torch.randn(cu[-1], heads * dim + padded, generator=gen) * spread).to(dtype).to(DEV)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)
    return dict(q=wide, keys=keys, values=values, table=table.to(DEV), host_table=table.tolist(), lengths=lengths, cu=cu, first=first,
                shared=shared, heads=heads, kv_heads=kv_heads, dim=dim, scale=dim ** -0.5, dtype=dtype,
                arrays=(ints(lengths), ints(cu), ints(first), ints(shared)),
                bounds=dict(max_new=max(max(new), 1), max_group=max(1, max(cu[first[g + 1]] - cu[first[g]] for g in range(len(shared)))),
                            max_shared=max(shared), max_own=max(max(n - p * PAGE for n, p in zip(
                                lengths, [p for p, m in groups for _ in m])), 1)))


def call(b, **more):
    return ops().prefix_attention(b["q"], b["keys"], b["values"], b["table"], *b["arrays"], b["heads"], b["kv_heads"], b["dim"], b["scale"],
                                  **b["bounds"], **more)


def check(b, got):
    """The whole result against the definition in 64 bits, each row within its own bound."""
    heads, dim, share, u = b["heads"], b["dim"], b["heads"] // b["kv_heads"], 2.0 ** -24
    half = 0.0 if b["dtype"] == F32 else 2.0 ** -8
    torch.cuda.synchronize()
    ops().check_device_status()                                        # no wait in a kernel has run out
    assert got.dtype == b["dtype"] and tuple(got.shape) == (b["cu"][-1], heads * dim)
    got = got.double().view(-1, heads, dim)
    for s, length in enumerate(b["lengths"]):
        t0, t1 = b["cu"][s], b["cu"][s + 1]
        if t0 == t1:
            continue
        pages = torch.tensor(b["host_table"][s][:-(-length // PAGE)], dtype=torch.long, device=DEV)
        seen = torch.arange(length, device=DEV)[None, :] <= torch.arange(length - (t1 - t0), length, device=DEV)[:, None]
        for kv in range(b["kv_heads"]):
            k = b["keys"][pages, kv].double().reshape(-1, dim)[:length]
            v = b["values"][pages, kv].double().reshape(-1, dim)[:length]
            for a in range(kv * share, (kv + 1) * share):
                q = b["q"][t0:t1, a * dim:(a + 1) * dim].double()
                scores = (q @ k.T * b["scale"]).masked_fill(~seen, -math.inf)
                want = torch.softmax(scores, -1) @ v
                size = torch.softmax(scores, -1) @ v.abs()
                worst = ((q.abs() @ k.abs().T) * b["scale"]).masked_fill(~seen, 0).amax(-1, keepdim=True)
                bound = (4 * (2 * (dim + 8) * worst + length + 16) * u + half) * size + half * want.abs() + 1e-30
                off = (got[t0:t1, a] - want).abs()
                assert bool((off <= bound).all()), (s, a, float((off / bound).max()))


SHARED = [                                  # (shared pages, members' (held, new)) of every group
    [(1, [(5, 1), (17, 1), (0, 1)])],
    [(3, [(0, 1)] * 2), (0, [(0, 1)]), (0, [(130, 1)]), (2, [(63, 1), (64, 1), (191, 1), (1, 1)])],       # ends in, at and behind a page
    [(5, [(i * 7, 1) for i in range(33)])],                                     # more rows than any tile has
    [(2, [(0, 3), (9, 65), (70, 1), (0, 0), (3, 40)]), (0, [(0, 0)]), (1, [(0, 130), (64, 2)])],      # unequal, some bring nothing
    [(0, [(0, 1)]), (0, [(62, 1)]), (0, [(0, 70)])],                            # nothing is shared
    [(40, [(200, 1), (10, 1), (1500, 1)])],                                     # long enough to be cut into parts
    [(9, [(i, 1) for i in range(5)]), (49, [(40 + i, 1) for i in range(7)]), (20, [(100 * i, 1) for i in range(9)]),
     (33, [(63, 1)] * 11)],                                                     # unequal groups, dealt out in slices of equal length
]
HEADS = [(4, 4, 64), (8, 2, 128), (6, 1, 32), (4, 2, 16), (12, 4, 80), (2, 2, 256), (40, 2, 64), (3, 1, 18), (8, 1, 96)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads, kv_heads, dim", HEADS)
@pytest.mark.parametrize("groups", range(len(SHARED)))
def test_against_the_definition(dtype, heads, kv_heads, dim, groups):
    b = make(SHARED[groups], heads, kv_heads, dim, dtype, seed=groups)
    check(b, call(b))


@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 16, 64), (48, 24, 128), (64, 32, 128), (8, 8, 64), (40, 10, 128)])
@pytest.mark.parametrize("members, new", [(9, 1), (24, 1), (70, 1), (4, 25), (3, 130)])
def test_slices_of_many_pages(heads, kv_heads, dim, members, new):
    """Many key heads leave few blocks for each: a block walks many pages, over every number of them."""
    for pages in (67, 130):
        b = make([(pages, [(17 * i % 90, new) for i in range(members)])], heads, kv_heads, dim, BF16, seed=pages, spread=1.5)
        check(b, call(b))
    b = make([(61 - 13 * g, [(11 * i % 140, new) for i in range(members // 3 + g)]) for g in range(4)], heads, kv_heads, dim, BF16, seed=12, spread=1.5)
    check(b, call(b))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_scores(dtype):
    """Scores of the order of hundreds: the running maximum decides, sums of one key."""
    b = make([(4, [(100, 1), (3, 5)])], 8, 2, 64, dtype, seed=3, spread=6.0)
    check(b, call(b))


@pytest.mark.parametrize("poison", [float("inf"), float("-inf"), 3e38])
@pytest.mark.parametrize("dim", [64, 80])
def test_what_is_left_in_pages_does_not_count(poison, dim):
    b = make(SHARED[1], 8, 2, dim, BF16, seed=4, poison=poison)
    check(b, call(b))
    b = make(SHARED[3], 8, 2, dim, BF16, seed=4, poison=poison)
    check(b, call(b))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_inside_wider_ones_and_a_given_result(dtype):
    b = make(SHARED[3], 8, 2, 64, dtype, seed=5, padded=256)
    out = torch.empty((b["cu"][-1], 512), dtype=dtype, device=DEV)
    assert call(b, out=out) is out
    check(b, out)
    b = make(SHARED[1], 8, 2, 64, dtype, seed=5, padded=3)            # rows on odd places
    check(b, call(b))


def test_bounds_that_are_too_large_change_nothing_but_the_launch():
    b = make(SHARED[3], 8, 2, 64, BF16, seed=6)
    b["bounds"] = dict(max_new=500, max_group=900, max_shared=b["table"].shape[1], max_own=1000)
    check(b, call(b))


@pytest.mark.parametrize("heads, kv_heads, dim", [(4, 2, 64), (8, 2, 128), (4, 2, 48)])
@pytest.mark.parametrize("new", [1, 40])
def test_a_sequence_that_is_not_finite_spoils_no_other(heads, kv_heads, dim, new):
    """Keys and values of one sequence's own pages are infinite or no numbers: the rows of the others, in the same tile, are as before."""
    groups = [(3, [(70, new), (20, new), (0, new), (130, new)])]
    b = make(groups, heads, kv_heads, dim, BF16, seed=20)
    before = call(b)
    check(b, before)
    own = [p for p in b["host_table"][1][3:] if p]
    b["keys"][own] = float("nan")
    b["values"][own] = float("inf")
    got = call(b)
    for s in (0, 2, 3):
        rows = slice(b["cu"][s], b["cu"][s + 1])
        assert torch.equal(got[rows], before[rows])
    assert not torch.isfinite(got[b["cu"][1]:b["cu"][2]].float()).any()


@pytest.mark.parametrize("heads, kv_heads, dim", [(4, 2, 64), (40, 2, 64), (4, 2, 32)])
def test_more_sequences_than_shared_memory_lists(heads, kv_heads, dim):
    """Above 512 sequences lengths and groups are read where they lie: single tokens, and tokens enough for whole walks."""
    b = make([(2, [(i % 70, 1) for i in range(60)]), (1, [(i % 9, 1) for i in range(200)])] + [(0, [(i % 50, 1)]) for i in range(290)],
             heads, kv_heads, dim, BF16, seed=21)
    check(b, call(b))
    b = make([(2, [(i % 70, 1 + 39 * (i % 16 == 0)) for i in range(400)]), (1, [(i % 9, 1) for i in range(130)])], heads, kv_heads, dim, BF16, seed=22)
    check(b, call(b))


@pytest.mark.parametrize("heads, kv_heads, dim", [(8, 2, 64), (32, 8, 128), (16, 2, 128), (4, 2, 64)])
@pytest.mark.parametrize("members, shared", [(9, 2), (9, 9), (9, 70), (40, 1), (40, 2), (40, 33), (70, 7), (70, 17), (140, 3), (140, 40)])
def test_shared_pages_read_by_every_sequence_or_once(heads, kv_heads, dim, members, shared):
    """Few shared pages are read by every sequence itself, many once for all: sizes on both sides, one group and several."""
    b = make([(shared, [(23 * i % 140, 1) for i in range(members)])], heads, kv_heads, dim, BF16, seed=30 + shared)
    check(b, call(b))
    b = make([(shared, [(31 * i % 90, 1) for i in range(members)]), (0, [(5, 1), (0, 0)]), (shared // 2, [(i, 1) for i in range(members // 2)])],
             heads, kv_heads, dim, BF16, seed=31 + shared)
    check(b, call(b))


@pytest.mark.parametrize("heads, kv_heads, dim", [(4, 2, 64), (16, 2, 128)])
def test_more_sequences_than_shared_memory_lists_behind_many_pages(heads, kv_heads, dim):
    """Shared pages that are read once: groups of more rows than a tile holds, and small ones."""
    b = make([(5, [(i % 70, 1) for i in range(300)]), (9, [(i % 40, 1) for i in range(200)])] + [(0, [(i % 50, 1)]) for i in range(60)],
             heads, kv_heads, dim, BF16, seed=41)
    check(b, call(b))
    b = make([(3 + g % 4, [(i * 9 + g, 1) for i in range(7 + g % 5)]) for g in range(62)], heads, kv_heads, dim, BF16, seed=42)
    check(b, call(b))


@pytest.mark.parametrize("members, shared", [(40, 17), (40, 1), (70, 33), (70, 2), (61, 0)])
def test_own_pages_of_unequal_sequences(members, shared):
    """One to two rounds of blocks for own pages, from none to many: long sequences start first, behind each way of reading the shared pages."""
    b = make([(shared, [(137 * i % 900, 1) for i in range(members)])], 16, 8, 64, BF16, seed=50 + shared)
    check(b, call(b))
    b = make([(shared, [(97 * i % 700, 1) for i in range(members - 20)]), (0, [(3, 1), (0, 0), (650, 1)]), (shared // 3, [(200 * i, 1) for i in range(4)])],
             16, 8, 64, BF16, seed=51 + shared)
    check(b, call(b))
    b = make([(shared, [(0, 1)] * (members - 1) + [(600, 1)])], 16, 8, 64, BF16, seed=52 + shared)
    check(b, call(b))


def test_same_result_twice_and_on_another_stream():
    b = make(SHARED[5], 32, 8, 128, BF16, seed=7)
    first = call(b)
    for _ in range(3):
        assert torch.equal(call(b), first)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = call(b)
    side.synchronize()
    assert torch.equal(other, first)


def test_replay_on_other_lengths():
    """A captured call reads lengths, tables and groups from the device: it serves another step of the same bounds."""
    b = make([(3, [(9, 1), (80, 1)]), (1, [(0, 1), (5, 1)])], 8, 2, 64, BF16, seed=8)
    c = make([(4, [(90, 1), (1, 1), (30, 1)]), (2, [(64, 1)])], 8, 2, 64, BF16, seed=9)
    n_pages = max(b["keys"].shape[0], c["keys"].shape[0])
    width = max(b["table"].shape[1], c["table"].shape[1])
    bounds = {k: max(b["bounds"][k], c["bounds"][k]) for k in b["bounds"]}
    held = dict(b, keys=torch.zeros((n_pages, 2, PAGE, 64), dtype=BF16, device=DEV), values=torch.zeros((n_pages, 2, PAGE, 64), dtype=BF16, device=DEV),
                table=torch.zeros((4, width), dtype=torch.int32, device=DEV), q=b["q"].clone(), bounds=bounds,
                arrays=tuple(t.clone() for t in b["arrays"]))

    def load(x):
        held["keys"][:x["keys"].shape[0]] = x["keys"]
        held["values"][:x["values"].shape[0]] = x["values"]
        held["table"].zero_()
        held["table"][:, :x["table"].shape[1]] = x["table"]
        held["q"].copy_(x["q"])
        for to, t in zip(held["arrays"], x["arrays"]):
            to.copy_(t)
    load(b)
    call(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(held)
    for x in (b, c, b):
        load(x)
        graph.replay()
        check(x, out)


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes (and 2^31 elements) of keys, its pages far apart."""
    b = make([(3, [(70, 1), (10, 2)])], 8, 8, 128, BF16, seed=10, n_pages=33500)
    assert b["keys"].numel() > 1 << 31
    check(b, call(b))


def test_refusals():
    from llm_b200.errors import KernelError
    b = make(SHARED[0], 4, 2, 64, BF16)

    def refuses(**change):
        c = dict(b)
        bounds = dict(b["bounds"])
        for k, v in change.items():
            if k in bounds:
                bounds[k] = v
            else:
                c[k] = v
        c["bounds"] = bounds
        with pytest.raises(KernelError):
            call(c)
    refuses(heads=3)                                                   # no multiple of the key heads
    refuses(heads=8)                                                   # more columns than the queries have
    refuses(dim=32)
    refuses(kv_heads=4)
    refuses(keys=b["keys"].float())
    refuses(values=b["values"][:, :, ::2])
    refuses(q=b["q"].half())
    refuses(q=b["q"].t())
    refuses(table=b["table"].long())
    refuses(table=b["table"][:2])
    refuses(arrays=(b["arrays"][0].long(), *b["arrays"][1:]))
    refuses(arrays=(b["arrays"][0], b["arrays"][1][:-1], *b["arrays"][2:]))
    refuses(arrays=(*b["arrays"][:3], b["arrays"][3][:0]))
    refuses(max_new=0)
    refuses(max_group=0)
    refuses(max_shared=-1)
    refuses(max_shared=99)                                             # wider than the table
    refuses(keys=b["keys"].cpu())
    with pytest.raises(KernelError):
        call(b, out=torch.empty((3, 64), dtype=BF16, device=DEV))
    with pytest.raises(KernelError):
        call(dict(b, q=torch.empty((3, 4 * 300), dtype=BF16, device=DEV), keys=torch.empty((2, 2, 64, 300), dtype=BF16, device=DEV),
                  values=torch.empty((2, 2, 64, 300), dtype=BF16, device=DEV), dim=300))


def test_no_token():
    b = make(SHARED[0], 4, 2, 64, BF16)
    assert call(dict(b, q=b["q"][:0])).shape == (0, 256)
