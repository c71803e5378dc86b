"""A cache held in 8 bits: appending to it and attention over it, against the definition in 64 bits.

Every batch is made so that a wrong page, key or row shows: shuffled pages, unequal sequences, and scales that are no number in every block
that no sequence holds.

Appending: a rotated element x in 32 bits is off by at most e = 2 u (|x0 c| + |x1 s|), u = 2^-24 (two products and a sum, each rounded by half a
step). So a whole number q is right when |q s - x| <= s / 2 + e, a new scale s when 63.5 s - e < max |x| <= 127 s + e, and what a block held before
is right to the last bit: its whole numbers times a power of two, rounded to even.

Attention, for each element of the result: a score of D products in 32 bits is off by at most (D + 8) u sum |q k| scale, so a weight by
twice that at most, relatively; sums over n keys, the parts' maxima and the division add (n + 16) u; tensor cores may drop bits below the largest term, so
all of this counts four times. In bfloat16 runs weights are rounded to fp16 (2^-11) and the result once (2^-8); values of a page
less than 2^-32 of its largest, and weights less than 2^-38 of the row's largest, may be lost, which adds n 2^-32 max |v|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
PAGE = 64
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def ops():
    import llm_b200.ops as o
    return o


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def pages_of(n_pages, kv_heads, dim, block, gen, low=-6, high=-3):
    """Whole numbers everywhere; scales that are no number everywhere."""
    whole = torch.randint(-127, 128, (n_pages, kv_heads, PAGE, dim), dtype=torch.int8, generator=gen).to(DEV)
    return ops().Int8Pages(whole, torch.full((n_pages, kv_heads, PAGE // block), math.nan, device=DEV))


def make(held, new, heads, kv_heads, dim, dtype, block=16, window=0, ring=None, seed=0, spread=1.0, low=-6, high=-3, padded=0):
    """A step of len(held) sequences. What the sequences hold, new tokens included, has scales 2^low .. 2^high."""
    gen = torch.Generator().manual_seed(seed)
    lengths = [h + n for h, n in zip(held, new)]
    width = ring or max(-(-n // PAGE) for n in lengths) + 1
    need = [min(-(-n // PAGE), width) for n in lengths]
    n_pages = sum(need) + 3
    free = (torch.randperm(n_pages - 3, generator=gen) + 3).tolist()
    table, at = torch.zeros((len(lengths), width), dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(free[at:at + n], dtype=torch.int32)
        at += n
    keys, values = (pages_of(n_pages, kv_heads, dim, block, gen) for _ in range(2))
    for s, length in enumerate(lengths):
        oldest = max(0, -(-length // PAGE) - width) * PAGE
        for p in range(oldest, length, block):
            for cache in (keys, values):
                cache.scales[table[s, p // PAGE % width], :, p % PAGE // block] = torch.exp2(torch.randint(low, high + 1, (kv_heads,), generator=gen).float()).to(DEV)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    wide = (torch.randn(cu[-1], heads * dim + padded, generator=gen) * spread).to(dtype).to(DEV)
    return dict(q=wide, keys=keys, values=values, table=table.to(DEV), ring=width, lengths=lengths, new=new, cu=cu, heads=heads, kv_heads=kv_heads, dim=dim,
                scale=dim ** -0.5, dtype=dtype, window=window, arrays=(ints(lengths), ints(cu)),
                bounds=dict(max_new=max(max(new), 1), max_len=max(max(lengths), 1)))


def call(b, **more):
    return ops().attention_int8(b["q"], b["keys"], b["values"], b["table"], b["ring"], *b["arrays"], b["heads"], b["kv_heads"], b["dim"], b["scale"],
                                b["window"], **{**b["bounds"], **more})


def check(b, got, where=None):
    """The whole result against the definition in 64 bits, each element within its own bound. `where`: the tokens that are looked at."""
    heads, dim, share, window = b["heads"], b["dim"], b["heads"] // b["kv_heads"], b["window"]
    weight, half = (0.0, 0.0) if b["dtype"] == F32 else (2.0 ** -11, 2.0 ** -8)
    torch.cuda.synchronize()
    ops().check_device_status()
    assert got.dtype == b["dtype"] and tuple(got.shape) == (b["cu"][-1], heads * dim)
    got, table = got.double().view(-1, heads, dim), b["table"].tolist()
    held = [cache.held(torch.float64) for cache in (b["keys"], b["values"])]
    for s, length in enumerate(b["lengths"]):
        t0, t1 = b["cu"][s], b["cu"][s + 1]
        if t0 == t1:
            continue
        first = max(0, length - (t1 - t0) - window + 1) if window else 0
        position, row = torch.arange(length - (t1 - t0), length, device=DEV), torch.arange(first, length, device=DEV)
        page = torch.tensor(table[s], device=DEV)[row // PAGE % b["ring"]]
        seen = row[None, :] <= position[:, None]
        if window:
            seen &= row[None, :] > position[:, None] - window
        for kv in range(b["kv_heads"]):
            k, v = (cache[page, kv, row % PAGE] for cache in held)
            for a in range(kv * share, (kv + 1) * share):
                q = b["q"][t0:t1, a * dim:(a + 1) * dim].double()
                scores = (q @ k.T * b["scale"]).masked_fill(~seen, -math.inf)
                weights = torch.softmax(scores, -1)
                want, size = weights @ v, weights @ v.abs()
                worst = ((q.abs() @ k.abs().T) * b["scale"]).masked_fill(~seen, 0).amax(-1, keepdim=True)
                bound = (4 * (2 * (dim + 8) * worst + length + 16) * U + weight + half) * size + half * want.abs() + 1e-30
                if weight:
                    bound = bound + length * 2.0 ** -32 * v.abs().max()
                off = (got[t0:t1, a] - want).abs()
                ok = off <= bound
                if where is not None:
                    ok = ok | ~torch.tensor([t in where for t in range(t0, t1)], device=DEV)[:, None]
                assert bool(ok.all()), (s, a, float((off / bound).max()))


STEPS = [                                   # (held, new) of every sequence, window
    ([0], [1], 0),
    ([5, 17, 0], [1, 1, 1], 0),
    ([62, 63, 64, 127, 1500], [1] * 5, 0),                                   # ends in, at and behind a page; cut into parts
    ([i * 7 for i in range(33)], [1] * 33, 0),
    ([0, 9, 70, 0, 3], [3, 65, 1, 0, 40], 0),                                 # unequal, one brings nothing
    ([0, 64], [130, 2], 0),
    ([1000, 0], [70, 300], 0),
    ([2300], [33], 0),
    ([200, 64, 1030, 3], [1] * 4, 65),
    ([200, 64, 1030, 0], [90, 1, 33, 150], 100),
    ([3000, 700], [1, 1], 1),
    ([130, 7], [4, 4], 0),                                                   # a few tokens each
    ([500, 0], [20, 9], 7),
]
HEADS = [(4, 4, 64), (8, 2, 128), (6, 1, 32), (4, 2, 16), (12, 4, 80), (2, 2, 256), (40, 2, 64), (3, 1, 18), (8, 1, 96), (32, 1, 128)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads, kv_heads, dim", HEADS)
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_attention_against_the_definition(dtype, heads, kv_heads, dim, step):
    held, new, window = STEPS[step]
    b = make(held, new, heads, kv_heads, dim, dtype, block=(16, 1, 64, 4)[step % 4], window=window, seed=step)
    check(b, call(b))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("block", [1, 2, 4, 8, 16, 32, 64])
def test_attention_blocks_of_every_size(dtype, block):
    """Scales that differ by 2^24 from block to block."""
    for held, new in (([300, 70], [1, 1]), ([100, 0], [50, 130])):
        b = make(held, new, 8, 2, 128, dtype, block=block, seed=block, low=-20, high=4, spread=0.02)
        check(b, call(b))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("spread", [1e-18, 40.0, 3e6])
def test_attention_small_and_large_queries(dtype, spread):
    """All weights alike, and one key that has all; 3e6: beyond what fp16 holds, with scales that bring the scores back."""
    low, high = (-30, -26) if spread > 1e6 else (-6, -3)
    for held, new in (([400, 65], [1, 1]), ([90], [60])):
        b = make(held, new, 8, 2, 64, dtype, seed=3, spread=spread, low=low, high=high)
        check(b, call(b))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_values_of_far_apart_pages(dtype, new):
    """The last pages' values are 2^60 times the first's, with weights of nothing: the first ones' still decide."""
    b = make([200], [new], 4, 1, 128, dtype, seed=5)
    q, share = torch.zeros_like(b["q"]), 4
    q[:] = 1.0
    b["q"] = q
    pages = b["table"][0].long()
    b["keys"].values[pages[0], 0] = 100                       # scores of the first page: large; of the others: far below
    b["keys"].values[pages[1:4], 0] = -100
    b["keys"].scales[pages[:4]] = 2.0 ** -4
    b["values"].scales[pages[0]] = 2.0 ** -30
    b["values"].scales[pages[1:4]] = 2.0 ** 30
    torch.cuda.synchronize()
    got = call(b).double()
    want = b["values"].held(torch.float64)[pages[0], 0].mean(0)
    size = b["values"].held(torch.float64)[pages[0], 0].abs().mean(0)
    assert bool(((got.view(new, share, 128) - want).abs() <= (2.0 ** -7) * size).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 3, 70])
def test_attention_scales_that_are_no_number(dtype, new):
    """A block whose scale is none spoils the rows that see it, and only those."""
    for which in ("keys", "values"):
        b = make([300, 150], [new, new], 8, 2, 128, dtype, seed=7, window=100)
        page = b["table"][0, 1]                               # positions 64 .. 127 of the first sequence: the last block is 112 .. 127
        b[which].scales[page, 1, 3] = math.nan
        got = call(b)
        torch.cuda.synchronize()
        spoilt = {t for t in range(new) if 300 + t - 99 <= 127}
        for t in range(2 * new):
            row = got[t].view(8, 128)
            assert bool(row[4:].isnan().all()) == (t in spoilt) and not bool(row[:4].isnan().any()), (which, t)
            if t not in spoilt:
                assert not bool(row.isnan().any())
        clean = {**b, which: ops().Int8Pages(b[which].values, b[which].scales.nan_to_num(2.0 ** -4))}
        check(clean, got, where=set(range(2 * new)) - spoilt)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_ring_of_pages(dtype):
    """A window's pages in a ring that has been gone round several times."""
    for held, new, window, ring in (([700, 333, 20], [1, 1, 1], 130, 4), ([500, 64], [60, 64], 100, 4), ([1000], [7], 64, 3)):
        b = make(held, new, 8, 2, 128, dtype, window=window, ring=ring, seed=11)
        check(b, call(b))


@pytest.mark.parametrize("dtype, dim", [(F32, 16), (BF16, 128), (BF16, 64), (BF16, 80)])
def test_attention_rows_of_a_projection_order_and_bounds(dtype, dim):
    """Queries as the first columns of wider rows; an order of the sequences; wide bounds; a given result: the same bits."""
    b = make([100, 0, 900], [1, 40, 3], 4, 2, dim, dtype, seed=13, padded=4 * dim)
    got = call(b)
    check(b, got)
    out = torch.empty_like(got)
    assert call(b, out=out, seq_order=ints([2, 0, 1])) is out and torch.equal(out, got)
    narrow = b["q"][:, :4 * dim].contiguous()
    assert torch.equal(call({**b, "q": narrow}), got)
    check(b, call(b, max_new=4096, max_len=100000))


def test_attention_on_another_stream_and_captured():
    """Captured once, replayed with other lengths, queries and pages; a call on another stream in between."""
    for dtype, new in ((BF16, [1, 1, 1]), (BF16, [30, 1, 5]), (F32, [1, 2, 1])):
        b = make([700, 80, 1000], new, 8, 2, 128, dtype, seed=17)
        other = make([900, 5, 600], new, 8, 2, 128, dtype, seed=18)
        check(b, call(b, max_len=1100))
        wide = max(b["table"].shape[1], other["table"].shape[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(b, max_len=1100)
        graph.replay()
        check(b, out)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            beside = call(other, max_len=1100)
        torch.cuda.current_stream().wait_stream(stream)
        check(other, beside)
        if other["table"].shape == b["table"].shape and other["keys"].values.shape[0] <= b["keys"].values.shape[0]:
            n = other["keys"].values.shape[0]
            b["q"].copy_(other["q"])
            b["table"].copy_(other["table"])
            b["arrays"][0].copy_(other["arrays"][0])
            for name in ("keys", "values"):
                b[name].values[:n].copy_(other[name].values)
                b[name].scales[:n].copy_(other[name].scales)
            graph.replay()
            check(other, out)
        del wide


def test_attention_same_bits_again():
    for held, new in (([3000, 100, 700], [1, 1, 1]), ([3000, 100], [40, 300])):
        b = make(held, new, 32, 8, 128, BF16, seed=19)
        first = call(b)
        for _ in range(3):
            assert torch.equal(call(b), first)


def test_attention_reports():
    """More tokens than max_new says, a page and an order that there are not: reported, and the next call is served."""
    from llm_b200.errors import KernelError
    for dtype in (F32, BF16):
        b = make([100, 10], [1, 40], 4, 2, 128, dtype, seed=23)
        good = call(b)
        for wrong in ("max_new", "page", "order", "scale"):
            c = dict(b)
            if wrong == "scale":
                c["keys"] = ops().Int8Pages(b["keys"].values, b["keys"].scales * 1.5)
            if wrong == "page":
                c["table"] = b["table"].clone()
                c["table"][0, 1] = 1 << 20
            more = {"max_new": 1} if wrong == "max_new" else {"seq_order": ints([0, 5])} if wrong == "order" else {}
            call(c, **more)
            torch.cuda.synchronize()
            with pytest.raises(KernelError, match="a step brought"):
                ops().check_device_status()
        assert torch.equal(call(b), good)
        check(b, good)


# ----------------------------------------------------------------------------- appending

def projection(b, n_rot, interleaved, seed, loud=1.0):
    gen = torch.Generator().manual_seed(seed)
    heads, kv, dim, n = b["heads"], b["kv_heads"], b["dim"], b["cu"][-1]
    x = torch.randn(n, heads + 2 * kv, dim, generator=gen) * torch.exp(torch.randn(n, heads + 2 * kv, 1, generator=gen)) * loud
    x = x.to(b["dtype"]).to(DEV)
    angles = None
    if n_rot:
        most = max(b["lengths"])
        a = torch.arange(most, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, n_rot, 2, dtype=torch.float64) / n_rot)
        angles = torch.cat([a.cos(), a.sin()], 1).float().to(DEV)
    return x, angles


def places(b):
    """(tok_pos, tok_seq) of the step."""
    return (ints([length - n + j for length, n in zip(b["lengths"], b["new"]) for j in range(n)]),
            ints([s for s, n in enumerate(b["new"]) for _ in range(n)]))


def append(b, x, angles, interleaved=False, **more):
    pos, seq = places(b)
    return ops().rope_cache_write_int8(x.flatten(1), angles, pos, seq, b["arrays"][1], b["table"], b["ring"], b["keys"], b["values"], b["heads"],
                                       b["kv_heads"], b["dim"], interleaved, **more)


def turned(b, x, angles, interleaved):
    """(rotated queries and keys in 64 bits, the bound of their error in 32)."""
    pos = places(b)[0].long()
    y = x[:, :b["heads"] + b["kv_heads"]].double()
    off = torch.zeros_like(y)
    if angles is not None:
        n = angles.shape[1]
        c, s = angles[pos, None, :n // 2].double(), angles[pos, None, n // 2:].double()
        at0 = torch.arange(0, n, 2) if interleaved else torch.arange(n // 2)
        at1 = at0 + (1 if interleaved else n // 2)
        low, high = y[..., at0].clone(), y[..., at1].clone()
        y[..., at0], y[..., at1] = low * c - high * s, high * c + low * s
        off[..., at0], off[..., at1] = 2 * U * ((low * c).abs() + (high * s).abs()), 2 * U * ((high * c).abs() + (low * s).abs())
    return y, off


def check_append(b, x, angles, interleaved, before, got):
    """`before`: (whole numbers, scales) of keys and values as they were."""
    torch.cuda.synchronize()
    ops().check_device_status()
    heads, kv, dim = b["heads"], b["kv_heads"], b["dim"]
    y, off = turned(b, x, angles, interleaved)
    half = 0.0 if b["dtype"] == F32 else 2.0 ** -8
    queries = got.double().view(-1, heads, dim)
    assert got.dtype == b["dtype"] and bool(((queries - y[:, :heads]).abs() <= half * y[:, :heads].abs() + (1 + half) * off[:, :heads] + 1e-40).all())
    table, v = b["table"].tolist(), x[:, heads + kv:].double()
    for cache, rows, error, (old_whole, old_scales) in ((b["keys"], y[:, heads:], off[:, heads:], before[0]), (b["values"], v, torch.zeros_like(v), before[1])):
        block, whole, scales = cache.block, cache.values.double(), cache.scales.double()
        untouched_rows = torch.ones(cache.values.shape[:3], dtype=torch.bool, device=DEV)
        untouched_blocks = torch.ones(cache.scales.shape, dtype=torch.bool, device=DEV)
        for s, (length, n) in enumerate(zip(b["lengths"], b["new"])):
            done = 0
            while done < n:
                p = length - n + done
                count = min(block - p % block, n - done)
                page, r, at = table[s][p // PAGE % b["ring"]], p % PAGE, p % PAGE // block
                t = b["cu"][s] + done
                new, e = rows[t:t + count].transpose(0, 1), error[t:t + count].transpose(0, 1)
                size, slack = new.abs().amax((1, 2)), e.amax((1, 2))
                scale, fresh = scales[page, :, at], torch.ones(kv, dtype=torch.bool, device=DEV)
                if p % block:
                    was = old_scales[page, :, at].double()
                    fresh = scale > was
                    assert bool((scale >= was).all())
                    begin = at * block
                    expect = torch.round(old_whole[page, :, begin:r].double() * (was / scale)[:, None, None])
                    assert torch.equal(whole[page, :, begin:r], expect)
                assert bool((torch.exp2(torch.round(torch.log2(scale))) == scale).all())
                assert bool((size <= 127 * scale + slack).all()) and bool((~fresh | (size > 63.5 * scale - slack) | (scale == 2.0 ** -126)).all())
                q = whole[page, :, r:r + count]
                assert bool(((q * scale[:, None, None] - new).abs() <= scale[:, None, None] / 2 + e).all())
                untouched_rows[page, :, at * block:r + count] = False
                untouched_blocks[page, :, at] = False
                done += count
        assert torch.equal(cache.values[untouched_rows], old_whole[untouched_rows])
        assert torch.equal(cache.scales[untouched_blocks].nan_to_num(7.0), old_scales[untouched_blocks].nan_to_num(7.0))


def copies(b):
    return [(c.values.clone(), c.scales.clone()) for c in (b["keys"], b["values"])]


APPENDS = [([0], [1]), ([5, 17, 0, 63, 64], [1] * 5), ([0, 9, 70, 0, 3, 15], [3, 65, 1, 0, 40, 17]), ([0, 30], [200, 129]), ([127, 1, 16], [2, 15, 16]),
           ([i * 3 for i in range(40)], [1] * 40)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads, kv_heads, dim, n_rot, interleaved", [
    (8, 2, 128, 128, False), (4, 4, 64, 64, True), (6, 1, 64, 0, False), (4, 2, 16, 16, False), (12, 4, 80, 32, True), (2, 2, 256, 128, False),
    (3, 1, 18, 10, False), (8, 2, 128, 96, True), (16, 16, 128, 128, False)])
@pytest.mark.parametrize("step", range(len(APPENDS)))
def test_append_against_the_definition(dtype, heads, kv_heads, dim, n_rot, interleaved, step):
    held, new = APPENDS[step]
    b = make(held, new, heads, kv_heads, dim, dtype, block=(16, 64, 1, 4, 32)[(step + heads) % 5], seed=step)
    x, angles = projection(b, n_rot, interleaved, step)
    before, kept = copies(b), x.clone()
    got = append(b, x, angles, interleaved)
    check_append(b, x, angles, interleaved, before, got)
    assert torch.equal(x, kept)


@pytest.mark.parametrize("block", [1, 2, 8, 64])
@pytest.mark.parametrize("loud", [1e-42, 1e-30, 1e-3, 1e3, 1e30])
def test_append_blocks_that_grow_or_stay(block, loud):
    """Rows far smaller and far larger than what their blocks hold, down to values that 32 bits hold in part."""
    b = make([3, 40, 70], [2, 30, 1], 4, 2, 64, F32, block=block, seed=3, low=-12, high=12)
    x, angles = projection(b, 64, False, 5, loud)
    before = copies(b)
    check_append(b, x, angles, False, before, append(b, x, angles))


def test_append_zeros_and_exact_steps():
    """Rows of zeros; magnitudes at 127 steps exactly and just above."""
    b = make([0, 0, 0], [1, 1, 1], 2, 1, 16, F32, block=16)
    x = torch.zeros(3, 4, 16, device=DEV)
    x[1] = 127 * 2.0 ** -3
    x[2] = 127 * 2.0 ** -3 * (1 + 2.0 ** -20)
    before = copies(b)
    check_append(b, x, None, False, before, append(b, x, None))
    at = [int(b["table"][s, 0]) for s in range(3)]
    assert [float(b["keys"].scales[p, 0, 0]) for p in at] == [2.0 ** -126, 2.0 ** -3, 2.0 ** -2]
    assert int(b["keys"].values[at[1], 0, 0].min()) == 127 and int(b["keys"].values[at[2], 0, 0].max()) == 64


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_values_that_are_not_finite(bad, dtype):
    """Their block's scale is no number, while it is continued too, and a number again when the block is begun anew. Other heads, blocks and
    sequences are as they are without them."""
    b = make([20, 5], [30, 4], 4, 2, 64, dtype, seed=29)
    x, _ = projection(b, 0, False, 7)
    x[3, 5, 10] = bad                                         # key head 1 of position 23: block 16 .. 31
    x[31, 6, 0] = bad                                         # value head 0 of the second sequence's position 6
    append(b, x, None)
    torch.cuda.synchronize()
    ops().check_device_status()
    p0, p1 = int(b["table"][0, 0]), int(b["table"][1, 0])
    assert b["keys"].scales[p0].isnan().tolist() == [[False] * 4, [False, True, False, False]]
    assert bool(b["values"].scales[p1, 0, 0].isnan()) and not bool(b["values"].scales[p1, 1, 0].isnan())
    more = make([9], [1], 4, 2, 64, dtype)
    y, _ = projection(more, 0, False, 8)
    more.update(keys=b["keys"], values=b["values"], table=b["table"][1:2], ring=b["ring"])
    append(more, y, None)                                     # continues the spoilt block
    assert bool(b["values"].scales[p1, 0, 0].isnan())
    more["lengths"], more["arrays"] = [1], (ints([1]), ints([0, 1]))
    append(more, y, None)                                     # the block is begun anew
    torch.cuda.synchronize()
    assert not bool(b["values"].scales[p1, 0, 0].isnan())


def test_append_queries_alone_and_given():
    b = make([70, 3], [5, 1], 8, 2, 128, BF16, seed=31)
    x, angles = projection(b, 128, False, 9)
    before = copies(b)
    out = torch.empty(6, 8 * 128, dtype=BF16, device=DEV)
    assert append(b, x, angles, write_cache=False, out=out) is out
    torch.cuda.synchronize()
    for cache, (whole, scales) in zip((b["keys"], b["values"]), before):
        assert torch.equal(cache.values, whole) and torch.equal(cache.scales.nan_to_num(7.0), scales.nan_to_num(7.0))
    check_append(b, x, angles, False, before, append(b, x, angles))
    assert torch.equal(out, append(b, x, angles))


def test_append_ring_and_reports():
    from llm_b200.errors import KernelError
    b = make([250, 500], [20, 1], 4, 2, 64, BF16, ring=3, window=60, seed=37)
    x, angles = projection(b, 64, False, 11)
    before = copies(b)
    check_append(b, x, angles, False, before, append(b, x, angles))
    for wrong in ("page", "angles"):
        c = dict(b)
        if wrong == "page":
            c["table"] = torch.full_like(b["table"], -5)
        append(c, x, angles[:100] if wrong == "angles" else angles)
        torch.cuda.synchronize()
        with pytest.raises(KernelError, match="a step brought"):
            ops().check_device_status()


@pytest.mark.parametrize("dtype, dim, n_rot", [(F32, 16, 16), (BF16, 128, 128), (BF16, 128, 64)])
def test_append_rows_behind_the_last_sequence(dtype, dim, n_rot):
    """A padded batch: the padding's queries and pages are left as they are, whatever its positions and sequences say."""
    b = make([5, 40], [3, 30], 4, 2, dim, dtype, seed=43)
    x, angles = projection(b, n_rot, False, 13)
    padded = torch.cat([x, torch.full((9, *x.shape[1:]), math.nan, dtype=dtype, device=DEV)])
    pos, seq = places(b)
    pos, seq = torch.cat([pos, ints([0, 16, 64, 3, -7, 1 << 30, 0, 1, 2])]), torch.cat([seq, ints([0, 1, 1, 0, 0, 1, 99, -1, 0])])
    out = torch.full((42, 4 * dim), 7.0, dtype=dtype, device=DEV)
    before = copies(b)
    ops().rope_cache_write_int8(padded.flatten(1), angles, pos, seq, b["arrays"][1], b["table"], b["ring"], b["keys"], b["values"], 4, 2, dim, out=out)
    check_append(b, x, angles, False, before, out[:33])
    assert bool((out[33:] == 7).all())


@pytest.mark.parametrize("dtype, dim", [(F32, 16), (BF16, 128), (BF16, 80)])
@pytest.mark.parametrize("new", [[1, 1, 1], [20, 1, 90]])
def test_attention_rows_behind_the_last_sequence_and_wide_tables(dtype, dim, new):
    """A padded batch, and a table inside a wider one."""
    b = make([200, 3, 70], new, 4, 2, dim, dtype, seed=47)
    n = b["cu"][-1]
    wide = torch.full((3, b["ring"] + 5), 1 << 20, dtype=torch.int32, device=DEV)
    wide[:, :b["ring"]] = b["table"]
    padded = torch.cat([b["q"], torch.full((6, 4 * dim), math.nan, dtype=dtype, device=DEV)])
    out = torch.full((n + 6, 4 * dim), 7.0, dtype=dtype, device=DEV)
    call({**b, "q": padded, "table": wide[:, :b["ring"]]}, out=out)
    check(b, out[:n].contiguous())
    assert bool((out[n:] == 7).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_attention_scales_of_the_scores(dtype, scale):
    for new in ([1, 2], [60, 1]):
        b = make([100, 30], new, 4, 2, 64, dtype, seed=53)
        b["scale"] = scale
        got = call(b)
        torch.cuda.synchronize()
        for s, length in enumerate(b["lengths"]):
            t = b["cu"][s]
            page = b["table"][s].long()[torch.arange(length, device=DEV) // PAGE]
            row = torch.arange(length, device=DEV) % PAGE
            seen = length - new[s] + 1                         # of the sequence's first new token
            k, v = (c.held(torch.float64)[page, 0, row][:seen] for c in (b["keys"], b["values"]))
            weights = torch.softmax(b["q"][t, :64].double() @ k.T * scale, -1)
            assert bool(((got[t, :64].double() - weights @ v).abs() <= 2.0 ** -7 * (weights @ v.abs())).all())


def test_pages_behind_two_to_the_31_bytes():
    """Pools of more than 2^31 whole numbers, whose last pages are in use."""
    n_pages, kv, dim = 34000, 8, 128                           # 2.2 * 10^9 whole numbers each of keys and values
    small = make([300, 90], [1, 1], 32, kv, dim, BF16, seed=59)
    big = []
    for cache in (small["keys"], small["values"]):
        n = cache.values.shape[0]
        whole = torch.zeros((n_pages, kv, PAGE, dim), dtype=torch.int8, device=DEV)
        scales = torch.full((n_pages, kv, cache.scales.shape[2]), math.nan, device=DEV)
        whole[-n:], scales[-n:] = cache.values, cache.scales
        big.append(ops().Int8Pages(whole, scales))
    shift = n_pages - small["keys"].values.shape[0]
    table = small["table"] + shift
    for new in (1, 20):
        b = make([301 - new, 91 - new], [new, new], 32, kv, dim, BF16, seed=61)
        b.update(keys=small["keys"], values=small["values"], table=small["table"], ring=small["ring"])
        want = call(b)
        check(b, want)
        assert torch.equal(call({**b, "keys": big[0], "values": big[1], "table": table}), want)
    x, angles = projection(b, dim, False, 15)
    append(b, x, angles)
    append({**b, "keys": big[0], "values": big[1], "table": table}, x, angles)
    for cache, whole in zip((b["keys"], b["values"]), big):
        n = cache.values.shape[0]
        assert torch.equal(whole.values[-n:], cache.values) and torch.equal(whole.scales[-n:].nan_to_num(7.0), cache.scales.nan_to_num(7.0))


# ----------------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype, heads, kv_heads, dim", [(F32, 4, 2, 16), (BF16, 8, 2, 128), (BF16, 8, 8, 64), (BF16, 6, 2, 80)])
@pytest.mark.parametrize("block", [1, 16, 64])
def test_a_prompt_and_its_next_tokens(dtype, heads, kv_heads, dim, block):
    """Prompts, questions behind them and single tokens, as a layer of the engine runs them. What is held after each step is near the
    unrounded keys and values, and attention is right for what is held."""
    lengths, b, exact = [0, 0, 0], make([0, 0, 0], [400, 400, 400], heads, kv_heads, dim, dtype, block=block, seed=41), [[], [], []]
    table, ring, keys, values = b["table"], b["ring"], b["keys"], b["values"]
    for i, new in enumerate(([90, 1, 33], [20, 50, 0], [1, 1, 1], [1, 1, 1], [1, 1, 1], [4, 60, 2], [1, 1, 1])):
        lengths = [a + n for a, n in zip(lengths, new)]
        cu = [sum(new[:j]) for j in range(4)]
        b = dict(b, lengths=lengths, new=new, cu=cu, arrays=(ints(lengths), ints(cu)), bounds=dict(max_new=max(new), max_len=max(lengths)), table=table)
        x, angles = projection(b, dim if dim != 80 else 64, False, 50 + i)
        b["q"] = append(b, x, angles)
        check(b, call(b))
        y = turned(b, x, angles, False)[0][:, heads:]
        for s in range(3):
            exact[s].append(y[cu[s]:cu[s + 1]])
    held = keys.held(torch.float64)
    for s, length in enumerate(lengths):
        row = torch.arange(length, device=DEV)
        got = held[table[s].long()[row // PAGE], :, row % PAGE]
        scale = keys.scales.double()[table[s].long()[row // PAGE], :, row % PAGE // block]
        # half a step, and half of each step that the block was in before it grew: less than one step in all
        assert bool(((got - torch.cat(exact[s])).abs() <= scale[..., None] * (0.5 if block == 1 else 1.0) + 1e-5).all())


# (held, new, heads, kv_heads, dim, window): sequences that many blocks share, one long one among many short, few heads, up to 8 rows and above
SHARED = [
    ([8190], [1], 32, 8, 128, 0),
    ([30000] + [3] * 20, [1] * 21, 16, 8, 64, 0),
    ([4000, 0, 900], [2, 1, 0], 32, 8, 128, 0),
    ([20000], [1], 8, 1, 128, 0),
    ([2000, 2500, 700], [1, 1, 1], 4, 4, 64, 1500),
    ([3000, 5000], [4, 2], 16, 4, 128, 0),
    ([640 + 7 * i for i in range(40)], [1] * 40, 8, 8, 64, 0),
]


def test_attention_parts_that_meet():
    """Parts of a pair are joined in their own order whichever block ends last, and counts of one shape's parts do not show in another's: calls of all
    shapes in turn, some of them captured, give the same bits each time."""
    batches = [make(held, new, heads, kv_heads, dim, BF16, window=window, seed=60 + i)
               for i, (held, new, heads, kv_heads, dim, window) in enumerate(SHARED)]
    first = [call(b) for b in batches]
    for b, got in zip(batches, first):
        check(b, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [call(b) for b in batches]
    for _ in range(10):
        graph.replay()
        for b, got, again in zip(batches, first, captured):
            assert torch.equal(again, got)
            again.zero_()
        for b, got in zip(batches, first):
            assert torch.equal(call(b), got)


@pytest.mark.parametrize("dtype, heads, kv_heads, dim", [(BF16, 8, 2, 128), (F32, 4, 2, 64)])
def test_steps_whose_lengths_are_counted_on_the_device(dtype, heads, kv_heads, dim):
    """Lengths, positions and the table written by a tensor operation right in front of the calls, as a loop on the device has them: the same as
    with everything waited for in between."""
    held = [700, 5, 60, 0]
    b = make(held, [1] * 4, heads, kv_heads, dim, dtype, seed=71)
    steps = 60
    n_pages, width = b["keys"].values.shape[0], 16
    start = torch.stack([torch.randperm(64)[:width] + 64 * s for s in range(4)]).to(torch.int32).to(DEV)
    x, angles = projection(dict(b, lengths=[1000]), dim, False, 72)
    more = torch.randn(steps, *x.flatten(1).shape, generator=torch.Generator().manual_seed(73)).to(dtype).to(DEV)
    _, seq = places(b)

    def loop(wait):
        gen = torch.Generator().manual_seed(74)
        keys, values = (pages_of(256, kv_heads, dim, 16, gen) for _ in range(2))
        for cache in (keys, values):
            cache.scales.fill_(2.0 ** -5)
        pos, lens, table, outs = ints(held), ints([h + 1 for h in held]), start.clone(), []
        for i in range(steps):
            if wait:
                torch.cuda.synchronize()
            q = ops().rope_cache_write_int8(more[i], angles, pos, seq, b["arrays"][1], table, width, keys, values, heads, kv_heads, dim)
            if wait:
                torch.cuda.synchronize()
            outs.append(ops().attention_int8(q, keys, values, table, width, lens, b["arrays"][1], heads, kv_heads, dim, b["scale"], max_new=1, max_len=1024))
            if wait:
                torch.cuda.synchronize()
            table.copy_((table + 1) % 256)                     # (other pages each time: what a stale table names holds something else)
            lens.add_(1)
            pos.add_(1)
        torch.cuda.synchronize()
        ops().check_device_status()
        return torch.stack(outs)

    want = loop(True)
    for _ in range(5):
        assert torch.equal(loop(False), want)


@pytest.mark.parametrize("dtype, new", [(BF16, [1, 1]), (BF16, [70, 3]), (F32, [2, 1])])
def test_attention_windows_beyond_all_positions(dtype, new):
    """A window that no sequence fills, whatever its number, is none."""
    b = make([900, 40], new, 8, 2, 64, dtype, seed=81)
    want = call(b)
    for window in (b["ring"] * PAGE + 1, 2 ** 31 - 1, 2 ** 32 + 5):
        assert torch.equal(call(dict(b, window=window)), want)
    check(dict(b, window=b["ring"] * PAGE), call(dict(b, window=b["ring"] * PAGE)))


@pytest.mark.parametrize("which", range(len(SHARED)))
def test_attention_parts_inside_a_step(which):
    """The same shapes inside a step's scope, where a launch of its own joins the parts."""
    held, new, heads, kv_heads, dim, window = SHARED[which]
    b = make(held, new, heads, kv_heads, dim, BF16, window=window, seed=90 + which)
    with ops().StepScope():
        check(b, call(b))
        first, graph = call(b), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            again = call(b)
    for _ in range(3):
        again.zero_()
        graph.replay()
        assert torch.equal(again, first)


# ----------------------------------------------------------------------------- long padded batches

def padded(b, rows):
    """The batch with `rows` rows behind its last sequence's, and a result whose every element is 7."""
    width = b["heads"] * b["dim"]
    q = torch.cat([b["q"], torch.full((rows, width), math.nan, dtype=b["dtype"], device=DEV)])
    return {**b, "q": q}, torch.full((q.shape[0], width), 7.0, dtype=b["dtype"], device=DEV)


@pytest.mark.parametrize("dtype, dim", [(F32, 16), (F32, 64), (F32, 128), (BF16, 80), (BF16, 256), (BF16, 64), (BF16, 128)])
@pytest.mark.parametrize("new", [[1, 1, 1], [20, 1, 90], [3, 0, 2]])
def test_attention_rows_behind_the_last_sequence_of_cut_ones(dtype, dim, new):
    """A padded batch whose sequences are cut into parts: the padding is left as it is by what joins them, in calls one by one, inside of a
    step, and in captured ones that are replayed on fewer tokens."""
    b = make([2000, 3, 700], new, 4, 2, dim, dtype, seed=101)
    n = b["cu"][-1]
    wide, out = padded(b, 6)
    call(wide, out=out)
    check(b, out[:n].contiguous())
    assert bool((out[n:] == 7).all())
    with ops().StepScope():
        out.fill_(7)
        call(wide, out=out)
        check(b, out[:n].contiguous())
        assert bool((out[n:] == 7).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(wide, out=out)
    kept = n - new[2]
    b["arrays"][1][3] = kept                                   # the last sequence brings nothing
    b["arrays"][0][2] = 700
    fewer = {**b, "new": new[:2] + [0], "cu": b["cu"][:3] + [kept], "lengths": b["lengths"][:2] + [700]}
    for _ in range(2):
        out.fill_(7)
        graph.replay()
        check(fewer, out[:kept].contiguous())
        assert bool((out[kept:] == 7).all())


@pytest.mark.parametrize("dtype, dim", [(F32, 16), (F32, 128), (BF16, 80), (BF16, 64), (BF16, 128)])
@pytest.mark.parametrize("held, new, window", [([1000, 20], [1, 1], 0), ([1000, 20], [40, 3], 0), ([700, 9], [1, 1], 300), ([190, 9], [70, 1], 0)])
def test_attention_reports_sequences_longer_than_their_ring(dtype, dim, held, new, window):
    """A sequence of which a step sees more pages than its ring has is reported, whichever kernel serves it; one that fits is not."""
    from llm_b200.errors import KernelError
    b = make(held, new, 4, 2, dim, dtype, window=window, seed=103)
    check(b, call(b))
    small = {**b, "ring": 4}                                   # (4 pages of the table)
    call(small)
    torch.cuda.synchronize()
    with pytest.raises(KernelError, match="a step brought"):
        ops().check_device_status()
    check(b, call(b))
    call({**small, "window": 50} if held[0] > 300 and max(new) < 50 else {**b, "ring": 5})
    torch.cuda.synchronize()
    ops().check_device_status()


@pytest.mark.parametrize("dtype, heads, kv_heads, dim, new", [
    (BF16, 8, 2, 128, [1, 1, 1]), (BF16, 8, 2, 128, [30, 1, 5]), (BF16, 4, 4, 64, [2, 1, 1]), (BF16, 4, 4, 64, [5, 300, 1]), (BF16, 4, 2, 80, [1, 1, 1]),
    (BF16, 4, 2, 80, [30, 1, 5]), (F32, 8, 2, 128, [1, 2, 1]), (F32, 8, 2, 64, [30, 1, 5])])
@pytest.mark.parametrize("inside", [False, True])
def test_attention_replayed_on_another_batch(dtype, heads, kv_heads, dim, new, inside):
    """A captured call replayed with other lengths, queries, pages and scales, and with the new tokens of the sequences dealt out another way."""
    import contextlib
    ring = 22
    b = make([700, 80, 1000], new, heads, kv_heads, dim, dtype, ring=ring, seed=107)
    others = [make([900, 5, 300], new, heads, kv_heads, dim, dtype, ring=ring, seed=108),
              make([3, 600, 70], new[1:] + new[:1], heads, kv_heads, dim, dtype, ring=ring, seed=109)]
    scope = ops().StepScope() if inside else contextlib.nullcontext()
    with scope:
        check(b, call(b, max_len=1300))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(b, max_len=1300)
    graph.replay()
    check(b, out)
    for other in others:
        n = other["keys"].values.shape[0]
        assert n <= b["keys"].values.shape[0] and other["table"].shape == b["table"].shape and other["cu"][-1] == b["cu"][-1]
        b["q"].copy_(other["q"])
        b["table"].copy_(other["table"])
        for mine, theirs in zip(b["arrays"], other["arrays"]):
            mine.copy_(theirs)
        for name in ("keys", "values"):
            b[name].values[:n].copy_(other[name].values)
            b[name].scales[:n].copy_(other[name].scales)
        out.zero_()
        graph.replay()
        check(other, out)


@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 8, 128), (8, 8, 64), (10, 2, 128)])
@pytest.mark.parametrize("window", [0, 2100])
def test_attention_single_tokens_beside_a_prompt(heads, kv_heads, dim, window):
    """Steps that two kernels serve, each with its work dealt out and its parts in the same scratch: sequences of a few tokens at long and short
    positions among prompts of 60 and 30."""
    share = heads // kv_heads
    held = [5000, 0, 3000, 4500, 200, 4000, 64, 2300] + [700 + 61 * i for i in range(24)]
    new = [1, 60, 1, 30, 1, 16 // share, 0, 1] + [1] * 24
    assert sum(new) < len(new) * (16 // share + 1)             # (some bring up to 16 rows for certain: both kernels are launched)
    b = make(held, new, heads, kv_heads, dim, BF16, window=window, seed=113)
    first = call(b)
    check(b, first)
    with ops().StepScope():
        check(b, call(b))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            again = call(b)
    for _ in range(2):
        again.zero_()
        graph.replay()
        assert torch.equal(again, first)
    b["arrays"][0][0] = 900                                    # (shorter, in the same captured launches)
    b["lengths"][0] = 900
    graph.replay()
    check(b, again)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads, kv_heads, dim", [(1, 1, 64), (4, 2, 64), (7, 7, 64), (3, 1, 128), (33, 1, 128)])
@pytest.mark.parametrize("new", [1, 700])
def test_append_queries_of_any_number_of_heads(dtype, heads, kv_heads, dim, new):
    """Queries alone (a layer that reads another's cache), of fewer heads than an instruction has rows, and more than a task has."""
    b = make([70, 3], [new, 1], heads, kv_heads, dim, dtype, seed=151)
    x, angles = projection(b, dim, False, 31)
    before = copies(b)
    alone = append(b, x, angles, write_cache=False)
    check_append(b, x, angles, False, before, append(b, x, angles))
    assert torch.equal(append(b, x, angles), alone)


# ----------------------------------------------------------------------------- appends that leave something out

def same_pages(a, b):
    return all(torch.equal(x.values, y.values) and torch.equal(x.scales.nan_to_num(7.0), y.scales.nan_to_num(7.0)) for x, y in zip(a, b))


def cloned(b):
    return [ops().Int8Pages(c.values.clone(), c.scales.clone()) for c in (b["keys"], b["values"])]


APPENDERS = [(F32, 16, 16), (F32, 128, 128), (BF16, 64, 64), (BF16, 128, 128), (BF16, 128, 64), (BF16, 80, 0)]


@pytest.mark.parametrize("dtype, dim, n_rot", APPENDERS)
@pytest.mark.parametrize("held, new", [(10, 300), (0, 257), (63, 194), (250, 2000)])
def test_append_of_more_than_a_ring_holds(dtype, dim, n_rot, held, new):
    """A sequence that brings more pages than its ring has is left out and reported; the others of the step, and all queries, are as without it."""
    from llm_b200.errors import KernelError
    b = make([held, 3], [new, 2], 4, 2, dim, dtype, ring=4, seed=127)
    x, angles = projection(b, n_rot, False, 17)
    keys, values = cloned(b)
    alone = dict(b, keys=keys, values=values, table=b["table"][1:], lengths=[5], new=[2], cu=[0, 2], arrays=(ints([5]), ints([0, 2])))
    want = append(alone, x[new:].contiguous(), angles)
    queries = append(b, x, angles, write_cache=False)
    torch.cuda.synchronize()
    ops().check_device_status()
    got = append(b, x, angles)
    torch.cuda.synchronize()
    with pytest.raises(KernelError, match="int8_cache: a step brought"):
        ops().check_device_status()
    assert torch.equal(got, queries) and torch.equal(got[new:], want)
    assert same_pages((b["keys"], b["values"]), (keys, values))


@pytest.mark.parametrize("dtype, dim, n_rot", APPENDERS)
@pytest.mark.parametrize("held, new", [(0, 256), (63, 193), (255, 1), (64 * 9 + 1, 200)])
def test_append_of_what_a_ring_just_holds(dtype, dim, n_rot, held, new):
    b = make([held, 3], [new, 2], 4, 2, dim, dtype, ring=4, seed=131)
    x, angles = projection(b, n_rot, False, 19)
    before = copies(b)
    check_append(b, x, angles, False, before, append(b, x, angles))


@pytest.mark.parametrize("dtype, dim, n_rot", APPENDERS)
def test_append_of_tokens_that_are_not_their_sequences(dtype, dim, n_rot):
    """A token whose sequence says other rows: reported, wherever it stands in its block."""
    from llm_b200.errors import KernelError
    b = make([5, 16], [20, 30], 4, 2, dim, dtype, seed=137)
    x, angles = projection(b, n_rot, False, 23)
    pos, seq = places(b)
    for token, says in ((3, 1), (11, 1), (0, 1), (20, 0), (40, 0)):       # in the middle of a block, at its beginning, a sequence's first
        wrong = seq.clone()
        wrong[token] = says
        ops().rope_cache_write_int8(x.flatten(1), angles, pos, wrong, b["arrays"][1], b["table"], b["ring"], b["keys"], b["values"], 4, 2, dim)
        torch.cuda.synchronize()
        with pytest.raises(KernelError, match="int8_cache: a step brought"):
            ops().check_device_status()


@pytest.mark.parametrize("dtype, dim, n_rot", APPENDERS)
def test_steps_without_sequences(dtype, dim, n_rot):
    """A padded batch that has no sequence at all: nothing is written."""
    b = make([5], [3], 4, 2, dim, dtype, seed=139)
    x, angles = projection(b, n_rot, False, 29)
    pos, seq = places(b)
    kept, out = cloned(b), torch.full((3, 4 * dim), 7.0, dtype=dtype, device=DEV)
    none, table = ints([0]), b["table"][:0]
    ops().rope_cache_write_int8(x.flatten(1), angles, pos, seq, none, table, b["ring"], b["keys"], b["values"], 4, 2, dim, out=out)
    ops().attention_int8(b["q"], b["keys"], b["values"], table, b["ring"], ints([]), none, 4, 2, dim, b["scale"], max_new=1, max_len=1, out=out)
    torch.cuda.synchronize()
    ops().check_device_status()
    assert bool((out == 7).all()) and same_pages((b["keys"], b["values"]), kept)


# ----------------------------------------------------------------------------- loud positions that a row does not see

def check_rows(b, got):
    """`check` with each row's own share of what may be lost: n 2^-32 times the largest value that the row itself sees."""
    heads, dim, share = b["heads"], b["dim"], b["heads"] // b["kv_heads"]
    weight, half = (0.0, 0.0) if b["dtype"] == F32 else (2.0 ** -11, 2.0 ** -8)
    torch.cuda.synchronize()
    ops().check_device_status()
    got, (length,), (n_new,) = got.double().view(-1, heads, dim), b["lengths"], b["new"]
    row = torch.arange(length, device=DEV)
    seen = row[None, :] <= torch.arange(length - n_new, length, device=DEV)[:, None]
    page = b["table"][0].long()[row // PAGE]
    for a in range(heads):
        k, v = (cache.held(torch.float64)[page, a // share, row % PAGE] for cache in (b["keys"], b["values"]))
        q = b["q"][:, a * dim:(a + 1) * dim].double()
        weights = torch.softmax((q @ k.T * b["scale"]).masked_fill(~seen, -math.inf), -1)
        want, size = weights @ v, weights @ v.abs()
        worst = ((q.abs() @ k.abs().T) * b["scale"]).masked_fill(~seen, 0).amax(-1, keepdim=True)
        bound = (4 * (2 * (dim + 8) * worst + length + 16) * U + weight + half) * size + half * want.abs() + 1e-30
        if weight:
            bound = bound + length * 2.0 ** -32 * (seen * v.abs().amax(-1)).amax(-1, keepdim=True)
        off = (got[:, a] - want).abs()
        assert bool((off <= bound).all()), (a, float((off / bound).max()))


@pytest.mark.parametrize("dtype, dim, apart", [(BF16, 64, 28), (BF16, 128, 28), (F32, 64, 28), (F32, 128, 90), (BF16, 80, 90)])
@pytest.mark.parametrize("held, new", [(14, 4), (0, 64), (100, 70), (0, 500)])
@pytest.mark.parametrize("which", ["keys", "values"])
def test_attention_loud_positions_that_a_row_does_not_see(dtype, dim, apart, held, new, which):
    """A block of later positions that is 2^apart times as loud as all others, in the same page, under the causal mask: rows in front of it are as near as
    without it, and those that see it are right. (The tensor cores' kernels hold scales within 29 powers of two of the largest that a row of the tile sees.)"""
    b = make([held], [new], 8, 2, dim, dtype, seed=157)
    first = -(-(held + new // 2) // 16) * 16                   # of the loud block
    assert held < first < held + new
    if which == "keys" and dtype == BF16 and dim != 80 and new > 4:
        apart = 17                                             # (scores beyond 2^23 are reported there: the next test)
    for name in ("keys", "values"):
        base = -6.0 if name == "keys" or apart < 60 else -50.0
        for p in range(0, held + new, 16):
            b[name].scales[b["table"][0, p // PAGE], :, p % PAGE // 16] = 2.0 ** (base + (apart if name == which and p == first else 0))
    got = call(b)
    check_rows(b, got)
    check(b, got)


@pytest.mark.parametrize("dtype, dim", [(BF16, 64), (BF16, 128), (F32, 64), (BF16, 80)])
@pytest.mark.parametrize("held, new", [(300, 1), (300, 3), (14, 4), (300, 40), (0, 70), (2500, 40)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_large_scores(dtype, dim, held, new, sign):
    """One key that has all of a row's weight by scores of up to 2^35: its value comes back, or the call is reported. At negative scores (all of a row's) the
    smallest wins."""
    from llm_b200.errors import KernelError
    for size in (14, 20, 26, 33):
        b = make([held], [new], 8, 2, dim, dtype, seed=167)
        b["q"].fill_(1.0)
        pages = b["table"][0].long()
        at = [min(5 + 64 * i, held) for i in range(2)] + [held]            # keys that stand out, a little more each time
        b["keys"].values.fill_(0 if sign > 0 else -64)
        for i, p in enumerate(at):
            b["keys"].values[pages[p // PAGE], :, p % PAGE] = int((64 + 8 * i) if sign > 0 else -(40 - 8 * i))
        b["keys"].scales[pages] = 2.0 ** (size - 6 - round(math.log2(dim * b["scale"])))
        b["values"].scales[pages] = 2.0 ** -9
        b["values"].scales[pages[-1:]] = 2.0 ** -3
        got = call(b)
        torch.cuda.synchronize()
        scores = 1.4427 * b["scale"] * dim * 64 * 2.0 ** (size - 6 - round(math.log2(dim * b["scale"])))
        if dtype == BF16 and dim != 80 and new > 4 and scores > 2.0 ** 23:
            with pytest.raises(KernelError, match="scores beyond"):
                ops().check_device_status()
            continue
        ops().check_device_status()
        got, want = got.double().view(new, 8, dim), b["values"].held(torch.float64)[pages[held // PAGE], :, held % PAGE]
        want = want.repeat_interleave(4, 0)
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -10 if size == 14 else 0.0)).all()), (size, float((got - want).abs().max()))


def test_attention_references_at_the_border_of_a_move():
    """Scores whose rounded product lies at the border of where a reference moves, and the unrounded one beyond it: both warps of a row decide alike."""
    import numpy as np
    log2e, held, new = np.float32(1.4426950408889634), 150, 50
    b = make([held], [new], 4, 1, 128, BF16, seed=173)
    pages = b["table"][0].long()
    b["keys"].scales[pages[:4]] = 2.0 ** -4
    b["values"].scales[pages[:4]] = 2.0 ** -3
    b["keys"].values.zero_()
    b["keys"].values[pages[2], 0, 7, 0] = 64                   # scores of 0, and one of 8 in the second step
    tried = 0
    for m in range(128):
        product = (1 + m / 128) * 64 * 2.0 ** -4
        at = int(np.float32(8 / product / float(log2e)).view(np.int32))
        scale = next((float(s) for s in (np.int32(at + d).view(np.float32) for d in range(-40, 41))
                      if 8 + 2.0 ** -22 < float(np.float32(s * log2e)) * product < 8 + 2.0 ** -21), None)
        if scale is None:
            continue
        b["q"].zero_()
        b["q"].view(new, 4, 128)[:, :, 0] = 1 + m / 128
        b["scale"] = scale
        check(b, call(b))
        tried += 1
    assert tried > 20


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("apart", [12, 28, 45])
@pytest.mark.parametrize("held, new, window", [(40, 4, 0), (0, 64, 0), (100, 90, 0), (300, 4, 30), (300, 90, 50), (1000, 60, 300)])
def test_attention_values_lost_beside_loud_ones(dim, apart, held, new, window):
    """Values beside much louder ones, some of which a row does not see: what is lost is small beside the largest that a row of the tile sees."""
    b = make([held], [new], 8, 2, dim, BF16, window=window, seed=163)
    for p in range(0, held + new, 16):
        loud = p // 16 % 3 == 1
        b["values"].scales[b["table"][0, p // PAGE], :, p % PAGE // 16] = 2.0 ** (-20 + (apart if loud else 0))
    check(b, call(b))


@pytest.mark.parametrize("dtype, dim", [(F32, 64), (F32, 128), (BF16, 64), (BF16, 128), (BF16, 80), (BF16, 256)])
@pytest.mark.parametrize("held, new", [([3000, 70], [1, 1]), ([300, 70], [4, 3]), ([300, 0], [60, 90]), ([9000], [33])])
def test_attention_queries_that_are_not_finite_and_extreme_scales(dtype, dim, held, new):
    """A query that is not finite has no number for a result, and no other query's result changes by a bit; whole numbers of -128, and scales at
    both ends of what 32 bits hold."""
    b = make(held, new, 8, 2, dim, dtype, seed=179)
    want, n = call(b).clone(), b["cu"][-1]
    spoilt = torch.zeros(n, 8, dtype=torch.bool, device=DEV)
    spoilt[0, 1] = spoilt[n - 1, 5] = True
    for bad in (math.nan, math.inf, -math.inf):
        q = b["q"].clone()
        q[0, dim + 3] = q[n - 1, 5 * dim + 3] = bad
        got = call({**b, "q": q}).view(n, 8, dim)
        torch.cuda.synchronize()
        ops().check_device_status()
        assert bool(got[spoilt].isnan().all()) and torch.equal(got[~spoilt], want.view(n, 8, dim)[~spoilt])
    for which, exponent in (("values", -126), ("values", 110), ("keys", -126)):
        c = make(held, new, 8, 2, dim, dtype, seed=181)
        c[which].values[:, :, ::3] = -128
        c[which].scales[~c[which].scales.isnan()] = 2.0 ** exponent
        check(c, call(c))
    c["values"].scales[~c["values"].scales.isnan()] = 0.0
    assert not bool(call(c).any())
