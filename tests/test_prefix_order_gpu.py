"""Prefix attention behind a kernel that lets its successor start early, and calls whose bounds are wider than the step: what is
read is what the kernel in front has written, whichever kernels the bounds choose and however little is left for them."""
import pytest
import torch

from test_prefix_attention_gpu import BF16, DEV, call, check, make, ops

pytestmark = pytest.mark.gpu

ROW = 131072                    # columns of the buffer that holds the queries: its kernel runs for some ten microseconds


def behind_a_kernel_in_front(b, launches):
    """The same queries and results as with the stream empty in front of every call. The rows are written by the gated activation,
    whose blocks let the next kernel start before they write (16 bytes at a time it does not: its input starts on odd places)."""
    n, width = b["cu"][-1], b["heads"] * b["dim"]
    inputs = [torch.empty(n * 2 * ROW + 1, dtype=BF16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(i))[1:].view(n, 2 * ROW) for i in range(2)]
    rows = torch.empty((n, ROW), dtype=BF16, device=DEV)
    b = dict(b, q=rows[:, :width])
    want = []
    for x in inputs:
        ops().swiglu(x, out=rows)
        torch.cuda.synchronize()
        before = ops().launch_count()
        want.append(call(b))
        assert ops().launch_count() - before == launches
        check(b, want[-1])
    got = []
    for i in range(12):
        ops().swiglu(inputs[i % 2], out=rows)
        got.append(call(b))
    torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2]), i


def with_bounds(b, **bounds):
    return dict(b, bounds=dict(b["bounds"], **bounds))


def test_groups_that_share_nothing_where_many_pages_are_allowed():
    """The bounds choose the kernel for many rows, which finds no page to read; the own parts behind it still start behind the kernel in front."""
    members = [(13 * i % 150, 1) for i in range(80)]
    b = make([(0, members[:40]), (0, members[40:])], 32, 8, 128, BF16, seed=60, extra_width=10)
    behind_a_kernel_in_front(with_bounds(b, max_shared=8), 3)
    b = make([(0, members)], 32, 8, 128, BF16, seed=61, extra_width=40)
    behind_a_kernel_in_front(with_bounds(b, max_shared=32), 3)


@pytest.mark.parametrize("members, new, bounds", [
    ([30, 1, 3], 1, dict(max_new=1, max_group=3)),                     # own parts of more rows than their kernel holds
    ([1] * 40, 1, dict(max_new=1, max_group=4)),                       # and groups, for each of the kernels that may be chosen
    ([1] * 40, 1, dict(max_new=1, max_group=16)),
    ([90] * 5, 90, dict(max_new=30, max_group=40)),
])
def test_a_step_beyond_its_bounds_is_reported(members, new, bounds):
    from llm_b200.errors import KernelError
    b = make([(9, [(17 * i % 100, n) for i, n in enumerate(members)])], 8, 2, 64, BF16, seed=62)
    call(with_bounds(b, **bounds))
    torch.cuda.synchronize()
    with pytest.raises(KernelError, match="max_new"):
        ops().check_device_status()
    check(b, call(b))                                                  # and the next call is as it was


@pytest.mark.parametrize("wide", [2 ** 31 - 1, 2 ** 32 + 1, 2 ** 40])
@pytest.mark.parametrize("new", [1, 30])
def test_bounds_of_any_size(wide, new):
    """Bounds are no sizes of anything: the widest serve."""
    b = make([(3, [(17 * i % 100, new) for i in range(7)]), (0, [(150, new)])], 8, 2, 64, BF16, seed=63)
    check(b, call(with_bounds(b, max_new=wide, max_group=wide, max_own=wide)))


def even(n, low, high):
    return [(low + (high - low) * (7 * i % n) // max(n - 1, 1), 1) for i in range(n)]


REPLAYED = {                    # kernel: heads, groups of the captured step and of others of the same bounds, launches
    "tile": ((8, 2, 64), [[(20, even(12, 0, 150))], [(31, even(12, 0, 30))], [(3, even(12, 60, 200))]], 3),
    "tile, dealt out": ((8, 2, 64), [[(20, even(12, 0, 150)), (9, even(7, 3, 70)), (0, even(1, 9, 9))], [(5, even(4, 0, 90)), (31, even(14, 0, 128)), (2, even(2, 1, 64))],
                                     [(0, even(15, 0, 150)), (30, even(1, 63, 63)), (7, even(4, 0, 20))]], 3),
    "wide": ((32, 8, 128), [[(33, even(40, 0, 200))], [(20, even(40, 3, 900))], [(1, even(40, 0, 66))]], 3),
    "wide, dealt out": ((32, 8, 128), [[(33, even(40, 0, 200)), (0, even(2, 5, 80)), (9, even(6, 0, 130))], [(4, even(10, 0, 128)), (40, even(37, 0, 64)), (0, even(1, 700, 700))],
                                       [(0, even(40, 0, 100)), (0, even(2, 0, 3)), (0, even(6, 1, 300))]], 3),
    "few": ((8, 2, 64), [[(20, even(4, 0, 150))], [(31, even(4, 0, 30))]], 2),
    "on the cuda cores": ((8, 2, 48), [[(20, even(4, 0, 150)), (3, even(9, 0, 90))], [(31, even(12, 0, 30)), (0, even(1, 70, 70))]], 2),
}


@pytest.mark.parametrize("which", REPLAYED)
def test_each_kernel_replays_on_other_lengths_and_groups(which):
    """The bounds of a captured call hold for all its replays and are loose for each: unequal groups, groups that share nothing, short and long own parts."""
    (heads, kv_heads, dim), steps, launches = REPLAYED[which]
    made = [make(groups, heads, kv_heads, dim, BF16, seed=70 + i) for i, groups in enumerate(steps)]
    n_pages, width = max(b["keys"].shape[0] for b in made), max(b["table"].shape[1] for b in made)
    n = made[0]["cu"][-1]
    held = dict(made[0], q=made[0]["q"].clone(), arrays=tuple(t.clone() for t in made[0]["arrays"]),
                table=torch.zeros((n, width), dtype=torch.int32, device=DEV),
                keys=torch.zeros((n_pages, kv_heads, 64, dim), dtype=BF16, device=DEV), values=torch.zeros((n_pages, kv_heads, 64, dim), dtype=BF16, device=DEV),
                bounds={k: max(b["bounds"][k] for b in made) for k in made[0]["bounds"]})

    def load(b):
        held["keys"][:b["keys"].shape[0]] = b["keys"]
        held["values"][:b["values"].shape[0]] = b["values"]
        held["table"].zero_()
        held["table"][:, :b["table"].shape[1]] = b["table"]
        held["q"].copy_(b["q"])
        for to, t in zip(held["arrays"], b["arrays"]):
            to.copy_(t)
    load(made[0])
    before = ops().launch_count()
    call(held)
    assert ops().launch_count() - before == launches
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(held)
    for b in made + made[:1]:
        load(b)
        graph.replay()
        check(b, out)


@pytest.mark.parametrize("groups", [[(33, even(40, 0, 300))], [(33, even(40, 0, 300)), (5, even(4, 0, 100))], [(20, even(12, 0, 150))], [(20, even(3, 0, 150))]])
def test_shared_and_own_parts_behind_a_kernel_in_front(groups):
    b = make(groups, 32, 8, 128, BF16, seed=64)
    behind_a_kernel_in_front(b, 2 if len(groups[0][1]) == 3 else 3)
