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
