"""Pages and per-sequence rows copied inside their pools: every byte of the pool afterwards, against indexing."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
PAGE = 64


def ops():
    import llm_b200.ops as o
    return o


def random(*shape, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).to(DEV)


def copied(pool, source, target, rows):
    want = pool.clone()
    for s, t, r in zip(source, target, rows):
        want[..., t, :, :r, :] = pool[..., s, :, :r, :]
    return want


LISTS = [
    ([3], [5], [1]),
    ([0] * 7, [1, 2, 3, 4, 5, 6, 7], [64, 1, 37, 63, 2, 64, 33]),                       # one page to many, unequal rows
    ([9, 0, 9, 4], [1, 11, 3, 2], [5, 64, 64, 17]),                                     # a source's pairs stand apart
    (list(range(20, 40)), list(range(20)), [64] * 20),
    ([], [], []),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, dim", [(8, 128), (1, 64), (3, 20), (2, 18), (5, 1), (2, 256)])
@pytest.mark.parametrize("lists", range(len(LISTS)))
def test_pages(dtype, heads, dim, lists):
    source, target, rows = LISTS[lists]
    pool = random(2, 2, 40, heads, PAGE, dim, dtype=dtype, seed=lists)
    want = copied(pool, source, target, rows)
    ops().copy_pages(pool, source, target, rows)
    assert torch.equal(pool, want)


def test_whole_pages_of_several_pools():
    pools = [random(3, 12, 2, PAGE, 32, seed=1), random(12, 4, PAGE, 24, dtype=torch.float32, seed=2), random(2, 12, 1, PAGE, 7, seed=3)]
    source, target = [11, 10, 11], [0, 5, 2]
    want = [copied(p, source, target, [PAGE] * 3) for p in pools]
    ops().copy_pages(pools, source, target)
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


def test_more_pairs_and_tensors_than_a_launch_takes():
    pools = [random(700, 1, PAGE, 8, seed=i) for i in range(19)]
    source, target = [i % 50 for i in range(600)], list(range(100, 700))
    want = [copied(p, source, target, [PAGE] * 600) for p in pools]
    before = ops().launch_count()
    ops().copy_pages(pools, source, target)
    assert ops().launch_count() - before == 6                          # 3 lists of pairs, 2 of tensors
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


def test_a_pool_that_does_not_start_on_16_bytes():
    flat = random(2 * 6 * 2 * PAGE * 8 + 1)
    pool = flat[1:].view(2, 6, 2, PAGE, 8)
    want = copied(pool, [0], [4], [9])
    ops().copy_pages(pool, [0], [4], [9])
    assert torch.equal(pool, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_slots(dtype):
    states = [random(9, 4, 128, 96, dtype=torch.float32, seed=1), random(9, 3, 1001, dtype=dtype, seed=2), random(9, 1, dtype=dtype, seed=3)]
    source, target = [2, 2, 2, 7], [0, 8, 3, 1]
    want = [s.clone() for s in states]
    for w, s in zip(want, states):
        w[torch.tensor(target)] = s[torch.tensor(source)]
    ops().copy_slots(states, source, target)
    for s, w in zip(states, want):
        assert torch.equal(s, w)


def test_offsets_beyond_32_bits():
    pool = torch.zeros((2, 40000, 8, PAGE, 64), dtype=torch.bfloat16, device=DEV)          # 5.2 GB
    pool[:, 39998] = random(2, 8, PAGE, 64)
    ops().copy_pages(pool, [39998, 39998], [39999, 1])
    assert torch.equal(pool[:, 39999], pool[:, 39998]) and torch.equal(pool[:, 1], pool[:, 39998])
    assert not pool[:, 2].any() and not pool[:, 39997].any() and not pool[:, 0].any()


def test_on_another_stream():
    pool = random(2, 2, 40, 4, PAGE, 64)
    want = copied(pool, [1], [2], [64])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops().copy_pages(pool, [1], [2])
    side.synchronize()
    assert torch.equal(pool, want)


def test_refusals():
    from llm_b200.errors import KernelError
    pool = random(2, 12, 2, PAGE, 32)
    held = pool.clone()
    for source, target, rows in [([0], [12], [64]), ([-1], [2], [64]), ([0], [-1], [64]), ([12], [0], [64]), ([0, 1], [2, 2], [64, 64]),
                                 ([0, 1], [1, 2], [64, 64]), ([3], [3], [64]), ([0], [1], [0]), ([0], [1], [65]), ([0], [1, 2], [64, 64]),
                                 ([0, 1], [2, 3], [64])]:
        with pytest.raises(KernelError):
            ops().copy_pages(pool, source, target, rows)
    for bad in (pool[:, ::2], pool[..., :16], random(2, 12, 2, 32, 32), pool.cpu(), [pool, random(11, 2, PAGE, 32)]):
        with pytest.raises(KernelError):
            ops().copy_pages(bad, [0], [1])
    with pytest.raises(KernelError):
        ops().copy_slots([random(4, 8), random(5, 8)], [0], [1])
    with pytest.raises(KernelError):
        ops().copy_slots([random(4, 8).t()], [0], [1])
    with pytest.raises(KernelError):
        ops().copy_slots([torch.zeros((4, 3), dtype=torch.uint8, device=DEV)], [0], [1])
    assert torch.equal(pool, held)
