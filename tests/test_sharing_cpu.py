"""Sequences that share pages, on the CPU: the cache's bookkeeping of forks and compaction, which sequences of a step and which
prompts of a batch stand together, and the engine and the generation loop over them with plain kernels."""
import random
import sys

import pytest
import torch

import plain_llama
from tiny import make_folder, random_tokens

from llm_b200.cache import PAGE, KvRequest, PagedCache, StateRequest
from llm_b200.engine import Engine, Entry, GenerationRequest, generate, load_model
from llm_b200.engine.generate import _Prompts
from llm_b200.errors import CacheFull, ContextFull, FormatError, LlmError
from llm_b200.sampling import SamplingParams


def make(requests=None, states=None, **options):
    requests = requests if requests is not None else [KvRequest(2, 16)] * 2
    defaults = dict(max_tokens=PAGE * 12, max_seq_len=PAGE * 6, max_slots=6, dtype=torch.float32, device="cpu")
    return PagedCache(requests, states or [None] * len(requests), **{**defaults, **options})


def fill(cache, slot, length):
    cache.reserve(slot, length)
    cache.set_length(slot, length)


# ----------------------------------------------------------------------------- the cache

@pytest.mark.parametrize("length, copied", [(0, 0), (1, 1), (PAGE - 1, 1), (PAGE, 0), (3 * PAGE, 0), (3 * PAGE + 17, 1)])
def test_a_fork_shares_full_pages_and_copies_the_last(plain_kernels, length, copied):
    cache = make()
    slot = cache.acquire()
    fill(cache, slot, length)
    group = cache.groups[0]
    group.storage.copy_(torch.arange(group.storage.numel()).view_as(group.storage))
    before = group.storage.clone()
    held = group.pool.n_held
    children = cache.fork(slot, 2)
    assert len(children) == 2 and all(cache.length(c) == length for c in children)
    assert group.pool.n_held == held + 2 * copied
    full = length // PAGE
    for child in children:
        mine, parents = group.slot_pages[child], group.slot_pages[slot]
        assert mine[:full] == parents[:full] and len(mine) == -(-length // PAGE)
        if copied:
            rows = length % PAGE
            assert mine[full] != parents[full]
            assert torch.equal(group.storage[:, :, mine[full], :, :rows], before[:, :, parents[full], :, :rows])
    cache.check()
    cache.release(slot)                                    # the parent may leave first
    cache.check()
    assert group.slot_pages[children[0]][:full] == group.slot_pages[children[1]][:full]
    cache.release(children[1])
    cache.release(children[0])
    cache.check()
    assert group.pool.n_held == 0 and cache.slots.n_held == 0


def test_a_fork_copies_rings_and_states(plain_kernels):
    cache = make([KvRequest(2, 16), KvRequest(2, 16, window=70), KvRequest(1, 8, value_dim=24), KvRequest(1, 8, values_are_keys=True)],
                 [StateRequest((3, 5)), None, StateRequest((7,)), None], max_tokens=PAGE * 24, step_tokens=PAGE)
    slot = cache.acquire()
    fill(cache, slot, 4 * PAGE + 9)
    for group in cache.groups:
        for t in (group.storage, group.keys, group.values):
            if t is not None:
                t.copy_(torch.randn(t.shape))
    for state in cache.states:
        if state is not None:
            state.copy_(torch.randn(state.shape))
    (child,) = cache.fork(slot)
    for group in cache.groups:
        mine, parents = group.slot_pages[child], group.slot_pages[slot]
        assert len(mine) == len(parents)
        if group.kind == "window":
            assert not set(mine) & set(parents)
            assert all(torch.equal(group.storage[:, :, a], group.storage[:, :, b]) for a, b in zip(mine, parents))
        else:
            assert mine[:4] == parents[:4] and mine[4] != parents[4]
            for t in ([group.storage] if group.storage is not None else [group.keys, group.values]):
                assert torch.equal(t[..., mine[4], :, :9, :], t[..., parents[4], :, :9, :])
    for state in cache.states:
        if state is not None:
            assert torch.equal(state[child], state[slot])
    cache.check()


def test_a_fork_that_does_not_fit_changes_nothing(plain_kernels):
    cache = make(max_tokens=PAGE * 4, max_slots=5)
    slot = cache.acquire()
    fill(cache, slot, 2 * PAGE + 1)                        # one page is left
    held, free = cache.groups[0].pool.n_held, cache.slots.n_free
    for count, error in ((2, CacheFull), (5, CacheFull), (0, LlmError), (-1, LlmError)):
        with pytest.raises(error):
            cache.fork(slot, count)
        assert cache.groups[0].pool.n_held == held and cache.slots.n_free == free
    with pytest.raises(LlmError):
        cache.fork(4)                                      # not held
    cache.fork(slot)
    cache.check()


def test_a_failing_copy_gives_the_children_back(plain_kernels, monkeypatch):
    import llm_b200.ops as ops
    cache = make()
    slot = cache.acquire()
    fill(cache, slot, 70)

    def fails(*_):
        raise RuntimeError("no")
    monkeypatch.setattr(ops, "copy_pages", fails)
    with pytest.raises(RuntimeError):
        cache.fork(slot, 3)
    cache.check()
    assert cache.slots.n_held == 1 and cache.groups[0].pool.n_held == 2


def test_random_forks_releases_and_compactions_lose_nothing(plain_kernels):
    """Every position of every sequence keeps the number that was written there, whatever is forked, released and moved."""
    cache = make([KvRequest(1, 4), KvRequest(1, 4, window=100)], max_tokens=PAGE * 20, max_slots=8, step_tokens=40)
    rng, live, stamp = random.Random(1), {}, 0

    def place(group, slot, position):
        page = group.slot_pages[slot][position // PAGE % group.ring_pages]
        return group.storage[0, :, page, 0, position % PAGE, 0]
    for _ in range(400):
        action = rng.random()
        if action < 0.2 and cache.slots.n_free:
            live[cache.acquire()] = []
        elif action < 0.55 and live:
            slot = rng.choice(list(live))
            n = rng.randint(1, 40)
            try:
                cache.reserve(slot, len(live[slot]) + n)
            except (CacheFull, ContextFull):
                continue
            for _ in range(n):
                stamp += 1
                for group in cache.groups:
                    place(group, slot, len(live[slot])).fill_(stamp)
                live[slot].append(stamp)
            cache.set_length(slot, len(live[slot]))
        elif action < 0.75 and live:
            slot = rng.choice(list(live))
            try:
                for child in cache.fork(slot, rng.randint(1, 2)):
                    live[child] = list(live[slot])
            except CacheFull:
                pass
        elif action < 0.9 and live:
            slot = rng.choice(list(live))
            cache.release(slot)
            del live[slot]
        else:
            cache.compact()
            for group in cache.groups:
                held = {p for pages in group.slot_pages.values() for p in pages}
                assert held == set(range(group.pool.n_held))
        cache.check()
        for slot, numbers in live.items():
            assert cache.length(slot) == len(numbers)
            for group in cache.groups:
                first = max(0, len(numbers) - group.window) if group.window else 0
                assert all(float(place(group, slot, j)[0]) == numbers[j] for j in range(first, len(numbers)))


def test_compact_moves_only_what_lies_behind(plain_kernels):
    cache = make()
    slots = [cache.acquire() for _ in range(4)]
    for slot in slots:
        fill(cache, slot, 2 * PAGE)
    cache.release(slots[0])
    cache.release(slots[2])
    assert cache.compact() == 2                            # pages 6 and 7 to 0 and 1; 2 and 3 stay
    assert [cache.groups[0].slot_pages[s] for s in (slots[1], slots[3])] == [[2, 3], [0, 1]]
    assert cache.compact() == 0
    cache.check()
    assert cache.block_table_rows(0, [slots[3]])[0, :2].tolist() == [0, 1]


# ----------------------------------------------------------------------------- what stands together

def test_prompts_that_begin_alike():
    a, b = list(range(500)), list(range(500, 1000))
    p = _Prompts([a[:300], a[:300], a[:200] + b, b[:100], a[:64], a[:64] + b[:3], a[:63], a[:63]])
    assert p.twin == [False, True, False, False, False, False, False, True]
    assert p.common == [192, 192, 192, 0, 0, 0, 0, 0]      # a prompt keeps a token of its own behind what is shared
    assert [p.shared(i) for i in range(8)] == [0, 256, 192, 0, 0, 0, 0, 0]
    p = _Prompts([a[:400] + [1], a[:400] + [2], a[:70] + [3]])         # three of 64, or two of 384: the sum decides
    assert p.common == [384, 384, 0] and p.run[0] == p.run[1] != p.run[2]
    p = _Prompts([a[:130] + [1]] + [a[:70] + [i] for i in range(5)])
    assert p.common == [64] * 6 and len(set(p.run)) == 1
    with pytest.raises(FormatError):
        _Prompts([["x"]])


# ----------------------------------------------------------------------------- the engine

def _setup(tmp_path, which, **engine_options):
    folder = make_folder(tmp_path, which, torch.float32)
    config, weights = plain_llama.read_model_folder(folder)
    model = load_model(folder, torch.float32, "cpu")
    return config, weights, Engine(model, **{"max_tokens": 1024, **engine_options})


def test_forked_sequences_go_their_own_ways(tmp_path, plain_kernels, monkeypatch):
    import llm_b200.ops as ops
    config, weights, engine = _setup(tmp_path, "A")
    calls = []
    plain = ops.prefix_attention                           # (32-bit steps always read shared pages once)
    monkeypatch.setattr(ops, "prefix_attention", lambda *a, **k: calls.append((a[6].tolist(), a[7].tolist(), k)) or plain(*a, **k))
    prompt = random_tokens(70, config["vocab_size"], 1)
    (slot,) = engine.acquire()
    engine.step([Entry(slot, prompt, [])])
    (other,) = engine.acquire()
    engine.step([Entry(other, prompt[:9], [])])
    assert not calls
    slots = [slot] + engine.fork(slot, 2) + [other]
    tails = [random_tokens(n, config["vocab_size"], 40 + i) for i, n in enumerate((3, 5, 1, 4))]
    texts = [prompt + tails[0], prompt + tails[1], prompt + tails[2], prompt[:9] + tails[3]]
    logits = engine.step([Entry(s, t, [len(t) - 1]) for s, t in zip(slots, tails)])
    layers = config["num_hidden_layers"]
    assert [c[:2] for c in calls] == [([0, 3, 4], [1, 0])] * layers
    assert calls[0][2]["max_new"] == 5 and calls[0][2]["max_group"] == 9 and calls[0][2]["max_shared"] == 1
    for row, text in zip(logits, texts):
        assert torch.allclose(row, plain_llama.forward(config, weights, text)[-1], atol=2e-5, rtol=1e-5)
    for k in range(3):                                     # decode steps, in another order: nothing stands together then
        new = [random_tokens(1, config["vocab_size"], 100 + 10 * k + i) for i in range(4)]
        texts = [t + n for t, n in zip(texts, new)]
        order = [0, 3, 1, 2] if k == 1 else [0, 1, 2, 3]
        logits = engine.step([Entry(slots[i], new[i], [0]) for i in order])
        for row, i in zip(logits, order):
            assert torch.allclose(row, plain_llama.forward(config, weights, texts[i])[-1], atol=2e-5, rtol=1e-5)
    engine.cache.compact()
    engine.release([slots[0]])
    logits = engine.step([Entry(s, [7], [0]) for s in slots[1:]])
    for row, text in zip(logits, texts[1:]):
        assert torch.allclose(row, plain_llama.forward(config, weights, text + [7])[-1], atol=2e-5, rtol=1e-5)
    engine.cache.check()


def test_a_step_does_not_write_on_a_shared_page(tmp_path, plain_kernels):
    config, _, engine = _setup(tmp_path, "A")
    (slot,) = engine.acquire()
    engine.step([Entry(slot, random_tokens(70, config["vocab_size"], 1), [])])
    (child,) = engine.fork(slot)
    engine.cache.set_length(slot, 30)                      # back onto page 0, which the child has too
    with pytest.raises(LlmError):
        engine.step([Entry(slot, [1], [0])])
    engine.step([Entry(child, [1], [0])])
    engine.release([child])
    engine.step([Entry(slot, [1], [0])])                   # nobody shares it any more
    engine.cache.check()


def _requests(prompts, **more):
    return [GenerationRequest(p, params=SamplingParams(temperature=0.8, seed=5 + i), **{"max_tokens": 6, **more}) for i, p in enumerate(prompts)]


def test_shared_generation_equals_separate_generation(tmp_path, plain_kernels):
    config, _, engine = _setup(tmp_path, "A", max_slots=5)
    system = random_tokens(70, config["vocab_size"], 1)
    prompts = [system + [3, 4], system + [3, 4], system + [3, 4], system + [9], random_tokens(5, config["vocab_size"], 2), system + [1] * 40, system + [2]]
    apart = generate(engine, _requests(prompts))
    fed = engine.cache.held_tokens()
    assert fed == 0
    steps = []
    step = engine.step

    def counted(entries, *a, **k):
        entries = list(entries)
        steps.append(sum(len(e.tokens) for e in entries))
        return step(entries, *a, **k)
    engine.step = counted
    together = generate(engine, _requests(prompts), share_prefix=True)
    assert [r.tokens for r in together] == [r.tokens for r in apart]
    assert [r.stop_reason for r in together] == [r.stop_reason for r in apart]
    assert steps[0] == 64 and steps[1] == 8 + 7 + 5        # the common page once, then what each distinct prompt of the first five has left
    assert engine.cache.slots.n_held == 0 and engine.cache.groups[0].pool.n_held == 0
    engine.cache.check()


def test_samples_of_a_prompt_and_what_the_cache_must_hold(tmp_path, plain_kernels):
    import llm_b200
    folder = make_folder(tmp_path, "A", torch.float32)
    config, _ = plain_llama.read_model_folder(folder)
    prompt = random_tokens(100, config["vocab_size"], 3)
    # room for the prompt once and a second page for each of four samples: five pages, not eight
    llm = llm_b200.LLM(str(folder), dtype="float32", device="cpu", context=128, batch=4, max_tokens_held=5 * PAGE)
    batches = []
    module = sys.modules["llm_b200.engine.generate"]
    run = module._run_batch
    module._run_batch = lambda engine, requests, batch, *rest: batches.append(len(batch)) or run(engine, requests, batch, *rest)
    try:
        results = llm.generate([prompt, prompt[:5]], samples=4, max_tokens=5, seed=11, stop_tokens=())
    finally:
        module._run_batch = run
    assert batches == [4, 4] and [len(r) for r in results] == [4, 4]
    for i, p in enumerate((prompt, prompt[:5])):
        for j in range(4):
            assert llm.generate([p], max_tokens=5, seed=11 + 4 * i + j, stop_tokens=())[0] == results[i][j]
    assert len({tuple(t) for t in results[1]}) > 1
    with pytest.raises(FormatError):
        llm.generate([prompt], samples=0)
    assert llm.generate([], samples=3) == []
    llm.engine.cache.check()


def test_a_prefill_that_fails_leaves_no_slot_behind(tmp_path, plain_kernels):
    config, _, engine = _setup(tmp_path, "A", max_slots=4)
    prompt = random_tokens(70, config["vocab_size"], 1)
    step = engine.step

    def fails(entries, *a, **k):
        entries = list(entries)
        if any(len(e.tokens) < 64 for e in entries):
            raise RuntimeError("no")
        return step(entries, *a, **k)
    engine.step = fails
    with pytest.raises(RuntimeError):
        generate(engine, _requests([prompt, prompt[:64] + [1], prompt]), share_prefix=True)
    assert engine.cache.slots.n_held == 0
    engine.cache.check()
