"""Which steps read shared pages once, and what captured steps are kept under, on the CPU."""
import pytest
import torch

from tiny import make_folder, random_tokens

from llm_b200.cache import PAGE, KvRequest, PagedCache
from llm_b200.engine import Engine, Entry, load_model
from llm_b200.engine import step as step_module


@pytest.fixture
def engine(tmp_path, plain_kernels):
    return Engine(load_model(make_folder(tmp_path, "F", torch.float32), torch.float32, "cpu"), max_tokens=64 * PAGE, max_slots=16)


def forked(engine, pages, members, behind=5):
    """`members` sequences that share `pages` pages and hold `behind` positions each behind them (nothing is computed)."""
    (slot,) = engine.acquire()
    engine.cache.reserve(slot, pages * PAGE + behind)
    engine.cache.set_length(slot, pages * PAGE + behind)
    return [slot] + (engine.fork(slot, members - 1) if members > 1 else [])


def sharing(engine, *groups, new=1):
    """What the engine makes of a step over groups of (pages, members)."""
    slots = [s for pages, members in groups for s in forked(engine, pages, members)]
    batch = step_module._Batch([Entry(s, [1] * new, [0]) for s in slots])
    room = torch.zeros(2 * engine._group_room(batch.n), dtype=torch.int32)
    found = engine._groups(batch, room)
    engine.release(slots)
    return found


def test_captured_steps_are_kept_under_what_launches_depend_on(engine):
    """Not under the pages that are saved: other numbers of pages within the same bounds are the same step."""
    first = sharing(engine, (5, 3))
    assert first == sharing(engine, (6, 3)) == sharing(engine, (8, 3)) and first != sharing(engine, (9, 3))
    assert sharing(engine, (5, 3), (2, 4)) == sharing(engine, (3, 3), (6, 4))
    assert sharing(engine, (5, 3), (2, 3), (2, 2)) == sharing(engine, (5, 4), (2, 2), (2, 2))     # groups of four at most
    # a prompt step's launches have a tile for every so many tokens of the largest group
    assert sharing(engine, (5, 3), (2, 3), new=30) != sharing(engine, (5, 4), (2, 2), new=30)


def test_the_rule_is_asked_once_for_every_kind_of_attention(engine, monkeypatch):
    from llm_b200 import ops
    asked = []
    monkeypatch.setattr(ops, "prefix_attention_pays", lambda *a: asked.append(a) or a[1] > 1)
    engine.sharing_shapes = ((4, 2, 64), (1, 1, 32), (8, 2, 64))
    found = sharing(engine, (5, 3), (2, 2))
    assert [a[1:4] for a in asked] == list(engine.sharing_shapes)
    assert all(a[0] == torch.float32 and a[4:8] == (5, 1, 5, 2 * 5 + 2) for a in asked)
    assert found[-1] == ((4, 2, 64), (8, 2, 64))


def test_a_step_that_gains_nothing_is_an_ordinary_one(engine, monkeypatch):
    """Nothing of the groups reaches the step, its buffer or its key."""
    from llm_b200 import ops
    seen, run = [], engine.model.forward

    def forward(tokens, ctx, rows):
        seen.append(ctx.sharing)
        return run(tokens, ctx, rows)
    monkeypatch.setattr(engine.model, "forward", forward)
    slots = forked(engine, 1, 3)
    engine.step([Entry(s, [3], [0]) for s in slots])
    assert seen[0].shapes == engine.sharing_shapes
    monkeypatch.setattr(ops, "prefix_attention_pays", lambda *a: False)
    assert sharing(engine, (5, 3)) is None
    engine.step([Entry(s, [3], [0]) for s in slots])
    assert seen[1] is None


def test_a_model_whose_attentions_read_for_themselves_asks_nothing(engine, monkeypatch):
    engine.sharing_shapes = ()
    monkeypatch.setattr(engine, "_groups", None)
    slots = forked(engine, 1, 3)
    engine.step([Entry(s, [3], [0]) for s in slots])
    engine.cache.check()


def test_what_is_counted_until_it_is_captured_is_bounded(engine):
    for i in range(step_module.MAX_SEEN + 50):
        assert engine._replay(i, 64, None, 0, None) is None
    assert 0 < len(engine._graph_seen) <= step_module.MAX_SEEN


def pays(*a):
    from llm_b200 import ops
    return ops.prefix_attention_pays(torch.bfloat16, *a)


def test_single_tokens_pay_where_reading_once_was_measured_faster():
    """(query heads, key heads, head size, sequences, 1, shared pages, saved pages, tokens of the largest group) on both sides of each line."""
    for heads, n, no, yes in [((32, 8, 128), 4, 8, 32), ((32, 8, 128), 16, 4, 8), ((32, 8, 128), 32, 4, 8), ((32, 32, 128), 16, 2, 4), ((32, 32, 128), 32, 2, 4),
                              ((32, 8, 64), 32, 8, 16), ((32, 1, 128), 16, 32, 128), ((40, 2, 64), 64, 8, 32),
                              ((32, 8, 128), 64, 1, 2), ((32, 8, 64), 64, 2, 8)]:            # these two are one launch
        assert not pays(*heads, n, 1, no, (n - 1) * no, n), (heads, n, no)
        assert pays(*heads, n, 1, yes, (n - 1) * yes, n), (heads, n, yes)
    # four groups of 16 behind 2, 4, 6 and 8 pages 21.5 / 24.3 us, behind 8 to 32 62 / 29; a pair among many sequences
    assert not pays(32, 8, 128, 64, 1, 8, 15 * 20, 16) and pays(32, 8, 128, 64, 1, 32, 15 * 80, 16)
    assert not pays(32, 8, 128, 64, 1, 128, 128, 2)


def test_few_tokens_a_sequence():
    assert pays(32, 8, 128, 64, 4, 32, 32, 8, None) and not pays(32, 8, 128, 64, 4, 16, 16, 8, None)
    assert not pays(32, 32, 128, 64, 16, 128, 128, 32, None) and pays(32, 32, 128, 32, 16, 128, 3 * 576, 64, None)


@pytest.mark.parametrize("heads", [(32, 8, 128), (32, 8, 64)])
def test_prompt_steps_of_several_groups_pay_where_their_tiles_fill_the_gpu(tmp_path, plain_kernels, heads):
    """A few questions behind a document among prompts that share nothing were slower read once (30 / 46, 101 / 148 us); several such groups were
    not (50 / 40, 269 / 185), nor questions alone."""
    engine = Engine(load_model(make_folder(tmp_path, "F", torch.float32), torch.float32, "cpu"), max_tokens=PAGE, max_slots=1)
    engine.dtype, engine.sharing_shapes = torch.bfloat16, (heads,)
    engine.cache = PagedCache([KvRequest(1, 2)], [None], max_tokens=2048 * PAGE, max_seq_len=100 * PAGE, max_slots=128, dtype=torch.float32, device="cpu")

    def taken(*groups):
        """groups: (pages, [new tokens, ...])."""
        slots, new = [], []
        for pages, counts in groups:
            slots += forked(engine, pages, len(counts)) if pages else engine.acquire(len(counts))
            new += counts
        batch = step_module._Batch([Entry(s, [1] * n, [0]) for s, n in zip(slots, new)])
        found = engine._groups(batch, torch.zeros(2 * engine._group_room(batch.n), dtype=torch.int32))
        engine.release(slots)
        return found is not None
    for pages in (32, 60):
        assert taken((pages, [40, 70]))
        for others in (6, 19, 62):
            assert not taken((pages, [17, 17]), *[(0, [17 + 29 * i % 134]) for i in range(others)])
        assert not taken((pages, [17, 17]), *[(0, [1000])] * 6)
        assert taken(*[(pages * (g + 1) // 4, [17, 54, 91, 51]) for g in range(4)])
        assert taken(*[(pages * (g + 1) // 16, [17, 54]) for g in range(16)])
        assert taken((pages, [50] * 64), *[(0, [30 + i]) for i in range(16)])
    assert not taken((0, [500]), (32, [1] * 8)) and taken((0, [500]), (32, [1] * 63))


def test_what_runs_of_prompts_begin_with_is_prefilled_in_one_step(engine, monkeypatch):
    """Two documents with their questions, a prompt alone and a repeated one: what is common once, in one step, then all the rest in another."""
    from llm_b200.engine import GenerationRequest, generate
    from llm_b200.sampling import SamplingParams
    one, two = [random_tokens(n, engine.vocab, 5 + n) for n in (130, 200)]
    prompts = [one + [3], one + [4, 5], [9, 8, 7], two + [1], two + [2], two + [2], two[:150] + [6]]
    requests = [GenerationRequest(p, max_tokens=4, params=SamplingParams(temperature=0.8, seed=i)) for i, p in enumerate(prompts)]
    apart = generate(engine, requests)
    steps, step = [], engine.step
    monkeypatch.setattr(engine, "step", lambda entries, *a, **k: steps.append([len(e.tokens) for e in entries]) or step(entries, *a, **k))
    together = generate(engine, requests, share_prefix=True)
    assert [r.tokens for r in together] == [r.tokens for r in apart]
    assert steps[0] == [128, 128] and steps[1] == [3, 4, 3, 73, 73, 23]
    assert engine.cache.slots.n_held == 0
    engine.cache.check()


def test_the_command_line_holds_a_prompt_once(tmp_path, plain_kernels, monkeypatch):
    """Whole contexts for every sample are more than a GPU has for a long prompt: what is asked for holds all samples at once, and no page more."""
    import sys
    import llm_b200
    from llm_b200.cli import _held_by_samples
    model = load_model(make_folder(tmp_path, "F", torch.float32), torch.float32, "cpu")
    held = _held_by_samples(model, 200, 8, 2048, 5)
    assert held == (3 + 5) * PAGE and _held_by_samples(model, 200, 100000, 2048, 5) == (3 + 5 * 29) * PAGE
    assert _held_by_samples(model, 192, 0, 2048, 5) == 3 * PAGE
    assert _held_by_samples(model, 200, 100000, 1 << 20, 5) == (3 + 5 * 29) * PAGE                    # the model's own limit
    batches, module = [], sys.modules["llm_b200.engine.generate"]
    run = module._run_batch
    monkeypatch.setattr(module, "_run_batch", lambda engine, requests, batch, *rest: batches.append(len(batch)) or run(engine, requests, batch, *rest))
    llm = llm_b200.LLM(model, context=2048, batch=5, max_tokens_held=held)
    results = llm.generate([random_tokens(200, 5000, 3)], samples=5, max_tokens=8, stop_tokens=())
    assert batches == [5] and [len(r) for r in results[0]] == [8] * 5
    model.cache_requests = lambda: ([KvRequest(1, 2, window=70)], [None])
    assert _held_by_samples(model, 200, 8, 2048, 5) == 5 * 4 * PAGE
