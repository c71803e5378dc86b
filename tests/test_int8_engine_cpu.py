"""The engine with a cache held in 8 bits: host logic on the CPU, the kernels replaced by their plain statements. What is under test is which rows,
pages, scales and slots the operators are given."""
import gc
import weakref

import pytest
import torch

import plain_int8
import plain_llama
from tiny import CONFIGS, make_folder, random_tokens

from llm_b200.cache import KvRequest, PagedCache
from llm_b200.engine import Engine, Entry, load_model
from llm_b200.errors import LlmError


def setup(tmp_path, monkeypatch, which, **options):
    plain_int8.install(monkeypatch)
    folder = make_folder(tmp_path, which, torch.float32)
    config, weights = plain_llama.read_model_folder(folder)
    return config, weights, Engine(load_model(folder, torch.float32, "cpu"), **{"max_tokens": 2048, "cache_dtype": "int8", **options})


@pytest.mark.parametrize("which", sorted(CONFIGS))
def test_without_the_rounding_the_plain_implementation(tmp_path, plain_kernels, monkeypatch, which):
    """Rows are read as they were before they were rounded: everything else of a step is then the plain implementation's."""
    monkeypatch.setattr(plain_int8, "exact", {})
    config, weights, engine = setup(tmp_path, monkeypatch, which, step_tokens=48)
    texts = [random_tokens(n, config["vocab_size"], 40 + n) for n in (60, 11)]
    expected = [plain_llama.forward(config, weights, t) for t in texts]
    slots = engine.acquire(2)
    logits = engine.step([Entry(s, t[:-3], list(range(len(t) - 3))) for s, t in zip(slots, texts)])
    got = [logits[:57], logits[57:]]
    for k in (3, 2, 1):
        last = engine.step([Entry(s, t[len(t) - k:len(t) - k + 1], [0]) for s, t in zip(slots, texts)])
        got = [torch.cat([a, b[None]]) for a, b in zip(got, last)]
    for a, b in zip(got, expected):
        assert torch.allclose(a, b, atol=5e-5 * max(1.0, float(b.abs().max())), rtol=1e-5)


@pytest.mark.parametrize("which", sorted(CONFIGS))
@pytest.mark.parametrize("block", [1, 16])
def test_unequal_batches_slots_and_cuts(tmp_path, plain_kernels, monkeypatch, which, block):
    """Sequences of a batch do not touch one another; with a scale for each position a cut prompt is the whole one's."""
    config, weights, engine = setup(tmp_path, monkeypatch, which, cache_block=block)
    vocab = config["vocab_size"]
    limit = min(config["max_position_embeddings"], 130)
    texts = [random_tokens(n, vocab, 20 + i) for i, n in enumerate((limit, 9, 65 if limit > 65 else 30))]
    alone = []
    for text in texts:
        (slot,) = engine.acquire()
        alone.append(engine.step([Entry(slot, text[:-2], []), ]))
        alone[-1] = torch.cat([engine.step([Entry(slot, text[-2:-1], [0])]), engine.step([Entry(slot, text[-1:], [0])])])
        engine.release([slot])
    slots = engine.acquire(3)
    engine.step([Entry(s, t[:-2], []) for s, t in zip(slots, texts)])
    first = engine.step([Entry(s, t[-2:-1], [0]) for s, t in zip(slots, texts)])
    second = engine.step([Entry(s, t[-1:], [0]) for s, t in zip(slots, texts)])
    for i in range(3):
        assert torch.allclose(torch.stack([first[i], second[i]]), alone[i], atol=2e-5, rtol=1e-5)
    engine.release(slots)
    if block == 1:
        text = texts[0]
        (slot,) = engine.acquire()
        whole = engine.step([Entry(slot, text, [len(text) - 1])])
        (other,) = engine.acquire()
        for at in range(0, len(text), 37):
            piece = text[at:at + 37]
            cut = engine.step([Entry(other, piece, [len(piece) - 1])])
        assert torch.allclose(cut, whole, atol=2e-4, rtol=1e-4)
    engine.cache.check()


@pytest.mark.parametrize("block", [1, 16, 64])
def test_forks_go_on_as_their_parent(tmp_path, plain_kernels, monkeypatch, block):
    config, weights, engine = setup(tmp_path, monkeypatch, sorted(CONFIGS)[0], cache_block=block)
    vocab = config["vocab_size"]
    tokens = random_tokens(70 if config["max_position_embeddings"] > 100 else 40, vocab, 5)
    (slot,) = engine.acquire()
    engine.step([Entry(slot, tokens, [])])
    children = engine.fork(slot, 3)
    tails = [random_tokens(4, vocab, 30 + i) for i in range(4)]
    apart = []
    for tail in tails:
        (one,) = engine.acquire()
        engine.step([Entry(one, tokens, [])])
        for t in tail:
            out = engine.step([Entry(one, [t], [0])])
        apart.append(out[0])
        engine.release([one])
    for step in zip(*tails):
        together = engine.step([Entry(s, [t], [0]) for s, t in zip([slot] + children, step)])
    assert torch.allclose(together, torch.stack(apart), atol=2e-5, rtol=1e-5)
    engine.release([children[0]])
    assert engine.cache.compact() >= 0
    engine.cache.check()
    more = engine.step([Entry(slot, [1], [0])])
    assert bool(torch.isfinite(more).all())


def test_half_the_bytes_and_refusals(tmp_path, plain_kernels, monkeypatch):
    config, weights, engine = setup(tmp_path, monkeypatch, sorted(CONFIGS)[0])
    plain = Engine(engine.model, max_tokens=2048)
    kv = [r for r in engine.model.cache_requests()[0] if r is not None]
    held = sum(2 * r.n_kv_heads * (r.head_dim + 4 / 16) for r in kv) * 2048
    assert engine.cache.bytes() == held and plain.cache.bytes() > 3.5 * held          # (32 bits)
    with pytest.raises(LlmError):
        Engine(engine.model, max_tokens=2048, cache_dtype="int4")
    with pytest.raises(LlmError):
        Engine(engine.model, max_tokens=2048, cache_dtype="int8", cache_block=3)
    sizes = dict(max_tokens=128, max_seq_len=128, max_slots=1, dtype=torch.float32, device="cpu", kv_dtype=torch.int8)
    for request in (KvRequest(2, 16, value_dim=32), KvRequest(2, 16, values_are_keys=True), KvRequest(2, 15)):
        with pytest.raises(LlmError):
            PagedCache([request], [None], **sizes)
    for mixer in {type(engine.model.blocks[item.layer].mixer) for item in engine.model.spec.schedule}:
        monkeypatch.setattr(mixer, "serves_int8_cache", False)
    with pytest.raises(LlmError, match="does not read"):
        Engine(engine.model, max_tokens=2048, cache_dtype="int8")


@pytest.mark.parametrize("options", [{}, {"cache_dtype": None}])
def test_an_engine_goes_with_its_last_name(tmp_path, plain_kernels, monkeypatch, options):
    """Captured steps that are destroyed by the garbage collector while another engine captures end that capture."""
    config, weights, engine = setup(tmp_path, monkeypatch, sorted(CONFIGS)[0], **options)
    (slot,) = engine.acquire()
    engine.step([Entry(slot, [1, 2, 3], [2])])
    gone = weakref.ref(engine)
    gc.collect()
    gc.disable()
    try:
        del engine
        assert gone() is None
    finally:
        gc.enable()


def test_mixers_of_other_designs_are_refused(tmp_path, plain_kernels):
    from tiny_zemozen import make_folder as zemozen_folder
    engine_of = lambda **o: Engine(load_model(zemozen_folder(tmp_path, "P", torch.float32), torch.float32, "cpu"), max_tokens=512, **o)
    engine_of()
    with pytest.raises(LlmError, match="does not read a cache in 8 bits"):
        engine_of(cache_dtype="int8")


@pytest.mark.parametrize("which", sorted(CONFIGS))
def test_queries_and_results_lie_in_the_arena(tmp_path, plain_kernels, monkeypatch, which):
    """The operators of a layer are given where to write to: buffers of the arena that do not overlap, and that an engine with a cache in the
    run's type has too. (A result that is allocated in each call would be kept once for each layer and recorded step.)"""
    from llm_b200 import ops
    config, weights, engine = setup(tmp_path, monkeypatch, which)
    seen = []

    def inside(t, n, width):
        begin, size = engine.workspace.arena.data_ptr(), engine.workspace.arena.numel()
        assert t is not None and tuple(t.shape) == (n, width) and t.is_contiguous()
        assert begin <= t.data_ptr() and t.data_ptr() + t.numel() * t.element_size() <= begin + size
        return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()

    def append(qkv, *args, out=None, **more):
        a, b = inside(out, qkv.shape[0], args[8] * args[10])
        assert b <= qkv.data_ptr() or qkv.data_ptr() + qkv.numel() * qkv.element_size() <= a
        seen.append("append")
        return plain_int8.rope_cache_write_int8(qkv, *args, out=out, **more)

    def attention(q, *args, out=None, **more):
        a, b = inside(out, q.shape[0], args[6] * args[8])
        assert b <= q.data_ptr() or q.data_ptr() + q.numel() * q.element_size() <= a
        seen.append("attention")
        return plain_int8.attention_int8(q, *args, out=out, **more)

    monkeypatch.setattr(ops, "rope_cache_write_int8", append)
    monkeypatch.setattr(ops, "attention_int8", attention)
    (slot,) = engine.acquire()
    engine.step([Entry(slot, [1, 2, 3], [2])])
    engine.step([Entry(slot, [4], [0])])
    assert seen.count("append") == seen.count("attention") > 0
    other = Engine(engine.model, max_tokens=2048)
    for n in (1, 3, 100):
        plan = engine.workspace.plan_for(n)
        plan.check()
        assert plan.total == other.workspace.plan_for(n).total


def test_sequences_go_back_to_where_a_block_begins(tmp_path, plain_kernels, monkeypatch):
    """Positions that are dropped keep their say in the scale of a block that is continued, and one that was not finite its block: going back into the
    middle of a block is refused, and what is dropped from a block's beginning on leaves nothing behind."""
    config, weights, engine = setup(tmp_path, monkeypatch, sorted(CONFIGS)[0], cache_block=16)
    tokens = random_tokens(40, config["vocab_size"], 3)
    (slot,) = engine.acquire()
    engine.step([Entry(slot, tokens[:32], [])])
    want = engine.step([Entry(slot, tokens[32:], list(range(8)))])
    for length in (39, 33, 31, 17, 1):
        with pytest.raises(LlmError, match="block"):
            engine.cache.set_length(slot, length)
        assert engine.length(slot) == 40
    engine.step([Entry(slot, random_tokens(5, config["vocab_size"], 4), [])])
    engine.cache.set_length(slot, 32)
    for group in engine.cache.groups:                          # (what the dropped positions may have left: no number at all)
        page = group.slot_pages[slot][0]
        group.scales[:, :, page, :, 2:] = float("nan")
    assert torch.equal(engine.step([Entry(slot, tokens[32:], list(range(8)))]), want)
    engine.cache.set_length(slot, 40)
    engine.cache.set_length(slot, 0)
    engine.cache.set_length(slot, 5)                           # (forward, as before)
    for options in ({"cache_block": 1}, {"cache_dtype": None}):
        other = Engine(engine.model, **{"max_tokens": 2048, "cache_dtype": "int8", **options})
        (slot,) = other.acquire()
        want = other.step([Entry(slot, tokens, [39])])
        other.cache.set_length(slot, 37)
        assert torch.allclose(other.step([Entry(slot, tokens[37:], [2])]), want, atol=2e-4, rtol=1e-4)
