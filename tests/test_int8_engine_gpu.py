"""The engine with a cache held in 8 bits on the GPU: what its layers ask of the operators is checked call by call against the definition, replayed and
recorded steps against plain ones bit for bit, forks against sequences that were never forked, and the ways a user has to it."""
import pytest
import torch

import test_int8_cache_gpu as definition
from tiny import CONFIGS, make_folder, random_tokens

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def engine_for(folder, dtype, **options):
    from llm_b200.engine import Engine, load_model
    return Engine(load_model(folder, dtype, DEV), **{"max_tokens": 8192, "cache_dtype": "int8", **options})


@pytest.fixture
def checked(monkeypatch):
    """Every call of the two operators is compared with the definition."""
    from llm_b200 import ops
    calls = {"append": 0, "attention": 0}
    append, attention = ops.rope_cache_write_int8, ops.attention_int8

    def batch(cu, lens, table, ring, keys, values, heads, kv, dim, dtype):
        cu, lens = cu.tolist(), lens.tolist()
        return dict(lengths=lens, cu=cu, new=[b - a for a, b in zip(cu, cu[1:])], table=table, ring=ring, keys=keys, values=values, heads=heads, kv_heads=kv,
                    dim=dim, dtype=dtype)

    def checked_append(qkv, angles, tok_pos, tok_seq, cu, table, ring, keys, values, heads, kv, dim, interleaved=False, write_cache=True, out=None):
        calls["append"] += 1
        lens = [int(tok_pos[int(cu[i + 1]) - 1]) + 1 for i in range(len(cu) - 1)]
        b = batch(cu, torch.tensor(lens), table, ring, keys, values, heads, kv, dim, qkv.dtype)
        before = definition.copies(b)
        got = append(qkv, angles, tok_pos, tok_seq, cu, table, ring, keys, values, heads, kv, dim, interleaved, write_cache, out)
        x = qkv.view(-1, heads + 2 * kv, dim)
        if write_cache:
            definition.check_append(b, x, angles, interleaved, before, got)
        return got

    def checked_attention(q, keys, values, table, ring, lens, cu, heads, kv, dim, scale, window=0, **more):
        calls["attention"] += 1
        got = attention(q, keys, values, table, ring, lens, cu, heads, kv, dim, scale, window, **more)
        b = batch(cu, lens, table, ring, keys, values, heads, kv, dim, q.dtype)
        definition.check(dict(b, q=q, scale=scale, window=window), got)
        return got
    monkeypatch.setattr(ops, "rope_cache_write_int8", checked_append)
    monkeypatch.setattr(ops, "attention_int8", checked_attention)
    return calls


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("which", sorted(CONFIGS))
def test_every_call_of_a_layer(tmp_path, checked, dtype, which):
    from llm_b200.engine import Entry
    engine = engine_for(make_folder(tmp_path, which, BF16), dtype, use_graphs=False, step_tokens=50)
    engine.use_records = False
    vocab = engine.vocab
    longest = min(engine.max_seq_len - 8, 140)
    texts = [random_tokens(n, vocab, 60 + n) for n in (longest, 17, 66 if longest > 66 else 20)]
    slots = engine.acquire(3)
    engine.step([Entry(s, t, [len(t) - 1]) for s, t in zip(slots, texts)])
    slots += engine.fork(slots[0], 1)
    for i in range(3):
        engine.step([Entry(s, random_tokens(1 + (i + j) % 2 * i, vocab, i), [0]) for j, s in enumerate(slots)])
    engine.check()
    assert checked["append"] == checked["attention"] > 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("which", sorted(CONFIGS))
def test_replayed_and_recorded_steps_are_plain_ones(tmp_path, dtype, which):
    """The same steps with graphs and records and without: the same bits, over a growing length, other slots and pages."""
    from llm_b200.engine import Entry
    folder = make_folder(tmp_path, which, BF16)
    quick, plain = engine_for(folder, dtype), engine_for(folder, dtype, use_graphs=False)
    plain.use_records = False
    vocab, steps = quick.vocab, min(quick.max_seq_len - 40, 40)
    results = []
    for engine in (quick, plain):
        logits = []
        for start in (5, 20, 20):                            # the third time in other slots and pages
            slots = engine.acquire(3)
            texts = [random_tokens(start + 7 * i, vocab, 70 + i) for i in range(3)]
            logits.append(engine.step([Entry(s, t, [len(t) - 1]) for s, t in zip(slots, texts)]))
            for k in range(min(steps, 12)):
                logits.append(engine.step([Entry(s, [(k * 13 + i) % vocab], [0]) for i, s in enumerate(slots)]))
            spare = engine.acquire(1)
            engine.release(slots)
            engine.step([Entry(spare[0], [1, 2, 3], [])])
        engine.check()
        results.append(logits)
    assert quick.graph_replays > 0 and quick.records_run > 0
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forks_and_compaction(tmp_path, dtype):
    """Forked sequences go on as ones that were never forked, in the same batch: the same bits."""
    from llm_b200.engine import Entry
    which = sorted(CONFIGS)[0]
    folder = make_folder(tmp_path, which, BF16)
    forked, apart = engine_for(folder, dtype), engine_for(folder, dtype)
    tokens = random_tokens(min(forked.max_seq_len - 12, 90), forked.vocab, 5)
    (slot,) = forked.acquire()
    forked.step([Entry(slot, tokens, [])])
    slots = [slot] + forked.fork(slot, 3)
    others = apart.acquire(4)
    for o in others:
        apart.step([Entry(o, tokens, [])])
    for k in range(6):
        new = [[(31 * k + 7 * i) % forked.vocab] for i in range(4)]
        a = forked.step([Entry(s, n, [0]) for s, n in zip(slots, new)])
        b = apart.step([Entry(s, n, [0]) for s, n in zip(others, new)])
        assert torch.equal(a, b)
        if k == 2:
            for engine, held in ((forked, slots), (apart, others)):
                (spare,) = engine.acquire()
                engine.step([Entry(spare, tokens[:70], [])])
                engine.release([spare])
            forked.cache.compact()
            forked.cache.check()
    forked.check()
    assert forked.cache.groups[0].pool.n_held < apart.cache.groups[0].pool.n_held or len(tokens) < 64


def test_generation_and_the_command_line(tmp_path, capsys):
    import llm_b200
    from llm_b200 import cli
    folder = make_folder(tmp_path, sorted(CONFIGS)[0], BF16)
    llm = llm_b200.LLM(str(folder), context=100, batch=4, cache_dtype="int8")
    prompt = random_tokens(30, llm.engine.vocab, 9)
    ids = llm.generate([prompt, prompt[:7]], max_tokens=12, temperature=0)
    assert llm.generate([prompt], max_tokens=12, temperature=0) == ids[:1]
    four = llm.generate([prompt], max_tokens=8, samples=4, temperature=0)
    assert [len(set(map(tuple, four[0])))] == [1] and four[0][0] == ids[0][:8]
    llm.engine.check()
    arguments = ["--model", str(folder), "--context", "100", "--max-tokens", "12", "--temperature", "0", "--cache-dtype", "int8"]
    capsys.readouterr()
    assert cli.main(arguments + [str(t) for t in prompt]) == 0
    assert [int(x) for x in capsys.readouterr().out.split()] == ids[0]
    assert cli.main(["bench", "-m", str(folder), "-c", "64", "-p", "16", "-n", "4", "-r", "1", "--cache-dtype", "int8"]) == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_recorded_passes_keep_no_results(tmp_path, dtype):
    """Passes recorded under many keys hold addresses of one arena: a record keeps no more than one of an engine with a cache in the run's type."""
    from llm_b200.engine import Entry
    folder = make_folder(tmp_path, sorted(CONFIGS)[0], BF16)

    def grown(cache_dtype):
        """What a record of a pass of n - 1 tokens adds to what the device has allocated, behind one of n."""
        engine = engine_for(folder, dtype, use_graphs=False, max_tokens=4096, cache_dtype=cache_dtype)
        longest, held = min(engine.max_seq_len - 8, 120), []
        for n in (longest, longest - 1):
            for _ in range(4):
                (slot,) = engine.acquire()
                engine.step([Entry(slot, random_tokens(n, engine.vocab, n), [n - 1])])
                engine.release([slot])
            torch.cuda.synchronize()
            held.append((torch.cuda.memory_allocated(), len(engine._records)))
        engine.check()
        (before, keys), (after, more) = held
        assert engine.records_run > 0 and more > keys
        queries = sum(block.mixer.q_width for block in engine.model.blocks) * (longest - 1) * torch.empty((), dtype=dtype).element_size()
        return after - before, queries

    (plain, queries), (int8, _) = grown(None), grown("int8")
    assert int8 - plain < queries


def test_blocks_of_the_command_line(tmp_path, capsys):
    """--cache-block reaches the engine: the same tokens as LLM(cache_block=...) gives, and numbers that are none refused."""
    import llm_b200
    from llm_b200 import cli
    from llm_b200.errors import LlmError
    folder = make_folder(tmp_path, sorted(CONFIGS)[0], BF16)
    prompt = random_tokens(30, llm_b200.LLM(str(folder), context=100).engine.vocab, 9)
    for block in (1, 64):
        (want,) = llm_b200.LLM(str(folder), context=100, batch=1, cache_dtype="int8", cache_block=block).generate([prompt], max_tokens=12, temperature=0)
        arguments = ["--model", str(folder), "--context", "100", "--max-tokens", "12", "--temperature", "0", "--cache-dtype", "int8", "--cache-block", str(block)]
        capsys.readouterr()
        assert cli.main(arguments + [str(t) for t in prompt]) == 0
        assert [int(x) for x in capsys.readouterr().out.split()] == want
    assert cli.main(["bench", "-m", str(folder), "-c", "64", "-p", "16", "-n", "4", "-r", "1", "--cache-dtype", "int8", "--cache-block", "32"]) == 0
    with pytest.raises(LlmError, match="blocks of 3 positions"):
        llm_b200.LLM(str(folder), context=100, cache_dtype="int8", cache_block=3)
