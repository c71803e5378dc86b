"""Sequences that share pages, on the GPU: forked sequences against the plain implementation (prompt steps and replayed decode
steps), every architecture's forks against sequences that were never forked, and the samples of a prompt."""
import importlib

import pytest
import torch

import plain_llama
from test_model_gpu import close
from tiny import CONFIGS, make_folder, random_tokens

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def engine_for(folder, dtype, **options):
    from llm_b200.engine import Engine, load_model
    return Engine(load_model(folder, dtype, DEV), **{"max_tokens": 8192, **options})


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("which", sorted(CONFIGS))
def test_forked_sequences_against_the_plain_implementation(tmp_path, monkeypatch, dtype, which):
    from llm_b200 import ops
    used = []
    kernel = ops.prefix_attention
    monkeypatch.setattr(ops, "prefix_attention", lambda *a, **k: used.append(1) or kernel(*a, **k))
    monkeypatch.setattr(ops, "prefix_attention_pays", lambda *a: not ops.tactics.is_disabled("prefix_attention"))      # however little is shared
    from llm_b200.engine import Entry
    folder = make_folder(tmp_path, which, BF16)
    config, weights = plain_llama.read_model_folder(folder)
    vocab, limit = config["vocab_size"], config["max_position_embeddings"]
    engine = engine_for(folder, dtype)
    common = random_tokens(70 if limit < 200 else 140, vocab, 1)
    (slot,) = engine.acquire()
    engine.step([Entry(slot, common, [])])
    (other,) = engine.acquire()
    engine.step([Entry(other, common[:11], [])])
    slots = [slot] + engine.fork(slot, 4) + [other]
    tails = [random_tokens(n, vocab, 40 + i) for i, n in enumerate((3, 25, 1, 9, 30, 2))]
    texts = [common + t for t in tails[:5]] + [common[:11] + tails[5]]

    def step(new):
        """One step with the new tokens of every sequence, against the plain implementation."""
        logits = engine.step([Entry(s, n, [len(n) - 1]) for s, n in zip(slots, new)])
        for row, text in zip(logits, texts):
            assert close(row[None], plain_llama.forward(config, weights, text)[-1:], dtype)
        return logits
    step(tails)
    for k in range(7):
        new = [random_tokens(1, vocab, 100 + 10 * k + i) for i in range(6)]
        texts = [t + n for t, n in zip(texts, new)]
        step(new)
    assert engine.graph_replays >= 4
    assert used
    new = [[5]] * 6
    texts = [t + [5] for t in texts]
    shared = step(new)
    del used[:]
    for s, t in zip(slots, texts):                         # the same step with every sequence's pages read for itself
        engine.cache.set_length(s, len(t) - 1)
    ops.tactics.disable("prefix_attention")
    engine._graphs.clear()
    try:
        apart = step(new)
    finally:
        ops.tactics.enable("prefix_attention")
    assert not used
    assert close(shared, apart.cpu(), dtype)
    engine.release(slots[:2])
    engine.cache.compact()
    slots, texts = slots[2:], [t + [7] for t in texts[2:]]
    engine._graphs.clear()
    step([[7]] * 4)
    engine.check()
    engine.cache.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name", ["guberax", "mefolorn", "zogapel", "zemozen", "duvozen", "renapel"])
def test_a_fork_continues_like_its_parent_in_every_architecture(tmp_path, dtype, name):
    """Two pairs: the parent with a sequence that had the same prompt, its child with another one; a pair's logits stay equal
    up to the order of sums while the pairs part."""
    from llm_b200.engine import Entry
    tiny = importlib.import_module("tiny_" + name)
    for which in sorted(tiny.CONFIGS):
        engine = engine_for(tiny.make_folder(tmp_path, which, dtype), dtype, max_slots=8)
        n = min(150, engine.max_seq_len - 12)
        prompt = tiny.random_tokens(n, engine.vocab, 3)
        alone = engine.acquire(2)
        (parent,) = engine.acquire()
        engine.step([Entry(s, prompt, []) for s in alone + [parent]])
        (child,) = engine.fork(parent)
        for k in range(6):
            a, b = tiny.random_tokens(1, engine.vocab, 50 + k), tiny.random_tokens(1, engine.vocab, 80 + k)
            logits = engine.step([Entry(parent, a, [0]), Entry(child, b, [0]), Entry(alone[0], a, [0]), Entry(alone[1], b, [0])]).float()
            for mine, theirs in ((0, 2), (1, 3)):
                scale = float(logits[theirs].abs().max())
                assert float((logits[mine] - logits[theirs]).abs().max()) <= (5e-5 if dtype == F32 else 0.04) * max(scale, 1.0), (which, k)
            assert k < 1 or float((logits[0] - logits[1]).abs().max()) > 1e-3
        engine.check()
        engine.cache.check()


@pytest.mark.parametrize("which", ["A", "D", "F"])
def test_samples_of_a_prompt(tmp_path, which):
    """In 32 bits the samples of a prompt drawn together are those that are drawn one by one."""
    import llm_b200
    folder = make_folder(tmp_path, which, F32)
    config, _ = plain_llama.read_model_folder(folder)
    prompt = random_tokens(80, config["vocab_size"], 3)
    llm = llm_b200.LLM(str(folder), dtype="float32", context=120, batch=6)
    options = dict(max_tokens=20, temperature=0.9, stop_tokens=())
    together = llm.generate([prompt, prompt[:70] + [1, 2]], samples=3, seed=7, share_prefix=True, **options)
    assert llm.engine.graph_replays > 0
    for i, p in enumerate((prompt, prompt[:70] + [1, 2])):
        for j in range(3):
            assert llm.generate([p], seed=7 + 3 * i + j, **options)[0] == together[i][j]
    llm.engine.cache.check()


def test_what_is_read_once_pays_from_some_bytes_on():
    from llm_b200 import ops
    pays = ops.prefix_attention_pays
    assert not pays(BF16, 32, 8, 128, 4, 1, 8, 24) and pays(BF16, 32, 8, 128, 4, 1, 32, 96)
    assert not pays(BF16, 32, 8, 128, 64, 1, 1, 63) and pays(BF16, 32, 8, 128, 64, 1, 4, 252) and pays(BF16, 32, 8, 128, 64, 1, 8, 504)
    assert not pays(BF16, 32, 8, 128, 8, 20, 16, 112) and pays(BF16, 32, 8, 128, 8, 20, 32, 224)
    assert not pays(BF16, 32, 32, 128, 8, 90, 64, 448) and pays(BF16, 32, 32, 128, 8, 90, 128, 896)
    assert pays(F32, 4, 2, 16, 2, 1, 1, 1) and not pays(F32, 4, 2, 16, 2, 1, 0, 0)
    assert not pays(BF16, 4, 2, 96, 8, 1, 128, 896) and pays(BF16, 4, 2, 80, 8, 1, 1, 7)


def test_a_long_prompt_is_read_once_by_rule(tmp_path):
    """Eight samples of 1,600 positions on the small model with heads of 128: the step chooses the kernel for itself, in a prompt step and
    in replayed decode steps."""
    from llm_b200 import ops
    from llm_b200.engine import Entry
    folder = make_folder(tmp_path, "F", BF16)
    config, weights = plain_llama.read_model_folder(folder)
    engine = engine_for(folder, F32)
    common = random_tokens(1600, config["vocab_size"], 1)
    (slot,) = engine.acquire()
    engine.step([Entry(slot, common, [])])
    slots = [slot] + engine.fork(slot, 7)
    want = plain_llama.forward(config, weights, common + [3, 4, 5])
    logits = engine.step([Entry(s, [3, 4], [0, 1]) for s in slots])
    for s in range(8):
        assert close(logits[2 * s:2 * s + 2], want[1600:1602], F32)
    for _ in range(4):
        logits = engine.step([Entry(s, [5], [0]) for s in slots])
        for s, row in zip(slots, logits):
            assert close(row[None], want[1602:1603], F32)
            engine.cache.set_length(s, 1602)
    engine.check()
    engine.cache.check()


def test_the_command_line_prints_a_line_a_sample(tmp_path, capsys):
    from llm_b200.cli import main
    import llm_b200
    folder = make_folder(tmp_path, "A", F32)
    assert main(["--model", str(folder), "--dtype", "float32", "--context", "100", "--max-tokens", "6", "--samples", "3", "--seed", "5", "7", "8", "9"]) == 0
    lines = [[int(t) for t in line.split()] for line in capsys.readouterr().out.splitlines()]
    llm = llm_b200.LLM(str(folder), dtype="float32", context=100, batch=1)
    assert lines == [llm.generate([[7, 8, 9]], max_tokens=6, seed=5 + j)[0] for j in range(3)]
    with pytest.raises(SystemExit):
        main(["--model", str(folder), "--samples", "0", "7"])
