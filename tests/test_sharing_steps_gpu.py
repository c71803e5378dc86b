"""Steps of forked sequences on the GPU by the engine's own rule: which of them read shared pages once, what is captured for them, and their logits."""
import pytest
import torch

import plain_llama
from test_model_gpu import close
from tiny import make_folder, random_tokens

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def engine_for(folder, dtype, **options):
    from llm_b200.engine import Engine, load_model
    return Engine(load_model(folder, dtype, DEV), **{"max_tokens": 16384, **options})


def test_another_number_of_shared_pages_replays_the_same_graph(tmp_path):
    from llm_b200.engine import Entry
    folder = make_folder(tmp_path, "F", F32)
    config, weights = plain_llama.read_model_folder(folder)
    engine = engine_for(folder, F32)
    graphs = []
    for pages in (5, 6, 7):
        prompt = random_tokens(pages * 64 + 9, config["vocab_size"], pages)
        (slot,) = engine.acquire()
        engine.step([Entry(slot, prompt, [])])
        slots, texts = [slot] + engine.fork(slot, 2), [prompt] * 3
        for k in range(5):
            new = [random_tokens(1, config["vocab_size"], 100 * pages + 10 * k + i) for i in range(3)]
            texts = [t + n for t, n in zip(texts, new)]
            logits = engine.step([Entry(s, n, [0]) for s, n in zip(slots, new)])
        for row, text in zip(logits, texts):
            assert close(row[None], plain_llama.forward(config, weights, text)[-1:], F32)
        engine.release(slots)
        graphs.append((len(engine._graphs), engine.graph_replays))
    assert graphs == [(1, 3), (1, 8), (1, 13)]
    engine.check()


@pytest.mark.parametrize("members, pages, once", [
    (32, 29, True), (32, 28, False),         # one tile of 128 rows
    (130, 21, True), (130, 20, False),       # more rows, own pages behind them
    (40, 9, True), (40, 8, False),           # each sequence reads the few pages itself, in one launch
])
def test_samples_in_bfloat16_by_the_rule(tmp_path, monkeypatch, members, pages, once):
    """Samples on both sides of the line: which kernel a step takes, in plain and in replayed steps, and its logits."""
    from llm_b200 import ops
    from llm_b200.engine import Entry
    calls = []
    kernel = ops.prefix_attention
    monkeypatch.setattr(ops, "prefix_attention", lambda *a, **k: calls.append(1) or kernel(*a, **k))
    folder = make_folder(tmp_path, "F", BF16)
    config, weights = plain_llama.read_model_folder(folder)
    engine = engine_for(folder, BF16)
    common = random_tokens(pages * 64 + 5, config["vocab_size"], 1)
    (slot,) = engine.acquire()
    engine.step([Entry(slot, common, [])])
    slots = [slot] + engine.fork(slot, members - 1)
    texts = [common + [3, 4, 5, 6, 7], common + [8, 9, 10, 11, 12]]
    want = [plain_llama.forward(config, weights, t)[-5:] for t in texts]
    for k in range(5):
        logits = engine.step([Entry(s, [texts[i % 2][len(common) + k]], [0]) for i, s in enumerate(slots)])
        for i in range(2):
            assert close(logits[i::2], want[i][k][None].expand(len(logits[i::2]), -1), BF16)
    assert engine.graph_replays == 3
    # two plain steps and the capture, in both layers
    assert len(calls) == (6 if once else 0)
    assert [key[2] is not None for key in engine._graphs] == [once]
    engine.check()
    engine.cache.check()
