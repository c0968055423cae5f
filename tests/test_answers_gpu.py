"""Forks, several answers to one prompt and scores through the engine, against the plain implementation."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import kefetar_kit as K
import plain_qwen3 as P

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOL = {"float32": 1e-5, "bfloat16": 2.0 ** -5}      # of the logits' scale (those of long decoding in test_engine_gpu.py)


def tokens(vocab, n, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def engine(folder, **kw):
    from llm_infer_rust_b200.engine import Engine
    kw.setdefault("cuda_graph_bs", 0)
    kw.setdefault("max_running_req", 12)
    kw.setdefault("max_total_tokens", 2048)
    return Engine(folder, **kw)


@pytest.fixture(autouse=True)
def always_shared(monkeypatch):
    """Small steps take the shared kernels too."""
    from llm_infer_rust_b200.engine import engine as module
    monkeypatch.setattr(module, "_SAVED_BYTES_AT_LEAST", 1)


@pytest.fixture(scope="module")
def folders(tiny, tiny_dirs, tmp_path_factory):
    """(folder, weights) of a configuration, stored in 32 or in 16 bits."""
    from llm_infer_rust_b200 import random_tensors, write_random_model
    made = {}

    def of(name, dtype):
        if (name, dtype) not in made:
            v = tiny[name]
            w = random_tensors(v["raw"], v["seed"], norm_std=v["norm_std"])
            folder = tiny_dirs[name]
            if dtype == "bfloat16":
                folder = write_random_model(str(tmp_path_factory.mktemp("answers")), v["raw"], v["seed"], norm_std=v["norm_std"], dtype="bfloat16")
                w = {n: t.to(torch.bfloat16) for n, t in w.items()}
            made[name, dtype] = folder, w
        return made[name, dtype]
    return of


def near(got, want, dtype):
    assert np.abs(got - want).max() <= TOL[dtype] * max(1.0, np.abs(want).max()), np.abs(got - want).max()


@pytest.mark.parametrize("graphs", [0, 12])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
def test_forked_requests_go_their_own_ways(name, dtype, graphs, tiny, folders):
    """A prompt, forks of it and of one of them, other requests beside them, prompts while they decode, ends: every row's logits are
    those of its own tokens."""
    from llm_infer_rust_b200.engine import StepEntry
    if graphs and dtype == "float32":
        pytest.skip("float32 engines have no graphs")
    raw = tiny[name]["raw"]
    vocab, page = raw["vocab_size"], tiny[name]["page_size"]
    folder, w = folders(name, dtype)
    eng = engine(folder, dtype=dtype, page_size=page, cuda_graph_bs=graphs)
    mgr = eng.cache.manager
    seq = {1: tokens(vocab, 5 * page + 3, 11), 2: tokens(vocab, 7, 12)}
    for r in (1, 2):
        eng.open_request(r)
        eng.step([StepEntry(r, seq[r], [])])

    def fork(parent, children):
        eng.fork_request(parent, children)
        for c in children:
            seq[c] = list(seq[parent])

    def decode(rows, seed, more=()):
        entries = []
        for i, r in enumerate(rows):
            new = tokens(vocab, 1, 100 * seed + i)
            seq[r] = seq.get(r, []) + new
            entries.append(StepEntry(r, new, [0]))
        for r, n in more:
            new = tokens(vocab, n, 7000 + seed)
            seq[r] = seq.get(r, []) + new
            entries.append(StepEntry(r, new, [n - 1]))
        got = eng.step(entries).float().cpu().numpy()
        for row, e in zip(got, entries):
            near(row, P.plain_forward(w, raw, seq[e.request]).numpy()[-1], dtype)
        eng.check_kernel_errors()
        assert mgr.check() == ""
    fork(1, [3, 4, 5, 6])
    assert mgr.shared_pages(eng._prefix_group) == 5
    for step in range(3):
        decode([2, 3, 1, 4, 6, 5], step)
    fork(4, [7])                                             # shares the first prompt's pages and none beyond them, or its own too
    fork(2, [8])
    for step in range(3, 3 + page):
        decode([7, 2, 5, 8, 4, 1], step)
    eng.open_request(9)
    decode([3, 4, 7], 90, more=[(9, page + 1)])              # a prompt beside decoded tokens
    eng.close_request(1)                                     # the parent ends first
    decode([7, 4, 3, 9], 91)
    decode([6], 92)
    if graphs:
        assert eng._prefix_graphs and all(g.graph is not None for g in eng._prefix_graphs.values())
    for r in (2, 3, 4, 5, 6, 7, 8, 9):
        eng.close_request(r)
    assert mgr.check() == "" and mgr.live_requests() == 0 and all(mgr.shared_pages(g) == 0 for g in range(mgr.num_groups()))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["K1", "K3", "K4"])
def test_states_of_layers_are_copied(name, dtype, tmp_path):
    """Convolutions and retention keep states beside the pages: a fork's go on from its parent's."""
    from llm_infer_rust_b200.engine import StepEntry
    raw = K.CONFIGS[name]
    w = K.random_weights(raw, 3)
    eng = K.make_engine(K.write_model(str(tmp_path / "m"), raw, w), dtype, max_requests=6)
    prompt = K.tokens(raw["vocab"], 41, 5)
    eng.open_request(1)
    eng.step([StepEntry(1, prompt, [])])
    eng.fork_request(1, [2, 3])
    seq = {r: list(prompt) for r in (1, 2, 3)}
    for step in range(6):
        entries = []
        for r in seq:
            new = K.tokens(raw["vocab"], 1, 50 * step + r)
            seq[r] += new
            entries.append(StepEntry(r, new, [0]))
        got = eng.step(entries).float().cpu().numpy()
        for row, r in zip(got, seq):
            want = K.oracle(raw, w, seq[r])[-1]
            tol = 2e-5 if dtype == "float32" else 8e-2
            assert np.abs(row - want).max() <= tol * max(1.0, np.abs(want).max())
    eng.check_kernel_errors()


def test_a_fork_without_room_and_forks_that_make_no_sense(folders):
    from llm_infer_rust_b200.engine import StepEntry
    folder, _ = folders("A", "float32")
    eng = engine(folder, dtype="float32", page_size=4, max_running_req=3, max_total_tokens=32)
    eng.open_request(1)
    eng.step([StepEntry(1, tokens(256, 27, 1), [])])           # seven of eight pages
    free = eng.cache.manager.free_pages(0)
    with pytest.raises(MemoryError, match="nothing has changed"):
        eng.fork_request(1, [2, 3])
    assert eng.cache.manager.free_pages(0) == free and eng.cache.manager.live_requests() == 1 and eng.cache.manager.check() == ""
    for parent, children in ((9, [2]), (1, [1]), (1, [2, 2])):
        with pytest.raises(ValueError):
            eng.fork_request(parent, children)
    eng.fork_request(1, [])
    eng.fork_request(1, [2])
    assert eng.request_length(2) == 27


@pytest.mark.parametrize("graphs", [0, 8])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_answers_are_what_generate_gives_with_their_seeds(dtype, graphs, folders):
    from llm_infer_rust_b200 import SamplingParams
    if graphs and dtype == "float32":
        pytest.skip("float32 engines have no graphs")
    folder, w = folders("E", dtype)
    eng = engine(folder, dtype=dtype, cuda_graph_bs=graphs)
    prompt = tokens(307, 70, 3)
    sp = SamplingParams(temperature=0.9, top_k=40, max_tokens=12, ignore_eos=True, seed=21, logprobs=3)
    got = eng.answers(prompt, 6, sp)
    assert eng.cache.manager.live_requests() == 0 and eng.cache.manager.check() == ""
    assert len({tuple(r.tokens) for r in got}) > 1
    for i, r in enumerate(got):
        assert r.finish_reason == "length" and len(r.tokens) == len(r.logprobs) == 12
        alone = eng.generate([prompt], SamplingParams(temperature=0.9, top_k=40, max_tokens=12, ignore_eos=True, seed=21 + i, logprobs=3))[0]
        # 32-bit logits leave a drawn token no choice; in bfloat16 another batch's products may move one that lies at a border
        same = next((n for n, (a, b) in enumerate(zip(r.tokens, alone.tokens)) if a != b), 12)
        assert same == 12 or dtype == "bfloat16"
        for a, b in zip(r.logprobs[:same], alone.logprobs[:same]):
            assert a.token == b.token and abs(a.logprob - b.logprob) <= 2 * TOL[dtype] * 10 and abs(a.entropy - b.entropy) <= 2 * TOL[dtype] * 10
    # what is reported is the model's own distribution
    for r in got:
        logits = P.plain_forward(w, json.load(open(os.path.join(folder, "config.json"))), prompt + r.tokens).double()
        lp = torch.log_softmax(logits, -1)[len(prompt) - 1:-1]
        scale = float(logits.abs().max())
        for t, (token, found) in enumerate(zip(r.tokens, r.logprobs)):
            assert found.token == token and len(found.top) == 3
            assert abs(found.logprob - float(lp[t, token])) <= 2 * TOL[dtype] * max(1.0, scale)
            assert all(abs(v - float(lp[t, i])) <= 2 * TOL[dtype] * max(1.0, scale) for i, v in found.top)
            assert found.top[0][1] >= found.top[1][1] >= found.top[2][1]


def test_answers_that_end_at_unlike_places(folders):
    from llm_infer_rust_b200 import SamplingParams
    folder, _ = folders("A", "float32")
    prompt = tokens(256, 30, 8)
    sp = SamplingParams(temperature=1.5, max_tokens=20, seed=4)
    stops = list(range(0, 256, 5))                              # an answer ends after five tokens or so, some at once
    eng = engine(folder, dtype="float32", page_size=4, eos_token_ids=stops)
    got = eng.answers(prompt, 12, sp)
    reasons = {r.finish_reason for r in got}
    assert "stop" in reasons and len({len(r.tokens) for r in got}) > 3 and any(len(r.tokens) == 1 for r in got)
    for i, r in enumerate(got):
        alone = eng.generate([prompt], SamplingParams(temperature=1.5, max_tokens=20, seed=4 + i))[0]
        assert (r.tokens, r.finish_reason) == (alone.tokens, alone.finish_reason) and r.logprobs is None
    assert eng.cache.manager.live_requests() == 0 and eng.cache.manager.check() == ""


def test_answers_at_their_limits(folders):
    from llm_infer_rust_b200 import SamplingParams
    folder, _ = folders("A", "float32")
    eng = engine(folder, dtype="float32", page_size=4, max_running_req=3, max_total_tokens=60, max_seq_len=40)
    one = eng.answers(tokens(256, 5, 1), 1, SamplingParams(max_tokens=6, ignore_eos=True))[0]
    assert one.tokens == eng.generate([tokens(256, 5, 1)], SamplingParams(max_tokens=6, ignore_eos=True))[0].tokens
    full = eng.answers(tokens(256, 40, 2), 2, SamplingParams(max_tokens=6, ignore_eos=True))
    assert [(len(r.tokens), r.finish_reason) for r in full] == [(1, "length")] * 2
    near_end = eng.answers(tokens(256, 38, 2), 2, SamplingParams(max_tokens=6, ignore_eos=True))
    alone = eng.generate([tokens(256, 38, 2)], SamplingParams(max_tokens=6, ignore_eos=True))[0]
    assert [r.tokens for r in near_end] == [alone.tokens] * 2 and near_end[0].finish_reason == alone.finish_reason == "length"
    for n, prompt in ((0, [1]), (4, [1]), (2, []), (2, [1] * 41)):
        with pytest.raises(ValueError):
            eng.answers(prompt, n)
    with pytest.raises(MemoryError):
        eng.answers(tokens(256, 30, 2), 3, SamplingParams(max_tokens=30, ignore_eos=True))      # 7 pages in common and 3 of each answer's own: 16, and there are 15
    assert eng.cache.manager.live_requests() == 0 and eng.cache.manager.check() == ""


@pytest.mark.parametrize("overlap", [False, True])
def test_logprobs_of_the_scheduler(overlap, folders):
    """Requests with and without log probabilities side by side, some ending before others."""
    from llm_infer_rust_b200 import SamplingParams
    folder, w = folders("B", "float32")
    raw = json.load(open(os.path.join(folder, "config.json")))
    eng = engine(folder, dtype="float32", cpu_gpu_overlap=overlap, max_running_req=3)
    prompts = [tokens(509, n, n) for n in (4, 33, 17, 9)]
    params = [SamplingParams(max_tokens=5, ignore_eos=True, logprobs=2), SamplingParams(max_tokens=9, ignore_eos=True),
              SamplingParams(max_tokens=7, ignore_eos=True, logprobs=0), SamplingParams(max_tokens=3, ignore_eos=True, logprobs=32)]
    plain = [SamplingParams(max_tokens=p.max_tokens, ignore_eos=True) for p in params]
    without = eng.generate(prompts, plain)
    got = eng.generate(prompts, params)
    assert [r.tokens for r in got] == [r.tokens for r in without] and all(r.logprobs is None for r in without)
    assert got[1].logprobs is None and not eng._logprobs
    for r, p, prompt in zip(got, params, prompts):
        if p.logprobs is None:
            continue
        lp = torch.log_softmax(P.plain_forward(w, raw, prompt + r.tokens).double(), -1)[len(prompt) - 1:-1]
        assert [t.token for t in r.logprobs] == r.tokens and all(len(t.top) == p.logprobs for t in r.logprobs)
        for t, found in enumerate(r.logprobs):
            assert abs(found.logprob - float(lp[t, found.token])) <= 4e-5
            assert abs(found.entropy + float((lp[t].exp() * lp[t]).sum())) <= 4e-4
            if found.top:
                assert found.top[0][0] == found.token                     # (greedy)
    uid = eng.add_request(prompts[0], params[0])
    while not eng.is_idle():
        eng.schedule_step()
    assert [t.token for t in eng.take_logprobs(uid)] == got[0].tokens and eng.take_logprobs(uid) == []


@pytest.mark.parametrize("portion", [1, 7, 1024])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores(dtype, portion, folders):
    folder, w = folders("E", dtype)
    raw = json.load(open(os.path.join(folder, "config.json")))
    eng = engine(folder, dtype=dtype)
    ids = tokens(307, 90, 2)
    found = eng.score(ids, top=4, portion=portion)
    logits = P.plain_forward(w, raw, ids).double()
    lp = torch.log_softmax(logits, -1)
    assert [f.token for f in found] == ids[1:]
    for t, f in enumerate(found):
        assert abs(f.logprob - float(lp[t, ids[t + 1]])) <= 2 * TOL[dtype] * max(1.0, float(logits.abs().max())) and len(f.top) == 4
    assert eng.score([5]) == [] and eng.cache.manager.live_requests() == 0
    for bad in (dict(tokens=[]), dict(tokens=[1, 2], top=33), dict(tokens=[1, 2], portion=0)):
        with pytest.raises(ValueError):
            eng.score(**bad)
    with pytest.raises(Exception, match="token id"):
        eng.score([1, 400, 2])
    assert eng.cache.manager.live_requests() == 0


def test_command_line(folders):
    folder, _ = folders("A", "float32")
    run = subprocess.run([sys.executable, "-m", "llm_infer_rust_b200", "--model-path", folder, "--prompt-ids", "1,2,3,4,5", "--max-tokens", "4",
                          "--ignore-eos", "--answers", "3", "--logprobs", "2", "--temperature", "1.0", "--seed", "3", "--max-total-tokens", "256",
                          "--max-running-req", "4", "--cuda-graph-bs", "0", "--log-level", "error"], cwd=ROOT, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    lines = [json.loads(line) for line in run.stdout.splitlines()]
    assert len(lines) == 3 and all(len(l["output_ids"]) == len(l["logprobs"]) == 4 and len(l["logprobs"][0]["top"]) == 2 for l in lines)


def test_large_groups_through_the_tcgen05_kernel(folders, monkeypatch):
    """Head size 128, 48 answers of two query heads a KV head behind 300 tokens: the engine's own step against decode attention's."""
    from llm_infer_rust_b200.engine import StepEntry
    from llm_infer_rust_b200.engine import engine as module
    from llm_infer_rust_b200.kernels import prefix
    for name in ("_TENSOR_CORE_BLOCKS", "_TENSOR_CORE_BLOCKS_A_STEP", "_TENSOR_CORE_BLOCKS_OF_GROUPS"):
        monkeypatch.setattr(prefix, name, 0)
    asked, load = [], prefix.load_entry_points
    monkeypatch.setattr(prefix, "load_entry_points", lambda source, *a: asked.append(source) or load(source, *a))
    prefix._plan.cache_clear()
    folder, _ = folders("E", "bfloat16")
    eng = engine(folder, dtype="bfloat16", max_running_req=50, max_total_tokens=4096)
    eng.open_request(1)
    eng.step([StepEntry(1, tokens(307, 300, 4), [])])
    eng.fork_request(1, list(range(2, 49)))
    ids = list(range(1, 49))
    for step in range(3):
        logits = []
        eng.step([StepEntry(r, tokens(307, 1, 60 * step + r), [0]) for r in ids])
    # one more token, by both ways on the same cache: forks of every request take it without sharing
    new = [tokens(307, 1, 999 + r)[0] for r in ids]
    twin = engine(folder, dtype="bfloat16", max_running_req=50, max_total_tokens=4096)
    twin.open_request(1)
    twin.step([StepEntry(1, tokens(307, 300, 4), [])])
    twin.fork_request(1, list(range(2, 49)))
    for least, e in ((1, eng), (1 << 60, twin)):
        module._SAVED_BYTES_AT_LEAST = least
        if e is twin:
            for step in range(3):
                e.step([StepEntry(r, tokens(307, 1, 60 * step + r), [0]) for r in ids])
        logits.append(e.step([StepEntry(r, [t], [0]) for r, t in zip(ids, new)]).float().cpu().numpy().copy())
        e.check_kernel_errors()
    prefix._plan.cache_clear()
    assert "prefix_tcgen05.cu" in asked
    near(logits[0], logits[1], "bfloat16")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_layers_whose_calls_are_made_again(head_dim, dtype):
    """Many rows without a graph: the first layer, which finds no residual yet, and the second go through Python, the third's and the
    fourth's calls are those that the second made."""
    from llm_infer_rust_b200 import Engine
    from llm_infer_rust_b200.engine import StepEntry
    from llm_infer_rust_b200.kernels import ops, prefix
    config = {"model_type": "qwen3", "architectures": ["Qwen3ForCausalLM"], "num_hidden_layers": 4, "hidden_size": 256,
              "num_attention_heads": 4, "num_key_value_heads": 2, "head_dim": head_dim, "intermediate_size": 512, "vocab_size": 300,
              "rope_theta": 10000.0, "rms_norm_eps": 1e-6, "tie_word_embeddings": True, "max_position_embeddings": 4096, "eos_token_id": None}
    eng = Engine(None, random_weights_config=config, random_weights_seed=3, dtype=dtype, max_running_req=160, max_seq_len=3000,
                 max_total_tokens=8000, cuda_graph_bs=0, log_level="warn")
    ids = list(range(1, 151))
    eng.open_request(1)
    eng.step([StepEntry(1, tokens(300, 2200, 5), [])])
    eng.fork_request(1, ids[1:])
    twins = [tokens(300, 1, r)[0] for r in ids]
    called, again = [], []
    inner, inner_again = prefix.prefix_attention, ops.LayerCalls.again
    prefix.prefix_attention = lambda *a, **kw: called.append(1) or inner(*a, **kw)
    ops.LayerCalls.again = lambda self, values: again.append(inner_again(self, values)) or again[-1]
    try:
        got = eng.step([StepEntry(r, [t], [0]) for r, t in zip(ids, twins)]).clone()
        assert len(called) == 2 and again == [True] * 2
        for r in ids:                                            # the same step again, every layer through Python
            eng.close_request(r)
        eng.open_request(1)
        eng.step([StepEntry(1, tokens(300, 2200, 5), [])])
        eng.fork_request(1, ids[1:])
        eng.model.repeats_layers = False
        want = eng.step([StepEntry(r, [t], [0]) for r, t in zip(ids, twins)]).clone()
        assert len(called) == 6
    finally:
        prefix.prefix_attention, ops.LayerCalls.again = inner, inner_again
    assert torch.equal(got, want)
    eng.check_kernel_errors()


def test_answers_whose_copies_fail_leave_nothing(folders, monkeypatch):
    from llm_infer_rust_b200 import SamplingParams
    folder, _ = folders("A", "float32")
    eng = engine(folder, dtype="float32", page_size=4)
    free = eng.cache.manager.free_pages(0)

    def fails(copies):
        raise RuntimeError("the copies fail")
    with monkeypatch.context() as m:
        m.setattr(eng.cache, "copy_fork", fails)
        with pytest.raises(RuntimeError, match="the copies fail"):
            eng.answers(tokens(256, 30, 2), 4, SamplingParams(max_tokens=5, ignore_eos=True))
    mgr = eng.cache.manager
    assert mgr.live_requests() == 0 and mgr.free_pages(0) == free and mgr.shared_pages(0) == 0 and mgr.check() == ""
    assert len(eng.answers(tokens(256, 30, 2), 4, SamplingParams(max_tokens=5, ignore_eos=True))) == 4


@pytest.mark.parametrize("name", ["K1", "K4"])
def test_layers_that_read_every_row_by_itself_have_no_graphs_of_shared_pages(name, tmp_path):
    """Their forks decode in the graphs that are there."""
    from llm_infer_rust_b200.engine import StepEntry
    raw = K.CONFIGS[name]
    w = K.random_weights(raw, 3)
    eng = K.make_engine(K.write_model(str(tmp_path / "m"), raw, w), "bfloat16", max_requests=4, cuda_graph_bs=4)
    captures = []
    capture = eng._capture
    eng._capture = lambda *a: captures.append(a) or capture(*a)
    prompt = K.tokens(raw["vocab"], 41, 5)
    eng.open_request(1)
    eng.step([StepEntry(1, prompt, [])])
    eng.fork_request(1, [2, 3])
    seq = {r: list(prompt) for r in (1, 2, 3)}
    for step in range(4):
        entries = []
        for r in seq:
            new = K.tokens(raw["vocab"], 1, 50 * step + r)
            seq[r] += new
            entries.append(StepEntry(r, new, [0]))
        got = eng.step(entries).float().cpu().numpy()
        for row, r in zip(got, seq):
            want = K.oracle(raw, w, seq[r])[-1]
            assert np.abs(row - want).max() <= 8e-2 * max(1.0, np.abs(want).max())
    eng.check_kernel_errors()
    assert not captures and not eng._prefix_graphs


@pytest.mark.parametrize("graphs", [0, 8])
def test_steps_of_more_rows_than_the_tensor_core_kernels_take_read_by_themselves(graphs, folders, monkeypatch):
    """The limit is lowered: six rows in three groups, a graph of eight rows in as many, are beyond it."""
    from llm_infer_rust_b200.engine import StepEntry
    from llm_infer_rust_b200.kernels import prefix
    folder, w = folders("E", "bfloat16")
    raw = json.load(open(os.path.join(folder, "config.json")))
    calls = []
    inner = prefix.prefix_attention
    monkeypatch.setattr(prefix, "prefix_attention", lambda *a, **k: calls.append(k) or inner(*a, **k))
    found = {}
    for limit in (8, 400):
        monkeypatch.setattr(prefix, "_MOST_ENTRIES", limit)
        prefix._plan.cache_clear()
        eng = engine(folder, dtype="bfloat16", cuda_graph_bs=graphs)
        prompts = {1: tokens(307, 70, 3), 2: tokens(307, 90, 4)}
        for r, prompt in prompts.items():
            eng.open_request(r)
            eng.step([StepEntry(r, prompt, [])])
        eng.fork_request(1, [3, 4])
        eng.fork_request(2, [5, 6])
        calls.clear()
        for step in range(3):
            rows = {r: tokens(307, 1, 60 * step + r) for r in range(1, 7)}
            logits = eng.step([StepEntry(r, t, [0]) for r, t in rows.items()]).float().cpu().numpy().copy()
        eng.check_kernel_errors()
        found[limit] = logits
        assert bool(calls) == (limit == 400)
    prefix._plan.cache_clear()
    near(found[8], found[400], "bfloat16")


def test_graphs_of_shared_pages_are_captured_when_they_come_again_and_kept(folders):
    from llm_infer_rust_b200 import SamplingParams
    from llm_infer_rust_b200.engine import StepEntry
    folder, _ = folders("A", "bfloat16")
    eng = engine(folder, dtype="bfloat16", cuda_graph_bs=12, eos_token_ids=list(range(0, 256, 11)))
    captures = []
    capture = eng._capture
    eng._capture = lambda g, *a: captures.append(g.bucket) or capture(g, *a)
    eng.open_request(1)
    eng.step([StepEntry(1, tokens(256, 40, 1), [])])
    eng.fork_request(1, [2, 3])
    counts = []
    for step in range(4):
        eng.step([StepEntry(r, tokens(256, 1, 10 * step + r), [0]) for r in (1, 2, 3)])
        counts.append(len(captures))
    assert counts == [0, 1, 1, 1]                             # (the first step went through the graph that was there)
    for r in (1, 2, 3):
        eng.close_request(r)
    # answers that end at unlike places pass through all buckets, with few and with many keys of their own
    sp = SamplingParams(temperature=1.5, max_tokens=200, seed=4)
    first = eng.answers(tokens(256, 30, 8), 12, sp)
    assert max(len(r.tokens) for r in first) > 1
    for _ in range(2):
        last = eng.answers(tokens(256, 30, 8), 12, sp)
    known = len(captures)
    assert 3 <= len(eng._prefix_graphs) <= eng._prefix_graph_limit == 10
    again = eng.answers(tokens(256, 30, 8), 12, sp)
    assert len(captures) == known and [r.tokens for r in again] == [r.tokens for r in last]
    # what is not asked for goes first
    eng._prefix_graph_limit = 2
    for bucket in (1, 2, 4):
        assert eng._prefix_graph(bucket, 1, 1 << 12, 7) is None and eng._prefix_graph(bucket, 1, 1 << 12, 7).bucket == bucket
    assert [key[0] for key in eng._prefix_graphs] == [2, 4]


def test_answers_and_scores_without_a_slot_for_their_request(folders):
    from llm_infer_rust_b200 import SamplingParams
    folder, _ = folders("A", "float32")
    eng = engine(folder, dtype="float32", page_size=4, max_running_req=2, max_total_tokens=64)
    eng.open_request(1)
    eng.open_request(2)
    for call in (lambda: eng.answers([1, 2, 3], 2, SamplingParams(max_tokens=2)), lambda: eng.score([1, 2, 3])):
        with pytest.raises(MemoryError, match="no request can be opened"):
            call()
    assert eng.cache.manager.live_requests() == 2 and eng.cache.manager.check() == ""
    eng.close_request(1)
    assert len(eng.score([1, 2, 3])) == 2 and len(eng.answers([1, 2, 3], 1, SamplingParams(max_tokens=2, ignore_eos=True))[0].tokens) == 2
    eng.close_request(2)
    assert len(eng.answers([1, 2, 3], 2, SamplingParams(max_tokens=2, ignore_eos=True))) == 2


def test_command_line_goes_on_behind_a_prompt_that_is_refused(folders):
    folder, _ = folders("A", "float32")
    long = ",".join(["7"] * 70)
    run = subprocess.run([sys.executable, "-m", "llm_infer_rust_b200", "--model-path", folder, "--prompt-ids", long, "--prompt-ids", "1,2,3", "--max-tokens",
                          "4", "--ignore-eos", "--answers", "2", "--max-seq-len", "64", "--max-total-tokens", "256", "--max-running-req", "4",
                          "--cuda-graph-bs", "0", "--log-level", "error"], cwd=ROOT, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    lines = [json.loads(line) for line in run.stdout.splitlines()]
    assert [(len(l["prompt_ids"]), len(l["output_ids"]), l["finish_reason"]) for l in lines] == [(70, 0, "abort")] * 2 + [(3, 4, "length")] * 2
