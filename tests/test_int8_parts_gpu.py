"""Parts and engines whose projections are in 8-bit integers, against the plain implementation with the same products: weights
and activations taken to 8 bits by the formula, the rest in 64 bits.

Weights are taken to 8 bits once, by the float formula, on both sides.  Where an activation lies within rounding of half a step,
float arithmetic and 64 bits take it to either side, and everything behind it moves by that step (in attention: every later token).
One element in some 100,000 does (2^-24 of up to 127 steps, a few times over), a part's single pass of up to 36,000 elements has
none or one.  Against what 8 bits do to the logits, where all elements are off by up to half a step, a handful of such elements is
below a tenth.
"""
import pytest
import torch

import plain_qwen3 as P

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


class EightBit:
    """Stands for a weight matrix in ``x @ w.T``: both sides in 8 bits."""

    def __init__(self, w):
        top = w.float().abs().amax(dim=1, keepdim=True)
        most = torch.full_like(top, 127.0)
        self.q, self.step = torch.round(w.float() * (most / top)).double(), (top / most).double()

    def to(self, dtype):
        return self

    @property
    def T(self):
        return self

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        x, w = args
        step = x.double().abs().amax(dim=-1, keepdim=True) / 127
        return ((torch.round(x.double() / step) @ w.q.T) * step * w.step[:, 0]).to(x.dtype)


def eight_bit(weights):
    return {n: EightBit(t) if "_proj." in n else t for n, t in weights.items()}


def engine(folder, **kw):
    from llm_infer_rust_b200.engine import Engine
    kw.setdefault("cuda_graph_bs", 0)
    kw.setdefault("max_running_req", 4)
    return Engine(folder, int8_projections=True, **kw)


def tokens(vocab, n, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
def test_engine_in_32_bits(name, tiny, tiny_weights, tiny_dirs):
    from llm_infer_rust_b200.engine import StepEntry
    raw = tiny[name]["raw"]
    seq = tokens(raw["vocab_size"], 100, 3)
    want = P.plain_forward(eight_bit(tiny_weights[name]), raw, seq)
    eng = engine(tiny_dirs[name], dtype="float32", page_size=tiny[name]["page_size"], max_total_tokens=512, max_seq_len=120)
    eng.open_request(1)
    got = [eng.step([StepEntry(1, seq[a:b], list(range(b - a)))]).double().cpu() for a, b in
           ((0, 70), (70, 90), (90, 91), (91, 99), (99, 100))]
    eng.check_kernel_errors()
    err, scale = (torch.cat(got) - want).abs(), want.abs().max()
    full = (torch.cat(got) - P.plain_forward(tiny_weights[name], raw, seq)).abs()
    assert err.max() <= 4e-2 * scale and err.median() <= 0.1 * full.median(), (float(err.max()), float(err.median()), float(full.median()))
    assert err[0].max() <= 2e-5 * scale and full.median() > 1e-4 * scale


@pytest.mark.parametrize("name", ["A", "E"])
def test_engine_in_16_bits_with_graphs(name, tiny, tiny_weights, tiny_dirs):
    from llm_infer_rust_b200 import SamplingParams
    from llm_infer_rust_b200.engine import StepEntry
    raw = tiny[name]["raw"]
    seq = tokens(raw["vocab_size"], 90, 5)
    weights = {n: t.bfloat16().float() for n, t in tiny_weights[name].items()}
    want = P.plain_forward(eight_bit(weights), raw, seq)
    eng = engine(tiny_dirs[name], dtype="bfloat16", page_size=tiny[name]["page_size"], max_total_tokens=512, max_seq_len=128, cuda_graph_bs=2)
    eng.open_request(1)
    got = torch.cat([eng.step([StepEntry(1, seq[a:b], list(range(b - a)))]).double().cpu() for a, b in ((0, 70), (70, 88), (88, 89), (89, 90))])
    assert (got - want).abs().max() <= 5e-2 * max(1.0, want.abs().max())
    eng.close_request(1)
    results = eng.generate([seq[:9], seq[:30], seq[:3]], SamplingParams(max_tokens=12, ignore_eos=True))
    assert [len(r.tokens) for r in results] == [12, 12, 12]
    eng.check_kernel_errors()
    assert eng.cache.manager.live_requests() == 0 and eng.cache.manager.check() == ""


def test_weights_take_half_the_memory(tiny_dirs):
    from llm_infer_rust_b200.engine import Engine
    full = Engine(tiny_dirs["E"], dtype="bfloat16", cuda_graph_bs=0, max_running_req=2, max_total_tokens=256, max_seq_len=128)
    held = engine(tiny_dirs["E"], dtype="bfloat16", max_running_req=2, max_total_tokens=256, max_seq_len=128)
    # (rows lie a multiple of 16 bytes apart; embedding, head and norms are as they were)
    projections = sum(p.numel() for block in full.model.blocks for part in (block.mixer, block.feed_forward)
                      for n, p in part.params.items() if n.endswith("proj"))
    assert full.model.parameter_bytes() - held.model.parameter_bytes() == projections
    for block in held.model.blocks:
        assert all(block.feed_forward.params[n].dtype == torch.int8 for n in ("gate_up_proj", "down_proj"))


@pytest.mark.parametrize("activation,limit", [("silu", 0.0), ("gelu_tanh", 0.0), ("clamped_swish", 7.0)])
@pytest.mark.parametrize("tokens_", [1, 5, 40, 300])
def test_gated_feed_forwards(activation, limit, tokens_):
    from llm_infer_rust_b200 import PartSpec
    from llm_infer_rust_b200.parts import BuildEnv, build_part
    g = torch.Generator().manual_seed(tokens_)
    gate_up, down = torch.randn(2 * 120, 88, generator=g) * 0.1, torch.randn(88, 120, generator=g) * 0.1
    x = torch.randn(tokens_, 88, generator=g)
    part = build_part("feed_forward", PartSpec("gated_act_int8", {"hidden_size": 88, "intermediate_size": 120, "activation": activation,
                                                                 "limit": limit}), BuildEnv(torch.float32, DEV, {}))
    part.bind("gate_up_proj", gate_up.to(DEV))
    part.bind("down_proj", down.to(DEV))
    got = part.forward(x.to(DEV)).double().cpu()
    u, v = (x.double() @ EightBit(gate_up).T).chunk(2, dim=1)
    if activation == "clamped_swish":
        u, v = u.clamp_max(limit), v.clamp(-limit, limit) + 1
        h = u * torch.sigmoid(1.702 * u) * v
    else:
        h = (u * torch.sigmoid(u) if activation == "silu" else torch.nn.functional.gelu(u, approximate="tanh")) * v
    want = h @ EightBit(down).T
    err, scale = (got - want).abs(), want.abs().max()
    assert err.median() <= 2e-5 * scale and err.max() <= 4e-2 * scale


def test_another_architectures_feed_forwards(tmp_path):
    """Bevuvik's clamped gate between its own mixers and norms (whose projections have no such form and stay as they are)."""
    import bevuvik_kit as K
    raw = K.config(97, 40, 1e-5, 0.4, [
        K.attention(4, 2, 12, 20, 0.28, 0.35, K.rot(50000.0, 8), 24, K.dense(36, 2.0)),
        K.pair((4, 2, 12, 14, 0.3, 8.0, K.rot(10000.0, 6)), (6, 2, 12, 16, 3), K.dense(28, 1.0))], (0, 2, 2))
    weights = K.random_weights(raw, 11)
    ids = K.tokens(97, 50, 2)
    want = K.P.forward(raw, {n: EightBit(t) if ".mlp." in n else t for n, t in weights.items()}, ids)
    eng = K.make_engine(K.write_model(str(tmp_path), raw, weights), "float32", int8_projections=True)
    got = torch.from_numpy(K.run_alone(eng, 1, ids, [30, 1, 19])).double()
    err, scale = (got - want).abs(), want.abs().max()
    full = (got - K.P.forward(raw, weights, ids)).abs()
    assert err.median() <= 0.1 * full.median() and err.max() <= 0.1 * scale, (float(err.median()), float(full.median()), float(err.max()))
