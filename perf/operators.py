"""The products in 8-bit integers, as cases that can be timed and checked.

A layer whose weights are held in 8 bits (one scale an output channel) takes its activations to 8 bits too (one scale a
token), multiplies integers and scales the sums.  Three operators, as a layer uses them:

* ``linear``       y = x . w^T (an output or down projection, with or without a bias);
* ``norm_linear``  the residual add and RMS norm before a block, then the product (the packed q, k, v projection): y and
                   the new residual;
* ``norm_glu``     the same with gate and up projections and silu(gate) * up behind the product: h and the new residual.

With a = max |x| of a token's row: scale s = a / 127, q = rint(x * (127 / a)); y[t, n] = s[t] c[n] sum_k q[t, k] w[n, k].  A
norm's factor is common to a row, so it goes into the row's scale alone: q comes from (x + residual) * gain.
"""
import math

import torch

own = False

EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------- cases
def _case(op, tokens, k, n, dtype="bfloat16", bias=False, apart=0):
    """``n``: outputs a token (norm_glu: of gate and of up each).  ``apart``: columns between a row's end and the next
    row's start (x is a range of columns of a wider matrix)."""
    return {"op": op, "tokens": tokens, "k": k, "n": n, "dtype": dtype, "bias": bias, "apart": apart}


def listed():
    return [dict(c, name=n) for n, c in (
        # one user, a small model: the output projection of a decode step, all latency
        ("linear-1-small", _case("linear", 1, 2048, 1024)),
        # one user, wide layers: q, k, v of a decode step and its gate and up
        ("norm-linear-1", _case("norm_linear", 1, 4096, 6144)),
        ("norm-glu-1", _case("norm_glu", 1, 4096, 12288)),
        # eight requests decode: the down projection of wide layers
        ("linear-8-down", _case("linear", 8, 12288, 4096)),
        # a server under load: 45 requests at the gate and up of wide layers, 64 at the widest q, k, v
        ("norm-glu-45", _case("norm_glu", 45, 4096, 12288)),
        ("norm-linear-64", _case("norm_linear", 64, 5120, 10240)),
        # no size is round, 32-bit activations out of a wider matrix, a bias
        ("linear-odd-float32", _case("linear", 77, 1999, 2501, "float32", True, 13)),
        # a question of no special length at a small model's feed-forward
        ("norm-glu-777", _case("norm_glu", 777, 1024, 2816)),
        # prompts: the down projection, 32-bit activations, q k v of a full portion and its gate and up (the largest)
        ("linear-2048-down", _case("linear", 2048, 12288, 4096)),
        ("linear-1500-float32", _case("linear", 1500, 5120, 8192, "float32")),
        ("norm-linear-8192", _case("norm_linear", 8192, 4096, 6144)),
        ("norm-glu-8192", _case("norm_glu", 8192, 4096, 12288)),
    )]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: 1 to 8,192 tokens, rows of 64 to 16,384, 64 to 28,672 outputs, at most the largest case's work."""
    op = rng.choice(("linear", "linear", "norm_linear", "norm_glu"))
    dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
    tokens, k = _log_int(rng, 1, 8192), _log_int(rng, 64, 16384)
    if rng.random() < 0.6:
        k = max(64, k // 64 * 64)
    most = 1.6e12 / (2.0 * tokens * k) / (2 if op == "norm_glu" else 1)
    n = _log_int(rng, 64, max(65, min(28672 if op != "norm_glu" else 14336, int(most), int(2.4e8 / k))))
    if rng.random() < 0.6:
        n = max(64, n // 64 * 64)
    return _case(op, tokens, k, n, dtype, op == "linear" and rng.random() < 0.3, rng.choice((0, 0, 64, 7)) if op == "linear" else 0)


# ------------------------------------------------------------------------------------------------------ the timed call
def _inputs(case, seed):
    device = "cuda"
    gen = torch.Generator(device).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    tokens, k = case["tokens"], case["k"]
    rows = case["n"] * (2 if case["op"] == "norm_glu" else 1)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    # activations: tokens of unlike size, a few channels far above the others
    channels = 1.0 + 15.0 * (torch.rand(k, generator=gen, device=device) < 0.01)
    size = torch.exp(0.5 * normal(tokens, 1))
    wide = torch.zeros(tokens, k + case["apart"], device=device, dtype=dtype)
    x = wide[:, :k]
    x.copy_(normal(tokens, k) * channels * size)
    # weights: 8-bit values with a scale a row, rows at multiples of 16 bytes
    w = normal(rows, k)
    scales = (w.abs().amax(dim=1) / 127.0 * (0.02 + 0.02 * torch.rand(rows, generator=gen, device=device))).contiguous()
    values = torch.zeros(rows, -(-k // 16) * 16, device=device, dtype=torch.int8)[:, :k]
    values.copy_(torch.round(w.mul_(127.0 / w.abs().amax(dim=1, keepdim=True))))
    found = {"x": x, "values": values, "scales": scales, "bias": None, "residual": None, "gain": None}
    if case["bias"]:
        found["bias"] = normal(rows)
    if case["op"] != "linear":
        found["residual"] = (normal(tokens, k) * channels * 3.0).to(dtype)
        found["gain"] = (0.2 + torch.rand(k, generator=gen, device=device)).to(dtype)
    return found


def prepare(case, seed):
    return dict(_inputs(case, seed), op=case["op"], half=case["n"])


def _plain(state):
    x, values, scales = state["x"].float(), state["values"].float(), state["scales"]
    factor, kept = None, None
    if state["op"] != "linear":
        x = x + state["residual"].float()
        kept = x.to(state["x"].dtype)
        factor = torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS)
        x = x * state["gain"].float()
    top = x.abs().amax(dim=1, keepdim=True)
    most = torch.full_like(top, 127.0)            # (one division each: torch takes a number's through a rounded reciprocal)
    q = torch.where(top > 0, torch.round(x * (most / top)), torch.zeros_like(x))
    scale = top / most
    if factor is not None:
        scale = scale * factor
    y = (q @ values.t()) * (scale * scales)
    if state["bias"] is not None:
        y = y + state["bias"]
    if state["op"] == "norm_glu":
        gate, up = y[:, :state["half"]], y[:, state["half"]:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    y = y.to(state["x"].dtype)
    return y if kept is None else (y, kept)


def _own(state):
    from llm_infer_rust_b200.kernels import int8, ops
    weight = int8.Int8Weight(state["values"], state["scales"])
    if state["op"] == "linear":
        return int8.int8_linear(state["x"], weight, bias=state["bias"])
    pending = ops.PendingNorm(state["x"], state["residual"], state["gain"], EPS)
    y = int8.int8_glu(pending, weight) if state["op"] == "norm_glu" else int8.int8_linear(pending, weight)
    return y, pending.residual_out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    e = 2 if case["dtype"] == "bfloat16" else 4
    tokens, k, n = case["tokens"], case["k"], case["n"]
    rows = 2 * n if case["op"] == "norm_glu" else n
    size = tokens * k * e + rows * k + 4 * rows + tokens * n * e
    if case["bias"]:
        size += 4 * rows
    if case["op"] != "linear":
        size += 2 * tokens * k * e + k * e
    return {"bytes": size, "flops": 2 * tokens * rows * k}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """From the definition: the norm's output is what is taken to 8 bits, all of it in 64 bits."""
    got = _inputs(case, seed)
    a = got["x"].double()
    kept = None
    if case["op"] != "linear":
        kept = a + got["residual"].double()
        a = kept / (kept.pow(2).mean(dim=-1, keepdim=True) + EPS).sqrt() * got["gain"].double()
    step = a.abs().max(dim=-1).values.unsqueeze(-1) / 127
    level = (a / step.clamp_min(1e-300)).round()
    out = torch.matmul(level, got["values"].double().transpose(0, 1)) * step * got["scales"].double()
    if got["bias"] is not None:
        out = out + got["bias"].double()
    if case["op"] == "norm_glu":
        gate, up = out.split(case["n"], dim=-1)
        out = gate * torch.sigmoid(gate) * up
    return out if kept is None else (out, kept)
