"""Products in 8-bit integers against their definition in 64 bits.

Taking rows to 8 bits is compared exactly: every step of it is one correctly rounded float operation.  Products: the integer
sum is exact, so what may differ is the sum's conversion to float, the product of the scales, their product and the bias (each
2^-24 relative), and the rounding to the output's type (2^-9 for bfloat16).  A norm's sum of squares is added up in chains of at
most 40 and trees of at most 21 additions, so the row's scale is off by at most about half of 61 * 2^-24 and a few
roundings: 2^-18 relative.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def int8():
    from llm_infer_rust_b200.kernels import int8 as m
    return m


def ops():
    from llm_infer_rust_b200.kernels import ops as m
    return m


def rnd(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def activations(tokens, k, dtype, seed=0, apart=0):
    """Tokens of unlike size with a few large channels; ``apart``: columns between rows."""
    g = torch.Generator().manual_seed(seed + tokens + 3 * k)
    v = torch.randn(tokens, k, generator=g) * torch.exp(torch.randn(tokens, 1, generator=g)) * \
        (1 + 20 * (torch.rand(k, generator=g) < 0.02).float())
    wide = torch.full((tokens, k + apart), float("nan"), dtype=dtype, device=DEV)
    wide[:, :k] = v.to(dtype).to(DEV)
    return wide[:, :k]


def plain_rows(v):
    """(values, scales) of float32 rows, operation by operation.  (torch divides by a number, and a number by a tensor, through
    a rounded reciprocal; tensor by tensor is one division.)"""
    top = v.abs().amax(dim=1, keepdim=True)
    most = torch.full_like(top, 127.0)
    pre = torch.where(top < 2.0 ** -100, 2.0 ** 100, 1.0)
    q = torch.round((v * pre) * (most / (top * pre)))
    q = torch.where((top > 0) & torch.isfinite(top), q, 0.0)
    s = torch.where(torch.isfinite(top), top / most, float("nan"))
    return q.to(torch.int8), s[:, 0]


def weight(n, k, seed=0, full=False):
    """8-bit weights with pitch padding that must not count; ``full``: -128 among the values."""
    g = torch.Generator().manual_seed(seed + n + 5 * k)
    m = int8()
    values = torch.randint(-128 if full else -127, 128, (n, m.row_pitch(k)), generator=g, dtype=torch.int8).to(DEV)[:, :k]
    return m.Int8Weight(values, (torch.rand(n, generator=g) * 0.01 + 1e-4).to(DEV))


def floats(rows, w, bias=None):
    """(the sums with their scales, their sizes for the tolerance) in 64 bits."""
    sums = (rows.values.double() @ w.values.double().t()) * rows.scales.double()[:, None] * w.scales.double()
    return (sums, sums.abs()) if bias is None else (sums + bias.double(), sums.abs() + bias.double().abs())


def check(got, want, size, dtype, rel=0.0):
    assert got.dtype == dtype and got.shape == want.shape
    tol = (2.0 ** -22 + rel) * size + (2.0 ** -8 if dtype == BF16 else 0.0) * want.abs() + 1e-37
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


def gated(y, glu, limit, alpha):
    g, u = y.chunk(2, dim=1)
    if glu == "silu":
        return g * torch.sigmoid(g) * u
    if glu == "gelu_tanh":
        return torch.nn.functional.gelu(g, approximate="tanh") * u
    g, u = g.clamp_max(limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(alpha * g) * (u + 1)


# ---------------------------------------------------------------------------------------------------- rows to 8 bits
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,k,apart", [(1, 1, 0), (3, 7, 0), (2, 8, 0), (5, 100, 3), (4, 1000, 8), (33, 1024, 0), (300, 4096, 0),
                                            (7, 12288, 64), (2, 16384, 0), (3, 16392, 0), (2, 40001, 0), (1, 131071, 0)])
def test_rows_in_8_bits_are_the_formulas(tokens, k, apart, dtype):
    x = activations(tokens, k, dtype, apart=apart)
    rows = int8().quantize_rows(x)
    q, s = plain_rows(x.float())
    assert rows.values.shape == (tokens, k) and rows.values.stride(0) % 16 == 0
    assert torch.equal(rows.values, q) and torch.equal(rows.scales, s)
    assert int(rows.values.abs().amax()) == 127


def test_rows_without_an_8_bit_form_and_rows_of_zeros_or_tiny_values():
    x = rnd(8, 200)
    x[0] = 0.0
    x[1, 5] = float("inf")
    x[2, 199] = float("nan")
    x[3] *= 1e-38
    x[4] = 0.0
    x[4, 17] = 1e-45                                      # the smallest float there is
    x[5] *= 3e37
    x[6, 0] = -float("inf")
    rows = int8().quantize_rows(x)
    q, s = plain_rows(x)
    assert torch.equal(rows.values, q)
    assert rows.scales.isnan().tolist() == [False, True, True, False, False, False, True, False]
    assert torch.equal(rows.scales.nan_to_num(-1.0), s.nan_to_num(-1.0)) and rows.scales[0] == 0
    assert int(rows.values[4, 17]) == 127 and int(rows.values[3].abs().amax()) == 127
    for n, tokens in ((40, 8), (40, 200)):
        w = weight(n, 200)
        y = int8().int8_linear(x.repeat(tokens // 8, 1), w)
        nan = y.isnan().all(dim=1)
        assert nan.view(-1, 8)[0].tolist() == [False, True, True, False, False, False, True, False]
        assert torch.equal(nan.view(-1, 8), nan.view(-1, 8)[:1].expand(tokens // 8, 8)) and (y[0] == 0).all()
        # (row 5's results are around the largest float: those beyond it are infinite, as the definition's are)
        want = floats(int8().Int8Rows(q, s), w)[0].repeat(tokens // 8, 1)[~nan]
        assert torch.equal(torch.isfinite(y[~nan]), want.abs() < torch.finfo(F32).max)


@pytest.mark.parametrize("dtype,gain_dtype", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("tokens,k", [(1, 3), (5, 100), (2, 1024), (130, 4096), (3, 20000)])
def test_a_norm_on_the_way_to_8_bits(tokens, k, dtype, gain_dtype):
    x, gain, eps = activations(tokens, k, dtype), (1.0 + 0.3 * rnd(k, seed=2)).to(gain_dtype), 1e-5
    for residual in (None, rnd(tokens, k, dtype=dtype, seed=3, scale=2.0)):
        pending = ops().PendingNorm(x.contiguous(), residual, gain, eps)
        rows = int8().quantize_rows(pending)
        v = x.float() if residual is None else x.float() + residual.float()
        q, s = plain_rows(v * gain.float())
        assert torch.equal(rows.values, q)
        want = s.double() * (v.double().square().mean(dim=1) + eps).rsqrt()
        assert ((rows.scales.double() - want).abs() <= 2.0 ** -18 * want).all()
        if residual is not None:
            assert torch.equal(pending.residual_out, v.to(dtype))


# ------------------------------------------------------------------------------------------------------------ products
SIZES = [(1, 1, 1), (1, 16, 16), (1, 17, 33), (2, 1024, 1000), (3, 1000, 100), (4, 2048, 64), (5, 100, 2501), (7, 4096, 130), (8, 12288, 48),
         (8, 64, 8), (9, 4096, 65), (16, 640, 256), (17, 1999, 127), (31, 15, 100), (64, 1024, 1024), (65, 129, 129), (100, 4096, 200),
         (128, 128, 128), (129, 257, 385), (200, 2050, 64), (255, 512, 511), (257, 1024, 640), (300, 96, 1544), (513, 4096, 384),
         (1000, 72, 80), (2, 40001, 24), (20, 40001, 24), (1, 131071, 3), (12, 131071, 5)]


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,k,n", SIZES)
def test_products(tokens, k, n, out_dtype):
    m = int8()
    rows, w = m.quantize_rows(activations(tokens, k, F32)), weight(n, k, full=True)
    for bias in (None, rnd(n, scale=3.0)):
        y = m.int8_linear(rows, w, bias=bias, out_dtype=out_dtype)
        check(y, *floats(rows, w, bias), out_dtype)
        assert torch.equal(y, m.int8_linear(rows, w, bias=bias, out_dtype=out_dtype))


def test_the_largest_sums_that_32_bits_hold():
    m = int8()
    for tokens in (1, 70):
        k = m.MAX_K
        rows = m.Int8Rows(torch.full((tokens, m.row_pitch(k)), -128, dtype=torch.int8, device=DEV)[:, :k], torch.ones(tokens, device=DEV))
        w = m.Int8Weight(torch.full((18, m.row_pitch(k)), -128, dtype=torch.int8, device=DEV)[:, :k], torch.ones(18, device=DEV))
        assert (m.int8_linear(rows, w, out_dtype=F32) == float(128 * 128 * k)).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,k,n,apart", [(1, 2048, 1024, 0), (2, 1000, 90, 5), (4, 4096, 300, 64), (8, 640, 128, 0), (8, 12288, 96, 0),
                                              (8, 16384, 64, 0), (3, 30000, 40, 0), (45, 1024, 200, 7), (128, 520, 520, 0), (700, 1024, 264, 8)])
def test_products_of_float_rows(tokens, k, n, apart, dtype):
    m = int8()
    x, w, bias = activations(tokens, k, dtype, apart=apart), weight(n, k), rnd(n)
    rows = m.Int8Rows(*plain_rows(x.float()))
    for out_dtype in (None, F32):
        y = m.int8_linear(x, w, bias=bias, out_dtype=out_dtype)
        check(y, *floats(rows, w, bias), out_dtype or dtype)
    assert torch.equal(m.int8_linear(x, w), m.int8_linear(m.quantize_rows(x), w, out_dtype=dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,k,n", [(1, 1024, 700), (2, 4096, 256), (4, 1000, 64), (8, 2048, 520), (8, 12288, 32), (20, 1024, 96),
                                        (129, 2048, 200), (600, 1024, 256)])
def test_products_behind_a_norm(tokens, k, n, dtype):
    m, o = int8(), ops()
    x, w, gain, eps = activations(tokens, k, dtype).contiguous(), weight(n, k), 1.0 + 0.3 * rnd(k, seed=2), 1e-6
    for residual in (None, rnd(tokens, k, dtype=dtype, seed=3, scale=2.0)):
        pending = o.PendingNorm(x, residual, gain, eps)
        y = m.int8_linear(pending, w)
        v = x.float() if residual is None else x.float() + residual.float()
        q, s = plain_rows(v * gain)
        rows = m.Int8Rows(q, s.double() * (v.double().square().mean(dim=1) + eps).rsqrt())
        check(y, *floats(rows, w), dtype, rel=2.0 ** -18)
        if residual is not None:
            assert torch.equal(pending.residual_out, v.to(dtype))
    # rows picked out of more, as a model's last norm does
    at = torch.arange(tokens - 1, -1, -2, dtype=torch.int32, device=DEV)
    y = m.int8_linear(o.PendingNorm(x, residual, gain, eps, rows=at, write_residual=False), w)
    normed = o.add_rms_norm(x, residual.clone(), gain, eps, rows=at, write_residual=False)
    assert torch.equal(y, m.int8_linear(normed, w))


GLUS = [("silu", 0.0, 1.0), ("gelu_tanh", 0.0, 1.0), ("clamped_swish", 7.0, 1.702)]


@pytest.mark.parametrize("glu,limit,alpha", GLUS)
@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,k,n", [(1, 4096, 1), (1, 1024, 300), (3, 100, 17), (8, 4096, 96), (16, 1000, 129), (45, 2048, 256),
                                        (128, 64, 65), (130, 1024, 192), (520, 640, 328), (1100, 256, 128)])
def test_gated_products(tokens, k, n, out_dtype, glu, limit, alpha):
    m = int8()
    rows, w = m.quantize_rows(activations(tokens, k, F32)), weight(2 * n, k)
    for bias in (None, rnd(2 * n)):
        h = m.int8_glu(rows, w, glu=glu, limit=limit, alpha=alpha, bias=bias, out_dtype=out_dtype)
        y, size = floats(rows, w, bias)
        # the gate's slope is below 1.2 (alpha g: 1.702 * 1.2) and each of its operations is off by a few 2^-24; so is up
        g, u = size.chunk(2, dim=1)
        size = g * (u + 1.0)
        want = gated(y, glu, limit, alpha)
        tol = 2.0 ** -18 * size + (2.0 ** -8 if out_dtype == BF16 else 0.0) * want.abs()
        assert h.shape == want.shape and h.dtype == out_dtype
        bad = ~((h.double() - want).abs() <= tol)
        assert not bad.any(), (int(bad.sum()), float(((h.double() - want).abs() / tol).max()))


def test_a_gated_product_behind_a_norm_is_the_steps_in_turn():
    m, o = int8(), ops()
    for tokens, k, n in ((1, 4096, 512), (2, 1024, 100), (8, 4096, 64), (45, 1024, 96), (300, 1024, 256)):
        x, residual, gain = activations(tokens, k, BF16).contiguous(), rnd(tokens, k, dtype=BF16), 1.0 + 0.2 * rnd(k).to(BF16)
        w = weight(2 * n, k)
        pending = o.PendingNorm(x, residual, gain, 1e-6)
        h = m.int8_glu(pending, w)
        v = x.float() + residual.float()
        q, s = plain_rows(v * gain.float())
        rows = m.Int8Rows(q, s.double() * (v.double().square().mean(dim=1) + 1e-6).rsqrt())
        y, size = floats(rows, w)
        want = gated(y, "silu", 0.0, 1.0)
        g, u = size.chunk(2, dim=1)
        assert ((h.double() - want).abs() <= 2.0 ** -16 * g * (u + 1.0) + 2.0 ** -8 * want.abs()).all()
        assert torch.equal(pending.residual_out, v.to(BF16))


# ------------------------------------------------------------------------------------------------- what is around them
@pytest.mark.parametrize("tokens,k,n,mode", [(1, 100, 37, 0), (8, 64, 50, 0), (5, 1000, 21, 1), (40, 200, 130, 0), (129, 64, 129, 1), (300, 256, 257, 0),
                                             (300, 256, 264, 0), (600, 1024, 520, 1)])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_nothing_is_written_beside_the_results(tokens, k, n, mode, out_dtype):
    m, o = int8(), ops()
    x, w = activations(tokens, k, BF16).contiguous(), weight(n * (1 + mode), k)
    pitch = m.row_pitch(k)
    whole = torch.full((tokens * n + 512,), 123.0, dtype=out_dtype, device=DEV)
    out = whole[256:256 + tokens * n].view(tokens, n)
    q = torch.full((tokens * pitch + 512,), 77, dtype=torch.int8, device=DEV)
    s = torch.full((tokens + 128,), 55.0, device=DEV)
    rc = m._lib().b200_int8_linear(x, None, None, None, q[256:], s[64:], w.values, w.scales, None, out, tokens, n, k, k, pitch,
                                   w.values.stride(0), 1, 0, o._code(out), mode, 0.0, 0.0, 1.0, o.error_word(out.device), o._stream())
    assert rc == 0
    assert (whole[:256] == 123).all() and (whole[256 + tokens * n:] == 123).all()
    assert (q[:256] == 77).all() and (q[256 + tokens * pitch:] == 77).all() and (s[:64] == 55).all() and (s[64 + tokens:] == 55).all()
    want = m.int8_glu(x, w, out_dtype=out_dtype) if mode else m.int8_linear(x, w, out_dtype=out_dtype)
    assert torch.equal(out, want)


def test_outputs_at_any_address():
    """The C entry takes outputs that are aligned to their elements alone."""
    m, o = int8(), ops()
    for tokens, k, n, mode in ((1, 64, 40, 0), (30, 128, 136, 0), (300, 256, 512, 0), (600, 512, 512, 1)):
        x, w = activations(tokens, k, BF16).contiguous(), weight(n * (1 + mode), k)
        rows = m.quantize_rows(x)
        for out_dtype in (BF16, F32):
            out = torch.zeros(tokens * n + 3, dtype=out_dtype, device=DEV)[1:1 + tokens * n].view(tokens, n)
            rc = m._lib().b200_int8_linear(None, None, None, None, rows.values, rows.scales, w.values, w.scales, None, out, tokens, n, k, 0,
                                           rows.values.stride(0), w.values.stride(0), 0, 0, o._code(out), mode, 0.0, 0.0, 1.0,
                                           o.error_word(out.device), o._stream())
            assert rc == 0
            assert torch.equal(out, m.int8_glu(rows, w, out_dtype=out_dtype) if mode else m.int8_linear(rows, w, out_dtype=out_dtype))


@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("tokens,k,n", [(300, 96, 1540), (300, 96, 1541), (300, 96, 1542), (700, 256, 324), (700, 256, 323), (2100, 64, 2052),
                                        (2100, 64, 2051)])
def test_results_of_any_width_at_any_address(tokens, k, n, mode):
    """Rows of results that begin at multiples of 16, 8, 4 and 2 bytes, against the definition, with nothing written beside them."""
    m, o = int8(), ops()
    rows, w = m.quantize_rows(activations(tokens, k, BF16)), weight(n * (1 + mode), k)
    want, size = floats(rows, w)
    if mode:
        want = gated(want, "silu", 0.0, 1.0)
    for out_dtype in (BF16, F32):
        first = None
        for at in (16, 20, 18, 17):
            space = torch.full((tokens * n + 64,), 123.0, dtype=out_dtype, device=DEV)
            out = space[at:at + tokens * n].view(tokens, n)
            rc = m._lib().b200_int8_linear(None, None, None, None, rows.values, rows.scales, w.values, w.scales, None, out, tokens, n, k, 0,
                                           rows.values.stride(0), w.values.stride(0), 0, 0, o._code(out), mode, 0.0, 0.0, 1.0,
                                           o.error_word(out.device), o._stream())
            assert rc == 0 and (space[:at] == 123).all() and (space[at + tokens * n:] == 123).all()
            if first is None:
                first = out
                if not mode:
                    check(out, want, size, out_dtype)
                else:                                           # both factors 2^-21, the gate's own functions 2^-19 of what they give
                    g, u = size.chunk(2, dim=1)
                    check(out, want, g * u + g + u, out_dtype, rel=2.0 ** -18)
            assert torch.equal(out, first)


def test_rows_are_alike_whatever_runs_beside_them():
    """A token's result has the same bits alone and among others (sums are exact, scales are its own)."""
    m = int8()
    x, w = activations(700, 1024, BF16).contiguous(), weight(384, 1024)
    whole = m.int8_linear(x, w)
    for a, b in ((0, 1), (5, 13), (20, 84), (100, 300), (699, 700)):
        assert torch.equal(m.int8_linear(x[a:b], w), whole[a:b])


def test_no_tokens_and_no_channels():
    m = int8()
    w = weight(20, 64)
    assert m.int8_linear(torch.empty(0, 64, device=DEV, dtype=BF16), w).shape == (0, 20)
    assert m.int8_glu(torch.empty(0, 64, device=DEV), w).shape == (0, 10)
    assert m.quantize_rows(torch.empty(0, 64, device=DEV)).values.shape == (0, 64)
    none = m.Int8Weight(w.values[:0], w.scales[:0])
    assert m.int8_linear(rnd(3, 64), none).shape == (3, 0)


def test_another_stream_than_the_default_and_a_graph():
    m, o = int8(), ops()
    side = torch.cuda.Stream()
    cases = [(activations(t, 1024, BF16).contiguous(), weight(512, 1024)) for t in (1, 8, 40, 300)]
    want = [(m.int8_linear(x, w), m.int8_glu(x, w)) for x, w in cases]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = [(m.int8_linear(x, w), m.int8_glu(x, w)) for x, w in cases]
    side.synchronize()
    assert all(torch.equal(a, b) for g, h in zip(got, want) for a, b in zip(g, h))
    inputs = [x.clone() for x, _ in cases]
    graph = torch.cuda.CUDAGraph()
    with o.graph_capture(graph):
        out = [(m.int8_linear(x, w), m.int8_glu(x, w)) for x, (_, w) in zip(inputs, cases)]
    for turn in range(3):
        for x, (was, _) in zip(inputs, cases):
            x.copy_(was.roll(turn, 1))
        graph.replay()
        torch.cuda.synchronize()
        for (a, b), x, (_, w) in zip(out, inputs, cases):
            assert torch.equal(a, m.int8_linear(x, w)) and torch.equal(b, m.int8_glu(x, w))
    del graph
    o.check_errors(torch.device(DEV, 0))


def test_what_was_written_just_before_is_what_is_read():
    """Weights and rows that the kernels before the product wrote: it may start early, but not read early."""
    m = int8()
    x = activations(4, 2048, F32).contiguous()
    first, second = rnd(1536, 2048, seed=1), rnd(1536, 2048, seed=2)
    want = [m.int8_linear(x, m.int8_weight(f)).clone() for f in (first, second)]
    torch.cuda.synchronize()
    w = m.int8_weight(first)
    for turn in range(20):
        source = (first, second)[turn % 2]
        fresh = m.int8_weight(source)
        w.values.copy_(fresh.values)
        w.scales.copy_(fresh.scales)
        assert torch.equal(m.int8_linear(x, w), want[turn % 2])
        assert torch.equal(m.int8_linear(x, m.int8_weight(source)), want[turn % 2])


def test_weights_in_8_bits():
    m = int8()
    for dtype in (BF16, F32):
        w = rnd(37, 500, dtype=dtype)
        held = m.int8_weight(w)
        q, s = plain_rows(w.float())
        assert torch.equal(held.values, q) and torch.equal(held.scales, s)
        assert ((held.dequantize() - w.float()).abs() <= 0.5001 * s[:, None]).all()
        again = m.int8_weight_from(q, s)
        assert torch.equal(again.values, q) and again.values.stride(0) % 16 == 0
        x = rnd(3, 500)
        assert torch.equal(m.int8_linear(x, again), m.int8_linear(x, held))
    laid = m.int8_weight_from(held.values, held.scales)
    assert laid.values.data_ptr() == held.values.data_ptr()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,k", [(2, 9), (3, 15), (5, 257), (400, 264), (64, 1999), (400, 2051), (1300, 1999), (7, 4095), (200, 4100), (1300, 4095),
                                      (3, 8191), (160, 8201), (160, 12289), (1200, 12288), (2, 33333), (170, 16395)])
def test_rows_that_begin_anywhere(tokens, k, dtype):
    """Row lengths that are no multiple of eight, with and without a norm; sums are written to their rows and nowhere else."""
    m, o = int8(), ops()
    x, residual, gain = activations(tokens, k, dtype).contiguous(), rnd(tokens, k, dtype=dtype, seed=3), 1.0 + 0.3 * rnd(k, seed=4)
    q, s = plain_rows(x.float())
    rows = m.quantize_rows(x)
    assert torch.equal(rows.values, q) and torch.equal(rows.scales, s)
    v = x.float() + residual.float()
    q, s = plain_rows(v * gain)
    want = s.double() * (v.double().square().mean(dim=1) + 1e-5).rsqrt()
    for lead in (16, 1):                                       # outputs at a multiple of 16 bytes and off it
        whole = torch.full((tokens * k + 64,), 99.0, dtype=dtype, device=DEV)
        kept = whole[lead:lead + tokens * k]
        pitch = m.row_pitch(k)
        values = torch.full((tokens * pitch + 32,), 77, dtype=torch.int8, device=DEV)
        scales = torch.zeros(tokens, device=DEV)
        rc = m._lib().b200_int8_rows(x, residual, gain, kept, values[16:], scales, tokens, k, k, pitch, o._code(x), 0, 1e-5, o._stream())
        assert rc == 0
        assert torch.equal(kept.view(tokens, k), v.to(dtype))
        assert (whole[:lead] == 99).all() and (whole[lead + tokens * k:] == 99).all()
        got = values[16:16 + tokens * pitch].view(tokens, pitch)[:, :k]
        assert torch.equal(got, q) and (values[:16] == 77).all() and (values[16 + tokens * pitch:] == 77).all()
        assert ((scales.double() - want).abs() <= 2.0 ** -18 * want).all()


@pytest.mark.parametrize("dtype,gain_dtype", [(BF16, BF16), (F32, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("tokens,k", [(200, 3), (700, 64), (700, 250), (700, 507), (2000, 512), (700, 533), (700, 536), (700, 767), (700, 1000),
                                      (2000, 1024), (700, 1001), (1300, 2049), (1300, 8187), (170, 16400)])
def test_rows_beside_anything(tokens, k, dtype, gain_dtype):
    """Short and long rows of many tokens; x, the residual, the gain and the sums begin at unlike places, between and beside them there
    is nothing but NaN, and none of it counts or is written."""
    m, o = int8(), ops()
    nan = float("nan")
    for apart, lead, begin in ((0, 8, (0, 0, 0)), (0, 3, (1, 1, 2)), (5, 2, (3, 6, 1)), (8, 8, (1, 0, 5))):
        pitch_x = k + apart
        space = torch.full((tokens * pitch_x + 32,), nan, dtype=dtype, device=DEV)
        x = space[lead:lead + tokens * pitch_x].view(tokens, pitch_x)[:, :k]
        x.copy_(activations(tokens, k, dtype))
        residual, gain, kept = (torch.full((size + 64,), nan, dtype=t, device=DEV)[16 + at:16 + at + size]
                                for size, t, at in zip((tokens * k, k, tokens * k), (dtype, gain_dtype, dtype), begin))
        residual.copy_(rnd(tokens * k, dtype=dtype, seed=3))
        gain.copy_((1.0 + 0.3 * rnd(k, seed=4)).to(gain_dtype))
        pitch, scales = m.row_pitch(k), torch.zeros(tokens, device=DEV)
        values = torch.full((tokens, pitch), 77, dtype=torch.int8, device=DEV)
        q, s = plain_rows(x.float())
        rc = m._lib().b200_int8_rows(x, None, None, None, values, scales, tokens, k, pitch_x, pitch, o._code(x), 0, 0.0, o._stream())
        assert rc == 0 and torch.equal(values[:, :k], q) and torch.equal(scales, s)
        v = x.float() + residual.float().view(tokens, k)
        q, s = plain_rows(v * gain.float())
        rc = m._lib().b200_int8_rows(x, residual, gain, kept, values, scales, tokens, k, pitch_x, pitch, o._code(x), o._code(gain), 1e-5,
                                     o._stream())
        want = s.double() * (v.double().square().mean(dim=1) + 1e-5).rsqrt()
        assert rc == 0 and torch.equal(values[:, :k], q) and torch.equal(kept.view(tokens, k), v.to(dtype))
        assert ((scales.double() - want).abs() <= 2.0 ** -18 * want).all()
        for t, at in ((residual, begin[0]), (kept, begin[2])):
            around = t.as_strided((tokens * k + 64,), (1,), 0)
            assert around[:16 + at].isnan().all() and around[16 + at + tokens * k:].isnan().all()


@pytest.mark.parametrize("tokens,k", [(1, 1999), (2, 1023), (4, 777), (7, 333), (8, 1001), (3, 5001)])
def test_few_rows_that_begin_anywhere_behind_a_norm(tokens, k):
    """The same inside the kernel for few tokens."""
    m, o = int8(), ops()
    for dtype in (BF16, F32):
        x, residual, gain = activations(tokens, k, dtype).contiguous(), rnd(tokens, k, dtype=dtype, seed=3), 1.0 + 0.3 * rnd(k, seed=4)
        w, pending = weight(70, k), o.PendingNorm(x, residual, gain, 1e-6)
        y = m.int8_linear(pending, w, out_dtype=F32)
        v = x.float() + residual.float()
        q, s = plain_rows(v * gain)
        rows = m.Int8Rows(q, s.double() * (v.double().square().mean(dim=1) + 1e-6).rsqrt())
        check(y, *floats(rows, w), F32, rel=2.0 ** -18)
        assert torch.equal(pending.residual_out, v.to(dtype))


def test_more_results_than_32_bits_count():
    """16,500 tokens x 131,200 columns: results, and 40,000 rows of 60,000: inputs, beyond 2^31 elements."""
    m = int8()
    x, w = activations(16500, 32, BF16).contiguous(), weight(131200, 32)
    y = m.int8_linear(x, w)
    assert y.numel() > 2 ** 31
    for a, b in ((0, 3), (8000, 8009), (16490, 16500)):
        assert torch.equal(y[a:b], m.int8_linear(x[a:b], w))
    del y, x
    x = torch.zeros(40000, 60000, dtype=BF16, device=DEV)
    x[39990:] = activations(10, 60000, BF16)
    rows = m.quantize_rows(x)
    q, s = plain_rows(x[39990:].float())
    assert torch.equal(rows.values[39990:], q) and torch.equal(rows.scales[39990:], s) and not rows.scales[:39990].any()
