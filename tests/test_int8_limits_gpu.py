"""Products in 8-bit integers on both sides of the sizes at which another kernel takes over, against their definition in 64 bits (the
tolerances are those of the other sizes: see test_int8_gpu.py)."""
import pytest
import torch

import test_int8_gpu as T

pytestmark = pytest.mark.gpu

# (rows of these widths: the last that the streaming kernel takes with so many tokens, and the first that it leaves to the tiled one)
EDGES = [(16, 6208), (16, 6209), (16, 6272), (16, 6336), (16, 6337), (15, 6592), (15, 6656), (15, 6721), (14, 7104), (14, 7168), (14, 7233),
         (13, 7616), (13, 7680), (12, 8256), (12, 8320), (11, 9088), (10, 9920), (10, 9984), (9, 11136), (8, 14528), (8, 14592), (8, 14657),
         (6, 19456), (1, 117000)]


@pytest.mark.parametrize("dtype", [T.BF16, T.F32])
@pytest.mark.parametrize("tokens,k", EDGES)
def test_products_where_another_kernel_takes_over(tokens, k, dtype):
    m, o = T.int8(), T.ops()
    x, w, gain, eps = T.activations(tokens, k, dtype).contiguous(), T.weight(96, k), 1.0 + 0.3 * T.rnd(k, seed=2), 1e-6
    residual = T.rnd(tokens, k, dtype=dtype, seed=3, scale=2.0)
    rows = m.Int8Rows(*T.plain_rows(x.float()))
    T.check(m.int8_linear(x, w), *T.floats(rows, w), dtype)
    T.check(m.int8_linear(m.quantize_rows(x), w, out_dtype=dtype), *T.floats(rows, w), dtype)
    v = x.float() + residual.float()
    q, s = T.plain_rows(v * gain)
    rows = m.Int8Rows(q, s.double() * (v.double().square().mean(dim=1) + eps).rsqrt())
    for glu in (False, True):
        pending = o.PendingNorm(x, residual, gain, eps)
        if not glu:
            T.check(m.int8_linear(pending, w), *T.floats(rows, w), dtype, rel=2.0 ** -18)
        else:
            y, size = T.floats(rows, w)
            g, u = size.chunk(2, dim=1)
            want, got = T.gated(y, "silu", 0.0, 1.0), m.int8_glu(pending, w)
            assert got.dtype == dtype
            assert ((got.double() - want).abs() <= 2.0 ** -16 * g * (u + 1.0) + (2.0 ** -8 if dtype == T.BF16 else 0.0) * want.abs()).all()
        assert torch.equal(pending.residual_out, v.to(dtype))


@pytest.mark.parametrize("dtype", [T.BF16, T.F32])
@pytest.mark.parametrize("tokens,k", [(148, 8200), (149, 8200), (300, 12288), (1184, 16384), (1185, 9000), (160, 16392), (150, 8192), (200, 8193), (500, 16377)])
def test_rows_where_another_kernel_takes_over(tokens, k, dtype):
    """Long rows: kept in registers in few or many threads, or read twice."""
    x = T.activations(tokens, k, dtype)
    rows = T.int8().quantize_rows(x)
    q, s = T.plain_rows(x.float())
    assert torch.equal(rows.values, q) and torch.equal(rows.scales, s)
