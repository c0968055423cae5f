"""What a token's results owe to the tokens beside it: nothing, but for the order of a norm's sum of squares."""
import pytest
import torch

import test_int8_gpu as T

pytestmark = pytest.mark.gpu
CUTS = [(0, 1), (3, 5), (5, 13), (20, 36), (20, 84), (100, 300), (699, 700)]


@pytest.mark.parametrize("out_dtype", [T.BF16, T.F32])
@pytest.mark.parametrize("glu,limit,alpha", T.GLUS)
@pytest.mark.parametrize("k,n", [(1024, 384), (100, 90), (4096, 520)])
def test_gated_rows_are_alike_whatever_runs_beside_them(k, n, glu, limit, alpha, out_dtype):
    m = T.int8()
    x, w = T.activations(700, k, T.BF16).contiguous(), T.weight(2 * n, k)
    for bias in (None, T.rnd(2 * n)):
        keep = dict(glu=glu, limit=limit, alpha=alpha, bias=bias, out_dtype=out_dtype)
        whole = m.int8_glu(x, w, **keep)
        for a, b in CUTS:
            assert torch.equal(m.int8_glu(x[a:b], w, **keep), whole[a:b]), (a, b)


@pytest.mark.parametrize("dtype", [T.BF16, T.F32])
@pytest.mark.parametrize("k", [100, 1024, 4096, 12288])
def test_rows_behind_a_norm_are_alike_but_for_its_sum(k, dtype):
    """Both scales are within 2^-18 of the true one; the sums' conversion and three products make another 2^-21."""
    m, o = T.int8(), T.ops()
    x, residual, gain = T.activations(700, k, dtype).contiguous(), T.rnd(700, k, dtype=dtype, seed=3), 1.0 + 0.3 * T.rnd(k, seed=2)
    w = T.weight(384, k)
    run = lambda a, b: m.int8_linear(o.PendingNorm(x[a:b], residual[a:b], gain, 1e-6), w, out_dtype=T.F32).double()
    whole = run(0, 700)
    for a, b in CUTS:
        assert ((run(a, b) - whole[a:b]).abs() <= (2.0 ** -17 + 2.0 ** -21) * whole[a:b].abs()).all(), (a, b)
