"""What the products in 8-bit integers refuse, where no GPU is needed to say so."""
import pytest
import torch

from llm_infer_rust_b200.kernels import int8, ops
from llm_infer_rust_b200.kernels.ops import KernelError


def weight(n=4, k=32):
    return int8.Int8Weight(torch.zeros(n, int8.row_pitch(k), dtype=torch.int8)[:, :k], torch.ones(n))


def aligned(w):
    return w.values.data_ptr() % 16 == 0


def test_row_pitch():
    assert [int8.row_pitch(k) for k in (1, 16, 17, 4096)] == [16, 16, 32, 4096]


@pytest.mark.parametrize("x", [torch.zeros(2, 32, dtype=torch.float16), torch.zeros(2, 32, dtype=torch.int8), torch.zeros(32),
                               torch.zeros(2, 64)[:, ::2], torch.zeros(32, 2).t(), torch.zeros(1, 32).expand(3, 32), torch.zeros(2, 0)])
def test_rows_that_are_refused(x):
    with pytest.raises(KernelError, match="dtype|unit inner stride|columns are refused"):
        int8.int8_linear(x, weight())
    with pytest.raises(KernelError, match="dtype|unit inner stride|columns are refused"):
        int8.quantize_rows(x)


def test_more_columns_than_32_bit_sums_hold():
    with pytest.raises(KernelError, match="131071"):
        int8.quantize_rows(torch.zeros(1, 131072))
    with pytest.raises(KernelError, match="131071"):
        int8.int8_linear(int8.Int8Rows(torch.zeros(1, 131072, dtype=torch.int8), torch.ones(1)), weight())


@pytest.mark.parametrize("w,what", [
    (int8.Int8Weight(torch.zeros(4, 32), torch.ones(4)), "int8 values"),
    (int8.Int8Weight(torch.zeros(4, 32, dtype=torch.int8), torch.ones(4, dtype=torch.bfloat16)), "float32 scales"),
    (int8.Int8Weight(torch.zeros(4, 32, dtype=torch.int8), torch.ones(5)), "one scale a row"),
    (int8.Int8Weight(torch.zeros(4, 32, dtype=torch.int8), torch.ones(8)[::2]), "one scale a row"),
    (int8.Int8Weight(torch.zeros(32, 4, dtype=torch.int8).t(), torch.ones(4)), "unit inner stride"),
    (int8.Int8Weight(torch.zeros(4, 33, dtype=torch.int8)[:, :32], torch.ones(4)), "multiple of 16"),
    (int8.Int8Weight(torch.zeros(1, 32, dtype=torch.int8).expand(4, 32), torch.ones(4)), "multiple of 16"),
    (int8.Int8Weight(torch.zeros(4, 48, dtype=torch.int8)[:, 1:33], torch.ones(4)), "multiple of 16")])
def test_weights_that_are_refused(w, what):
    with pytest.raises(KernelError, match=what):
        int8.int8_linear(torch.zeros(2, 32), w)


def test_sizes_that_do_not_fit(monkeypatch):
    monkeypatch.setattr(ops, "_cuda", lambda *tensors: None)
    with pytest.raises(KernelError, match="the rows have 16 columns, the weight has 32"):
        int8.int8_linear(torch.zeros(2, 16), weight())
    with pytest.raises(KernelError, match="gate and up rows"):
        int8.int8_glu(torch.zeros(2, 32), weight(5))
    for bias in (torch.zeros(4, dtype=torch.bfloat16), torch.zeros(3), torch.zeros(8)[::2]):
        with pytest.raises(KernelError, match="the bias is float32"):
            int8.int8_linear(torch.zeros(2, 32), weight(), bias=bias)
    with pytest.raises(KernelError, match="gate 'relu' is refused"):
        int8.int8_glu(torch.zeros(2, 32), weight(), glu="relu")
    with pytest.raises(KernelError, match="dtype"):
        int8.int8_linear(torch.zeros(2, 32), weight(), out_dtype=torch.float16)


def test_norms_that_do_not_fit():
    x, gain = torch.zeros(2, 32), torch.ones(32)
    for pending in (ops.PendingNorm(x, None, torch.ones(31), 1e-6), ops.PendingNorm(x, torch.zeros(2, 32, dtype=torch.bfloat16), gain, 1e-6),
                    ops.PendingNorm(x, torch.zeros(3, 32), gain, 1e-6), ops.PendingNorm(x, None, torch.ones(64)[::2], 1e-6)):
        with pytest.raises(KernelError, match="norm weight|residual"):
            int8.int8_linear(pending, weight())


def test_there_is_no_cpu_path():
    with pytest.raises(KernelError, match="CUDA tensors only"):
        int8.int8_linear(torch.zeros(2, 32), weight())
    with pytest.raises(KernelError, match="CUDA tensors only"):
        int8.quantize_rows(torch.zeros(2, 32))


def test_8_bit_values_of_a_checkpoint_are_laid_out():
    values = torch.arange(-60, 60, dtype=torch.int8).view(6, 20)
    w = int8.int8_weight_from(values, torch.ones(6, 1, dtype=torch.float64))
    assert torch.equal(w.values, values) and w.values.stride() == (32, 1) and w.scales.shape == (6,) and w.scales.dtype == torch.float32
    with pytest.raises(KernelError, match="N scales"):
        int8.int8_weight_from(values, torch.ones(5))
    assert torch.equal(w.dequantize(), values.float())


def test_which_parts_have_a_form_in_8_bits():
    from llm_infer_rust_b200 import ConfigError, LayerSpec, ModelSpec, PartSpec, Qwen3Config, RunEntry
    from llm_infer_rust_b200.parts import int8_projections, registered
    raw = {"model_type": "qwen3", "architectures": ["Qwen3ForCausalLM"], "num_hidden_layers": 2, "hidden_size": 32,
           "num_attention_heads": 2, "num_key_value_heads": 1, "head_dim": 16, "intermediate_size": 48, "vocab_size": 61}
    spec = Qwen3Config.parse(raw).model_spec()
    held = int8_projections(spec)
    for before, layer in zip(spec.layers, held.layers):
        assert layer["mixer"].kind == "gqa_attention_int8" and layer["mixer"].params == before["mixer"].params
        assert layer["feed_forward"].kind == "swiglu_int8" and layer["input_norm"] == before["input_norm"]
        assert layer["mixer"].kind in registered("mixer") and layer["feed_forward"].kind in registered("feed_forward")
    assert held.lm_head == spec.lm_head and held.run_list == spec.run_list and held != spec
    other = LayerSpec(PartSpec("pre_norm_input_conv"), {"mixer": PartSpec("decay_retention", {})})
    with pytest.raises(ConfigError, match="no layer of X has projections with a form in 8-bit"):
        int8_projections(ModelSpec("X", 10, 8, 16, PartSpec("token_embedding"), (other,), (RunEntry(0),), PartSpec("rms_norm"),
                                   PartSpec("linear_head")))


def test_the_command_line_names_them():
    from llm_infer_rust_b200 import cli
    assert cli.parse_args(["--model-path", "m", "--int8-projections"]).int8_projections
    assert not cli.parse_args(["--model-path", "m"]).int8_projections and "--int8-projections" in cli.USAGE


def plan(*sizes):
    """(CTAs that share a tile's k, 0: pairs, columns of a tile) on 148 SMs that hold 36 clusters of four."""
    import llm_infer_rust_b200.kernels.build as build
    got = build.load_cuda_library("int8_linear.cu").b200_int8_plan(*sizes, 148, 36)
    return got // 1000, got % 1000


def test_how_products_are_cut_up():
    """The ways that were fastest, or within a few hundredths of it, of all that were measured; (tokens, columns, k, gated)."""
    assert plan(8192, 6144, 4096, 0) == plan(2048, 4096, 12288, 0) == (0, 256)          # many tiles: pairs of CTAs
    assert plan(190, 12288, 4096, 1)[0] == plan(777, 2816, 1024, 1)[0] == 0
    assert plan(1500, 8192, 5120, 0) == (0, 224)                                        # (three rounds of narrower tiles)
    assert plan(100, 4096, 12288, 0) == (4, 128)                                        # long k, few columns: shared
    assert plan(64, 4096, 4096, 0)[0] == 2 and plan(300, 4096, 4096, 0)[1] == 128
    assert plan(45, 12288, 4096, 1)[0] == plan(64, 10240, 5120, 0)[0] == 1              # one round over the SMs


def test_plans_are_ones_that_the_kernels_take():
    import random
    rng = random.Random(5)
    for _ in range(400):
        mode = rng.randint(0, 1)
        tokens, n, k = (int(2 ** rng.uniform(0, b)) for b in (14, 15, 17))
        way, bn = plan(tokens, n, min(k, 131071), mode)
        assert way in (0, 1, 2, 4) and 32 <= bn <= 256
        assert bn % 32 == 0 and tokens > 128 if way == 0 else bn % 16 == 0 and bn % (4 * way * (1 + mode)) == 0
        assert way <= max(1, -(-k // 128))


def test_which_tokens_need_no_kernel_in_front():
    import llm_infer_rust_b200.kernels.build as build
    alone = build.load_cuda_library("int8_linear.cu").b200_int8_alone
    assert all(alone(t, k) for t, k in ((1, 1), (1, 16384), (2, 8192), (3, 4096), (4, 4096), (8, 2048)))
    assert not any(alone(t, k) for t, k in ((1, 16392), (2, 8200), (5, 2056), (8, 2056), (9, 64), (0, 0), (1, 131072)))


def test_the_compiled_call_asks_for_its_arguments():
    from llm_infer_rust_b200.kernels.build import load_call_binding, load_entry_points
    lib, call = load_entry_points("int8_linear.cu"), load_call_binding().byte_product
    x, w = torch.zeros(2, 32), weight()
    good = [lib.b200_int8_linear, lib.b200_int8_alone, x, w.values, w.scales, None, None, None, None, None, 0, 0.0, 0.0, 1.0,
            torch.zeros(1, dtype=torch.int32), 0]
    assert call(*good) is None                               # (nothing is on a GPU: the wrapper says so)
    for at, wrong in ((0, len), (1, None), (9, "float32"), (10, 0.5), (11, 1), (14, None), (15, None)):
        with pytest.raises(TypeError):
            call(*good[:at], wrong, *good[at + 1:])
    with pytest.raises(TypeError):
        call(*good[:-1])


def test_entry_points_refuse_what_they_cannot_run():
    from llm_infer_rust_b200.kernels.build import load_entry_points
    lib = load_entry_points("int8_linear.cu")
    x, q, s, w, c, out = torch.zeros(2, 32), torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2), torch.zeros(4, 32, dtype=torch.int8), torch.ones(4), torch.zeros(2, 4)

    def call(tokens=2, n=4, k=32, x_pitch=32, q_pitch=32, w_pitch=32, x_code=0, gain_code=0, out_code=0, mode=0, x=x, q=q, w=w, gain=None):
        return lib.b200_int8_linear(x, None, gain, None, q, s, w, c, None, out, tokens, n, k, x_pitch, q_pitch, w_pitch, x_code, gain_code, out_code,
                                    mode, 0.0, 0.0, 1.0, None, 0)
    assert call(tokens=0) == 0
    assert call(x_code=2, tokens=20) == -1 and call(out_code=7) == -1 and call(gain=c, gain_code=3, tokens=20) == -1
    assert call(k=0) == call(k=131072) == call(tokens=-1) == call(n=-1) == call(mode=2) == call(w_pitch=16) == call(q_pitch=16) == -2
    assert call(x=None, q=None) == -2
    assert call(w=w.view(-1)[1:]) == -3 and call(q_pitch=40) == -3 and call(w_pitch=40) == -3
    assert lib.b200_int8_rows(x, None, None, None, q, s, 0, 32, 32, 32, 0, 0, 0.0, 0) == 0
    assert lib.b200_int8_rows(x, None, None, None, q, s, 2, 32, 31, 32, 0, 0, 0.0, 0) == -2
    assert lib.b200_int8_rows(x, None, None, None, q, s, 2, 32, 32, 33, 0, 0, 0.0, 0) == -3
