"""What a model whose projections are in 8-bit integers holds."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def matrices(model):
    """(rows, columns) of every projection."""
    return [tuple(part.param_decls()[n].shape) for block in model.blocks for part in (block.mixer, block.feed_forward)
            for n in part.params if n.endswith("proj")]


@pytest.mark.parametrize("name", ["A", "E"])
def test_scales_and_padding_are_counted(name, tiny_dirs):
    """Each projection in 16 bits is two bytes an element; in 8 bits rows of a multiple of 16 bytes and a float32 scale a row."""
    from llm_infer_rust_b200.engine import Engine
    keep = dict(dtype="bfloat16", cuda_graph_bs=0, max_running_req=2, max_total_tokens=256, max_seq_len=128)
    full = Engine(tiny_dirs[name], **keep).model
    held = Engine(tiny_dirs[name], int8_projections=True, **keep).model
    assert matrices(full) == matrices(held)
    in_16 = sum(2 * n * k for n, k in matrices(full))
    in_8 = sum(n * (-(-k // 16) * 16 + 4) for n, k in matrices(full))
    assert full.held_bytes() - held.held_bytes() == in_16 - in_8
    assert full.held_bytes() >= full.parameter_bytes() and held.held_bytes() > held.parameter_bytes()


def test_rows_of_odd_widths_are_counted_with_their_padding():
    from llm_infer_rust_b200 import PartSpec
    from llm_infer_rust_b200.kernels import int8
    from llm_infer_rust_b200.parts import BuildEnv, build_part
    part = build_part("feed_forward", PartSpec("swiglu_int8", {"hidden_size": 37, "intermediate_size": 53}), BuildEnv(torch.float32, torch.device("cuda"), {}))
    for n, shape in (("gate_up_proj", (106, 37)), ("down_proj", (37, 53))):
        part.bind(n, torch.randn(*shape, device="cuda"))
        assert part.params[n].untyped_storage().nbytes() == shape[0] * int8.row_pitch(shape[1])
        assert part.int8[n].scales.untyped_storage().nbytes() == 4 * shape[0]
