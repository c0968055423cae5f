"""Products in 8-bit integers at the edges of what their kernels take, as far as no GPU is needed to say."""
import pytest
import torch

import llm_infer_rust_b200.kernels.build as build

STATIC = (16 + 16 + 16) * 4           # the streaming kernel's own arrays: 16 tokens' scales, 16 warps' sums and maxima
BLOCK = 227 * 1024                    # what a block may have of shared memory


def test_what_the_streaming_kernel_takes_fits_its_launch():
    """Every number of tokens that it has a form for and every length of a row: nothing is taken that its launch would refuse."""
    lib = build.load_cuda_library("int8_linear.cu")
    asks, limit = lib.b200_int8_stream_bytes, lib.b200_int8_stream_limit()
    assert limit + STATIC <= BLOCK
    for tokens in range(1, 17):
        most = max(asks(tokens, k) for k in range(1, 131072))
        assert 0 < most <= limit, (tokens, most)
    assert all(asks(t, k) == 0 for t, k in ((0, 64), (17, 64), (1, 0), (1, 131072), (16, 131071)))
    # rows of these widths lie between what a block has and what a launch may ask for: the tiled kernel takes them
    assert all(asks(t, k) == 0 for t, k in ((16, 6272), (15, 6656), (14, 7168), (13, 7680), (10, 9984), (8, 14592)))
    assert all(asks(t, k) > 0 for t, k in ((16, 6208), (15, 6592), (14, 7104), (13, 7616), (10, 9920), (8, 14528)))


def entry_points():
    return build.load_entry_points("int8_linear.cu")


def linear_call(**kw):
    """b200_int8_linear on two rows of 32 (memory of the host: nothing may be launched)."""
    a = dict(x=torch.zeros(2, 32), residual=None, gain=None, kept=None, q=torch.zeros(2, 32, dtype=torch.int8), s=torch.zeros(2),
             w=torch.zeros(4, 32, dtype=torch.int8), c=torch.ones(4), bias=None, out=torch.zeros(2, 4), tokens=2, n=4, k=32, x_pitch=32, q_pitch=32,
             w_pitch=32, x_code=0, gain_code=0, out_code=0, mode=0, eps=0.0, limit=0.0, alpha=1.0, err=torch.zeros(1, dtype=torch.int32), stream=0)
    a.update(kw)
    return entry_points().b200_int8_linear(*a.values())


def test_entry_points_refuse_more_rows_than_they_count():
    """A step past the last row must stay below 2^31 too."""
    for many in (2 ** 31 - 1, 2 ** 31 - 65536):
        assert linear_call(tokens=many) == linear_call(n=many) == -2
        assert entry_points().b200_int8_rows(torch.zeros(2, 32), None, None, None, torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2), many, 32, 32, 32,
                                             0, 0, 0.0, 0) == -2
    assert linear_call(n=2 ** 30, mode=1) == -2                   # (gate and up rows together)


def test_more_rows_than_the_kernels_count_are_refused():
    from llm_infer_rust_b200.kernels import int8
    from llm_infer_rust_b200.kernels.ops import KernelError
    w = int8.Int8Weight(torch.zeros(4, 16, dtype=torch.int8)[:, :1], torch.ones(4))
    for many in (2 ** 31 - 65536, 2 ** 32 + 5):                   # (memory of no device: the sizes alone count)
        x = torch.empty(many, 1, dtype=torch.bfloat16, device="meta")
        rows = int8.Int8Rows(torch.empty(many, 16, dtype=torch.int8, device="meta")[:, :1], torch.empty(many, device="meta"))
        for call in (lambda: int8.int8_linear(x, w), lambda: int8.quantize_rows(x), lambda: int8.int8_linear(rows, w),
                     lambda: int8.int8_linear(torch.zeros(2, 1), int8.Int8Weight(*rows))):
            with pytest.raises(KernelError, match="rows are refused"):
                call()


def test_entry_points_refuse_null_operands():
    rows = lambda x=torch.zeros(2, 32), q=torch.zeros(2, 32, dtype=torch.int8), s=torch.zeros(2): \
        entry_points().b200_int8_rows(x, None, None, None, q, s, 2, 32, 32, 32, 0, 0, 0.0, 0)
    assert rows(x=None) == rows(q=None) == rows(s=None) == -2
    for tokens in (2, 20):                                        # (the streaming kernel and the tiled one)
        for name in ("w", "c", "out", "err"):
            assert linear_call(tokens=tokens, **{name: None}) == -2, (tokens, name)
        assert linear_call(tokens=tokens, x=None, s=None) == linear_call(tokens=tokens, x=None, q=None) == -2
    assert linear_call(tokens=20, q=None) == linear_call(tokens=20, s=None) == -2      # (two tokens alone need no place for them)
    assert linear_call(tokens=0, x=None, q=None, s=None, w=None, c=None, out=None, err=None) == 0


FAKE = r"""
#include <cuda_runtime.h>
#include <cstdio>
static int calls = 0, refuse = 0;
template <typename K> static cudaError_t fake_attribute(K, cudaFuncAttribute, int) { ++calls; return refuse ? cudaErrorInvalidValue : cudaSuccess; }
#define cudaFuncSetAttribute fake_attribute
#include "int8_common.cuh"
__global__ void kernel() {}
int main() {
  bool set[64] = {};
  for (int device : {0, 0, 1, 0, 63, 1, 63, 64, 64, -1, 2, 2}) {
    refuse = device == 2 && calls == 6;
    const int rc = int8_launch_limit(kernel, 1000, Int8Device{device, 148}, set);
    std::printf("%d:%d ", rc, calls);
  }
}
"""


def test_a_launch_limit_is_set_once_a_device(tmp_path):
    """Against a fake of the runtime's call: every device that a kernel is launched on has its limit, one that was refused is asked again."""
    import subprocess
    source, program = tmp_path / "limit.cu", tmp_path / "limit"
    source.write_text(FAKE)
    subprocess.run([build.find_nvcc(), *build.ARCH_FLAGS, "-std=c++17", "-I", build.CSRC, "-o", str(program), str(source)], check=True,
                   stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    said = subprocess.run([str(program)], check=True, stdout=subprocess.PIPE, text=True).stdout
    assert said.split() == "0:1 0:1 0:2 0:2 0:3 0:3 0:3 0:4 0:5 0:6 1:7 0:8".split()
