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
