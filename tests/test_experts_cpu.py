"""CPU: what the operators of layers of experts refuse, through Python and through the C ABI."""
import ctypes

import pytest
import torch


def test_ops_refuse_cpu_tensors_and_wrong_types():
    from weather_model_amd import ops
    x, w, off = torch.zeros(4, 8), torch.zeros(2, 6, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ops.dense_grouped(x, w, off), lambda: ops.dropout(x, 0.1, 1), lambda: ops.quantize_rows(x),
                 lambda: ops.dense_i8(x, w[0].to(torch.int8), torch.zeros(6))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.dropout([1.0], 0.1, 1)


def test_expert_stack_refuses_layers_that_do_not_fit():
    from weather_model_amd.experts import ExpertStack
    with pytest.raises(ValueError, match="one bias per weight"):
        ExpertStack([], [])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ExpertStack([torch.zeros(2, 3, 4)], [torch.zeros(2, 3)])


def test_dropout_arguments():
    from weather_model_amd import ops
    x = torch.zeros(4)
    for p, seed, offset, error, text in ((-0.1, 0, 0, ValueError, "probability"), (1.5, 0, 0, ValueError, "probability"),
                                         (float("nan"), 0, 0, ValueError, "probability"), (0.1, -1, 0, ValueError, "seed"),
                                         (0.1, 1 << 32, 0, ValueError, "seed"), (0.1, 0, -1, ValueError, "offset"),
                                         (0.1, 0, 1 << 63, ValueError, "offset"),
                                         (0.1, 0, torch.zeros(1, dtype=torch.int64), TypeError, "device offset"),
                                         (0.1, 0, torch.zeros(2), TypeError, "device offset")):
        with pytest.raises(error, match=text):
            ops._dropout_args(p, seed, offset, x)


def test_c_abi_refusals():
    """Argument checks come before any device work."""
    from weather_model_amd import _lib
    L = _lib.lib()
    buf = ctypes.create_string_buffer(64)
    p = ctypes.cast(buf, ctypes.c_void_p)

    def refused(rc, code, text):
        assert rc == code and text in L.wm_last_error(), (rc, L.wm_last_error())
    refused(L.wm_dropout(p, 0, p, -1, 0, 0.1, 0, 0, 0, 0), -1, b"element count")
    refused(L.wm_dropout(p, 0, p, 4, 0, 1.1, 0, 0, 0, 0), -1, b"probability")
    refused(L.wm_dropout(p, 0, p, 4, 0, float("nan"), 0, 0, 0, 0), -1, b"probability")
    refused(L.wm_dropout(p, 0, p, 4, 1, 0.1, 0, 0, 0, 0), -1, b"dtype")
    refused(L.wm_dropout(0, 0, p, 4, 0, 0.1, 0, 0, 0, 0), -1, b"null pointer")
    refused(L.wm_dense_grouped_fwd(p, p, 0, p, 0, 0, p, 0, 4, 4, 4, 0, 0, 0), -1, b"bad sizes")
    refused(L.wm_dense_grouped_fwd(p, p, 0, p, 0, 0, p, 1, -1, 4, 4, 0, 0, 0), -1, b"bad sizes")
    refused(L.wm_dense_grouped_fwd(p, p, 0, p, 0, 0, p, 1, 4, 4, (1 << 20) + 1, 0, 0, 0), -2, b"beyond")
    refused(L.wm_dense_grouped_fwd(p, p, 0, p, 0, 0, p, 4097, 4, 4, 4, 0, 0, 0), -2, b"4096 groups")
    refused(L.wm_dense_grouped_bwd_data(p, p, 0, p, 0, 0, p, 1, 4, 4, 4, 1, 0), -1, b"dtype")
    refused(L.wm_dense_grouped_bwd_wb(p, p, p, 0, 0, 0, p, 1, 4, 0, 4, 0, 0), -1, b"bad sizes")
    refused(L.wm_quantize_rows_i8(p, 4, (1 << 17) + 1, 0, p, p, 0), -2, b"32 bits")
    refused(L.wm_quantize_rows_i8(p, 4, 0, 0, p, p, 0), -1, b"bad sizes")
    refused(L.wm_dense_i8(p, p, p, 0, p, 0, 1, 4, 4, 4, 7, 0, p, 64, 0), -1, b"dtype")
    assert L.wm_dense_i8_workspace_bytes(0, 4, 4) == 0 and L.wm_dense_i8_workspace_bytes(3, 4, 0) == 0
    assert L.wm_dense_grouped_bwd_wb_workspace_bytes(0, 4, 4, 4, 0) == 0
    assert L.wm_dense_grouped_fwd_workspace_bytes(1, 16, 8192, 8192, 0) == 0          # few rows
    assert L.wm_dense_grouped_fwd_workspace_bytes(1, 200, 64, 500, 0) == 0          # no long contraction
    assert L.wm_dense_grouped_fwd_workspace_bytes(1, 200, 64, 8192, 0) >= 200 * 64 * 4 * 2
    assert L.wm_dense_grouped_bwd_data_workspace_bytes(1, 16, 8192, 64, 2) >= 16 * 64 * 4 * 2


def test_product_sizes_do_not_overflow_the_workspace_query():
    from weather_model_amd import _lib
    L = _lib.lib()
    assert L.wm_dense_i8_workspace_bytes(1, 8, 8192) == 0 and L.wm_dense_i8_workspace_bytes(1, 8, 8193) > 0
    assert L.wm_dense_i8_workspace_bytes(4, 8, 2048) == 0 and L.wm_dense_i8_workspace_bytes(4, 8000, 2048) > 0
    assert L.wm_dense_i8_workspace_bytes(1 << 24, 8, 1 << 17) >= (1 << 24) * (1 << 17)
    assert L.wm_dense_grouped_bwd_wb_workspace_bytes(1, 1 << 30, 8, 8, 0) >= 8 * 8 * 4


def test_group_offsets():
    from weather_model_amd import ops
    for dtype in (torch.int32, torch.int64):
        off = ops.group_offsets(torch.tensor([3, 0, 5, 0], dtype=dtype))
        assert off.dtype == torch.int64 and off.tolist() == [0, 3, 3, 8, 8]
    assert ops.group_offsets(torch.zeros((0,), dtype=torch.int64)).tolist() == [0]
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.group_offsets(torch.ones(3))
    with pytest.raises(ValueError, match="counts must be"):
        ops.group_offsets(torch.ones((2, 2), dtype=torch.int64))


def test_sizes_beyond_32_bits_are_refused():
    """Views of one element: nothing is allocated."""
    from weather_model_amd import ops
    n = 2 ** 32 + 4
    for shape in ((n, 1), (1, n), (3, 2 ** 31), (1, n, 1), (n, 1, 2)):
        with pytest.raises(ValueError, match="beyond 32 bits"):
            ops._in_32_bits(torch.zeros((1,) * len(shape)).expand(shape), "input")
    for shape in ((2 ** 31 - 1, 4), (2 ** 31 - 1,), (0, 5), (), (70000, 70000)):
        ops._in_32_bits(torch.zeros((1,) * len(shape)).expand(shape) if shape else torch.zeros(()), "input")


def test_expert_stack_refuses_what_is_no_probability_and_no_seed():
    """When it is made: a negative p or a NaN would train without dropout, and a seed would only be looked at by the first step."""
    from weather_model_amd.experts import ExpertStack
    w, b = [torch.zeros(2, 3, 4)], [torch.zeros(2, 3)]
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            ExpertStack(w, b, p=p)
    for seed in (-1, 1 << 32):
        with pytest.raises(ValueError, match="seed"):
            ExpertStack(w, b, seed=seed)
