"""The native calls that take a function's own tensors, of several types and any row stride: what they leave to the function's checks.
No device: a call ends before anything is launched."""
import numpy as np
import pytest
import torch

from pixienn_amd import capi, ops


@pytest.fixture(scope="module")
def functions():
    capi.load()
    if not capi.functions:
        capi.bind_calls()
    return capi.functions


def test_they_are_entry_points_of_the_binding(functions):
    assert set(functions) == {"pxh_rms_norm_forward", "pxh_rms_norm_backward", "pxh_token_logprobs_forward", "pxh_token_logprobs_backward",
                              "pxh_token_logprobs_forward_train"}
    assert set(functions) <= set(capi.SIGNATURES) and not set(functions) & set(capi.native)


def test_what_is_no_tensor_of_the_device_is_left(functions):
    x = torch.zeros(2, 8)
    calls = {"pxh_rms_norm_forward": (x, x, x[0], None, None, None, None, 1e-6, 0, None),
             "pxh_rms_norm_backward": (x, x, x[0], x[:, 0], x, x[0], None, 0, None, None),
             "pxh_token_logprobs_forward": (x, None, None, None, None, None, None, 1.0, None, None),
             "pxh_token_logprobs_backward": (x, None, None, None, x, None, None, 1.0, None),
             "pxh_token_logprobs_forward_train": (x, None, None, x, None, None, None, None, 1.0, None)}
    assert set(calls) == set(functions)
    for name, args in calls.items():
        assert functions[name](*args) is None, name
        for other in (np.zeros((2, 8)), 7, "x"):
            assert functions[name](other, *args[1:]) is None, name
        assert functions[name](*args, None) is None and functions[name](*args[:-1]) is None, name


def test_no_tensor_at_all_is_refused_by_the_entry_point(functions):
    none = [None] * 7
    assert functions["pxh_rms_norm_forward"](*none, 1e-6, 0, None) is None          # the weights have a type: they are looked at
    assert functions["pxh_token_logprobs_forward"](*none, 1.0, None, None) == -1
    assert "logits" in capi.last_error()


def test_the_functions_say_what_is_wrong():
    x = torch.zeros(2, 8)
    with pytest.raises(capi.PxError, match="must live on the GPU"):
        ops.rms_norm_forward(x, x, x[0])
    with pytest.raises(capi.PxError, match="logits is required"):
        ops.token_logprobs_forward(None, None, None)


def test_a_workspace_is_packed_memory_of_the_device():
    """Kernels write to it: anything else is refused before its address is taken."""
    assert ops._space(None) == (None, 0)
    with pytest.raises(capi.PxError, match="workspace must live on the GPU"):
        ops._space(torch.zeros(1 << 20))
    with pytest.raises(capi.PxError, match="workspace: torch.Tensor expected"):
        ops._space(np.zeros(1 << 20))
