"""The native calls that also look at the tensors' device, and what the entry points behind them refuse.  No device: a call ends before
anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

from pixienn_amd import capi, ops


@pytest.fixture(scope="module")
def layers():
    capi.load()
    if not capi.layers:
        capi.bind_calls()
    return capi.layers


X = torch.zeros(2, 8)
TOKENS = torch.zeros(2, dtype=torch.int32)
CALLS = {"pxh_embedding_forward": (X, TOKENS, X, 1.0),
         "pxh_embedding_backward": (X, TOKENS, X, 1.0, 0, None),
         "pxh_layer_norm_forward": (X, X, X[0], None, None, None, None, None, 1e-5),
         "pxh_layer_norm_backward": (X, X, X[0], X[:, 0], X[:, 0], X, X[0], None, None, 0, None),
         "pxh_gated_scan_forward": (X, X, X, None, None, None, None, None, None, None, None),
         "pxh_gated_scan_backward": (X, X, X, X, X, X, None, None, None, None, None, None, None, None, None),
         "pxh_gated_scan_step": (X, X, X, X, None, None),
         "pxh_beam_select": (X, X[:, :1], X[:, :1], TOKENS, TOKENS, None, 0, 1.0, None),
         "pxh_beam_reorder": ([X], TOKENS)}


def test_they_are_entry_points_of_the_binding(layers):
    assert set(layers) == set(CALLS)
    assert set(layers) <= set(capi.SIGNATURES) and not set(layers) & (set(capi.native) | set(capi.functions))


def test_what_is_no_tensor_of_the_device_is_left(layers):
    for name, args in CALLS.items():
        assert layers[name](*args, 0, 0) is None, name
        for other in (np.zeros((2, 8)), 7, "x"):
            assert layers[name](other, *args[1:], 0, 0) is None, name
        assert layers[name](*args, 0, 0, None) is None and layers[name](*args, 0) is None, name


def test_the_functions_say_what_is_wrong():
    for f, match in [(lambda: ops.embedding_forward(X, TOKENS, X), "must live on the GPU"),
                     (lambda: ops.embedding_backward(np.zeros((2, 8)), TOKENS, X), "torch.Tensor expected"),
                     (lambda: ops.layer_norm_forward(X, X, X[0]), "must live on the GPU"),
                     (lambda: ops.layer_norm_backward(X, X, X[0], X[:, 0], X[:, 0], X, X[0]), "must live on the GPU"),
                     (lambda: ops.gated_scan_forward(X, X, X), "must live on the GPU"),
                     (lambda: ops.gated_scan_backward(X, X, X, X, X, X), "must live on the GPU"),
                     (lambda: ops.gated_scan_step(X, X, X, X), "must live on the GPU"),
                     (lambda: ops.beam_select(X, X, X, X, X), "must live on the GPU"),
                     (lambda: ops.beam_reorder([X], None), "parents is required"),
                     (lambda: ops.beam_reorder([X], TOKENS.view(1, 2)), "must live on the GPU")]:
        with pytest.raises(capi.PxError, match=match):
            f()


F32, BF16, E4M3 = 0, 1, 3
HERE = 64            # an address that no refused call reads


def refused(name, *args):
    assert capi.call_raw(name, *args) == -1, name
    return capi.last_error()


def test_the_entry_points_refuse():
    def embedding(type=F32, wide=0, rows=2, vocab=8, width=4, stride=4, y_stride=4, at=HERE):
        return "pxh_embedding_forward", HERE, at, HERE, type, wide, rows, vocab, width, stride, y_stride, 1.0, None
    for change in (dict(type=9), dict(rows=-1), dict(vocab=0), dict(width=0), dict(stride=3), dict(y_stride=3), dict(at=None)):
        assert "pxh_embedding_forward" in refused(*embedding(**change)), change
    assert capi.call_raw(*embedding(rows=0)) == 0

    def gradient(type=BF16, d_type=BF16, rows=2, vocab=8, width=4, stride=4, d_stride=4, at=HERE):
        return "pxh_embedding_backward", HERE, at, HERE, type, d_type, 0, rows, vocab, width, stride, d_stride, 1.0, 0, HERE, 1 << 30, None
    for change in (dict(type=9), dict(d_type=9), dict(type=F32, d_type=BF16), dict(rows=-1), dict(rows=1 << 31), dict(vocab=0), dict(width=0),
                   dict(stride=3), dict(d_stride=3), dict(at=None)):
        assert "pxh_embedding_backward" in refused(*gradient(**change)), change

    def norm(type=F32, weight_type=F32, rows=2, width=4, strides=(4, 4, 4, 4), x=HERE, residual=HERE, sum=HERE):
        return "pxh_layer_norm_forward", x, residual, sum, HERE, None, HERE, None, None, type, weight_type, rows, width, *strides, 1e-5, None
    for change in (dict(type=9), dict(weight_type=BF16), dict(rows=-1), dict(width=0), dict(strides=(3, 4, 4, 4)), dict(strides=(4, 3, 4, 4)),
                   dict(strides=(4, 4, 3, 4)), dict(strides=(4, 4, 4, 3)), dict(x=None), dict(residual=None)):
        assert "pxh_layer_norm_forward" in refused(*norm(**change)), change
    assert capi.call_raw(*norm(rows=0)) == 0

    def scan(type=F32, rows=4, width=8, sequences=2, slots=0, starts=None, x=HERE, strides=(8, 8, 8, 8), state=None):
        return ("pxh_gated_scan_forward", x, HERE, None, HERE, starts, state, None, None, None, type, rows, width, sequences, slots, *strides,
                HERE, 1 << 30, None)
    for change in (dict(type=9), dict(rows=-1), dict(width=0), dict(sequences=-1), dict(sequences=3), dict(x=None), dict(strides=(7, 8, 8, 8)),
                   dict(strides=(8, 7, 8, 8)), dict(strides=(8, 8, 8, 7)), dict(sequences=0), dict(slots=-1, state=HERE)):
        assert "pxh_gated_scan_forward" in refused(*scan(**change)), change
    assert "pxh_gated_scan_step" in refused("pxh_gated_scan_step", HERE, HERE, None, HERE, None, None, F32, 2, 8, 2, 8, 8, 8, 8, None)

    def select(type=F32, batch=2, beams=3, vocab=9, stride=9, count=3, scale=1.0, logits=HERE):
        return "pxh_beam_select", logits, HERE, None, HERE, HERE, HERE, type, batch, beams, vocab, stride, count, 0, scale, HERE, 1 << 30, None
    for change in (dict(type=E4M3), dict(batch=-1), dict(beams=0), dict(beams=65), dict(vocab=0), dict(stride=8), dict(count=0), dict(count=65),
                   dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(logits=None)):
        assert "pxh_beam_select" in refused(*select(**change)), change
    assert capi.call_raw(*select(batch=0)) == 0
    assert "pxh_beam_reorder" in refused("pxh_beam_reorder", 1, None, None, None, HERE, 2, 3, None)

    def reorder(tensors=(HERE, 2 * HERE), row_bytes=(8, 8), strides=(8, 8), batch=2, beams=3, parents=HERE):
        n = len(tensors)
        return ("pxh_beam_reorder", n, (ctypes.c_void_p * n)(*tensors), (ctypes.c_longlong * n)(*row_bytes), (ctypes.c_longlong * n)(*strides),
                parents, batch, beams, None)
    # (the second tensor is looked at before the first is touched)
    for change in (dict(row_bytes=(8, -1)), dict(strides=(8, 7)), dict(tensors=(HERE, None)), dict(tensors=(HERE, HERE)), dict(parents=None),
                   dict(beams=0), dict(beams=65), dict(batch=-1), dict(batch=1 << 20, beams=64, row_bytes=(8, 1 << 20), strides=(8, 1 << 20))):
        assert "pxh_beam_reorder" in refused(*reorder(**change)), change
    assert capi.call_raw(*reorder(batch=0)) == 0 and capi.call_raw(*reorder(row_bytes=(0, 0), tensors=(None, None))) == 0


def test_a_workspace_that_is_too_small_or_askew_is_refused():
    lib = capi.load()
    for name, args, need in [
            ("pxh_embedding_backward", (HERE, HERE, HERE, F32, F32, 0, 600, 8, 4, 4, 4, 1.0, 0), lib.pxh_embedding_workspace_bytes(600, 4)),
            ("pxh_layer_norm_backward", (HERE, HERE, HERE, HERE, HERE, None, HERE, HERE, HERE, F32, F32, 600, 40, 40, 40, 40, 40, 0),
             lib.pxh_layer_norm_workspace_bytes(600, 40)),
            ("pxh_gated_scan_forward", (HERE, HERE, None, HERE, None, None, None, None, None, F32, 600, 8, 1, 0, 8, 8, 8, 8),
             lib.pxh_gated_scan_workspace_bytes(600, 8)),
            ("pxh_beam_select", (HERE, HERE, None, HERE, HERE, HERE, F32, 2, 3, 9, 9, 3, 0, 1.0), lib.pxh_beam_select_workspace_bytes(2, 3, 9, 3))]:
        assert need > 0
        assert capi.call_raw(name, *args, HERE, 8, None) != 0 and "too small" in capi.last_error(), name
        assert capi.call_raw(name, *args, HERE + 4, 1 << 40, None) != 0 and "aligned" in capi.last_error(), name


def test_a_workspace_serves_smaller_calls():
    lib = capi.load()
    sizes = [1, 2, 15, 16, 17, 31, 63, 64, 255, 256, 257, 999, 2047, 2048, 2049, 4099, 30011, 70001]
    for f in (lib.pxh_embedding_workspace_bytes, lib.pxh_layer_norm_workspace_bytes, lib.pxh_gated_scan_workspace_bytes):
        for a, b in zip(sizes, sizes[1:]):
            for other in (1, 7, 64, 1000, 2561, 4097, 16385, 40001):
                assert 0 < f(a, other) <= f(b, other), (a, other)
                assert f(other, a) <= f(other, b), (other, a)
    f = lib.pxh_beam_select_workspace_bytes
    for a, b in zip(sizes, sizes[1:]):
        for count in (1, 8, 64):
            assert 0 < f(1, 4, a, count) <= f(1, 4, b, count) and f(a, 1, 777, count) <= f(b, 1, 777, count)
            assert f(3, min(a, 64), 5001, count) <= f(3, min(b, 64), 5001, count) and f(2, 2, 333, min(a, 64)) <= f(2, 2, 333, min(b, 64))
