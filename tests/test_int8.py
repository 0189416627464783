"""Refusals of the int8 operators and of their C entry points, which need no GPU."""

import pytest
import torch

from sigcomp_b200 import _lib
from sigcomp_b200.int8 import dequantize_tokens, int8_linear, int8_linear_requant, quantize_tokens

X = torch.zeros((4, 32))
Q = torch.zeros((4, 32), dtype=torch.int8)
S = torch.ones(4)
W = torch.zeros((8, 32), dtype=torch.int8)
T = torch.ones(8)
B = torch.zeros(8)


def _refused(text, call, *args, **kwargs):
    with pytest.raises(ValueError, match=text):
        call(*args, **kwargs)


def test_arrays_off_the_gpu_are_refused():
    _refused("run on a GPU", quantize_tokens, X)
    _refused("run on a GPU", dequantize_tokens, Q, S)
    _refused("run on a GPU", int8_linear, X, W, T, B)
    _refused("run on a GPU", int8_linear_requant, Q, S, W, T, B)


@pytest.mark.parametrize("text,call", [
    ("torch tensor", lambda: quantize_tokens([1.0])),
    ("of type", lambda: quantize_tokens(X.double())),
    ("of type", lambda: quantize_tokens(Q)),
    ("at least one element", lambda: quantize_tokens(torch.zeros((3, 0)))),
    ("at least one element", lambda: quantize_tokens(torch.tensor(1.0))),
    ("gradient", lambda: quantize_tokens(X.clone().requires_grad_())),
    ("dense", lambda: quantize_tokens(torch.zeros(3, 4).to_sparse())),
    ("dense", lambda: quantize_tokens(torch.zeros(3, 4, dtype=torch.complex64).conj().imag)),
    ("of type", lambda: dequantize_tokens(X, S)),
    ("dtype must be", lambda: dequantize_tokens(Q, S, dtype=torch.int8)),
    ("shape", lambda: dequantize_tokens(Q, S[:3])),
    ("of type", lambda: dequantize_tokens(Q, S.double())),
    ("of type", lambda: int8_linear(X.double(), W, T)),
    ("of type", lambda: int8_linear(X, W.float(), T)),
    ("torch tensor", lambda: int8_linear(None, W, T)),
    ("rows of 32", lambda: int8_linear(X[:, :31], W, T)),
    ("out, in", lambda: int8_linear(X, W[0], T)),
    ("out, in", lambda: int8_linear(X, W[:0], T[:0])),
    ("elements", lambda: int8_linear(X, W, T[:7])),
    ("elements", lambda: int8_linear(X, W, T, B[:7])),
    ("of type", lambda: int8_linear(X, W, T, B.half())),
    ("need x_scales", lambda: int8_linear(Q, W, T)),
    ("belong to int8", lambda: int8_linear(X, W, T, x_scales=S)),
    ("shape", lambda: int8_linear(Q, W, T, x_scales=S[:, None])),
    ("dtype must be", lambda: int8_linear(X, W, T, dtype=torch.int8)),
    ("gradient", lambda: int8_linear(X.clone().requires_grad_(), W, T)),
    ("gradient", lambda: int8_linear(X, W, T.clone().requires_grad_())),
    ("overflow", lambda: int8_linear(torch.zeros((1, 131072)), torch.zeros((1, 131072), dtype=torch.int8), T[:1])),
    ("of type", lambda: int8_linear_requant(X, S, W, T)),
    ("finite positive", lambda: int8_linear_requant(Q, S, W, T, output_scale=0.0)),
    ("finite positive", lambda: int8_linear_requant(Q, S, W, T, output_scale=float("nan"))),
    ("finite positive", lambda: int8_linear_requant(Q, S, W, T, output_scale=-1.0)),
])
def test_wrong_arguments_are_refused(text, call):
    _refused(text, call)


def test_gradients_are_refused_only_where_one_is_recorded():
    with torch.no_grad():
        _refused("run on a GPU", quantize_tokens, X.clone().requires_grad_())


def _linear_status(**over):
    """The status of sc_int8_linear_device for arguments that it has to refuse before any GPU work."""
    a = dict(device=0, x=4096, x_type=3, x_stride=32, x_scales=4096, w=4096, w_stride=32, w_scales=4096, bias=None,
             rows=4, n=8, k=32, relu=0, y=4096, y_type=0, y_stride=8, y_scales=None, output_scale=0.0, workspace=None,
             workspace_bytes=0, stream=None)
    a.update(over)
    return _lib.load().sc_int8_linear_device(*a.values())


@pytest.mark.parametrize("over", [
    {"x_type": 4}, {"x_type": -1}, {"y_type": 4}, {"rows": -1}, {"n": 0}, {"k": 0}, {"k": 131072, "w_stride": 131072},
    {"w_stride": 31}, {"y_stride": 7}, {"x_stride": -1}, {"x": None}, {"y": None}, {"w": None}, {"w_scales": None},
    {"x_scales": None}, {"x_type": 0}, {"rows": 2 ** 31}, {"y_type": 3}, {"y_type": 3, "output_scale": float("inf")},
    {"y_type": 3, "output_scale": -1.0},
    # arrays that do not start on an element
    {"x_type": 0, "x_scales": None, "x": 4098}, {"x_type": 1, "x_scales": None, "x": 4097}, {"y": 4098},
    {"y_type": 2, "y": 4097}, {"x_scales": 4097}, {"w_scales": 4098}, {"bias": 4099}, {"y_type": 3, "y_scales": 4098},
    # workspace missing, too small or misaligned
    {"x_type": 0, "x_scales": None}, {"x_type": 0, "x_scales": None, "workspace": 4096, "workspace_bytes": 16},
    {"x_type": 0, "x_scales": None, "workspace": 4097, "workspace_bytes": 1 << 20},
])
def test_c_entry_point_refuses(over):
    assert _linear_status(**over) == _lib.SC_ERR_INVALID_ARGUMENT
    assert _lib.last_error()


def test_c_entry_points_do_nothing_for_no_rows():
    assert _linear_status(rows=0, x=None, y=None, x_scales=None) == _lib.SC_OK
    L = _lib.load()
    assert L.sc_quantize_tokens_device(0, None, 0, 0, 5, 5, None, 5, None, None) == _lib.SC_OK
    assert L.sc_dequantize_tokens_device(0, None, 5, None, 1.0, 0, 5, None, 0, 5, None) == _lib.SC_OK
    assert L.sc_int8_linear_workspace(0, 1, 1, 0, 8, 32, 3, 1) == 0


@pytest.mark.parametrize("args", [
    (0, 4096, 3, 4, 8, 8, 4096, 8, 4096, None),      # int8 in
    (0, 4096, 0, 4, 8, 8, 4096, 7, 4096, None),      # rows of q overlap
    (0, 4096, 0, 4, 0, 8, 4096, 8, 4096, None),      # no columns
    (0, None, 0, 4, 8, 8, 4096, 8, 4096, None),
    (0, 4096, 0, 4, 8, 8, 4096, 8, None, None),
    (0, 4096, 0, -1, 8, 8, 4096, 8, 4096, None),
    (0, 4098, 0, 4, 8, 8, 4096, 8, 4096, None),      # x within an element
    (0, 4096, 0, 4, 8, 8, 4096, 8, 4097, None),
])
def test_quantise_entry_point_refuses(args):
    assert _lib.load().sc_quantize_tokens_device(*args) == _lib.SC_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("args", [
    (0, 4096, 8, None, 1.0, 4, 8, 4096, 3, 8, None),
    (0, 4096, 8, None, 1.0, 4, 8, 4096, 0, 7, None),
    (0, None, 8, None, 1.0, 4, 8, 4096, 0, 8, None),
    (0, 4096, -8, None, 1.0, 4, 8, 4096, 0, 8, None),
    (0, 4096, 8, None, 1.0, 4, 8, 4097, 2, 8, None),
    (0, 4096, 8, 4098, 1.0, 4, 8, 4096, 2, 8, None),
])
def test_dequantise_entry_point_refuses(args):
    assert _lib.load().sc_dequantize_tokens_device(*args) == _lib.SC_ERR_INVALID_ARGUMENT


def test_workspace_size_is_a_whole_number_of_bytes():
    assert isinstance(_lib.load().sc_int8_linear_workspace(1, 1, 1, 1, 512, 8192, 2, 0), int)


@pytest.mark.parametrize("args", [
    (3, 1, 1, 4, 0, 32, 0, 0), (3, 1, 1, 4, 8, 0, 0, 0), (3, 1, 1, -4, 8, 32, 0, 0), (3, 1, 1, 4, -1, 32, 3, 1),
    (9, 1, 1, 4, 8, 32, 0, 0), (3, 1, 1, 4, 8, 32, -1, 0), (0, 1, 1, 4, 8, 1 << 40, 0, 0), (0, 0, 0, 1 << 60, 8, 8, 3, 1),
])
def test_workspace_of_refused_arguments(args):
    assert _lib.load().sc_int8_linear_workspace(*args) == 0


def test_workspace_sizes():
    """Rows of 8 bits and their scales, spread arrays, a product in 32 bits: each where it is needed."""
    size = _lib.load().sc_int8_linear_workspace
    assert size(3, 1, 1, 1000, 512, 512, 0, 0) == 0
    assert size(0, 0, 1, 1000, 512, 500, 0, 0) == 1000 * 512 + 4096                     # rounded to 256 bytes
    assert size(3, 0, 1, 1000, 512, 500, 0, 0) == 1000 * 512
    assert size(3, 1, 0, 1000, 512, 500, 0, 0) == 512 * 512
    assert size(0, 0, 1, 1, 512, 500, 0, 0) == 0                                        # one token: quantised on the way
    for rows in (1, 16, 300, 5000, 100000):
        for n in (3, 512, 2000):
            assert 0 <= size(3, 1, 1, rows, n, 256, 3, 1) <= rows * (n + 3) * 4 + 256
