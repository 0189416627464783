"""int8 operators with a scale for each token and each channel.

The bundled entropy models have one fixed-point multiplier per layer (``B200Compression``, and
``sc_linear_layer_device`` for a layer alone).  A model whose weights are quantised per channel,
and whose activations are quantised token by token as they come, is computed with these:

* :func:`quantize_tokens` / :func:`dequantize_tokens` - rows held in 8 bits with a scale each;
* :func:`int8_linear` - a linear layer on such rows, results in 16 or 32 bits;
* :func:`int8_linear_requant` - the same with int8 results: rows with a scale each for the next
  layer, or with one given scale, the int8 logits that the range coder takes
  (``sc_encode_logits_device``).

A row's result depends neither on the rows beside it nor on their number: sums of products are
whole numbers, exact in 32 bits, and the roundings after them are fixed (include/sigcomp_b200.h
writes them out).  So teacher-forced coding in large batches and decoding token by token agree bit
for bit.

Arrays are torch tensors on one GPU; leading dimensions are batch dimensions.  Work is put into the
current stream of that GPU and not waited for, so calls can be captured into CUDA graphs.  The
operators serve coding, not training: a tensor that asks for a gradient is refused.
"""

import functools
import math

import torch

from . import _lib

MAX_K = 131071

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _tensor(name, t, dtypes, device=None):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be of type {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other arrays are on {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} asks for a gradient, which the int8 operators do not have")
    return t


def _rows(name, t):
    """``t`` as rows: a view where its strides allow one, else a copy."""
    if t.dim() == 0 or t.shape[-1] == 0:
        raise ValueError(f"{name} must have rows of at least one element")
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _on_gpu(t):
    if not t.is_cuda:
        raise ValueError("the int8 operators run on a GPU: move the arrays there")


def _vector(name, t, length, device):
    _tensor(name, t, (torch.float32,), device)
    if t.dim() != 1 or t.shape[0] != length:
        raise ValueError(f"{name} must have {length} elements, not shape {tuple(t.shape)}")
    return t.contiguous()


def _scales(name, t, shape, device):
    _tensor(name, t, (torch.float32,), device)
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, one scale for each row, not {tuple(t.shape)}")
    return t.contiguous()


def _int8_out(rows, cols, device):
    """int8 rows that start a multiple of 16 bytes apart, as the matrix kernels read them."""
    return torch.empty((rows, -(-cols // 16) * 16), dtype=torch.int8, device=device)[:, :cols]


def _shaped(t, lead):
    return t if t.dim() - 1 == len(lead) else t.unflatten(0, lead) if lead else t[0]


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def quantize_tokens(x):
    """Quantise every row of ``x`` (``[..., k]``, float32, float16 or bfloat16) to int8.

    Returns ``(q, scales)``: int8 of x's shape and float32 of its leading shape.  With
    ``a = max(max|row|, 2**-100)``, ``scale = a / 127`` and ``q = rint(row * (127 / a))``; both
    quotients are rounded to float32, the product is not, and ties go to the even number.  A row
    holding an infinity or a NaN gets the scale NaN and zeros, so what is computed from it is NaN.
    Rows of ``q`` start a multiple of 16 bytes apart.
    """
    _tensor("x", x, _FLOATS)
    lead = x.shape[:-1]
    rows = _rows("x", x)
    _on_gpu(x)
    q = _int8_out(rows.shape[0], rows.shape[1], x.device)
    scales = torch.empty(rows.shape[0], dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().sc_quantize_tokens_device(
        x.device.index, rows.data_ptr(), _TYPES[x.dtype], rows.shape[0], rows.shape[1], rows.stride(0), q.data_ptr(),
        q.stride(0), scales.data_ptr(), _stream(x.device)), "sc_quantize_tokens_device")
    return _shaped(q, lead), scales.reshape(lead)


def dequantize_tokens(q, scales, dtype=torch.float32):
    """The values that int8 rows stand for: ``q * scales`` in float32, rounded once to ``dtype``.

    ``scales`` holds one scale for each row, or is one number for all of them.
    """
    _tensor("q", q, (torch.int8,))
    if dtype not in _FLOATS:
        raise ValueError(f"dtype must be one of {_FLOATS}")
    rows = _rows("q", q)
    if isinstance(scales, torch.Tensor):
        per_row, one = _scales("scales", scales, q.shape[:-1], q.device).data_ptr(), 0.0
    else:
        per_row, one = None, float(scales)
    _on_gpu(q)
    y = torch.empty(q.shape, dtype=dtype, device=q.device)
    _lib.check(_lib.load().sc_dequantize_tokens_device(
        q.device.index, rows.data_ptr(), rows.stride(0), per_row, one, rows.shape[0], rows.shape[1], y.data_ptr(),
        _TYPES[dtype], rows.shape[1], _stream(q.device)), "sc_dequantize_tokens_device")
    return y


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(*sizes):
    return _lib.load().sc_int8_linear_workspace(*sizes)


def _packed(t, stride, k):
    return t.data_ptr() % 16 == 0 and stride % 16 == 0 and stride >= k


def _linear(x, x_scales, weight, weight_scales, bias, relu, y_type, output_scale):
    """Checks, output and call shared by the two linear operators; y_type is a torch type."""
    _tensor("x", x, _TYPES)
    device = x.device
    _tensor("weight", weight, (torch.int8,), device)
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError("weight must be [out, in], both at least 1")
    n, k = weight.shape
    if k > MAX_K:
        raise ValueError(f"rows of more than {MAX_K} elements could overflow a 32-bit sum")
    if x.dim() == 0 or x.shape[-1] != k:
        raise ValueError(f"x has shape {tuple(x.shape)}, weight takes rows of {k}")
    lead = x.shape[:-1]
    weight_scales = _vector("weight_scales", weight_scales, n, device)
    if bias is not None:
        bias = _vector("bias", bias, n, device)
    if x.dtype is torch.int8:
        if x_scales is None:
            raise ValueError("int8 rows need x_scales")
        x_scales = _scales("x_scales", x_scales, lead, device)
    elif x_scales is not None:
        raise ValueError("x_scales belong to int8 rows; float rows are quantised here")
    _on_gpu(x)
    rows, weight = _rows("x", x), _rows("weight", weight)
    if n > 1 and weight.stride(0) < k:      # rows that overlap, as those of an expanded row do
        weight = weight.contiguous()
    m = rows.shape[0]
    y_scales = None
    if y_type is torch.int8:
        y = _int8_out(m, n, device)
        if output_scale is None:
            y_scales = torch.empty(m, dtype=torch.float32, device=device)
    else:
        y = torch.empty((m, n), dtype=y_type, device=device)
    xt, yt = _TYPES[x.dtype], _TYPES[y_type]
    x_stride, w_stride = rows.stride(0), max(weight.stride(0), k)
    size = _workspace_bytes(xt, _packed(rows, x_stride, k), _packed(weight, w_stride, k), m, n, k, yt, y_scales is not None)
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.check(_lib.load().sc_int8_linear_device(
        device.index, rows.data_ptr(), xt, x_stride, None if x_scales is None else x_scales.data_ptr(),
        weight.data_ptr(), w_stride, weight_scales.data_ptr(), None if bias is None else bias.data_ptr(), m, n, k,
        1 if relu else 0, y.data_ptr(), yt, y.stride(0), None if y_scales is None else y_scales.data_ptr(),
        output_scale or 0.0, None if work is None else work.data_ptr(), size, _stream(device)),
        "sc_int8_linear_device")
    return _shaped(y, lead), None if y_scales is None else y_scales.reshape(lead)


def int8_linear(x, weight, weight_scales, bias=None, *, x_scales=None, relu=False, dtype=None):
    """A linear layer in 8-bit integers: ``x`` ``[..., k]`` and ``weight`` ``[n, k]`` give ``[..., n]``.

    ``x`` is int8 with ``x_scales`` (one for each row, as :func:`quantize_tokens` gives them), or
    float, then quantised here in the same way.  ``weight`` is int8 with ``weight_scales`` ``[n]``;
    rows that start a multiple of 16 bytes apart are used as they lie, others are copied in each
    call.  With a whole sum ``c``, ``y = fma(c * x_scale, weight_scale, bias)`` in float32, then ReLU
    (a NaN stays), then one rounding to ``dtype``: x's type by default, float32 for an int8 ``x``.
    """
    if dtype is None:
        dtype = torch.float32 if isinstance(x, torch.Tensor) and x.dtype is torch.int8 else getattr(x, "dtype", None)
        if dtype not in _FLOATS:
            _tensor("x", x, _TYPES)
    elif dtype not in _FLOATS:
        raise ValueError(f"dtype must be one of {_FLOATS}; int8_linear_requant gives int8")
    return _linear(x, x_scales, weight, weight_scales, bias, relu, dtype, None)[0]


def int8_linear_requant(q, scales, weight, weight_scales, bias=None, *, relu=False, output_scale=None):
    """:func:`int8_linear` on int8 rows with int8 results.

    Returns ``(q, scales)``, the float32 results quantised as by :func:`quantize_tokens`; or, with
    ``output_scale``, only ``q = rint(y / output_scale)`` saturated to int8 (a NaN becomes 0), the form
    of an entropy model's logits.
    """
    _tensor("q", q, (torch.int8,))
    if output_scale is not None:
        output_scale = float(output_scale)
        if not math.isfinite(output_scale) or output_scale <= 0:
            raise ValueError("output_scale must be a finite positive number")
    y, y_scales = _linear(q, scales, weight, weight_scales, bias, relu, torch.int8, output_scale)
    return y if y_scales is None else (y, y_scales)


def check_waits(device=None):
    """Wait for the current stream of ``device`` and raise if a kernel of these operators gave up a wait
    there (2 s, see ``sc_int8_status_device``) since the last such check."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    _lib.check(_lib.load().sc_int8_status_device(device.index or 0, _stream(device)), "sc_int8_status_device")
