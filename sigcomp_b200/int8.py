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
writes them out).  So logits computed in large batches for coding and row by row for decoding agree
bit for bit.  (``sc_decode_logits_device`` starts every stream anew, so a decoder whose next logits
depend on the last symbol passes the rows of all steps so far.)

Arrays are torch tensors on one GPU; leading dimensions are batch dimensions.  Rows of every result
start a multiple of 16 bytes apart, so results are contiguous where their width is such a multiple, and
strided otherwise (rows of odd widths side by side took two to five times as long to write).  Work is put into the
current stream of that GPU and not waited for, so calls can be captured into CUDA graphs.  The
operators serve coding, not training: a tensor that asks for a gradient, or carries a tangent
(``torch.autograd.forward_ad``), is refused.
"""

import torch

from . import _lib

try:
    from . import _int8
except ImportError as exc:
    raise ImportError("sigcomp_b200/_int8.so is missing or does not load: build it with "
                      "`python -m sigcomp_b200.build_ext`") from exc
if _int8.torch_version != torch.__version__:
    raise ImportError(f"sigcomp_b200/_int8.so was built for torch {_int8.torch_version}, not {torch.__version__}: "
                      "build it with `python -m sigcomp_b200.build_ext`")

MAX_K = 131071


def quantize_tokens(x):
    """Quantise every row of ``x`` (``[..., k]``, float32, float16 or bfloat16) to int8.

    Returns ``(q, scales)``: int8 of x's shape and float32 of its leading shape.  With
    ``a = max(max|row|, 2**-100)``, ``scale = a / 127`` and ``q = rint(row * (127 / a))``; both
    quotients are rounded to float32, the product is not, and ties go to the even number.  A row
    holding an infinity or a NaN gets the scale NaN and zeros, so what is computed from it is NaN.
    """
    return _int8.quantize_tokens(x)


def dequantize_tokens(q, scales, dtype=torch.float32):
    """The values that int8 rows stand for: ``q * scales`` in float32, rounded once to ``dtype``.

    ``scales`` holds one scale for each row, or is one number for all of them.
    """
    return _int8.dequantize_tokens(q, scales, dtype)


def int8_linear(x, weight, weight_scales, bias=None, *, x_scales=None, relu=False, dtype=None):
    """A linear layer in 8-bit integers: ``x`` ``[..., k]`` and ``weight`` ``[n, k]`` give ``[..., n]``.

    ``x`` is int8 with ``x_scales`` (one for each row, as :func:`quantize_tokens` gives them), or
    float, then quantised here in the same way.  ``weight`` is int8 with ``weight_scales`` ``[n]``;
    rows that start a multiple of 16 bytes apart are used as they lie, others are copied in each
    call.  With a whole sum ``c``, ``y = fma(c * x_scale, weight_scale, bias)`` in float32, then ReLU
    (a NaN stays), then one rounding to ``dtype``: x's type by default, float32 for an int8 ``x``.
    """
    return _int8.int8_linear(x, x_scales, weight, weight_scales, bias, relu, dtype)


def int8_linear_requant(q, scales, weight, weight_scales, bias=None, *, relu=False, output_scale=None):
    """:func:`int8_linear` on int8 rows with int8 results.

    Returns ``(q, scales)``, the float32 results quantised as by :func:`quantize_tokens`; or, with
    ``output_scale``, only ``q = rint(y / output_scale)`` saturated to int8 (a NaN becomes 0), the form
    of an entropy model's logits.
    """
    return _int8.int8_linear_requant(q, scales, weight, weight_scales, bias, relu, output_scale)


def check_waits(device=None):
    """Wait for the current stream of ``device`` and raise if a kernel of these operators gave up a wait
    there (2 s, see ``sc_int8_status_device``) since this thread's last such check, or, in its first, at any
    time before.  Refused while that stream is captured."""
    device = torch.device("cuda" if device is None else device)
    index = torch.cuda.current_device() if device.index is None else device.index
    _lib.check(_lib.load().sc_int8_status_device(index, torch.cuda.current_stream(index).cuda_stream),
               "sc_int8_status_device")
