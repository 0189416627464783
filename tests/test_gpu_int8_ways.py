"""The int8 linear operators on every way that a call's sizes can choose: each kernel, each tile, and rows that are cut in
two parts.  tests/test_int8_edges.py asserts, without a GPU, that the shapes here and in test_gpu_int8.py reach them all."""

import numpy as np
import pytest
import torch

from sigcomp_b200 import _lib
from test_gpu_int8 import DEV, add_to_odd, float_rows, host, int8_rows, layer, same, scales_of, want_quantized

pytestmark = pytest.mark.gpu

# one part: tiles of 16 to 128 tokens, K split over one to eight CTAs
WHOLE = [(1000, 8192, 512), (1000, 4096, 700), (200, 64, 4096), (200, 2048, 1300), (60, 4096, 2304), (200, 8192, 300),
         (200, 64, 2304), (20, 2048, 2304), (20, 4096, 1300), (3, 2048, 1300), (1, 64, 2304), (1, 512, 700)]
# full waves of the pair kernel and a rest, from one row on
CUT = [(9473, 2048, 300), (19000, 2048, 512), (10000, 4096, 512), (10000, 4096, 300), (10000, 8192, 512), (9473, 4096, 1300),
       (19000, 4096, 700), (19000, 4096, 1300), (10000, 8192, 1300), (19000, 2048, 700), (18945, 8192, 300),
       (19200, 4096, 256), (19200, 2048, 512), (20480, 2048, 512), (20480, 4096, 512), (19200, 512, 256),
       (38000, 2048, 700), (20480, 8192, 512)]


@pytest.fixture(scope="module")
def ops():
    from sigcomp_b200 import int8
    return int8


def want_of(q, s, w, ws, b, relu):
    """want_linear with its whole sums taken on the GPU in float64, where they are exact."""
    total = torch.cat([part.double() @ w.double().t() for part in q.split(4096)]).float().cpu().numpy()
    p = (total * host(s)[:, None]).astype(np.float64) * host(ws).astype(np.float64)
    y = add_to_odd(p, np.broadcast_to(host(b).astype(np.float64), p.shape)).astype(np.float32)
    return np.where(y < 0, np.float32(0), y) if relu else y


@pytest.mark.parametrize("rows,k,n", WHOLE + CUT)
def test_each_way(ops, rows, k, n):
    """int8 rows: results in 32 and 16 bits, with a scale for each row, and by one scale."""
    q, s = int8_rows(rows, k, rows + k), scales_of(rows, n)
    relu = (rows + n) % 3 == 0
    w, ws, b = layer(n, k, n)
    y = want_of(q, s, w, ws, b, relu)
    same(ops.int8_linear(q, w, ws, b, x_scales=s, relu=relu), y)
    same(ops.int8_linear(q, w, ws, b, x_scales=s, relu=relu, dtype=torch.bfloat16),
         torch.from_numpy(y).to(torch.bfloat16).float().numpy())
    wq, wscale = want_quantized(y)
    yq, ys = ops.int8_linear_requant(q, s, w, ws, b, relu=relu)
    same(ys, wscale)
    same(yq, wq)
    same(ops.int8_linear_requant(q, s, w, ws, b, relu=relu, output_scale=0.011),
         np.clip(np.rint(y / np.float32(0.011)), -128, 127).astype(np.int8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k,n,pad", [(1000, 8192, 512, 0), (9473, 2048, 300, 3), (10000, 8192, 512, 0), (20480, 4096, 512, 8)])
def test_each_way_from_float_rows(ops, rows, k, n, pad, dtype):
    """Float rows, quantised into the workspace: the second part's rows are int8 there."""
    x = float_rows(rows, k, dtype, rows + n, pad)
    w, ws, b = layer(n, k, 5)
    q, s = want_quantized(host(x))
    y = want_of(torch.from_numpy(q).to(DEV), torch.from_numpy(s).to(DEV), w, ws, b, False)
    with np.errstate(over="ignore"):
        same(ops.int8_linear(x, w, ws, b), torch.from_numpy(y).to(dtype).float().numpy())


@pytest.mark.parametrize("y_type", [0, 2, 3, "rows"])
@pytest.mark.parametrize("rows,k,n", [(1000, 8192, 512), (9473, 2048, 300), (10000, 4096, 300), (10000, 8192, 512), (18945, 8192, 300),
                                      (19000, 2048, 700), (38000, 2048, 700)])
@pytest.mark.parametrize("x_gap,shift,gap", [(0, 3, 5), (7, 0, 3), (16, 16, 16)])
def test_each_way_at_any_address(rows, k, n, y_type, x_gap, shift, gap):
    """Rows of x and y any distance apart, y from any element on; the gaps stay."""
    q, s = int8_rows(rows, k, 4, k + x_gap), scales_of(rows, 5)
    w, ws, b = layer(n, k, 6)
    by_rows = y_type == "rows"
    code = 3 if by_rows else y_type
    dtype = {0: torch.float32, 2: torch.bfloat16, 3: torch.int8}[code]
    out = torch.full((shift + rows * (n + gap) + 9,), 5, dtype=dtype, device=DEV)
    scales = torch.full((rows + 2,), 7.0, device=DEV)
    L = _lib.load()
    size = L.sc_int8_linear_workspace(3, int(x_gap % 16 == 0), 1, rows, n, k, code, int(by_rows))
    work = torch.empty(max(size, 1), dtype=torch.uint8, device=DEV)
    _lib.check(L.sc_int8_linear_device(0, q.data_ptr(), 3, q.stride(0), s.data_ptr(), w.data_ptr(), w.stride(0), ws.data_ptr(),
                                       b.data_ptr(), rows, n, k, 0, out.data_ptr() + shift * out.element_size(), code,
                                       n + gap, scales.data_ptr() + 4 if by_rows else None, 0.02,
                                       work.data_ptr() if size else None, size, torch.cuda.current_stream().cuda_stream))
    y = want_of(q, s, w, ws, b, False)
    got = out[shift:shift + rows * (n + gap)].view(rows, n + gap)
    if by_rows:
        wq, wscale = want_quantized(y)
        same(got[:, :n], wq)
        same(scales[1:-1], wscale)
    elif code == 3:
        same(got[:, :n], np.clip(np.rint(y / np.float32(0.02)), -128, 127))
    else:
        same(got[:, :n], torch.from_numpy(y).to(dtype).float().numpy())
    assert scales[0] == 7 and scales[-1] == 7
    assert (got[:, n:] == 5).all() and (out[:shift] == 5).all() and (out[shift + rows * (n + gap):] == 5).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(300, 4096), (301, 4093), (300, 2049), (297, 1025), (300, 1521), (299, 2048), (400, 8192)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (1, 0), (8, 8), (5, 3)])
def test_many_wide_rows_quantised(ops, dtype, rows, cols, pad, offset):
    """Rows of 65 to 1,024 vectors in more than a wave of the kernels for few rows."""
    x = float_rows(rows, cols, dtype, rows + cols, pad, offset)
    q, s = ops.quantize_tokens(x)
    wq, wscale = want_quantized(host(x))
    same(q, wq)
    same(s, wscale)
    flat = torch.full((rows * cols + 40,), float("nan"), dtype=dtype, device=DEV)
    view = flat[offset:offset + rows * cols].view(rows, cols)
    view.copy_(x)
    q, s = ops.quantize_tokens(view)
    same(q, wq)
    same(s, wscale)
